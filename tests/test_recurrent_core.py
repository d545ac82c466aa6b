"""The selective core and the clipped policy loss together, as a user has
them: episodes played step by step, then trained on as windows."""

import random

import pytest
import torch
import torch.nn as nn

from handyrl_amd.batch import EpisodeBuffer, make_batch
from handyrl_amd.envs import tictactoe
from handyrl_amd.generation import Generator
from handyrl_amd.model import ModelWrapper
from handyrl_amd.models.selective import SelectiveCore
from handyrl_amd.train import Trainer, compute_loss
from handyrl_amd.util import map_r


class StepNet(nn.Module):
    """Recurrent policy for TicTacToe that only knows single steps."""

    def __init__(self):
        super().__init__()
        self.encode = nn.Linear(27, 32)
        self.core = SelectiveCore(32, states=8)
        self.policy, self.value = nn.Linear(32, 9), nn.Linear(32, 1)

    def init_hidden(self, batch_size=()):
        return self.core.init_hidden(batch_size)

    def heads(self, h, hidden):
        return {'policy': self.policy(h), 'value': torch.tanh(self.value(h)), 'hidden': hidden}

    def forward(self, x, hidden):
        return self.heads(*self.core(torch.relu(self.encode(x.flatten(1))), hidden))


class WindowNet(StepNet):
    def forward_window(self, x, hidden, mask):
        return self.heads(*self.core.window(torch.relu(self.encode(x.flatten(2))), hidden, mask))


def make_args(**over):
    return {'turn_based_training': True, 'observation': False, 'gamma': 0.8, 'forward_steps': 6,
            'burn_in_steps': 0, 'compress_steps': 4, 'entropy_regularization': 0.1,
            'entropy_regularization_decay': 0.1, 'batch_size': 4, 'minimum_episodes': 2,
            'maximum_episodes': 100, 'num_batchers': 1, 'lambda': 0.7, 'policy_target': 'UPGO',
            'value_target': 'TD', 'seed': 0, 'bf16': False, 'compress_episodes': True,
            'policy_loss': 'CLIP', 'clip_ratio': 0.2, 'kl_regularization': 0.3, **over}


def played(net, args, n=4):
    env = tictactoe.Environment()
    models = {p: ModelWrapper(net) for p in env.players()}
    job = {'player': env.players(), 'model_id': {p: 1 for p in env.players()}}
    episodes = []
    for i in range(n):
        random.seed(i)
        episodes.append(Generator(env, args).generate(models, job))
    random.seed(100)
    store = EpisodeBuffer(args)
    store.extend(episodes)
    return make_batch([store.select_episode() for _ in range(args['batch_size'])], args)


def loss_of(net, batch, args, device):
    model = ModelWrapper(net)
    batch = map_r(batch, lambda v: v.to(device))
    hidden = model.init_hidden([batch['value'].size(0), batch['value'].size(2)])
    net.zero_grad()
    losses, dcnt = compute_loss(batch, model, hidden, args)
    losses['total'].backward()
    return losses, [p.grad.clone() for p in net.parameters()]


def check_windows(device, over):
    torch.manual_seed(3)
    steps, windows = StepNet(), WindowNet()
    windows.load_state_dict(steps.state_dict())
    args = make_args(**over)
    batch = played(steps, args)
    steps, windows = steps.to(device), windows.to(device)
    one, grads_one = loss_of(steps, batch, args, device)
    two, grads_two = loss_of(windows, batch, args, device)
    assert set(one) == set(two)
    for k in one:       # sums of some 50 terms of order 1, through a few products over 32 to 64 terms
        torch.testing.assert_close(one[k].float(), two[k].float(), rtol=1e-4, atol=1e-4)
    for a, b in zip(grads_one, grads_two):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-3 * float(a.abs().max()) + 1e-6)
    assert all(g.isfinite().all() for g in grads_two)


CASES = [dict(), dict(observation=True), dict(burn_in_steps=2), dict(policy_loss='PG'),
         dict(policy_target='VTRACE', value_target='VTRACE', burn_in_steps=2, observation=True)]


@pytest.mark.parametrize('over', CASES)
def test_windows_give_what_steps_give(over):
    check_windows('cpu', over)


@pytest.mark.gpu
@pytest.mark.parametrize('over', CASES)
def test_windows_give_what_steps_give_gpu(over):
    check_windows('cuda', over)


def test_clip_is_the_policy_gradient_at_ratio_one():
    """Where the policy still is the acting one, the surrogate's gradient is the
    policy gradient's, and the KL term's is zero."""
    torch.manual_seed(3)
    net = StepNet()
    with torch.no_grad():                       # an even policy: probabilities of 1 / legal moves
        net.policy.weight.zero_()
        net.policy.bias.zero_()
    grads = []
    for loss in ('CLIP', 'PG'):
        args = make_args(policy_loss=loss)
        batch = played(net, args)
        losses, g = loss_of(net, batch, args, 'cpu')
        grads.append(g)
    assert losses['total'].isfinite()
    for a, b in zip(*grads):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_unknown_policy_loss():
    net = StepNet()
    args = make_args()
    batch = played(net, args)
    with pytest.raises(ValueError, match='policy_loss'):
        loss_of(net, batch, {**args, 'policy_loss': 'TRPO'}, 'cpu')


def check_training(device, bf16):
    torch.manual_seed(1)
    args = make_args(bf16=bf16)
    net = WindowNet()
    batch = played(net, args, n=6)
    trainer = Trainer(args, net, device=torch.device(device), batcher=False)
    before = [p.detach().clone() for p in trainer.model.parameters()]
    for _ in range(3):
        losses, dcnt = trainer.train_step(batch)
        assert dcnt > 0 and all(l.isfinite() for l in losses.values())
    assert {'p', 'v', 'kl', 'clip', 'ent', 'total'} == set(losses)
    moved = [not torch.equal(a, b) for a, b in zip(before, trainer.model.parameters())]
    assert sum(moved) >= len(moved) - 1         # a bias of the value head may stay in place


def test_training_step():
    check_training('cpu', False)


@pytest.mark.gpu
@pytest.mark.parametrize('bf16', [False, True])
def test_training_step_gpu(bf16):
    check_training('cuda', bf16)


@pytest.mark.gpu
@pytest.mark.parametrize('bf16', [False, True])
def test_captured_window_training_gpu(bf16):
    """The core, the heads and the clipped loss with all gradients in one graph,
    replayed on batches of other episodes, against the eager passes."""
    torch.manual_seed(5)
    args = make_args(burn_in_steps=2)
    net = WindowNet()
    batches = []
    for k in range(3):
        random.seed(k)
        batch = played(net, {**args, 'seed': k}, n=3 + k)
        batches.append(map_r(batch, lambda v: v.cuda()))
    net = net.cuda()
    model = ModelWrapper(net)
    static = map_r(batches[0], lambda v: v.clone())
    hidden = model.init_hidden([static['value'].size(0), static['value'].size(2)])

    def run():
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=bf16, cache_enabled=False):
            losses, dcnt = compute_loss(static, model, hidden, args)
        grads = torch.autograd.grad(losses['total'], list(net.parameters()))
        return [v.detach() for v in (*losses.values(), dcnt, *grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for batch in (batches[1], batches[2], batches[0]):
        for k in static:
            static[k].copy_(batch[k])
        eager = [v.clone() for v in run()]
        torch.cuda.synchronize()
        graph.replay()
        assert len(out) == len(eager) and all(v.isfinite().all() for v in eager)
        for a, b in zip(out, eager):
            # library products may be taken in another order by the graph: sums of some
            # 50 terms of order 1 in the losses, of as many rows in the gradients
            torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4 + 1e-3 * float(b.abs().max()))


@pytest.mark.gpu
def test_clipped_loss_in_the_captured_learner_gpu():
    """The learner's captured step on the device replay with policy_loss 'CLIP'."""
    from handyrl_amd.actor import GeeseActorPool
    from handyrl_amd.hipgraph import GraphedReplayTrainStep
    from handyrl_amd.models.geese_net import GeeseNet
    from handyrl_amd.replay import DeviceReplay
    args = make_args(turn_based_training=False, forward_steps=8, batch_size=16, bf16=True,
                     policy_target='VTRACE', value_target='VTRACE', compress_episodes=False,
                     maximum_episodes=500)
    device = torch.device('cuda', 0)
    trainer = Trainer(args, GeeseNet(), device=device, batcher=False)
    pool = GeeseActorPool(trainer.model, args, n_games=64, device=device, seed=0)
    trainer.model.eval()
    for _ in range(40000):
        pool.step_once()
        if pool.episodes_done >= 40:
            break
    assert pool.episodes_done >= 40, 'no episodes finished'
    replay = DeviceReplay(args, device, bytes_budget=256 << 20)
    replay.extend(pool.harvest())
    step = GraphedReplayTrainStep(trainer, replay, args['batch_size'])
    assert step.graph is not None, 'capture must succeed at world_size 1'
    before = [p.detach().clone() for p in trainer.params]
    for _ in range(3):
        losses, dcnt = step.step()
        torch.cuda.synchronize()
        assert all(v.isfinite() for v in losses.values()) and float(dcnt) > 0
    assert {'p', 'v', 'kl', 'clip', 'ent', 'total'} == set(losses)
    assert any(not torch.equal(b, p.detach()) for b, p in zip(before, trainer.params))
