"""Clipped policy loss: the eager path against the formula written out row by
row in 64 bits, its gradient against differences, its refusals, and (gpu) the
HIP kernels against the eager path in 64 bits."""

import math

import pytest
import torch

from handyrl_amd.losses import POLICY_LOSS_STATS, clipped_policy_loss

STEP = 2.0 ** -24            # half a step of float32, relative to the value


def make(rows, width, seed=0, dtype=torch.float32, legal=1.0, device='cpu'):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*rows, width, generator=g) * 2).to(dtype)
    actions = torch.randint(0, width, rows, generator=g)
    if legal < 1:
        illegal = torch.rand(*rows, width, generator=g) > legal
        illegal.scatter_(-1, actions.unsqueeze(-1), False)
        logits = logits.masked_fill(illegal, -1e32)
    logp = torch.log_softmax(logits.double(), -1).gather(-1, actions.unsqueeze(-1)).squeeze(-1)
    x = torch.randn(rows, generator=g).double() * 0.25
    for border in (math.log(0.8), math.log(1.3)):   # a rounding must not decide a side
        x = torch.where((x - border).abs() < 1e-4, x + 1e-3, x)
    args = dict(logits=logits, actions=actions, old_log_probs=(logp - x).float(),
                advantages=torch.randn(rows, generator=g),
                mask=(torch.rand(rows, generator=g) < 0.8).float() * torch.rand(rows, generator=g),
                entropy_scale=torch.rand(rows, generator=g))
    return {k: v.to(device) for k, v in args.items()}


COEFS = dict(clip=0.2, clip_high=0.3, kl_coef=0.7, entropy_coef=0.05)


def by_hand(logits, actions, old_log_probs, advantages, mask, entropy_scale,
            clip, clip_high, kl_coef, entropy_coef):
    sums = [0.0] * 6
    for z, a, old, adv, m, e in zip(logits.double(), actions.tolist(), old_log_probs.tolist(),
                                    advantages.tolist(), mask.tolist(), entropy_scale.tolist()):
        if m == 0:
            continue
        p = (z - z.max()).exp()
        p = (p / p.sum()).tolist()
        x = math.log(p[a]) - old
        r = math.exp(x)
        s = min(r * adv, min(max(r, 1 - clip), 1 + clip_high) * adv)
        entropy = -sum(v * math.log(v) for v in p if v > 0)
        sums[0] -= m * s
        sums[1] += m * (r - 1 - x)
        sums[2] += m * entropy
        sums[3] += m * e * entropy
        sums[4] += (adv > 0 and r > 1 + clip_high) or (adv < 0 and r < 1 - clip)
        sums[5] += m
    return sums[0] + kl_coef * sums[1] - entropy_coef * sums[3], sums


def in64(args):
    return {k: v.detach().cpu().double() if v.is_floating_point() else v.cpu()
            for k, v in args.items()}


@pytest.mark.parametrize('legal', [1.0, 0.3])
@pytest.mark.parametrize('width', [1, 2, 9, 214])
def test_eager_matches_formula(width, legal):
    args = in64(make((57,), width, legal=legal))
    loss, stats = clipped_policy_loss(**args, **COEFS)
    want, sums = by_hand(**args, **COEFS)
    assert len(stats) == len(POLICY_LOSS_STATS) and not stats.requires_grad
    # 64-bit sums of 57 rows of order 1
    torch.testing.assert_close(stats, torch.tensor(sums, dtype=torch.float64), rtol=1e-11, atol=1e-11)
    assert abs(loss.item() - want) < 1e-11 * (1 + abs(want))


def test_eager_gradient_matches_differences():
    args = in64(make((12,), 7))
    z = args.pop('logits').requires_grad_()
    assert torch.autograd.gradcheck(lambda v: clipped_policy_loss(v, **args, **COEFS)[0], (z,))


def test_rows_of_weight_zero_are_left_out():
    args = in64(make((20,), 5))
    args['mask'][::2] = 0
    want, _ = clipped_policy_loss(**args, **COEFS)
    spoilt = {k: v.clone() for k, v in args.items()}
    spoilt['logits'][::2] = float('nan')
    spoilt['logits'][2] = -float('inf')
    spoilt['actions'][::2] = 99
    for k in ('old_log_probs', 'advantages', 'entropy_scale'):
        spoilt[k][::2] = float('inf')
    z = spoilt['logits'].requires_grad_()
    loss, _ = clipped_policy_loss(**spoilt, **COEFS)
    loss.backward()
    assert loss.item() == want.item()
    assert (z.grad[::2] == 0).all() and z.grad[1::2].isfinite().all()


def test_illegal_actions_may_be_minus_infinity():
    args = in64(make((20,), 6, legal=0.5))
    want, _ = clipped_policy_loss(**args, **COEFS)
    args['logits'][args['logits'] < -1e31] = -float('inf')
    z = args['logits'].requires_grad_()
    loss, _ = clipped_policy_loss(**args, **COEFS)
    loss.backward()
    assert abs(loss.item() - want.item()) < 1e-12 and z.grad.isfinite().all()


def test_broadcasts_and_trailing_axis():
    args = in64(make((4, 6, 2), 5))
    args['entropy_scale'] = args['entropy_scale'][:, :, :1]
    want, _ = clipped_policy_loss(**args, **COEFS)
    args = {k: v if k == 'logits' else v.unsqueeze(-1) for k, v in args.items()}
    loss, _ = clipped_policy_loss(**args, **COEFS)
    assert loss.item() == want.item()


def check_overflow(device):
    """Without a KL term a ratio that overflows counts as the clipped one where
    the surrogate is flat."""
    args = make((8,), 5, device=device)
    args['mask'][:] = 1
    args['advantages'][2], args['old_log_probs'][2] = 1.5, -500.0
    z = args['logits'].requires_grad_()
    loss, stats = clipped_policy_loss(**args, clip=0.2, kl_coef=0.0, entropy_coef=0.1)
    loss.backward()
    assert loss.isfinite() and z.grad.isfinite().all() and math.isinf(stats[1].item())


def test_eager_overflow():
    check_overflow('cpu')


REFUSALS = [
    (dict(clip=-0.1), 'clip must be'), (dict(clip=1.5), 'clip must be'),
    (dict(clip_high=-1.0), 'clip_high'),
    (dict(actions=torch.zeros(3)), 'actions has type'),
    (dict(actions=torch.zeros(4, dtype=torch.int64)), 'actions of shape'),
    (dict(old_log_probs=torch.zeros(3, dtype=torch.int64)), 'old_log_probs has type'),
    (dict(advantages=torch.zeros(3, 2)), 'advantages of shape'),
    (dict(advantages=torch.zeros(3).requires_grad_()), 'detach'),
    (dict(mask=torch.zeros(5)), 'mask of shape'),
    (dict(logits=torch.zeros(3, 0)), 'logits must be'),
    (dict(logits=torch.zeros(3, 2, dtype=torch.int64)), 'logits must be'),
]


def refuse(change, match, device):
    args = dict(logits=torch.zeros(3, 2), actions=torch.zeros(3, dtype=torch.int64),
                old_log_probs=torch.zeros(3), advantages=torch.zeros(3))
    args.update(change)
    args = {k: v.detach().to(device).requires_grad_(v.requires_grad) if torch.is_tensor(v) else v
            for k, v in args.items()}
    with pytest.raises(ValueError, match=match):
        clipped_policy_loss(**args)


@pytest.mark.parametrize('change, match', REFUSALS)
def test_refusals(change, match):
    refuse(change, match, 'cpu')


# ------------------------------------------------------------------- GPU

gpu = pytest.mark.gpu


def assert_matches_64_bits(args, grad_out=1.0):
    """Tolerances: log p(a) comes from a difference of numbers up to max|z| and a
    sum over the width, an exponential of it carries that error as a relative
    one, and each of the few operations behind adds half a step."""
    z = args['logits'].detach().requires_grad_()
    loss, stats = clipped_policy_loss(**{**args, 'logits': z}, **COEFS)
    (loss * grad_out).backward()
    ref = in64(args)
    z64 = ref['logits'].requires_grad_()
    want, sums = clipped_policy_loss(**ref, **COEFS)
    (want * grad_out).backward()

    width = z.size(-1)
    rel = relative_error(ref)
    adv = ref['advantages'].abs() + 1
    m = ref['mask'].abs()
    size = float((m * (2 * adv + 3 + math.log(width + 1))).sum()) if m.numel() else 0
    assert abs(loss.item() - want.item()) <= 4 * rel * size + STEP * abs(want.item())
    assert torch.all((stats.cpu().double() - sums).abs() <= 4 * rel * size + STEP * sums.abs())
    assert z.grad.dtype == z.dtype and z.grad.shape == z.shape
    assert_gradient(z.grad, z64.grad, ref, grad_out)
    return loss, z.grad


def relative_error(ref):
    """Of one row's ratio or probability."""
    finite = ref['logits'].detach().clamp(min=-60)
    reach = float(finite.max() - finite.min()) + float(ref['old_log_probs'].abs().max()) \
        if finite.numel() else 0
    return STEP * (8 + 2 * reach + finite.size(-1) / 64)


def assert_gradient(grad, want, ref, grad_out=1.0):
    adv, m = ref['advantages'].abs() + 1, ref['mask'].abs()
    per = (m * (3 * adv + math.log(grad.size(-1) + 1))).unsqueeze(-1) * abs(grad_out)
    off = (grad.cpu().double() - want).abs()
    out = torch.finfo(grad.dtype).eps / 2
    assert torch.all(off <= 4 * relative_error(ref) * per + out * want.abs()), \
        float((off / per).nan_to_num().max())


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows, width', [
    ((1,), 1), ((3,), 2), ((2048,), 4), ((77,), 9), ((65,), 63), ((64,), 64), ((33,), 65),
    ((16, 8, 2), 214), ((9,), 1025), ((5,), 4099), ((3,), 20001), ((2,), 70001), ((2,), 140003)])
def test_kernel_matches_64_bits(rows, width, dtype):
    assert_matches_64_bits(make(rows, width, dtype=dtype, device='cuda'))
    assert_matches_64_bits(make(rows, width, seed=1, dtype=dtype, legal=0.3, device='cuda'), grad_out=-1.7)


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('width', [5, 300, 5000])
def test_kernel_left_out_rows_and_infinities(width, dtype):
    args = make((40,), width, dtype=dtype, legal=0.5, device='cuda')
    args['logits'][args['logits'] < -1e31] = -float('inf')
    args['mask'][::2] = 0
    want, grad = assert_matches_64_bits(args)
    args['logits'][::4] = float('nan')
    args['logits'][2::4] = -float('inf')
    args['actions'][::2] = -5
    for k in ('old_log_probs', 'advantages', 'entropy_scale'):
        args[k][::2] = float('nan')
    z = args['logits'].requires_grad_()
    loss, _ = clipped_policy_loss(**args, **COEFS)
    loss.backward()
    assert loss.item() == want.item() and torch.equal(z.grad, grad)


@gpu
def test_kernel_strides_and_offsets():
    wide = make((50,), 40, device='cuda')
    for low, high in ((0, 8), (3, 17), (1, 40)):
        base = make((50,), high - low, seed=low, device='cuda')
        wide['logits'][:, low:high] = base['logits']
        for view in (wide['logits'][:, low:high], base['logits'].t().contiguous().t()):
            assert_matches_64_bits({**base, 'logits': view})


@gpu
def test_kernel_empty_and_defaults():
    z = torch.zeros(0, 4, device='cuda', requires_grad=True)
    none = torch.zeros(0, device='cuda')
    loss, stats = clipped_policy_loss(z, none.long(), none, none)
    loss.backward()
    assert loss.item() == 0 and (stats == 0).all() and z.grad.shape == (0, 4)
    args = make((30,), 9, device='cuda')
    del args['mask'], args['entropy_scale']
    ref = in64(args)
    loss, stats = clipped_policy_loss(**args, **COEFS)
    want, sums = clipped_policy_loss(**ref, **COEFS)
    torch.testing.assert_close(stats.cpu().double(), sums, rtol=1e-5, atol=1e-5)
    assert stats[5].item() == 30 and abs(loss.item() - want.item()) < 1e-4


@gpu
def test_kernel_action_out_of_range_is_nan():
    args = make((30,), 9, device='cuda')
    args['mask'][:] = 1
    args['actions'][3] = 9
    z = args['logits'].requires_grad_()
    loss, _ = clipped_policy_loss(**args, **COEFS)
    loss.backward()
    assert math.isnan(loss.item()) and z.grad[3].isnan().all()
    assert z.grad[:3].isfinite().all() and z.grad[4:].isfinite().all()


@gpu
@pytest.mark.parametrize('change, match', REFUSALS)
def test_kernel_refusals(change, match):
    refuse(change, match, 'cuda')


@gpu
def test_kernel_backward_twice_scaled_and_not_again():
    args = make((100,), 214, device='cuda')
    z = args['logits'].requires_grad_()
    loss, _ = clipped_policy_loss(**args, **COEFS)
    one, = torch.autograd.grad(loss, z, retain_graph=True)
    kept = one.clone()
    two, = torch.autograd.grad(loss, z, torch.tensor(-3.0, device='cuda'), retain_graph=True)
    three, = torch.autograd.grad(loss, z)
    assert torch.equal(one, kept) and torch.equal(three, kept)
    # a product by -3: the two sides round it once each
    torch.testing.assert_close(two, -3 * kept, rtol=2 * STEP, atol=0)
    loss, _ = clipped_policy_loss(**args, **COEFS)
    with pytest.raises(RuntimeError, match='not differentiable again'):
        torch.autograd.grad(loss, z, create_graph=True)


@gpu
@pytest.mark.parametrize('rows, width', [((300,), 4), ((64,), 214), ((6,), 9000)])
def test_kernel_in_a_graph(rows, width):
    first, second = (make(rows, width, seed=s, device='cuda') for s in (0, 1))
    held = {k: v.clone() for k, v in first.items()}
    z = held['logits'].requires_grad_()

    def step():
        loss, stats = clipped_policy_loss(**held, **COEFS)
        grad, = torch.autograd.grad(loss * 0.5, z)
        return loss, stats, grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in (second, first, second):
        with torch.no_grad():
            for k, v in held.items():
                v.copy_(new[k])
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


@gpu
def test_kernel_overflow():
    check_overflow('cuda')


@gpu
def test_kernel_forward_and_backward_in_graphs_of_their_own():
    """As make_graphed_callables has them, with one upstream gradient and another."""
    args = make((64,), 214, device='cuda')
    logits = args.pop('logits')

    class Loss(torch.nn.Module):
        def forward(self, z):
            return clipped_policy_loss(z, **args, **COEFS)[0]

    z = logits.clone().requires_grad_()
    want, = torch.autograd.grad(Loss()(z), z)
    graphed = torch.cuda.make_graphed_callables(Loss(), (torch.zeros_like(logits).requires_grad_(),))
    for scale in (1.0, 2.0, 1.0, -0.5):          # powers of two: products without rounding
        z = logits.clone().requires_grad_()
        got, = torch.autograd.grad(graphed(z) * scale, z)
        assert torch.equal(got, want * scale)


@gpu
def test_kernel_results_repeat():
    args = make((5000,), 37, device='cuda')
    runs = [clipped_policy_loss(**args, **COEFS) for _ in range(3)]
    assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1]) for r in runs)


@gpu
def test_kernel_past_32_bit_offsets():
    """2.2e9 logits: the last rows as they come alone."""
    rows, width = 70000, 32003
    z = torch.empty(rows, width, device='cuda', dtype=torch.bfloat16).normal_().requires_grad_()
    args = dict(actions=torch.randint(0, width, (rows,), device='cuda'),
                old_log_probs=torch.full((rows,), -10.5, device='cuda'),
                advantages=torch.randn(rows, device='cuda'),
                mask=(torch.arange(rows, device='cuda') % 3 > 0).float())
    loss, stats = clipped_policy_loss(z, **args, **COEFS)
    grad, = torch.autograd.grad(loss, z)
    # alone, a row may begin elsewhere between 16 byte borders and be summed in another
    # order, so the last rows are held to the formula in 64 bits
    tail = slice(rows - 40, rows)
    ref = in64({'logits': z[tail], **{k: v[tail] for k, v in args.items()}})
    z64 = ref['logits'].requires_grad_()
    want, _ = clipped_policy_loss(**ref, **COEFS)
    want.backward()
    assert_gradient(grad[tail], z64.grad, ref)
    assert stats[5].item() == args['mask'].sum().item()
    assert (grad[::3][:5] == 0).all() and grad[1].abs().sum() > 0
