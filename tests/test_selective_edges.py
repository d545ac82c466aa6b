"""Selective scan and short convolution where they are easiest to get wrong:
growth past a float's range, rates without bound, plans of several chunks a
segment and of several rows a lane.  Helpers and tolerances are those of
test_selective.py."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd

from handyrl_amd import ops
from handyrl_amd.models.selective import (
    SelectiveCore, causal_conv, causal_conv_step, selective_scan, selective_step)
from test_selective import (
    STEP, assert_conv, assert_scan, make_conv, make_scan, move, run_scan, scan_by_hand)

gpu = pytest.mark.gpu


def assert_results(got, want, size, a):
    """As assert_scan has it: k half steps of each result's sum of magnitudes."""
    steps, width = a['x'].shape[1:]
    for k, v in got.items():
        out = torch.finfo(v.dtype).eps / 2
        off = (v.double().cpu() - want[k]).abs()
        tol = STEP * (4 * steps + 64 + width / 8) * size[k] + out * want[k].abs() + 1e-37
        assert torch.all(off <= tol), (k, float((off / tol).max()))


def growing(what, sign):
    """States that grow by e^4 a step (or e^3.125), past a float's range within a
    segment of 32 steps, where all results stay in it: zeros, with inputs in the
    last 16 steps and gradients in the first 16; or a tiny state (or a tiny
    gradient of the last one) that meets 32 observed steps.  Sign 1: rates above
    0; sign -1: steps below it."""
    zeros = what == 'zeros'
    a, (dy, dlast) = make_scan(1, 1100, 24, 16, gate=False, state=not zeros, share=1.0, plain=True)
    a['A'] = torch.full_like(a['A'], sign)
    a['dt'] = torch.full_like(a['dt'], sign * (4.0 if zeros else 3.125))
    if zeros:
        a['x'][:, :-16] = 0
        dy[:, 16:] = 0
        return a, dy, torch.zeros_like(dlast)
    a['mask'] = torch.zeros(1, 1100, dtype=torch.bool)
    a['mask'][:, slice(0, 32) if what == 'tiny state' else slice(1056, 1088)] = True
    a['x'] = torch.zeros_like(a['x'])
    a['state'] *= 1e-36 if what == 'tiny state' else 1e-30
    dlast *= 1e-30 if what == 'tiny state' else 1e-36
    return a, torch.zeros_like(dy), dlast


@gpu
@pytest.mark.parametrize('sign', [1.0, -1.0])
@pytest.mark.parametrize('what', ['zeros', 'tiny state', 'tiny gradient'])
def test_scan_of_growing_states(what, sign):
    a, dy, dlast = growing(what, sign)
    want = run_scan(move(a, double=True), dy.double(), dlast.double())
    assert all(v.float().isfinite().all() for v in want.values())
    # the magnitudes are the same for either sign
    size = scan_by_hand(growing(what, 1.0)[0], dy, dlast, absolute=True)
    assert_results(run_scan(move(a, 'cuda'), dy.cuda(), dlast.cuda()), want, size, a)


@gpu
@pytest.mark.parametrize('rate', [-float('inf'), -3e38])
@pytest.mark.parametrize('steps', [21, 700])
def test_scan_forgets_at_once(rate, steps):
    """States whose rate has no bound hold the last observed step alone, past
    holes and behind an end within a chunk.  With rates of -1e30 instead, 64
    bits give the same: decays of 0, times a rate that is finite."""
    a, (dy, dlast) = make_scan(2, steps, 40, 8)
    a['A'][::2, 1::3] = rate
    finite = {**a, 'A': a['A'].clamp(min=-1e30)}
    got = run_scan(move(a, 'cuda'), dy.cuda(), dlast.cuda())
    want = run_scan(move(finite, double=True), dy.double(), dlast.double())
    assert_results(got, want, scan_by_hand(finite, dy, dlast, absolute=True), a)
    held, t = a['state'].cuda(), int(a['mask'][0].nonzero()[0])
    row = {k: a[k][:, t].cuda() for k in ('x', 'dt', 'B', 'C', 'z', 'mask')}
    rest = {k: a[k].cuda() if torch.is_tensor(a[k]) else a[k] for k in ('A', 'D', 'dt_bias', 'dt_softplus')}
    _, last = selective_scan(**{k: v[:, None] for k, v in row.items()}, **rest, state=held)
    selective_step(held, **row, **rest)
    assert held.isfinite().all()
    torch.testing.assert_close(held, last, rtol=64 * STEP, atol=64 * STEP * 10)


def calls(device):
    """Each operator's entry with its arguments, and those that carry derivatives."""
    a, c = (move(make(2, 3, 8, 4)[0], device) for make in (make_scan, make_conv))
    row = {k: v[:, 0] if k in ('x', 'dt', 'B', 'C', 'z', 'mask') else v for k, v in a.items()}
    step = {k: v[:, 0] if k in ('x', 'mask') else v for k, v in c.items()}
    scan = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'state')
    conv = ('x', 'weight', 'bias', 'state')
    return [(selective_scan, a, scan), (selective_step, row, scan),
            (causal_conv, c, conv), (causal_conv_step, step, conv)]


def refuse_duals(device):
    for call, args, names in calls(device):
        for name in names:
            with fwd.dual_level():
                dual = fwd.make_dual(args[name].clone(), torch.ones_like(args[name]))
                with torch.no_grad(), pytest.raises(ValueError, match='forward-mode'):
                    call(**{**args, name: dual})
        assert call(**args) is not None


@pytest.mark.skipif(not ops.available(), reason='extension not built')
def test_extension_refuses_forward_mode():
    """The refusal comes before the extension looks at the device."""
    ext = ops.require()
    x = torch.zeros(2, 8)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match='causal_conv_step: has no forward-mode'):
            ext.causal_conv_step(torch.zeros(2, 3, 8), dual, torch.zeros(8, 4), None, None, True)
    with pytest.raises(ValueError, match='must be on the GPU'):
        ext.causal_conv_step(torch.zeros(2, 3, 8), x, torch.zeros(8, 4), None, None, True)


def test_eager_forward_mode():
    """On the CPU the derivative is the formula's: as one step's difference of a linear map."""
    a, _ = make_scan(2, 3, 8, 4)
    a = move(a, double=True)
    moved = torch.ones_like(a['x'])
    with fwd.dual_level():
        y, _ = selective_scan(**{**a, 'x': fwd.make_dual(a['x'], moved)})
        got = fwd.unpack_dual(y).tangent
    want = selective_scan(**{**a, 'x': a['x'] + moved})[0] - selective_scan(**a)[0]
    torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-10)


@gpu
def test_kernels_refuse_forward_mode():
    refuse_duals('cuda')


@gpu
@pytest.mark.parametrize('which', ['scan', 'conv'])
def test_captured_backward_beside_an_eager_graph(which):
    """Refused while the eager graph of the same leaf lives, and right once it is gone."""
    make, call = (make_scan, selective_scan) if which == 'scan' else (make_conv, causal_conv)
    a, (dy, _) = make(2, 21, 16, 4)
    a, dy = move(a, 'cuda'), dy.cuda()
    leaf = a['x'].requires_grad_()
    kept = call(**a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(**a)
        with pytest.raises(RuntimeError, match='living eager graph'):
            torch.autograd.grad(out[0], leaf, dy)
    want, = torch.autograd.grad(kept[0], leaf, dy)
    del kept, out, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(call(**a)[0], leaf, dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_launches_past_their_limit():
    """2^32 threads: refused before anything is allocated."""
    x = torch.zeros(1, 1, 2048, device='cuda', dtype=torch.bfloat16).expand(1 << 22, 1, 2048)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(ValueError, match='causal_conv: too large for one launch'):
        causal_conv(x, torch.zeros(2048, 4, device='cuda'))
    x = x[:, :, :8]
    for rows, groups in ((1 << 22, 8), (1 << 24, 1)):
        b = torch.zeros(1, 1, 1, 1, device='cuda', dtype=x.dtype).expand(rows, 1, groups, 1)
        u = x[:1].expand(rows, 1, 8)
        with pytest.raises(ValueError, match='selective_scan: too large for one launch'):
            selective_scan(u, u, -torch.ones(8, 1, device='cuda'), b, b)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


@gpu
def test_gradients_of_more_parts_than_a_launch_holds():
    """2^28 rates in the sums that finish the backward pass: as two halves of them."""
    g = torch.Generator('cuda').manual_seed(0)
    width = (1 << 22) + 64
    r = lambda *s: torch.randn(*s, device='cuda', generator=g)
    a = dict(x=r(1, 1, width), dt=r(1, 1, width).abs(), A=-r(width, 64).abs(), B=r(1, 1, 64),
             C=r(1, 1, 64), D=r(width), state=r(1, width, 64))
    dy, dlast = r(1, 1, width), r(1, width, 64)
    got = run_scan(a, dy, dlast)
    half = width // 2
    for part in (slice(0, half), slice(half, width)):
        cut = {k: v if k in 'BC' else v[part] if k in 'AD' else v[:, part] if k == 'state'
               else v[:, :, part] for k, v in a.items()}
        one = run_scan(cut, dy[:, :, part], dlast[:, part])
        for k, v in one.items():
            if k in ('x', 'dt', 'y'):
                assert torch.equal(got[k][:, :, part], v), k
            elif k in ('state', 'last'):
                assert torch.equal(got[k][:, part], v), k
            elif k in 'AD':
                assert torch.equal(got[k][part], v), k
        del one, cut


def check_core_type(dtype, device):
    """Parameters of another type, against a core in 64 bits that holds the same
    values.  Some nine roundings to `dtype` stand between an input and its output
    (projections, convolution, B, C, dt, y), each of half a step, and what follows
    makes at most twice as much of it (the slopes of silu and softplus are below
    1.1, products take two factors): 18 half steps of the outputs' size; for
    sums over 32 bits inside as many again."""
    torch.manual_seed(0)
    core = SelectiveCore(24, states=8).to(device).to(dtype)
    exact = SelectiveCore(24, states=8).double()
    exact.load_state_dict({k: v.double().cpu() for k, v in core.state_dict().items()})
    x = torch.randn(6, 17, 24, device=device, dtype=dtype)
    mask = torch.rand(6, 17, device=device) < 0.8
    hidden = core.init_hidden([6])
    real = torch.float64 if dtype == torch.float64 else torch.float32
    assert hidden[0].dtype == dtype and hidden[1].dtype == real
    y, end = core.window(x, hidden, mask)
    assert y.dtype == end[0].dtype == dtype and end[1].dtype == real
    want, last = exact.window(x.double().cpu(), exact.init_hidden([6]), mask.cpu())
    y.float().square().sum().backward()
    want.square().sum().backward()
    half = torch.finfo(dtype).eps / 2
    near = lambda a, b, k: (a.double().cpu() - b).norm() <= (k * half + 1e-6) * b.norm()
    assert near(y, want, 36) and near(end[0], last[0], 36) and near(end[1], last[1], 36)
    for (name, p), q in zip(core.named_parameters(), exact.parameters()):
        # y^2 doubles what y is off by, and the gradient walks the same way back
        assert p.grad.dtype == dtype and near(p.grad, q.grad, 108), name
    with torch.no_grad():
        held = core.init_hidden([6])
        for t in range(17):
            one = core.step_(x[:, t], held, mask[:, t])
            assert one.dtype == dtype
            assert near(one[mask[:, t]], want[:, t][mask[:, t].cpu()], 72)
        assert near(held[0], last[0], 36) and near(held[1], last[1], 36)
        assert core(x[:, 0])[0].dtype == dtype


@pytest.mark.parametrize('dtype', [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_core_type(dtype):
    check_core_type(dtype, 'cpu')


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_kernel_core_type(dtype):
    check_core_type(dtype, 'cuda')


# ---- steps of so many rows that a lane takes several: from 2^20 lanes (scan) and
# 2^20 values (convolution) on

def row_mask(kind, batch):
    return dict(none=None, alternate=torch.arange(batch) % 2 == 1, runs=torch.arange(batch) % 7 < 3,
                few=torch.arange(batch) % 64 == 63)[kind]


def check_rows(state, before, y, mask):
    """Rows of mask 0 keep every bit of their state and give 0."""
    if mask is not None:
        assert torch.equal(state[~mask], before[~mask]) and (y[~mask] == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('kind', ['none', 'alternate', 'runs', 'few'])
@pytest.mark.parametrize('batch, width, states, groups', [
    (4099, 64, 16, 1), (8191, 33, 16, 3), (4099, 128, 5, 2), (8191, 40, 13, 1), (4097, 17, 64, 1)])
def test_scan_steps_of_many_rows(batch, width, states, groups, kind, dtype):
    a, (dy, dlast) = make_scan(batch, 1, width, states, groups, share=1.0, dtype=dtype)
    if (mask := row_mask(kind, batch)) is not None:
        a['mask'] = mask[:, None]
    y, last = selective_scan(**move(a, double=True))
    size = scan_by_hand(a, dy, dlast, absolute=True)
    row = {k: v[:, 0] if k in ('x', 'dt', 'B', 'C', 'z', 'mask') else v for k, v in move(a, 'cuda').items()}
    held = row['state'].clone()
    got = selective_step(**{**row, 'state': held})
    check_rows(held, row['state'], got, row.get('mask'))
    assert_results(dict(y=got[:, None], last=held), dict(y=y, last=last), size, a)


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('kind', ['none', 'alternate', 'runs', 'few'])
@pytest.mark.parametrize('batch, width, taps', [(4099, 256, 4), (8191, 129, 3), (8190, 130, 2)])
def test_conv_steps_of_many_rows(batch, width, taps, kind, dtype):
    a, _ = make_conv(batch, 1, width, taps, share=1.0, dtype=dtype)
    mask = row_mask(kind, batch)
    row = {k: v[:, 0] if k == 'x' else v for k, v in a.items()}
    wide = move(row, double=True)
    want = wide['state'].clone()
    y = causal_conv_step(**{**wide, 'state': want}, mask=mask)
    row = move(row, 'cuda')
    held = row['state'].clone()
    got = causal_conv_step(**{**row, 'state': held}, mask=None if mask is None else mask.cuda())
    check_rows(held, row['state'], got, None if mask is None else mask.cuda())
    assert torch.equal(held.double().cpu(), want)           # inputs move on as they are
    terms = torch.cat([wide['state'], wide['x'][:, None]], 1).abs() * wide['weight'].abs().t()
    # a few operations on each term; silu moves by at most 1.1 of what it takes
    tol = STEP * 24 * 1.1 * (terms.sum(1) + wide['bias'].abs()) + torch.finfo(dtype).eps / 2 * y.abs()
    assert ((got.double().cpu() - y).abs() <= tol).all()


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('case', [
    dict(batch=1, steps=1100, width=24, states=16),             # 35 segments of 2 chunks, the last of 1
    dict(batch=1, steps=3300, width=6, states=3, groups=2),     # 52 of 4, the last of 3
    dict(batch=2, steps=1500, width=20, states=30, share=1.0, gate=False),      # 47 of 2
    dict(batch=12, steps=940, width=33, states=36),             # 20 of 3, the last of 2, 3 tiles
    dict(batch=6, steps=2100, width=70, states=8, groups=2, state=False, plain=True)])   # 44 of 3
def test_segments_of_several_chunks(case, dtype):
    a, grads = make_scan(dtype=dtype, **case)
    assert_scan(a, *grads)


@gpu
@pytest.mark.parametrize('case', [
    # more items than parts: a lane walks several
    dict(batch=300, steps=100, width=6, taps=4), dict(batch=300, steps=100, width=5, taps=3, share=0.2),
    dict(batch=40, steps=130, width=1030, taps=2, share=1.0, state=False),
    # 2^18 lanes: tiles of 32 and 64 steps, the last one short, two channels a lane and one
    dict(batch=100, steps=130, width=1200, taps=4), dict(batch=100, steps=130, width=1752, taps=4, share=0.2),
    dict(batch=64, steps=130, width=1367, taps=3), dict(batch=64, steps=167, width=1367, taps=4, share=1.0)])
def test_conv_of_many_tiles(case):
    dtype = torch.bfloat16 if case['taps'] == 4 else torch.float32
    a, grads = make_conv(dtype=dtype, **case)
    assert_conv(a, *grads)


@gpu
def test_eager_passes_while_another_thread_captures():
    """As the learner trains while an actor thread captures its graph."""
    made = [make_scan(2, 40, 32, 8, seed=s) for s in (0, 1)]
    (a, dy, dlast), (b, ey, elast) = (
        (move(a, 'cuda'), dy.cuda(), dlast.cuda()) for a, (dy, dlast) in made)
    want, there = run_scan(a, dy, dlast), run_scan(b, ey, elast)
    got, failed = [], []

    def train():
        try:
            got.extend(run_scan(a, dy, dlast) for _ in range(3))
        except Exception as e:          # noqa: BLE001 - raised again below
            failed.append(e)

    thread = threading.Thread(target=train)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode='thread_local'):
        one = run_scan(b, ey, elast)
        thread.start()
        thread.join()
        two = run_scan(b, ey, elast)
    assert not failed, failed
    graph.replay()
    torch.cuda.synchronize()
    for run in got:
        assert all(torch.equal(run[k], v) for k, v in want.items())
    for run in (one, two):
        assert all(torch.equal(run[k], v) for k, v in there.items())


@gpu
def test_scan_past_32_bit_offsets_to_the_bit():
    """2.4e9 values a tensor.  Three rows are cut as one is, 64 segments of 1024
    chunks, so the last row gives every bit that it gives alone."""
    shape = (3, 1 << 20, 768)
    g = torch.Generator('cuda').manual_seed(0)
    wide = torch.randn(shape[1:], device='cuda', generator=g).bfloat16()
    x = torch.empty(shape, device='cuda', dtype=torch.bfloat16)
    for b in range(3):
        x[b] = wide.roll(b, 0)
    A = -torch.rand(768, 2, device='cuda', generator=g) - 0.5
    B = torch.randn(3, shape[1], 2, device='cuda', generator=g).bfloat16()

    def run(x, B):
        leaves = x.detach().requires_grad_(), B.detach().requires_grad_()
        y, last = selective_scan(leaves[0], x, A, leaves[1], B, dt_softplus=True)
        return y.detach(), last.detach(), *torch.autograd.grad(y, leaves, x)

    alone = run(x[2:], B[2:])
    for a, b in zip(run(x, B), alone):
        assert torch.equal(a[2:], b)
