"""Short causal convolution and selective scan: the eager path against the
formulas written out in 64 bits (and their gradients by hand and by
differences), refusals, and (gpu) the HIP kernels against the eager path in
64 bits.

Tolerances.  ``scan_by_hand(absolute=True)`` sums the magnitudes of all terms
of a result, so that an error of k half steps (2^-24) in each term and in the
sums' order is at most k * 2^-24 times it.  A step's decay exp(d A) adds 2 half
steps and those of d A, which count at most once over a whole decay; two
recurrences follow each other in a gradient: k = 4 T + 64, and the sum over
channels (in trees over 64 and then over tiles) adds D / 8.
"""

import pytest
import torch

from handyrl_amd.models.selective import (
    SelectiveCore, causal_conv, causal_conv_step, selective_scan, selective_step)

STEP = 2.0 ** -24


def seen(batch, steps, share, g):
    """Random holes, padding behind an end, and one row that sees nothing."""
    if share >= 1:
        return None
    m = torch.rand(batch, steps, generator=g) < share
    m &= torch.arange(steps) < torch.randint(1, steps + 1, (batch, 1), generator=g)
    m[-1] = False
    return m


def make_scan(batch, steps, width, states, groups=1, *, gate=True, state=True, share=0.7,
              plain=False, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    a = dict(x=r(batch, steps, width).to(dtype), dt=(r(batch, steps, width) - 2).to(dtype),
             A=-torch.rand(width, states, generator=g) * 4 - 0.05,
             B=r(batch, steps, groups, states).to(dtype), C=r(batch, steps, groups, states).to(dtype))
    if plain:
        a['dt'] = torch.nn.functional.softplus(a['dt'].float()).to(dtype)
    else:
        a.update(D=r(width), dt_bias=r(width) * 0.3, dt_softplus=True)
    if gate:
        a['z'] = r(batch, steps, width).to(dtype)
    if state:
        a['state'] = r(batch, width, states)
    if (m := seen(batch, steps, share, g)) is not None:
        a['mask'] = m
    grads = r(batch, steps, width).to(dtype), r(batch, width, states)
    return a, grads


def move(a, device=None, double=False):
    def one(v):
        if not torch.is_tensor(v):
            return v
        v = v.detach()
        v = v.double() if double and v.is_floating_point() else v
        return v.to(device) if device else v
    return {k: one(v) for k, v in a.items()}


def scan_by_hand(a, dy, dlast, absolute=False):
    """Outputs and gradients step by step in 64 bits; or the sums of magnitudes."""
    a = move(a, 'cpu', True)
    mag = torch.abs if absolute else (lambda v: v)
    x, B, C = mag(a['x']), mag(a['B']), mag(a['C'])
    A, dy, dlast = a['A'], mag(dy.double().cpu()), mag(dlast.double().cpu())
    batch, steps, width = x.shape
    groups, states = B.shape[2:]
    D = mag(a['D']) if 'D' in a else torch.zeros(width, dtype=torch.float64)
    mask = a.get('mask', torch.ones(batch, steps, dtype=torch.bool))
    raw = a['dt'] + a.get('dt_bias', 0)
    soft = a.get('dt_softplus', False)
    d = torch.log1p(torch.exp(raw)) if soft else raw
    wide = lambda v: v.repeat_interleave(width // groups, 1)
    h = mag(a['state']) if 'state' in a else torch.zeros(batch, width, states, dtype=torch.float64)
    hs, pre = [h], torch.zeros_like(x)
    for t in range(steps):
        new = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * wide(B[:, t])
        h = torch.where(mask[:, t, None, None], new, h)
        hs.append(h)
        pre[:, t] = (h * wide(C[:, t])).sum(-1) + D * x[:, t]
    on = mask[..., None]
    z = a.get('z')
    sig = torch.sigmoid(z) if z is not None else None
    gate = mag(z * sig) if z is not None else torch.ones_like(x)
    out = dict(y=torch.where(on, pre * gate, 0), last=h)
    g = torch.where(on, dy * gate, 0)
    out.update(x=g * D, dt=torch.zeros_like(x), B=torch.zeros_like(B), C=torch.zeros_like(C),
               A=torch.zeros_like(A), D=(g * torch.where(on, x, 0)).sum((0, 1)))
    if z is not None:
        # silu'(z) = sig + sig z (1 - sig): two terms, of opposite sign for z < 0, whose
        # magnitudes add up to sig (1 + |z| (1 - sig)) while their sum passes 0 at z = -1.28
        out['z'] = torch.where(on, dy * pre * sig * (1 + mag(z) * (1 - sig)), 0)
    carry = dlast
    for t in reversed(range(steps)):
        here = mask[:, t, None, None]
        e, u, b = d[:, t, :, None], x[:, t, :, None], wide(B[:, t])
        decay = torch.exp(e * A)
        lam = torch.where(here, carry + wide(C[:, t]) * g[:, t, :, None], 0)
        fold = lambda v: v.view(batch, groups, -1, states).sum(2)
        out['C'][:, t] = fold(g[:, t, :, None] * hs[t + 1])
        out['B'][:, t] = fold(lam * e * u)
        out['x'][:, t] += (lam * e * b).sum(-1)
        out['dt'][:, t] = (lam * (mag(A) * decay * hs[t] + u * b)).sum(-1)
        out['A'] += (lam * e * decay * hs[t]).sum(0)
        carry = torch.where(here, decay * lam, carry)
    if soft:
        out['dt'] = out['dt'] * torch.sigmoid(raw)
    out.update(dt_bias=out['dt'].sum((0, 1)), state=carry)
    return out


def run_scan(a, dy, dlast, names=('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'state')):
    leaves = {k: a[k].detach().requires_grad_() for k in names if k in a}
    y, last = selective_scan(**{**a, **leaves})
    grads = torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])
    return dict(y=y.detach(), last=last.detach(), **dict(zip(leaves, grads)))


SMALL = [dict(batch=2, steps=5, width=6, states=3, groups=2),
         dict(batch=3, steps=4, width=3, states=1, gate=False, state=False, share=1.0),
         dict(batch=2, steps=3, width=4, states=2, plain=True)]


@pytest.mark.parametrize('case', SMALL)
def test_eager_scan_matches_formula(case):
    a, (dy, dlast) = make_scan(**case)
    a, dy, dlast = move(a, double=True), dy.double(), dlast.double()
    want = scan_by_hand(a, dy, dlast)
    for k, v in run_scan(a, dy, dlast).items():
        # 64-bit sums of a few terms of order 1
        torch.testing.assert_close(v, want[k], rtol=1e-12, atol=1e-12, msg=k)


@pytest.mark.parametrize('case', SMALL)
def test_eager_scan_gradient_matches_differences(case):
    a, _ = make_scan(**case)
    a = move(a, double=True)
    names = [k for k in a if torch.is_tensor(a[k]) and a[k].is_floating_point()]
    assert torch.autograd.gradcheck(
        lambda *v: selective_scan(**{**a, **dict(zip(names, v))}),
        [a[k].requires_grad_() for k in names])


def make_conv(batch, steps, width, taps, *, bias=True, state=True, share=0.7, silu=True,
              dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    a = dict(x=r(batch, steps, width).to(dtype), weight=r(width, taps),
             activation='silu' if silu else None)
    if bias:
        a['bias'] = r(width)
    if state:
        a['state'] = r(batch, taps - 1, width).to(dtype)
    if (m := seen(batch, steps, share, g)) is not None:
        a['mask'] = m
    return a, (r(batch, steps, width).to(dtype), r(batch, taps - 1, width).to(dtype))


def conv_by_hand(a, dy, dlast, absolute=False):
    """Row by row over the observed inputs alone; or the sums of magnitudes."""
    a = move(a, 'cpu', True)
    mag = torch.abs if absolute else (lambda v: v)
    x, w, dy, dlast = a['x'], a['weight'], dy.double().cpu(), dlast.double().cpu()
    batch, steps, width = x.shape
    taps = w.size(1)
    bias = a.get('bias', torch.zeros(width, dtype=torch.float64))
    state = a.get('state', torch.zeros(batch, taps - 1, width, dtype=torch.float64))
    mask = a.get('mask', torch.ones(batch, steps, dtype=torch.bool))
    out = {k: torch.zeros_like(v) for k, v in
           dict(y=x, last=state, x=x, weight=w, bias=bias, state=state).items()}
    for b in range(batch):
        at = mask[b].nonzero()[:, 0].tolist()
        u = torch.cat([state[b], x[b, at]])
        du = torch.zeros_like(u)
        for i, t in enumerate(at):
            terms = u[i:i + taps] * w.t()
            pre = terms.sum(0) + bias
            sig = torch.sigmoid(pre)
            silu = a['activation'] == 'silu'
            size = mag(terms).sum(0) + mag(bias)
            slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
            if absolute:
                # silu and its slope move by at most 1.1 and 0.5 of what `pre` does
                out['y'][b, t] = 1.1 * size if silu else size
                g = dy[b, t].abs() * (slope.abs() + (0.5 * size if silu else 0))
            else:
                out['y'][b, t] = pre * sig if silu else pre
                g = dy[b, t] * slope
            out['weight'] += (g * mag(u[i:i + taps])).t()
            out['bias'] += g
            du[i:i + taps] += g * mag(w.t())
        du[len(at):] += mag(dlast[b])
        out['last'][b] = mag(u[len(at):])
        out['state'][b] = du[:taps - 1]
        out['x'][b, at] = du[taps - 1:]
    return out


def run_conv(a, dy, dlast):
    leaves = {k: a[k].detach().requires_grad_() for k in ('x', 'weight', 'bias', 'state') if k in a}
    y, last = causal_conv(**{**a, **leaves})
    grads = torch.autograd.grad([y, last], list(leaves.values()), [dy, dlast])
    return dict(y=y.detach(), last=last.detach(), **dict(zip(leaves, grads)))


CONVS = [dict(batch=3, steps=7, width=5, taps=4), dict(batch=2, steps=2, width=3, taps=4),
         dict(batch=2, steps=6, width=2, taps=2, silu=False, bias=False, state=False, share=1.0),
         dict(batch=4, steps=9, width=3, taps=3, share=0.3)]


@pytest.mark.parametrize('case', CONVS)
def test_eager_conv_matches_formula(case):
    a, (dy, dlast) = make_conv(**case)
    a, dy, dlast = move(a, double=True), dy.double(), dlast.double()
    want = conv_by_hand(a, dy, dlast)
    for k, v in run_conv(a, dy, dlast).items():
        torch.testing.assert_close(v, want[k], rtol=1e-12, atol=1e-12, msg=k)


def without_holes(a, names, value=float('nan')):
    """The same call with NaN wherever nothing is observed."""
    a = dict(a)
    for k in names:
        if k in a:
            a[k] = a[k].clone()
            a[k][~a['mask']] = value
    return a


def check_holes(device):
    a, (dy, dlast) = make_scan(3, 21, 12, 5, groups=2)
    a, dy, dlast = move(a, device), dy.to(device), dlast.to(device)
    want = run_scan(a, dy, dlast)
    for value in (float('nan'), float('inf'), torch.finfo(torch.float32).min):
        spoilt = without_holes(a, ('x', 'dt', 'B', 'C', 'z'), value)
        got = run_scan(spoilt, torch.where(a['mask'][..., None], dy, value), dlast)
        for k, v in want.items():
            assert torch.equal(got[k], v), k
    a, (dy, dlast) = make_conv(3, 21, 12, 4)
    a, dy, dlast = move(a, device), dy.to(device), dlast.to(device)
    want = run_conv(a, dy, dlast)
    got = run_conv(without_holes(a, ('x',)), torch.where(a['mask'][..., None], dy, float('nan')), dlast)
    for k, v in want.items():
        assert torch.equal(got[k], v), k
    # nothing observed: the state passes through, and its gradient back
    assert torch.equal(want['last'][-1], a['state'][-1]) and (want['y'][-1] == 0).all()
    assert torch.equal(want['state'][-1], dlast[-1])


def test_eager_holes():
    check_holes('cpu')


def check_steps(device, dtype, make=None):
    """The step forms give what the windows give, and so does a cut window."""
    out = torch.finfo(dtype).eps / 2
    a, _ = make_scan(5, 19, 40, 16, groups=2, dtype=dtype)
    a = move(a, device)
    y, last = selective_scan(**a)
    held, state = a['state'].clone(), a['state']
    for t in range(19):
        row = {k: a[k][:, t] for k in ('x', 'dt', 'B', 'C', 'z', 'mask')}
        step = selective_step(held, A=a['A'], D=a['D'], dt_bias=a['dt_bias'], dt_softplus=True, **row)
        one, state = selective_scan(
            **{**a, **{k: v[:, None] for k, v in row.items()}, 'state': state})
        # the same operations in the same order up to contraction: 64 half steps of values of order 10
        tol = dict(rtol=2 * out, atol=64 * STEP * 10)
        torch.testing.assert_close(step, y[:, t], **tol)
        torch.testing.assert_close(one[:, 0], y[:, t], **tol)
    for h in (held, state):
        torch.testing.assert_close(h, last, rtol=64 * STEP, atol=64 * STEP * 10)
    a, _ = make_conv(5, 19, 40, 4, dtype=dtype)
    a = move(a, device)
    y, last = causal_conv(**a)
    held = a['state'].clone()
    params = {k: a[k] for k in ('weight', 'bias', 'activation')}
    for t in range(19):
        step = causal_conv_step(held, a['x'][:, t], mask=a['mask'][:, t], **params)
        torch.testing.assert_close(step, y[:, t], rtol=2 * out, atol=64 * STEP * 10)
    assert torch.equal(held, last)
    cut, mid = causal_conv(a['x'][:, :7], mask=a['mask'][:, :7], state=a['state'], **params)
    rest, end = causal_conv(a['x'][:, 7:], mask=a['mask'][:, 7:], state=mid, **params)
    torch.testing.assert_close(torch.cat([cut, rest], 1), y, rtol=2 * out, atol=64 * STEP * 10)
    assert torch.equal(end, last)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_eager_steps(dtype):
    check_steps('cpu', dtype)


def check_empty(device):
    for batch, steps in ((0, 3), (2, 0)):
        a, (dy, dlast) = make_scan(batch, steps, 8, 4, share=1.0)
        a, dy, dlast = move(a, device), dy.to(device), dlast.to(device)
        if device != 'cpu':                     # the eager loop leaves what it never meets unused
            got = run_scan(a, dy, dlast)
            assert torch.equal(got['state'], dlast) and (got['A'] == 0).all()
            assert got['y'].shape == a['x'].shape and torch.equal(got['last'], a['state'])
        y, last = selective_scan(**a)
        assert y.shape == a['x'].shape and torch.equal(last, a['state'])
        a, (dy, dlast) = make_conv(batch, steps, 8, 3, share=1.0)
        a, dy, dlast = move(a, device), dy.to(device), dlast.to(device)
        y, last = causal_conv(**a)
        assert y.shape == a['x'].shape and torch.equal(last, a['state'])
    a, _ = make_scan(0, 1, 8, 4, share=1.0)
    a = move(a, device)
    row = {k: a[k][:, 0] for k in ('x', 'dt', 'B', 'C', 'z')}
    assert selective_step(a['state'], A=a['A'], **row).shape == (0, 8)


def test_eager_empty():
    check_empty('cpu')


def refusals():
    z = torch.zeros
    scan = dict(x=z(2, 3, 4), dt=z(2, 3, 4), A=z(4, 5), B=z(2, 3, 5), C=z(2, 3, 5))
    step = dict(state=z(2, 4, 5), x=z(2, 4), dt=z(2, 4), A=z(4, 5), B=z(2, 5), C=z(2, 5))
    conv = dict(x=z(2, 3, 4), weight=z(4, 3))
    conv_step = dict(state=z(2, 2, 4), x=z(2, 4), weight=z(4, 3))
    for call, base, changes in [
        (selective_scan, scan, [
            (dict(x=z(2, 3)), 'x must be'), (dict(x=z(2, 3, 4).long()), 'x must be'),
            (dict(dt=z(2, 3, 1)), 'dt must have shape'), (dict(dt=z(2, 3, 4).half()), 'dt must be'),
            (dict(A=z(4, 65)), '1 to 64 states'), (dict(A=z(4, 0)), '1 to 64 states'),
            (dict(A=z(3, 5)), 'A must have shape'), (dict(A=z(4, 5).half()), 'A must be'),
            (dict(B=z(2, 3, 3, 5)), 'groups that divide'), (dict(B=z(2, 3, 0, 5)), 'groups that divide'),
            (dict(B=z(2, 3, 4)), 'B must have shape'), (dict(C=z(2, 3, 2, 5)), 'C must have shape'),
            (dict(C=z(2, 3, 5).half()), 'C must be'), (dict(D=z(5)), 'D must have shape'),
            (dict(z=z(2, 3, 5)), 'z must have shape'), (dict(dt_bias=z(1)), 'dt_bias must have shape'),
            (dict(state=z(2, 4, 4)), 'state must have shape'),
            (dict(state=z(2, 4, 5).half()), 'state must be'),
            (dict(mask=z(2, 4)), 'mask must have shape')]),
        (selective_step, step, [
            (dict(state=z(2, 5, 4).mT), 'contiguous'), (dict(state=z(3, 4, 5)), 'state must have shape'),
            (dict(x=z(2, 4).requires_grad_()), 'has no gradient'), (dict(mask=z(3)), 'mask must have')]),
        (causal_conv, conv, [
            (dict(x=z(3, 4)), 'x must be'), (dict(weight=z(4, 5)), '2 to 4 taps'),
            (dict(weight=z(4, 1)), '2 to 4 taps'), (dict(weight=z(3, 3)), 'weight must have shape'),
            (dict(bias=z(3)), 'bias must have shape'), (dict(weight=z(4, 3).half()), 'weight must be'),
            (dict(state=z(2, 3, 4)), 'state must have shape'),
            (dict(state=z(2, 2, 4).half()), 'state must be'),
            (dict(mask=z(3, 3)), 'mask must have shape'), (dict(activation='relu'), 'activation')]),
        (causal_conv_step, conv_step, [
            (dict(state=z(2, 4, 2).mT), 'contiguous'), (dict(state=z(2, 3, 4)), 'state must have shape'),
            (dict(weight=z(4, 3).requires_grad_()), 'has no gradient')]),
    ]:
        for change, match in changes:
            yield pytest.param(call, {**base, **change}, match, id='%s-%s' % (call.__name__, match))


def refuse(call, args, match, device):
    args = {k: v.detach().to(device).requires_grad_(v.requires_grad) if torch.is_tensor(v) else v
            for k, v in args.items()}
    if match == 'contiguous':                   # a copy to the GPU keeps the strides
        assert not args['state'].is_contiguous()
    with pytest.raises(ValueError, match=match):
        call(**args)


@pytest.mark.parametrize('call, args, match', refusals())
def test_refusals(call, args, match):
    refuse(call, args, match, 'cpu')


def check_core(device):
    """A window through the core is its steps; its gradients reach everything."""
    torch.manual_seed(0)
    core = SelectiveCore(24, states=8).to(device)
    x = torch.randn(6, 17, 24, device=device)
    mask = torch.rand(6, 17, device=device) < 0.8
    hidden = core.init_hidden([6])
    y, end = core.window(x, hidden, mask)
    (y.square().sum() + end[1].sum()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.abs().sum() > 0
               for p in core.parameters())
    with torch.no_grad():
        held = tuple(h.clone() for h in hidden)
        for t in range(17):
            one = core.step_(x[:, t], held, mask[:, t])
            both, after = core(x[:, t], hidden)
            # values of order 1 through products over 24 to 56 terms on either side
            torch.testing.assert_close(one[mask[:, t]], y[:, t][mask[:, t]], rtol=1e-4, atol=1e-5)
            torch.testing.assert_close(both[mask[:, t]], one[mask[:, t]], rtol=1e-4, atol=1e-5)
            on = mask[:, t, None, None]
            hidden = tuple(torch.where(on, n, o) for n, o in zip(after, hidden))
        for a, b, c in zip(held, end, hidden):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)
            torch.testing.assert_close(c, b, rtol=1e-4, atol=1e-5)
    with torch.enable_grad():
        one, _ = core(x[:, 0], hidden)
        assert one.requires_grad


def test_core():
    check_core('cpu')


# ------------------------------------------------------------------- GPU

gpu = pytest.mark.gpu


def assert_scan(a, dy, dlast):
    steps, width = a['x'].shape[1:]
    got = run_scan(move(a, 'cuda'), dy.cuda(), dlast.cuda())
    want = run_scan(move(a, double=True), dy.double(), dlast.double())
    size = scan_by_hand(a, dy, dlast, absolute=True)
    for k, v in got.items():
        assert v.dtype == (a['x'].dtype if k in ('y', 'last') and k == 'y' else
                           torch.float32 if k == 'last' else a[k].dtype), k
        out = torch.finfo(v.dtype).eps / 2
        off = (v.double().cpu() - want[k]).abs()
        tol = STEP * (4 * steps + 64 + width / 8) * size[k] + out * want[k].abs() + 1e-37
        assert torch.all(off <= tol), (k, float((off / tol).max()))


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('case', [
    dict(batch=1, steps=1, width=1, states=1), dict(batch=2, steps=1, width=64, states=16),
    dict(batch=3, steps=15, width=5, states=3, share=1.0),
    dict(batch=2, steps=16, width=64, states=16, share=1.0, state=False),
    dict(batch=2, steps=17, width=65, states=4), dict(batch=3, steps=33, width=130, states=5, groups=2),
    dict(batch=2, steps=50, width=257, states=8, gate=False),
    dict(batch=2, steps=40, width=48, states=24, groups=3), dict(batch=2, steps=37, width=36, states=33),
    dict(batch=2, steps=70, width=40, states=64, groups=2), dict(batch=2, steps=20, width=300, states=2),
    dict(batch=2, steps=30, width=20, states=16, plain=True, state=False, gate=False, share=1.0),
    dict(batch=1, steps=301, width=24, states=16), dict(batch=40, steps=19, width=72, states=16)])
def test_scan_matches_64_bits(case, dtype):
    a, grads = make_scan(dtype=dtype, **case)
    assert_scan(a, *grads)


def assert_conv(a, dy, dlast):
    batch, steps, _ = a['x'].shape
    got = run_conv(move(a, 'cuda'), dy.cuda(), dlast.cuda())
    want = run_conv(move(a, double=True), dy.double(), dlast.double())
    size = conv_by_hand(a, dy, dlast, absolute=True)
    for k, v in got.items():
        out = torch.finfo(v.dtype).eps / 2
        off = (v.double().cpu() - want[k]).abs()
        # a few operations on each term; a lane adds up its share of the steps in order
        serial = batch * steps if k in ('weight', 'bias') else 0
        tol = STEP * (24 + serial) * size[k] + out * want[k].abs()
        assert torch.all(off <= tol), (k, float((off / tol).max()))


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('case', [
    dict(batch=1, steps=1, width=1, taps=2), dict(batch=3, steps=2, width=8, taps=4),
    dict(batch=2, steps=16, width=64, taps=4, share=1.0), dict(batch=2, steps=17, width=65, taps=3),
    dict(batch=5, steps=130, width=24, taps=4, share=0.2), dict(batch=2, steps=70, width=256, taps=3),
    dict(batch=2, steps=40, width=16, taps=4, silu=False, bias=False, state=False),
    dict(batch=70, steps=19, width=40, taps=2)])
def test_conv_matches_64_bits(case, dtype):
    a, grads = make_conv(dtype=dtype, **case)
    assert_conv(a, *grads)


@gpu
@pytest.mark.parametrize('where', [[], [0], [3, 4, 5, 6], [0, 1, 399], [2, 150, 151, 290], [399]])
def test_conv_through_long_gaps(where):
    a, grads = make_conv(2, 400, 6, 4)
    a['mask'][0] = False
    a['mask'][0, where] = True
    assert_conv(a, *grads)
    a, grads = make_conv(3, 413, 3, 3)          # rows of the mask begin at odd addresses
    a['mask'][1] = False
    a['mask'][1, where] = True
    assert_conv(a, *grads)
    a, grads = make_scan(2, 400, 6, 4)
    a['mask'][0] = False
    a['mask'][0, where] = True
    assert_scan(a, *grads)


@gpu
def test_kernel_holes():
    check_holes('cuda')


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_kernel_steps(dtype):
    check_steps('cuda', dtype)


@gpu
def test_kernel_empty():
    check_empty('cuda')


@gpu
@pytest.mark.parametrize('call, args, match', refusals())
def test_kernel_refusals(call, args, match):
    refuse(call, args, match, 'cuda')


@gpu
def test_kernel_core():
    check_core('cuda')


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_kernel_strides(dtype):
    """Slices of wider tensors, steps-first layouts, odd offsets: as their copies."""
    a, (dy, dlast) = make_scan(3, 21, 32, 8, groups=2, dtype=dtype)
    a, dy, dlast = move(a, 'cuda'), dy.cuda(), dlast.cuda()
    want = run_scan(a, dy, dlast)
    for pad in (4, 3):
        b = dict(a)
        for k in ('x', 'dt', 'z', 'B', 'C'):
            wide = torch.full((*a[k].shape[:-1], a[k].shape[-1] + 2 * pad), float('nan'),
                              device='cuda', dtype=dtype)
            b[k] = wide[..., pad:-pad]
            b[k].copy_(a[k])
        got = run_scan(b, dy, dlast)
        assert all(torch.equal(got[k], v) for k, v in want.items())
    b = {**a, **{k: a[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ('x', 'dt', 'z', 'B')},
         'A': a['A'].t().contiguous().t(), 'C': a['C'].transpose(2, 3).contiguous().transpose(2, 3),
         'mask': a['mask'].float().unsqueeze(-1)}
    got = run_scan(b, dy.transpose(0, 1).contiguous().transpose(0, 1), dlast)
    assert all(torch.equal(got[k], v) for k, v in want.items())
    # an expanded gradient, as a sum's
    got = run_scan(a, dy[:1, :1, :1].expand_as(dy), dlast)
    flat = run_scan(a, dy[:1, :1, :1].expand_as(dy).contiguous(), dlast)
    assert all(torch.equal(got[k], v) for k, v in flat.items())

    a, (dy, dlast) = make_conv(3, 21, 32, 4, dtype=dtype)
    a, dy, dlast = move(a, 'cuda'), dy.cuda(), dlast.cuda()
    want = run_conv(a, dy, dlast)
    for pad in (8, 3):
        wide = torch.full((3, 21, 32 + 2 * pad), float('nan'), device='cuda', dtype=dtype)
        wide[..., pad:-pad] = a['x']
        got = run_conv({**a, 'x': wide[..., pad:-pad]}, dy, dlast)
        for k, v in want.items():       # lanes of another width share the steps out differently
            torch.testing.assert_close(got[k], v, rtol=1e-5, atol=1e-4)


@gpu
def test_kernel_unused_outputs_and_inputs():
    """Gradients of y alone, of the state alone, and of some inputs alone."""
    a, (dy, dlast) = make_scan(3, 21, 32, 8)
    a, dy, dlast = move(a, 'cuda'), dy.cuda(), dlast.cuda()
    full = [run_scan(a, dy, torch.zeros_like(dlast)), run_scan(a, torch.zeros_like(dy), dlast)]
    for which, g in enumerate((dy, dlast)):
        x = a['x'].requires_grad_()
        got, = torch.autograd.grad(selective_scan(**a)[which], x, g)
        assert torch.equal(got, full[which]['x'])
        x.requires_grad_(False)
    w = a['A'].requires_grad_()
    got, = torch.autograd.grad(selective_scan(**a)[0], w, dy)
    assert torch.equal(got, full[0]['A'])
    with pytest.raises(RuntimeError, match='not differentiable again'):
        torch.autograd.grad(selective_scan(**a)[0], w, dy, create_graph=True)
    c, (dy, dlast) = make_conv(3, 21, 32, 4)
    c, dy = move(c, 'cuda'), dy.cuda()
    x = c['x'].requires_grad_()
    with pytest.raises(RuntimeError, match='not differentiable again'):
        torch.autograd.grad(causal_conv(**c)[0], x, dy, create_graph=True)


@gpu
def test_kernel_step_tells_autograd():
    state = torch.zeros(2, 8, 4, device='cuda')
    w = torch.ones(2, 8, 4, device='cuda', requires_grad=True)
    out = (w * state).sum()
    row = torch.zeros(2, 8, device='cuda')
    selective_step(state, row, row, -torch.ones(8, 4, device='cuda'),
                   row[:, :4], row[:, :4])
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.backward()
    with torch.inference_mode():
        state = torch.zeros(2, 8, 4, device='cuda')
        selective_step(state, row, row, -torch.ones(8, 4, device='cuda'), row[:, :4], row[:, :4])


@gpu
def test_kernels_in_a_graph_and_on_a_side_stream():
    made = [make_scan(4, 40, 64, 16, dtype=torch.bfloat16, seed=s) for s in (0, 1)]
    sets = [dict(move(a, 'cuda'), dy=dy.cuda(), dlast=dl.cuda()) for a, (dy, dl) in made]
    taps = make_conv(1, 1, 64, 4)[0]['weight'].cuda()
    held = {k: v.clone() if torch.is_tensor(v) else v for k, v in sets[0].items()}

    def step():
        a = {k: v for k, v in held.items() if k not in ('dy', 'dlast')}
        u = a['x'].detach().requires_grad_()
        w = taps.detach().requires_grad_()
        x, last = causal_conv(u, w, activation='silu', mask=a['mask'])
        y, state = selective_scan(**{**a, 'x': x})
        grads = torch.autograd.grad([y, state], [u, w], [held['dy'], held['dlast']])
        return [y.detach(), state.detach(), last.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(there, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in (sets[1], sets[0], sets[1]):
        for k, v in held.items():
            if torch.is_tensor(v):
                v.copy_(new[k])
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


@gpu
def test_kernels_past_32_bit_offsets():
    """2.4e9 values a tensor: the last row as it comes alone."""
    shape = (3, 1 << 20, 768)
    g = torch.Generator('cuda').manual_seed(0)
    wide = torch.randn(shape[1:], device='cuda', generator=g).bfloat16()
    x = torch.empty(shape, device='cuda', dtype=torch.bfloat16)
    for b in range(3):
        x[b] = wide.roll(b, 0)
    weight = torch.randn(768, 4, device='cuda', generator=g)
    y, last = causal_conv(x, weight, activation='silu')
    one, end = causal_conv(x[2:], weight, activation='silu')
    assert torch.equal(y[2], one[0]) and torch.equal(last[2], end[0])
    del one
    A = -torch.rand(768, 2, device='cuda', generator=g) - 0.5
    B = torch.randn(3, shape[1], 2, device='cuda', generator=g).bfloat16()
    leaf = x.requires_grad_()
    out, state = selective_scan(leaf, y, A, B, B, dt_softplus=True)
    dx, = torch.autograd.grad(out, leaf, y)
    alone = x.detach()[2:].requires_grad_()
    one, end = selective_scan(alone, y[2:], A, B[2:], B[2:], dt_softplus=True)
    d_one, = torch.autograd.grad(one, alone, y[2:])
    # another cut into segments: a rounding to bfloat16 may fall the other way
    for a, b in ((out[2], one[0]), (dx[2], d_one[0])):
        for part in (slice(0, 4096), slice(-4096, None)):
            torch.testing.assert_close(a[part], b[part], rtol=2 ** -6, atol=1e-3)
    torch.testing.assert_close(state[2], end[0], rtol=1e-4, atol=1e-4)


@gpu
@pytest.mark.parametrize('share', [0.01, 0.05, 0.5, 0.98])
@pytest.mark.parametrize('steps', [63, 64, 65, 127, 200])
@pytest.mark.parametrize('taps', [2, 3, 4])
def test_conv_through_sparse_masks(share, steps, taps):
    a, grads = make_conv(5, steps, 5, taps, share=share, state=taps != 3, seed=steps)
    assert_conv(a, *grads)
