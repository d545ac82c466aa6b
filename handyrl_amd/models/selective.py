"""Selective state space core: a short causal convolution and a selective
scan (arXiv:2312.00752), over windows of steps for the learner and as single
steps for actors.

Next to the ConvLSTM core (models/geister_net.py) this is the recurrent core
whose whole training window is one call: the state moves linearly, so the
steps of a window need not be launched one by one.

Layouts are (batch, steps, channels), channels last; one row of the batch is
one player's view of one episode.  ``mask`` (batch, steps) marks the observed
steps, as ``observation_mask`` does: an unobserved step leaves the carried
state as it is and gives 0, whatever it holds.  Its padding behind an
episode's end is of that kind.

GPU tensors go through the HIP kernels (ops/src/selective.hip), which take
float32 or bfloat16 inputs beside float32 parameters and keep the scan's state
in float32.  CPU tensors take the eager path below, which is the kernels'
oracle in tests.  On the GPU the gradients cannot be differentiated again, there
is no forward-mode derivative, and a backward pass can only be captured into a
graph if its forward pass was and no eager pass over the same inputs lives on.
"""

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops

__all__ = ['causal_conv', 'causal_conv_step', 'selective_scan', 'selective_step',
           'SelectiveCore']


def causal_conv(x, weight, bias=None, *, activation=None, state=None, mask=None):
    """y_t = act(bias + sum_k weight[:, k] u_{t-K+1+k}) over each row's
    observed steps, u being the carried inputs and then x.

    x (batch, steps, channels); weight (channels, K) with K of 2 to 4; bias
    (channels); activation None or 'silu'; state (batch, K-1, channels), the
    last inputs observed before the window, oldest first (zeros if None).
    Returns (y, last): y like x, and the state behind the window.
    """
    silu = _silu('causal_conv', activation)
    if x.is_cuda:
        ext = ops.require()
        if ext is not None:
            y, last = ext.causal_conv(x, weight, bias, state, mask, silu)
            return y, last
    mask = _check_conv('causal_conv', 3, x, weight, bias, state, mask)
    real = weight.dtype
    batch, steps, width = x.shape
    held = [] if state is None else list(state.to(real).unbind(1))
    held = held or [x.new_zeros(batch, width, dtype=real)] * (weight.size(1) - 1)
    out = []
    for t in range(steps):
        held, y = _conv_eager(held, x[:, t], weight, bias, silu, None if mask is None else mask[:, t])
        out.append(y)
    y = torch.stack(out, 1) if out else x.new_zeros(x.shape, dtype=real)
    return y.to(x.dtype), torch.stack(held, 1).to(x.dtype)


def causal_conv_step(state, x, weight, bias=None, *, activation=None, mask=None):
    """One step of ``causal_conv``: x (batch, channels), mask (batch).  Moves
    ``state`` (batch, K-1, channels; contiguous, x's type) on in place and
    returns y.  Rows of mask 0 keep their state and give 0.  Without gradient.
    """
    silu = _silu('causal_conv_step', activation)
    if x.is_cuda:
        ext = ops.require()
        if ext is not None:
            return ext.causal_conv_step(state, x, weight, bias, mask, silu)
    mask = _check_conv('causal_conv_step', 2, x, weight, bias, state, mask)
    _check_step('causal_conv_step', state, x, weight, bias)
    with torch.no_grad():
        held, y = _conv_eager(list(state.to(weight.dtype).unbind(1)), x, weight, bias, silu, mask)
        state.copy_(torch.stack(held, 1))
    return y.to(x.dtype)


def selective_scan(x, dt, A, B, C, D=None, *, z=None, dt_bias=None, dt_softplus=False,
                   state=None, mask=None):
    """With d = dt + dt_bias (softplus of it if ``dt_softplus``), per channel:

        h_t = exp(d_t A) * h_{t-1} + d_t x_t B_t
        y_t = (C_t . h_t + D x_t) * silu(z_t)

    x, dt, z (batch, steps, channels); A (channels, states) with 1 to 64
    states; B, C (batch, steps, states), or (batch, steps, groups, states)
    where each group serves channels / groups neighbouring channels; D,
    dt_bias (channels); state (batch, channels, states), float32, zeros if
    None.  Without z there is no gate.  Returns (y, last): y like x, and the
    state behind the window.
    """
    B, C = _grouped(B, x), _grouped(C, x)
    if x.is_cuda:
        ext = ops.require()
        if ext is not None:
            y, last = ext.selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, mask)
            return y, last
    mask = _check_scan('selective_scan', 3, x, dt, A, B, C, D, z, dt_bias, state, mask)
    batch, steps, width = x.shape
    h = x.new_zeros(batch, width, A.size(1), dtype=A.dtype) if state is None else state
    out = []
    for t in range(steps):
        h, y = _scan_eager(h, x[:, t], dt[:, t], A, B[:, t], C[:, t], D,
                           None if z is None else z[:, t], dt_bias, dt_softplus,
                           None if mask is None else mask[:, t])
        out.append(y)
    y = torch.stack(out, 1) if out else x.new_zeros(x.shape)
    return y.to(x.dtype), h.clone() if h is state else h


def selective_step(state, x, dt, A, B, C, D=None, *, z=None, dt_bias=None, dt_softplus=False,
                   mask=None):
    """One step of ``selective_scan``: x, dt, z (batch, channels), B, C
    (batch, states) or (batch, groups, states), mask (batch).  Moves ``state``
    (batch, channels, states; contiguous, float32) on in place and returns y.
    Rows of mask 0 keep their state and give 0.  Without gradient.
    """
    B, C = _grouped(B, x), _grouped(C, x)
    if x.is_cuda:
        ext = ops.require()
        if ext is not None:
            return ext.selective_step(state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, mask)
    mask = _check_scan('selective_step', 2, x, dt, A, B, C, D, z, dt_bias, state, mask)
    _check_step('selective_step', state, x, dt, A, B, C, D, z, dt_bias)
    with torch.no_grad():
        h, y = _scan_eager(state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, mask)
        state.copy_(h)
    return y.to(x.dtype)


class SelectiveCore(nn.Module):
    """Recurrent core of a policy network, used as the ConvLSTM core is:

        core = SelectiveCore(width)
        hidden = core.init_hidden([batch])
        y, hidden = core(x, hidden)                 # x (batch, width): a step
        y, hidden = core.window(x, hidden, mask)    # x (batch, steps, width)

    ``window`` gives what ``forward`` gives step by step where the mask is 1,
    and carries ``hidden`` past the other steps.  Without gradient ``forward``
    takes the step kernels on a copy of ``hidden``; ``step_`` moves it on in
    place, for actors that keep it resident.

    Parameters may be of any floating type: the operators take them, and carry
    the scan's state, in 64 bits if they are that wide and in 32 bits otherwise.
    """

    def __init__(self, width, expand=2, states=16, taps=4, dt_rank=None):
        super().__init__()
        inner = expand * width
        self.inner, self.states, self.taps = inner, states, taps
        self.dt_rank = dt_rank if dt_rank is not None else max(1, -(-width // 16))
        self.proj_in = nn.Linear(width, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, taps).uniform_(-1, 1) * taps ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.proj_select = nn.Linear(inner, self.dt_rank + 2 * states, bias=False)
        self.proj_dt = nn.Linear(self.dt_rank, inner, bias=False)
        # steps spread from 1e-3 to 1e-1 at the start, rates from 1 to `states`
        step = torch.exp(torch.empty(inner).uniform_(-6.9, -2.3))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.log_rate = nn.Parameter(torch.log(torch.arange(1, states + 1).float()).repeat(inner, 1))
        self.skip = nn.Parameter(torch.ones(inner))
        self.proj_out = nn.Linear(inner, width, bias=False)

    def init_hidden(self, batch_size=()):
        like = self.proj_in.weight
        return (like.new_zeros(*batch_size, self.taps - 1, self.inner),
                like.new_zeros(*batch_size, self.inner, self.states, dtype=_real(like)))

    def _select(self, u):
        r, n = self.dt_rank, self.states
        dt, B, C = self.proj_select(u).split([r, n, n], -1)
        real = _real(u)
        return dict(x=u, dt=self.proj_dt(dt), A=-torch.exp(self.log_rate.to(real)), B=B, C=C,
                    D=self.skip.to(real), dt_bias=self.dt_bias.to(real), dt_softplus=True)

    def _taps(self, u):
        real = _real(u)
        return self.conv_weight.to(real), self.conv_bias.to(real)

    def window(self, x, hidden=None, mask=None):
        taken, state = (None, None) if hidden is None else hidden
        u, z = self.proj_in(x).chunk(2, -1)
        u, last = causal_conv(u, *self._taps(u), activation='silu',
                              state=None if taken is None else taken.to(u.dtype), mask=mask)
        y, state = selective_scan(**self._select(u), z=z, state=state, mask=mask)
        if taken is not None:
            last = last.to(taken.dtype)
        return self.proj_out(y), (last, state)

    def step_(self, x, hidden, mask=None):
        """One step without gradient; ``hidden`` moves on in place."""
        with torch.no_grad():
            u, z = self.proj_in(x).chunk(2, -1)
            taken = hidden[0] if hidden[0].dtype == u.dtype else hidden[0].to(u.dtype)
            u = causal_conv_step(taken, u, *self._taps(u), activation='silu', mask=mask)
            if taken is not hidden[0]:
                hidden[0].copy_(taken)
            y = selective_step(hidden[1], **self._select(u), z=z, mask=mask)
            return self.proj_out(y)

    def forward(self, x, hidden=None):
        if hidden is None:
            hidden = self.init_hidden(x.shape[:-1])
        if torch.is_grad_enabled():
            y, hidden = self.window(x.unsqueeze(1), hidden)
            return y.squeeze(1), hidden
        hidden = tuple(h.clone(memory_format=torch.contiguous_format) for h in hidden)
        return self.step_(x, hidden), hidden


# ------------------------------------------------------------- eager path

def _silu(op, activation):
    if activation not in (None, 'silu'):
        raise ValueError("%s: activation must be None or 'silu', got %r" % (op, activation))
    return activation == 'silu'


def _grouped(v, x):
    return v.unsqueeze(-2) if v.dim() == x.dim() else v


def _conv_eager(held, x, weight, bias, silu, mask):
    held = held + [x.to(weight.dtype)]
    if mask is not None:                # what unobserved steps hold is not used
        held[-1] = torch.where(mask[:, None], held[-1], 0)
    y = sum(h * weight[:, k] for k, h in enumerate(held))
    y = y if bias is None else y + bias
    y = F.silu(y) if silu else y
    if mask is None:
        return held[1:], y
    on = mask[:, None]
    return ([torch.where(on, new, old) for old, new in zip(held[:-1], held[1:])],
            torch.where(on, y, 0))


def _scan_eager(h, x, dt, A, B, C, D, z, dt_bias, dt_softplus, mask):
    real, width = A.dtype, x.size(-1)
    x, dt, B, C = (v.to(real) for v in (x, dt, B, C))
    if mask is not None:
        on = mask[:, None]
        x, dt = torch.where(on, x, 0), torch.where(on, dt, 0)
        B, C = (torch.where(on[..., None], v, 0) for v in (B, C))
    B, C = (v.repeat_interleave(width // v.size(-2), -2) for v in (B, C))
    d = dt if dt_bias is None else dt + dt_bias
    if dt_softplus:
        d = torch.logaddexp(d, torch.zeros_like(d))
    new = torch.exp(d.unsqueeze(-1) * A) * h + (d * x).unsqueeze(-1) * B
    y = (new * C).sum(-1)
    if D is not None:
        y = y + D * x
    if z is not None:
        z = z.to(real) if mask is None else torch.where(on, z.to(real), 0)
        y = y * F.silu(z)
    if mask is None:
        return new, y
    return torch.where(on[..., None], new, h), torch.where(on, y, 0)


def _want(op, name, t, shape, dtype=None):
    if tuple(t.shape) != tuple(shape):
        raise ValueError('%s: %s must have shape %s, got %s' % (op, name, tuple(shape), tuple(t.shape)))
    if dtype is not None and t.dtype != dtype:
        raise ValueError('%s: %s must be %s, got %s' % (op, name, dtype, t.dtype))


def _check_x(op, dim, x, mask):
    if x.dim() != dim or x.size(-1) < 1 or not x.is_floating_point():
        raise ValueError('%s: x must be %s, got %s %s' % (
            op, '(batch, steps, channels)' if dim == 3 else '(batch, channels)',
            tuple(x.shape), x.dtype))
    if mask is None:
        return None
    if mask.dim() == x.dim() and mask.size(-1) == 1:
        mask = mask.squeeze(-1)
    _want(op, 'mask', mask, x.shape[:-1])
    return mask if mask.dtype == torch.bool else mask != 0


def _real(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _check_conv(op, dim, x, weight, bias, state, mask):
    mask = _check_x(op, dim, x, mask)
    if weight.dim() != 2 or not 2 <= weight.size(1) <= 4:
        raise ValueError('%s: weight must be (channels, taps) with 2 to 4 taps, got %s'
                         % (op, tuple(weight.shape)))
    _want(op, 'weight', weight, (x.size(-1), weight.size(1)), _real(x))
    if bias is not None:
        _want(op, 'bias', bias, (x.size(-1),), _real(x))
    if state is not None:
        _want(op, 'state', state, (x.size(0), weight.size(1) - 1, x.size(-1)), x.dtype)
    return mask


def _check_scan(op, dim, x, dt, A, B, C, D, z, dt_bias, state, mask):
    mask = _check_x(op, dim, x, mask)
    _want(op, 'dt', dt, x.shape, x.dtype)
    if A.dim() != 2 or not 1 <= A.size(1) <= 64:
        raise ValueError('%s: A must be (channels, states) with 1 to 64 states, got %s'
                         % (op, tuple(A.shape)))
    _want(op, 'A', A, (x.size(-1), A.size(1)), _real(x))
    if B.dim() != dim + 1 or B.size(-2) < 1 or x.size(-1) % B.size(-2):
        raise ValueError('%s: B must be (..., groups, states) with groups that divide the '
                         'channels, got %s' % (op, tuple(B.shape)))
    for name, v in (('B', B), ('C', C)):
        _want(op, name, v, (*x.shape[:-1], B.size(-2), A.size(1)), x.dtype)
    for name, v in (('D', D), ('dt_bias', dt_bias)):
        if v is not None:
            _want(op, name, v, (x.size(-1),), _real(x))
    if z is not None:
        _want(op, 'z', z, x.shape, x.dtype)
    if state is not None:
        _want(op, 'state', state, (x.size(0), x.size(-1), A.size(1)), _real(x))
    return mask


def _check_step(op, state, *inputs):
    if not state.is_contiguous():
        raise ValueError('%s: state must be contiguous' % op)
    if torch.is_grad_enabled() and any(
            v is not None and v.requires_grad for v in (state, *inputs)):
        raise ValueError('%s: has no gradient; use %s over one step'
                         % (op, 'causal_conv' if 'conv' in op else 'selective_scan'))
