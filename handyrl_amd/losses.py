"""Off-policy target algorithms: Monte-Carlo, TD(lambda), UPGO, V-Trace;
and the clipped policy loss that may use their advantages.

Semantics match reference handyrl/losses.py:16-81 (V-Trace per
arXiv:1802.01561).  All tensors are (B, T, P, 1); the recurrence runs
backward over T.

Dispatch: on CUDA tensors the whole backward scan runs as ONE CDNA4 HIP
kernel (handyrl_amd/ops/src/scan.hip) with (B*P) lanes scanning T serially
in registers — replacing the reference's Python-level loop of ~3*T tiny
kernel launches per call (reference losses.py:20-29, 45-60).  The eager
loops below are the CPU path and the parity oracle for tests.
"""

import torch
import torch.nn.functional as F

from . import ops


def monte_carlo(values, returns):
    return returns, returns - values


def temporal_difference(values, returns, rewards, lambda_, gamma):
    """tv_t = r_t + gamma * ((1-lambda_{t+1}) V_{t+1} + lambda_{t+1} tv_{t+1})."""
    T = values.size(1)
    tv = returns[:, -1]
    out = [tv]
    for t in range(T - 2, -1, -1):
        r = rewards[:, t] if rewards is not None else 0
        lam = lambda_[:, t + 1]
        tv = r + gamma * ((1 - lam) * values[:, t + 1] + lam * tv)
        out.append(tv)
    targets = torch.stack(out[::-1], dim=1)
    return targets, targets - values


def upgo(values, returns, rewards, lambda_, gamma):
    """TD scan with a max(V, lambda-mixture) bootstrap (AlphaStar UPGO)."""
    T = values.size(1)
    tv = returns[:, -1]
    out = [tv]
    for t in range(T - 2, -1, -1):
        v_next = values[:, t + 1]
        r = rewards[:, t] if rewards is not None else 0
        lam = lambda_[:, t + 1]
        tv = r + gamma * torch.max(v_next, (1 - lam) * v_next + lam * tv)
        out.append(tv)
    targets = torch.stack(out[::-1], dim=1)
    return targets, targets - values


def vtrace(values, returns, rewards, lambda_, gamma, rhos, cs):
    """IMPALA V-Trace: delta scan then vs / advantage construction."""
    r = rewards if rewards is not None else 0
    v_next = torch.cat([values[:, 1:], returns[:, -1:]], dim=1)
    deltas = rhos * (r + gamma * v_next - values)

    T = values.size(1)
    acc = deltas[:, -1]
    out = [acc]
    for t in range(T - 2, -1, -1):
        acc = deltas[:, t] + gamma * lambda_[:, t + 1] * cs[:, t] * acc
        out.append(acc)
    vs_minus_v = torch.stack(out[::-1], dim=1)
    vs = vs_minus_v + values
    vs_next = torch.cat([vs[:, 1:], returns[:, -1:]], dim=1)
    advantages = r + gamma * vs_next - values
    return vs, advantages


def compute_target(algorithm, values, returns, rewards, lmb, gamma, rhos, cs, masks):
    if values is None:
        # no baseline: Monte-Carlo returns serve as target and advantage
        return returns, returns

    if algorithm == 'MC':
        return monte_carlo(values, returns)

    # outside the episode mask the scan degrades to lambda = 1 pass-through
    lambda_ = lmb + (1 - lmb) * (1 - masks)

    if values.is_cuda and ops.available():
        return ops.target_scan(algorithm, values, returns, rewards, lambda_, gamma, rhos, cs)

    if algorithm == 'TD':
        return temporal_difference(values, returns, rewards, lambda_, gamma)
    if algorithm == 'UPGO':
        return upgo(values, returns, rewards, lambda_, gamma)
    if algorithm == 'VTRACE':
        return vtrace(values, returns, rewards, lambda_, gamma, rhos, cs)
    raise ValueError('unknown target algorithm %r' % (algorithm,))


POLICY_LOSS_STATS = ('p', 'kl', 'ent', 'ent_scaled', 'clipped', 'rows')


def clipped_policy_loss(logits, actions, old_log_probs, advantages, mask=None,
                        entropy_scale=None, *, clip=0.2, clip_high=None,
                        kl_coef=0.0, entropy_coef=0.0):
    """Clipped policy loss (PPO, arXiv:1707.06347) with a KL term and an
    entropy bonus, summed (not averaged) over rows like the framework's
    other losses:

        sum_i mask_i * (-min(r adv, clamp(r, 1 - clip, 1 + clip_high) adv)
                        + kl_coef * (r - 1 - log r)
                        - entropy_coef * entropy_scale_i * H(policy_i))

    with r = exp(log policy(action) - old_log_prob).  As the actions come
    from the old policy, r - 1 - log r estimates KL(old || new) without bias.

    logits (..., A), float32 or bfloat16, carries the gradient.  actions
    (int64) and the float tensors hold one value a row: shape (...), or
    (..., 1), or one that broadcasts to it; they are constants of the loss.
    Rows of mask 0 are left out altogether, whatever their values.  An
    illegal action may have a logit of -inf or of a large negative number.
    An action outside [0, A) makes the loss NaN on the GPU (and raises on
    the CPU).

    Returns (loss, stats): a float32 scalar and the detached sums
    ``POLICY_LOSS_STATS``: surrogate loss, KL, entropy and scaled entropy
    (weighted by the mask), the number of clipped rows, and the mask's sum.
    On the GPU the gradient cannot be differentiated again, there is no
    forward-mode derivative, and a backward pass can only be captured into a
    graph if its forward pass was and no eager pass over the same logits lives on.
    """
    clip_high = clip if clip_high is None else clip_high
    if not 0 <= clip <= 1 or not clip_high >= 0:
        raise ValueError('clipped_policy_loss: clip must be in [0, 1] and clip_high '
                         'at least 0, got %r and %r' % (clip, clip_high))
    if logits.is_cuda:
        ext = ops.require()
        if ext is not None:
            return ext.clipped_policy_loss(logits, actions, old_log_probs,
                                           advantages, mask, entropy_scale,
                                           clip, clip_high, kl_coef, entropy_coef)

    if not logits.is_floating_point() or logits.dim() < 1 or logits.size(-1) < 1:
        raise ValueError('clipped_policy_loss: logits must be (..., actions), got %s %s'
                         % (tuple(logits.shape), logits.dtype))
    rows = logits.shape[:-1]

    def per_row(t, name, dtype):
        if torch.is_grad_enabled() and t.requires_grad:
            raise ValueError('clipped_policy_loss: %s is a constant of the loss: detach it' % name)
        if (dtype == torch.int64) != (t.dtype == torch.int64):
            raise ValueError('clipped_policy_loss: %s has type %s' % (name, t.dtype))
        v = t.squeeze(-1) if t.dim() == len(rows) + 1 and t.size(-1) == 1 else t
        try:
            return v.expand(rows).to(dtype)
        except RuntimeError:
            raise ValueError('clipped_policy_loss: %s of shape %s does not fit rows of shape %s'
                             % (name, tuple(t.shape), tuple(rows))) from None

    real = torch.float64 if logits.dtype == torch.float64 else torch.float32
    actions = per_row(actions, 'actions', torch.int64)
    old = per_row(old_log_probs, 'old_log_probs', real)
    adv = per_row(advantages, 'advantages', real)
    one = torch.ones((), dtype=real, device=logits.device)
    mask = per_row(one if mask is None else mask, 'mask', real)
    scale = per_row(one if entropy_scale is None else entropy_scale, 'entropy_scale', real)

    # the rows left out hold a plain value from here on, so that neither
    # they nor their gradients can spoil a sum
    on = mask != 0
    logp = F.log_softmax(torch.where(on.unsqueeze(-1), logits.to(real), 0), dim=-1)
    taken = torch.where(on, actions, 0).unsqueeze(-1)
    x = torch.where(on, logp.gather(-1, taken).squeeze(-1) - old, 0)
    adv = torch.where(on, adv, 0)
    now = x.detach().exp()
    flat = ((adv > 0) & (now > 1 + clip_high)) | ((adv < 0) & (now < 1 - clip))
    # the minimum, written so that a ratio without a part in it cannot spoil
    # the gradient by overflowing
    surrogate = adv * torch.where(flat, now.clamp(1 - clip, 1 + clip_high),
                                  torch.where(flat, 0, x).exp())
    kl = torch.expm1(x) - x
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp.clamp(min=torch.finfo(real).min), 0).sum(-1)
    scale = torch.where(on, scale, 0)
    terms = [-surrogate * mask, kl * mask, entropy * mask, entropy * mask * scale]
    p_sum, kl_sum, ent_sum, scaled_sum = [t.sum() for t in terms]
    loss = p_sum - entropy_coef * scaled_sum
    if kl_coef != 0:                # a ratio that overflows only counts where it is asked for
        loss = loss + kl_coef * kl_sum
    stats = torch.stack([p_sum, kl_sum, ent_sum, scaled_sum,
                         flat.sum().to(real), mask.sum()]).detach()
    return loss, stats
