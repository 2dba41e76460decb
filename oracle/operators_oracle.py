"""Plain restatements of the causal attention with a decay and of the layer norm, from their definitions: differentiable torch code
for any dtype (float64 in the tests)."""
import math

import torch


def _weights(log_decay, n, device):
    """exp(g (s - t)) for t <= s, 0 above: (H, n, n).  -inf: the token itself alone."""
    at = torch.arange(n, dtype=torch.float64, device=device)
    apart = (at[:, None] - at[None, :]).clamp(min=0)
    g = log_decay.double().clamp(min=-1e30).view(-1, 1, 1)
    return torch.exp(g * apart).tril()


def decay_attention(q, k, v, log_decay, scale=None, initial_state=None, seq_lens=None):
    """(out, final state), every pair of rows by itself.  Rows past a length are never read."""
    B, H, N, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    outs, states = [], []
    g = log_decay.double().clamp(min=-1e30).to(q.dtype)
    for b in range(B):
        n = N if seq_lens is None else max(0, min(N, int(seq_lens[b])))
        qb, kb, vb = q[b, :, :n], k[b, :, :n], v[b, :, :n]
        w = _weights(log_decay, n, q.device).to(q.dtype)
        out = scale * ((qb @ kb.transpose(-1, -2)) * w) @ vb
        at = torch.arange(n, dtype=q.dtype, device=q.device)
        last = torch.exp(g[:, None] * (n - 1 - at)[None]).unsqueeze(-1)
        state = (kb * last).transpose(-1, -2) @ vb
        if initial_state is not None:
            first = torch.exp(g[:, None] * (at + 1)[None]).unsqueeze(-1)
            out = out + scale * first * (qb @ initial_state[b])
            state = state + torch.exp(g * n).view(-1, 1, 1) * initial_state[b]
        outs.append(torch.cat([out, torch.zeros(H, N - n, D, dtype=q.dtype, device=q.device)], 1))
        states.append(state)
    return torch.stack(outs), torch.stack(states)


def decay_step(q, k, v, state, log_decay, scale=None, slots=None):
    """One token a row, in the order of the batch; returns (out, new states)."""
    B, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    state = state.clone()
    g = torch.exp(log_decay.double()).to(q.dtype).view(-1, 1, 1)
    out = torch.zeros_like(q)
    for b in range(B):
        s = b if slots is None else int(slots[b])
        if 0 <= s < state.shape[0]:
            state[s] = torch.where(g == 0, torch.zeros_like(g), g * state[s]) + k[b].unsqueeze(-1) * v[b].unsqueeze(-2)
            out[b] = scale * (q[b].unsqueeze(-2) @ state[s]).squeeze(-2)
    return out, state


def layer_norm(x, weight=None, bias=None, eps=1e-5, num_groups=1):
    runs = x.unflatten(-1, (num_groups, -1))
    mean = runs.mean(-1, keepdim=True)
    y = (runs - mean) / torch.sqrt(((runs - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = y.flatten(-2)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias


def half_step(dtype):
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def _small_steps(x, y, z, log_decay, scale, seq_lens, backwards):
    """What fp16's smallest step adds to the bound of A(x, y, z).  A pair's score, or the pair's part of y' in the state, is off by up to
    2^-25 (half that step) where it lies below the normal numbers, and never by more than it is: min(pair, 2^-25 (1 + scale |x|_1)) |z|
    summed over the pairs; the state's own 16-bit terms are off by 2^-25 an element: 2^-25 |x|_1 (1 or scale)."""
    u = 2.0 ** -25
    out = torch.zeros_like(x)
    for b in range(x.shape[0]):
        n = x.shape[2] if seq_lens is None else max(0, min(x.shape[2], int(seq_lens[b])))
        xb, yb, zb = x[b, :, :n].abs(), y[b, :, :n].abs(), z[b, :, :n].abs()
        w = _weights(log_decay, n, x.device)
        w = w.transpose(-1, -2) if backwards else w
        length = xb.sum(-1, keepdim=True)
        pair = scale * (xb @ yb.transpose(-1, -2)) * w
        out[b, :, :n] = torch.minimum(pair, u * (1 + scale * length)) @ zb + u * max(1.0, scale) * length
    return out


def _small_state_steps(y, z, log_decay, scale, seq_lens, backwards):
    """The same of the sum of weight * y z^T: min(weight |y|, 2^-25) |z|."""
    out = []
    for b in range(y.shape[0]):
        n = y.shape[2] if seq_lens is None else max(0, min(y.shape[2], int(seq_lens[b])))
        at = torch.arange(n, dtype=torch.float64, device=y.device)
        w = torch.exp(log_decay.double().clamp(min=-1e30)[:, None] * (at + 1 if backwards else n - 1 - at)[None]).unsqueeze(-1)
        out.append(scale * (y[b, :, :n].abs() * w).clamp(max=2.0 ** -25).transpose(-1, -2) @ z[b, :, :n].abs())
    return torch.stack(out)


def _range_steps(x, y, z, state, scale):
    """The same where a row's scores and the terms of the state are taken into fp16's range by a power of two of their largest, so that what is lost lies 2^-39 below
    that, and a tile of y' where its largest is below 2^-7: 2^-25 / 2^-7 of it is lost otherwise.  A score is at most scale |x|_1 max|y|, the state at most
    max|y| sum|z| more than what enters."""
    pairs = y.abs().amax((2, 3), keepdim=True) * z.abs().sum(2, keepdim=True).amax(3, keepdim=True)
    entered = 0 if state is None else state.abs().amax((2, 3), keepdim=True)
    return scale * x.abs().sum(-1, keepdim=True) * (2.0 ** -18 * pairs + 2 * 2.0 ** -39 * (pairs + entered))


def decay_bounds(q, k, v, d, log_decay, scale, initial_state, d_state, seq_lens, dtype, in_range=False):
    """How far the kernels' (out, state, dq, dk, dv, d_initial) may be off, element by element, given the float64 inputs.

    Every output is a sum of products of three factors (a pair of rows) or four (with a weight); `mass` is the same sum of absolute values.
    A float32 sum of n terms in any order is off by at most n 2^-24 mass; the tensor cores cut off where others round, two half
    steps.  n is at most the head size, the rows of a chunk and the number of chunks, as a sum of sums.  16-bit calls round each
    pair's score, or the key's part of the state, once to their type (half a step of mass), and the result once; fp16 has a smallest step
    on top (_small_steps; in_range: _range_steps, and of a state that is handed out 2^-25 of the largest key, as its sums' tiles are brought to 1 and more)."""
    a = lambda t: None if t is None else t.abs()  # noqa: E731
    D, N = q.shape[-1], q.shape[2]
    n = 2 * (D + 128 + N / 64 + 8) * 2.0 ** -24
    qa, ka, va = (a(t).requires_grad_(True) for t in (q, k, v))
    ia = None if initial_state is None else a(initial_state).requires_grad_(True)
    scale = abs(scale)
    out, state = decay_attention(qa, ka, va, log_decay, scale, ia, seq_lens)
    grads = [None] * 4
    if d is not None:
        wanted = [qa, ka, va] + ([ia] if ia is not None else [])
        top = (out * a(d)).sum() + (0 if d_state is None else (state * a(d_state)).sum())
        grads = list(torch.autograd.grad(top, wanted, allow_unused=True)) + [None] * (4 - len(wanted))
    u = half_step(dtype) if dtype != torch.float32 else 0.0
    big = lambda t: None if t is None else (n + 1.01 * u) * t.detach()  # noqa: E731
    small = lambda t: None if t is None else n * t.detach()  # noqa: E731
    bounds = [big(out), small(state), big(grads[0]), big(grads[1]), big(grads[2]), small(grads[3])]
    if dtype == torch.float16 and in_range:
        s0, ds = initial_state, None if d_state is None else d_state / scale      # (the gradient of the state has the scale in it)
        bounds[0] = bounds[0] + _range_steps(q, k, v, s0, scale)
        bounds[1] = bounds[1] + 2.0 ** -25 * k.abs().amax((2, 3), keepdim=True) * v.abs().sum(2).unsqueeze(2)
        if d is not None:
            for i, f, s in ((2, (d, v, k), s0), (3, (v, d, q), ds), (4, (k, q, d), ds)):
                bounds[i] = bounds[i] + _range_steps(*f, s, scale)
            if bounds[5] is not None:
                bounds[5] = bounds[5] + 2.0 ** -25 * scale * q.abs().amax((2, 3), keepdim=True) * d.abs().sum(2).unsqueeze(2)
    elif dtype == torch.float16:
        forms = [(0, (q, k, v), False)] + ([(2, (d, v, k), False), (3, (v, d, q), True), (4, (k, q, d), True)] if d is not None else [])
        for i, f, backwards in forms:
            bounds[i] = bounds[i] + _small_steps(*f, log_decay, scale, seq_lens, backwards)
        bounds[1] = bounds[1] + _small_state_steps(k, v, log_decay, 1.0, seq_lens, False)
        if bounds[5] is not None:
            bounds[5] = bounds[5] + _small_state_steps(q, d, log_decay, scale, seq_lens, True)
    return bounds


def within(got, ref, bound, dtype):
    """got is within `bound` of ref, with one rounding to its type on top (and what lies below its smallest normal number)."""
    ref = ref.detach().to(got.device)
    room = bound.to(got.device) * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + torch.finfo(dtype).tiny * half_step(dtype) * 2 + 1e-37
    off = (got.detach().double() - ref).abs()
    assert bool(torch.isfinite(got.detach()).all()), "not finite"
    worst = float((off / room).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound (largest error {float(off.max()):.3g})"
    return worst


def isqrt(D):
    return 1.0 / math.sqrt(D)
