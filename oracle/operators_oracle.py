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


def decay_bounds(q, k, v, d, log_decay, scale, initial_state, d_state, seq_lens, dtype):
    """How far the kernels' (out, state, dq, dk, dv, d_initial) may be off, element by element, given the float64 inputs.

    Every output is a sum of products of three factors (a pair of rows) or four (with a weight); `mass` is the same sum of absolute values.
    A float32 sum of n terms in any order is off by at most n 2^-24 mass; the tensor cores cut off where others round, two half
    steps.  n is at most the head size, the rows of a chunk and the number of chunks, as a sum of sums.  16-bit calls round each
    pair's score, or the key's part of the state, once to their type (half a step of mass), and the result once."""
    a = lambda t: None if t is None else t.abs()  # noqa: E731
    D, N = q.shape[-1], q.shape[2]
    n = 2 * (D + 128 + N / 64 + 8) * 2.0 ** -24
    qa, ka, va = (a(t).requires_grad_(True) for t in (q, k, v))
    ia = None if initial_state is None else a(initial_state).requires_grad_(True)
    out, state = decay_attention(qa, ka, va, log_decay, abs(scale), ia, seq_lens)
    grads = [None] * 4
    if d is not None:
        wanted = [qa, ka, va] + ([ia] if ia is not None else [])
        top = (out * a(d)).sum() + (0 if d_state is None else (state * a(d_state)).sum())
        grads = list(torch.autograd.grad(top, wanted, allow_unused=True)) + [None] * (4 - len(wanted))
    u = half_step(dtype) if dtype != torch.float32 else 0.0
    big = lambda t: None if t is None else (n + 1.01 * u) * t.detach() + 2.0 ** -24 * (dtype == torch.float16)  # noqa: E731
    small = lambda t: None if t is None else n * t.detach()  # noqa: E731
    return big(out), small(state), big(grads[0]), big(grads[1]), big(grads[2]), small(grads[3])


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
