"""torch.library registration of the forward and backward as custom operators, so that
torch.compile / torch.export trace through `flash_nystrom_attention` without a graph break (the
reference lists this as future work, README.md:387; its autograd.Function behind pybind breaks the
graph).

    torch.ops.flashnystrom_b200.nystrom_fwd(q, k, v, num_landmarks, newton_iter, kappa_star)
        -> (out, q_landmarks, k_landmarks, k2_inv, step2, lse1, lse2, lse3, ns_iterates, k2, bmat)
    torch.ops.flashnystrom_b200.nystrom_bwd(d_out, q, k, v, <the ten saved tensors>, ...)
        -> (dq, dk, dv)

    torch.ops.flashnystrom_b200.decay_fwd(q, k, v, log_decay, scale, initial_state, seq_lens) -> (out, final_state, states at the cuts)
    torch.ops.flashnystrom_b200.decay_bwd(...) -> (dq, dk, dv, d_initial_state)
    torch.ops.flashnystrom_b200.decay_step(q, k, v, state, log_decay, scale, slots) -> out, with state written
    torch.ops.flashnystrom_b200.norm_fwd(x, weight, bias, eps, num_groups) -> (y, mean, rstd)
    torch.ops.flashnystrom_b200.norm_bwd(...) -> (dx, d_weight, d_bias)

All have fake (meta) implementations, and the forward ones have their autograd formulas registered, so the
operators work under FakeTensorMode, AOT autograd and opcheck.  Eager calls go through the C++ module
(csrc/native.cpp) and, where that hands them back, through the autograd functions of flash_nystrom.py (less dispatcher
overhead per call); `flash_nystrom_attention` switches to the operators while a compiler is tracing."""
from typing import Optional, Tuple

import torch

from . import _C

_LIB = "flashnystrom_b200"


@torch.library.custom_op(f"{_LIB}::nystrom_fwd", mutates_args=(), device_types="cuda")
def nystrom_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_landmarks: int, newton_iter: int,
                kappa_star: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                            torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                            torch.Tensor]:
    r = _C.forward(q.contiguous(), k.contiguous(), v.contiguous(), num_landmarks, newton_iter, kappa_star, False, True)
    # r = [out, q, k, qt, kt, k2inv, step2, lse1, lse2, lse3, iterates, k2, bmat]; q and k are the
    # caller's own tensors and an operator must not return its inputs
    return (r[0], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10], r[11], r[12])


@nystrom_fwd.register_fake
def _(q, k, v, num_landmarks, newton_iter, kappa_star):
    B, H, N, D = q.shape
    m, J = num_landmarks, newton_iter
    f32 = dict(dtype=torch.float32, device=q.device)
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            torch.empty(B, H, m, D, **f32), torch.empty(B, H, m, D, **f32), torch.empty(B, H, m, m, **f32),
            torch.empty(B, H, m, D, **f32), torch.empty(B, H, N, **f32), torch.empty(B, H, m, **f32),
            torch.empty(B, H, m, **f32), torch.empty(B, H, J + 1, m, m, **f32), torch.empty(B, H, m, m, **f32),
            torch.empty(B, H, m, D, **f32))


@torch.library.custom_op(f"{_LIB}::nystrom_bwd", mutates_args=(), device_types="cuda")
def nystrom_bwd(d_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                q_landmarks: torch.Tensor, k_landmarks: torch.Tensor, k2_inv: torch.Tensor, step2: torch.Tensor,
                lse1: torch.Tensor, lse2: torch.Tensor, lse3: torch.Tensor, ns_iterates: torch.Tensor,
                k2: torch.Tensor, bmat: torch.Tensor, num_landmarks: int, newton_iter: int,
                kappa_star: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dq, dk, dv = _C.backward(d_out.contiguous(), q.contiguous(), k.contiguous(), q_landmarks, k_landmarks, k2_inv, step2,
                             lse1, lse2, lse3, ns_iterates, k2, bmat, v.contiguous(), out, num_landmarks, newton_iter,
                             True, kappa_star)
    return dq, dk, dv


@nystrom_bwd.register_fake
def _(d_out, q, k, v, out, q_landmarks, k_landmarks, k2_inv, step2, lse1, lse2, lse3, ns_iterates, k2, bmat,
      num_landmarks, newton_iter, kappa_star):
    c = torch.contiguous_format
    return (torch.empty_like(q, memory_format=c), torch.empty_like(k, memory_format=c),
            torch.empty_like(v, memory_format=c))


def _setup_context(ctx, inputs, output):
    q, k, v, m, J, kappa = inputs
    ctx.save_for_backward(q, k, v, *output)
    ctx.m, ctx.J, ctx.kappa = m, J, kappa


def _backward(ctx, d_out, *unused_saved_grads):
    q, k, v, out, qt, kt, k2inv, step2, lse1, lse2, lse3, iters, k2, bmat = ctx.saved_tensors
    dq, dk, dv = nystrom_bwd(d_out, q, k, v, out, qt, kt, k2inv, step2, lse1, lse2, lse3, iters, k2, bmat,
                             ctx.m, ctx.J, ctx.kappa)
    return dq, dk, dv, None, None, None


nystrom_fwd.register_autograd(_backward, setup_context=_setup_context)


def attention_via_ops(q, k, v, num_landmarks, newton_iter, kappa_star):
    """The attention output through the registered operators (differentiable, traceable)."""
    return nystrom_fwd(q, k, v, int(num_landmarks), int(newton_iter), float(kappa_star))[0]


# ---- causal attention with a decay ------------------------------------------------------------------------
# (an operator's outputs have one layout, whatever its inputs': contiguous)
@torch.library.custom_op(f"{_LIB}::decay_fwd", mutates_args=(), device_types="cuda")
def decay_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
              initial_state: Optional[torch.Tensor], seq_lens: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().decay_forward(q.contiguous(), k.contiguous(), v.contiguous(), log_decay, scale, initial_state, seq_lens, _C._status(q.device))


def _segment_floats(q):
    from . import _lib
    import ctypes as C
    shape = _lib.DecayShape(q.shape[0], q.shape[1], q.shape[2], q.shape[3], _C._DTYPES[q.dtype], 1.0, _C._flags & _lib.FNB_FLAG_FORCE_GENERIC)
    with _C._on_device(q.device):
        return _lib.load().fnb_decay_segment_floats(C.byref(shape))


@decay_fwd.register_fake
def _(q, k, v, log_decay, scale, initial_state, seq_lens):
    B, H, N, D = q.shape
    return (torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty(B, H, D, D, dtype=torch.float32, device=q.device),
            torch.empty(_segment_floats(q), dtype=torch.float32, device=q.device))


@torch.library.custom_op(f"{_LIB}::decay_bwd", mutates_args=(), device_types="cuda")
def decay_bwd(d_out: torch.Tensor, d_state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
              initial_state: Optional[torch.Tensor], seq_lens: Optional[torch.Tensor],
              segments: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().decay_backward(d_out.contiguous(), d_state.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), log_decay, scale, initial_state, seq_lens,
                                      segments, _C._status(q.device))


@decay_bwd.register_fake
def _(d_out, d_state, q, k, v, log_decay, scale, initial_state, seq_lens, segments):
    c = torch.contiguous_format
    return (torch.empty_like(q, memory_format=c), torch.empty_like(k, memory_format=c), torch.empty_like(v, memory_format=c),
            torch.empty_like(d_state, memory_format=c))


def _decay_context(ctx, inputs, output):
    q, k, v, log_decay, scale, initial_state, seq_lens = inputs
    ctx.save_for_backward(q, k, v, log_decay, initial_state, seq_lens, output[2])
    ctx.scale = scale


def _decay_backward(ctx, d_out, d_state, _unused):
    q, k, v, log_decay, initial_state, seq_lens, segments = ctx.saved_tensors
    dq, dk, dv, ds = decay_bwd(d_out, d_state, q, k, v, log_decay, ctx.scale, initial_state, seq_lens, segments)
    return dq, dk, dv, None, None, ds if initial_state is not None else None, None


decay_fwd.register_autograd(_decay_backward, setup_context=_decay_context)


def decay_attention_via_ops(q, k, v, log_decay, scale, initial_state, seq_lens):
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay is a constant here: it has no gradient")
    out, state, _ = decay_fwd(q, k, v, log_decay, scale, initial_state, seq_lens)
    return out, state


@torch.library.custom_op(f"{_LIB}::decay_step", mutates_args=("state",), device_types="cuda")
def decay_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: torch.Tensor, log_decay: torch.Tensor, scale: float,
               slots: Optional[torch.Tensor]) -> torch.Tensor:
    return _C.native().decay_step(q, k, v, state, log_decay, scale, slots)


@decay_step.register_fake
def _(q, k, v, state, log_decay, scale, slots):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


# ---- layer norm -------------------------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::norm_fwd", mutates_args=(), device_types="cuda")
def norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
             num_groups: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().norm_forward(x, weight, bias, eps, num_groups)


@norm_fwd.register_fake
def _(x, weight, bias, eps, num_groups):
    runs = x.numel() // x.shape[-1] * num_groups
    f32 = dict(dtype=torch.float32, device=x.device)
    return torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty(runs, **f32), torch.empty(runs, **f32)


@torch.library.custom_op(f"{_LIB}::norm_bwd", mutates_args=(), device_types="cuda")
def norm_bwd(d_y: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, eps: float, num_groups: int,
             param_f32: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _C.native().norm_backward(d_y, x, weight, mean, rstd, eps, num_groups, param_f32)


@norm_bwd.register_fake
def _(d_y, x, weight, mean, rstd, eps, num_groups, param_f32):
    p = dict(dtype=torch.float32 if param_f32 else x.dtype, device=x.device)
    return torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty(x.shape[-1], **p), torch.empty(x.shape[-1], **p)


def _norm_context(ctx, inputs, output):
    x, weight, bias, eps, num_groups = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.eps, ctx.num_groups, ctx.has_bias = eps, num_groups, bias is not None
    param = weight if weight is not None else bias
    ctx.param_f32 = param is None or param.dtype == torch.float32


def _norm_backward(ctx, d_y, _mean, _rstd):
    x, weight, mean, rstd = ctx.saved_tensors
    dx, dw, db = norm_bwd(d_y, x, weight, mean, rstd, ctx.eps, ctx.num_groups, ctx.param_f32)
    return dx, dw if weight is not None else None, db if ctx.has_bias else None, None, None


norm_fwd.register_autograd(_norm_backward, setup_context=_norm_context)


def layer_norm_via_ops(x, weight, bias, eps, num_groups):
    return norm_fwd(x, weight, bias, eps, num_groups)[0]
