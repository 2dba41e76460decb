"""Causal attention with a decay for each head: over sequences (forward and backward) and token by token, and a block around it.

    S_t = exp(g_h) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t

One float32 D x D state for each (batch, head) takes the place of a cache of keys and values, so that a token costs the same after any
number of others, and a sequence of N tokens costs N."""
import torch
import torch.nn as nn
from torch.autograd import forward_ad as _forward_ad

from . import _C
from .norm import layer_norm


def _scale(scale, D):
    scale = float(D) ** -0.5 if scale is None and D > 0 else 1.0 if scale is None else float(scale)
    if not 2.0 ** -64 <= abs(scale) <= 2.0 ** 64:
        raise RuntimeError(f"scale must be finite and not 0, between 2^-64 and 2^64 in magnitude (got {scale})")
    return scale


def _check_tensors(name, **tensors):
    for key, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name}: {key} must be a tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{name}: {key} must be a CUDA tensor (flashnystrom_b200 has no CPU path)")


def decay_attention(q, k, v, log_decay, scale=None, initial_state=None, seq_lens=None, return_state=False):
    """Attention of every token to itself and the tokens before it, weighted by exp(log_decay[head] * distance), without a
    normaliser; forward and exact backward on the GPU.

    q, k, v: (B, H, N, D) CUDA tensors of one dtype (fp16 / bf16 / fp32), D 16, 32, 64 or 128, any strides (the head-split view of a
    (B, N, H * D) projection is read in place, and the output and the gradients come back in that order of memory).
    log_decay: (H,) float32, <= 0: 0 keeps everything, -inf only the token itself; a constant, without a gradient.
    scale: D ** -0.5 unless given; 2^-64 to 2^64 in magnitude.
    initial_state: (B, H, D, D) float32, S[i, j] = sum k_i v_j, or None for zeros.  Differentiable.
    seq_lens: (B,) int32 on the GPU: rows past a sequence's length take no part, whatever they hold (infinities and NaN too), and
        come out as zeros; values outside 0..N count as the nearest of these.  None: all sequences have N rows.
    return_state: also return the state behind each sequence's last row (B, H, D, D), float32, differentiable: what the next
        call takes as initial_state, or decay_attention_step as its state.

    Sums and states are float32.  fp16 and bf16 calls round each pair's score, or the key's share of the state, once to their type on the way: outputs and gradients are off by
    1.25 to 1.45 times what rounding the result alone leaves.  A state that is handed out does not have that rounding, and asking for it may change the last
    bit of the output of long sequences.  Scores, states and tensors may lie far above or below fp16's range as long as the result does not.  fp16 and bf16 tensors whose start or
    strides are not multiples of 16 bytes take float32 arithmetic on the CUDA cores, several times slower.  A row of q, k or v that counts and holds an
    infinity or NaN reaches the rows after it by definition, and may reach up to 127 rows before it; rows behind a length stay zeros.  There is no second
    derivative, no forward-mode one, and no CPU path."""
    _check_tensors("decay_attention", q=q, k=k, v=v, log_decay=log_decay)
    scale = _scale(scale, q.shape[-1] if q.dim() else 0)
    r = None
    if not torch.compiler.is_compiling():
        if _forward_ad._current_level >= 0:
            _C.refuse_tangents("decay_attention", q, k, v, log_decay, initial_state)
        if not _C.wants_operators():
            r = _C.native().decay_attention(q, k, v, log_decay, scale, initial_state, seq_lens, bool(return_state), _C._status(q.device))
    if r is None:
        from . import _ops
        r = _ops.decay_attention_via_ops(q, k, v, log_decay, scale, initial_state, seq_lens, bool(return_state))
    out, state = r
    return (out, state) if return_state else out


def decay_attention_step(q, k, v, state, log_decay, scale=None, slots=None):
    """One token of decay_attention for each row of a batch: updates the states in place, returns the outputs.

    q, k, v: (B, H, D) CUDA tensors of one dtype, any strides.  state: (S, H, D, D) float32, contiguous, written.
    slots: (B,) int32 on the GPU, the state of each row; a row whose slot is not in 0..S-1 (-1, say) is idle: its output is zero and no state
        is touched.  Rows that name the same slot are taken in the order of the batch, as tokens that follow one another.
        None: row b has state b, and S is B.
    Returns (B, H, D).  No gradient: with one wanted, or a tangent given, the call is refused (decay_attention has a gradient)."""
    _check_tensors("decay_attention_step", q=q, k=k, v=v, state=state, log_decay=log_decay)
    scale = _scale(scale, q.shape[-1] if q.dim() else 0)
    if not torch.compiler.is_compiling():
        if _forward_ad._current_level >= 0:
            _C.refuse_tangents("decay_attention_step", q, k, v, state, log_decay)
        if not _C.wants_operators():
            out = _C.native().decay_step(q, k, v, state, log_decay, scale, slots)
            if out is not None:
                return out
    from . import _ops
    return _ops.decay_step(q, k, v, state, log_decay, scale, slots)


def default_log_decay(heads):
    """log(1 - 2^-e) with e from 5 to 12 over the heads: memories of about 32 to 4096 tokens."""
    e = torch.linspace(5.0, 12.0, heads, dtype=torch.float64) if heads > 1 else torch.tensor([5.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float()


class DecayAttention(nn.Module):
    """Multi-head causal self-attention block: bias-free q/k/v/out projections (named as in FlashNystromAttention) around
    decay_attention, whose outputs, sums without a normaliser, go through a layer norm for each head.

    log_decay: (heads,) values <= 0, default_log_decay(heads) unless given; a buffer."""

    def __init__(self, dim, heads=8, log_decay=None, head_norm=True, eps=1e-5):
        super().__init__()
        if dim <= 0 or heads <= 0 or dim % heads:
            raise ValueError(f"heads ({heads}) must divide dim ({dim})")
        self.dim, self.heads, self.head_dim, self.eps = dim, heads, dim // heads, eps
        if self.head_dim not in (16, 32, 64, 128):
            raise ValueError(f"head_dim must be 16, 32, 64 or 128, got {self.head_dim}")
        g = default_log_decay(heads) if log_decay is None else torch.as_tensor(log_decay, dtype=torch.float32).detach().clone()
        if g.shape != (heads,) or not (g.is_meta or bool((g <= 0).all())):
            raise ValueError("log_decay must hold one value <= 0 for each head")
        self.register_buffer("log_decay", g)
        self.q_proj = nn.Linear(dim, dim, bias=False)
        self.k_proj = nn.Linear(dim, dim, bias=False)
        self.v_proj = nn.Linear(dim, dim, bias=False)
        self.out_proj = nn.Linear(dim, dim, bias=False)
        self.register_parameter("norm_weight", nn.Parameter(torch.ones(dim)) if head_norm else None)
        self.register_parameter("norm_bias", nn.Parameter(torch.zeros(dim)) if head_norm else None)

    def _apply(self, fn, recurse=True):
        # (.half() and .bfloat16() are for the weights: decays close to 1 would round to it)
        g = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:
            self.log_decay = g.to(self.log_decay.device)
        return self

    def _finish(self, o):
        if self.norm_weight is not None:
            o = layer_norm(o, self.norm_weight, self.norm_bias, self.eps, num_groups=self.heads)
        return self.out_proj(o)

    def new_state(self, batch):
        """Zero states for `batch` sequences: what step() starts from."""
        return torch.zeros(batch, self.heads, self.head_dim, self.head_dim, device=self.log_decay.device)

    def forward(self, x, state=None, seq_lens=None, return_state=False):
        """x: (B, N, dim).  state, seq_lens, return_state as in decay_attention."""
        B, N, _ = x.shape
        q, k, v = (p(x).view(B, N, self.heads, self.head_dim).transpose(1, 2) for p in (self.q_proj, self.k_proj, self.v_proj))
        o = decay_attention(q, k, v, self.log_decay, initial_state=state, seq_lens=seq_lens, return_state=return_state)
        o, state = o if return_state else (o, None)
        y = self._finish(o.transpose(1, 2).reshape(B, N, self.dim))
        return (y, state) if return_state else y

    def step(self, x, state, slots=None):
        """One token a row: x (B, dim) -> (B, dim), the states updated in place (see decay_attention_step).  Under torch.no_grad()."""
        B = x.shape[0]
        q, k, v = (p(x).view(B, self.heads, self.head_dim) for p in (self.q_proj, self.k_proj, self.v_proj))
        return self._finish(decay_attention_step(q, k, v, state, self.log_decay, slots=slots).view(B, self.dim))
