"""The causal attention with a decay and the layer norm, as cases that can be prepared, run and timed.

Two families, each in the forms that a user's program calls:

  prompt   `decay_attention` over whole sequences (inference): output and the state behind the last row
  train    the same with its backward pass: output and the gradients of q, k, v (and of the initial state)
  decode   `decay_attention_step`: one token for each row of a batch, the states updated in place
  norm     `layer_norm` over the last dimension, whole or in groups (one group for each head)
  norm_train  the same with its backward pass: output and the gradients of x, weight and bias

With S_t = exp(g_h) S_{t-1} + k_t v_t^T (float32, one D x D state for each head) the attention is
o_t = scale * S_t^T q_t.  Sizes come from the repository's configurations, tests and benchmark: sequences of 1 to 65536
rows, head sizes 16 to 128, up to 64 (batch, head) slices of 16384 rows of 128, widths of 512 to 2048 and odd ones.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU, from the seed alone
    run(state)           one pass, returning everything that it computes
    work(case)           bytes and operations that the pass cannot do without
    exact(case, seed)    what run() returns, in 64 bits and from the definition
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _attention(name, kind, dtype, B, H, N, D, split=False, state=False, padded=False):
    """split: q, k, v are head-split views of (B, N, H * D) tensors, as projections leave them; state: an initial state is given and the
    last one is wanted; padded: sequences of their own lengths in a padded batch."""
    return {"name": name, "kind": kind, "dtype": dtype, "B": B, "H": H, "N": N, "D": D, "split": split, "state": state, "padded": padded}


def _decode(name, dtype, B, H, D, pool=0):
    """pool: number of states that the batch's rows pick theirs from, 0 for one state a row."""
    return {"name": name, "kind": "decode", "dtype": dtype, "B": B, "H": H, "D": D, "pool": pool}


def _norm(name, kind, dtype, rows, width, groups=1, params="same"):
    """params: type of weight and bias, that of x or fp32."""
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "width": width, "groups": groups, "params": params}


def listed():
    return [
        # one short prompt through a small model: launches and host time are all there is
        _attention("prompt_short", "prompt", "fp16", 1, 2, 256, 64, state=True),
        # a padded batch of prompts of odd lengths that go on from earlier states
        _attention("prompt_padded", "prompt", "bf16", 8, 8, 2000, 64, split=True, state=True, padded=True),
        # one long document, the benchmark's size
        _attention("prompt_64k", "prompt", "fp16", 1, 16, 65536, 64),
        # an ordinary training batch, tensors as the projections leave them
        _attention("train_4k", "train", "fp16", 4, 8, 4096, 64, split=True),
        # wide heads at the size of the reference's latency table
        _attention("train_wide_heads", "train", "bf16", 4, 16, 16384, 128),
        # full precision, an odd length, gradients of the states too
        _attention("train_fp32", "train", "fp32", 2, 8, 5001, 64, state=True),
        # one token for one user
        _decode("decode_one", "fp16", 1, 8, 64),
        # a serving batch with its states in a pool, some rows idle
        _decode("decode_pool", "bf16", 256, 16, 128, pool=320),
        # the norm of the heads of the benchmark's sequence, behind the attention
        _norm("norm_heads", "norm", "fp16", 65536, 1024, groups=16),
        # one token's activations
        _norm("norm_one", "norm", "bf16", 1, 512),
        # an ordinary training batch of the module's width, weights kept in full precision
        _norm("norm_train", "norm_train", "bf16", 16384, 512, params="fp32"),
        # the benchmark's sequence at the width of its heads together, one group for each head
        _norm("norm_train_heads", "norm_train", "fp16", 65536, 1024, groups=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# a drawn case stays below the largest listed ones: elements of one (B, H, N, D) tensor, or of one (rows, width) matrix
_MAX_ELEMENTS = 4 * 16 * 16384 * 128
_MAX_NORM = 65536 * 1024


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "decode", "norm", "norm_train"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if kind in ("prompt", "train"):
        D = rng.choice([16, 32, 64, 64, 128, 128])
        N = _log_int(rng, 1, 65536)
        H = rng.randint(1, 16)
        B = _log_int(rng, 1, 32)
        most = _MAX_ELEMENTS // (8 if dtype == "fp32" else 1)
        while B * H * N * D > most:
            if B > 1:
                B = B // 2
            elif H > 1:
                H = H // 2
            else:
                N = N // 2
        return {"kind": kind, "dtype": dtype, "B": B, "H": H, "N": N, "D": D, "split": rng.random() < 0.5, "state": rng.random() < 0.5,
                "padded": rng.random() < 0.4}
    if kind == "decode":
        B = _log_int(rng, 1, 256)
        return {"kind": kind, "dtype": dtype, "B": B, "H": rng.randint(1, 16), "D": rng.choice([16, 32, 64, 64, 128]),
                "pool": B + rng.randint(0, B) if rng.random() < 0.5 else 0}
    groups = rng.choice([1, 1, 1, 4, 8, 16])
    width = groups * (rng.choice([16, 32, 64, 128]) if groups > 1 else _log_int(rng, 16, 8192))
    rows = min(_log_int(rng, 1, 65536), _MAX_NORM // width)
    return {"kind": kind, "dtype": dtype, "rows": rows, "width": width, "groups": groups, "params": rng.choice(["same", "fp32"])}


# ---- inputs --------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _decays(H, gen):
    """exp(g) from 1 - 2^-4 to about 1 - 2^-12 over the heads, from short memory to long; a little off these by the seed."""
    octaves = 4.0 + 8.0 * torch.arange(H, device="cuda", dtype=torch.float64) / max(1, H - 1)
    octaves += 0.2 * torch.rand(H, device="cuda", dtype=torch.float64, generator=gen)
    return torch.log1p(-torch.exp2(-octaves)).float()


def prepare(case, seed):
    gen = _generator(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, mul=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * mul).to(dtype)

    kind = case["kind"]
    s = {"case": case}
    if kind in ("prompt", "train"):
        B, H, N, D = (case[n] for n in "BHND")

        def rows():
            return normal(B, N, H, D).transpose(1, 2) if case["split"] else normal(B, H, N, D)

        s["q"], s["k"], s["v"] = rows(), rows(), rows()
        s["log_decay"] = _decays(H, gen)
        s["initial"] = normal(B, H, D, D, dtype=torch.float32) if case["state"] else None
        s["lens"] = None
        if case["padded"]:
            s["lens"] = torch.randint(0, N + 1, (B,), device="cuda", generator=gen).to(torch.int32)
            s["lens"][0] = N
        if kind == "train":
            s["d_out"] = rows()
            s["d_final"] = normal(B, H, D, D, dtype=torch.float32) if case["state"] else None
            for n in ("q", "k", "v", "initial"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    elif kind == "decode":
        B, H, D, pool = (case[n] for n in ("B", "H", "D", "pool"))
        s["q"], s["k"], s["v"] = (normal(B, H, D) for _ in range(3))
        s["log_decay"] = _decays(H, gen)
        s["states"] = normal(pool or B, H, D, D, dtype=torch.float32, mul=4.0)
        s["slots"] = None
        if pool:
            s["slots"] = torch.randperm(pool, device="cuda", generator=gen)[:B].to(torch.int32)
            s["slots"][torch.rand(B, device="cuda", generator=gen) < 0.1] = -1     # idle rows
    else:
        rows, width = case["rows"], case["width"]
        pt = dt if case["params"] == "same" else torch.float32
        # activations: a mean and a spread of their own for each row
        x = torch.randn(rows, width, device="cuda", generator=gen)
        x = x * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)) + torch.randn(rows, 1, device="cuda", generator=gen)
        s["x"] = x.to(dt)
        s["weight"] = (1.0 + 0.2 * torch.randn(width, device="cuda", generator=gen)).to(pt)
        s["bias"] = (0.2 * torch.randn(width, device="cuda", generator=gen)).to(pt)
        if kind == "norm_train":
            s["d_out"] = normal(rows, width)
            for n in ("x", "weight", "bias"):
                s[n].requires_grad_(True)
    return s


EPS = 1e-5


# ---- the plain forms -----------------------------------------------------------------------------------------
CHUNK = 128


def _powers(g, n):
    """exp(g n) for exponents n >= 0 (any shape), one leading dimension for the heads; formed in 64 bits."""
    e = g.double().view(-1, *([1] * n.dim())) * n.double()
    return torch.exp(e).float()


def _causal(x, y, z, g):
    """sum over t <= s of exp(g (s - t)) (x_s . y_t) z_t for (B, H, N, D) tensors in 32 bits: within chunks by the masked product, from
    chunk to chunk by the sums of y z^T."""
    B, H, N, D = x.shape
    n = -(-N // CHUNK)
    if n * CHUNK != N:
        x, y, z = (torch.nn.functional.pad(t, (0, 0, 0, n * CHUNK - N)) for t in (x, y, z))
    x, y, z = (t.reshape(B, H, n, CHUNK, D) for t in (x, y, z))
    i = torch.arange(CHUNK, device=x.device)
    apart = i[:, None] - i[None, :]
    inside = torch.where(apart >= 0, _powers(g, apart.clamp(min=0)), 0.0)
    out = (x @ y.transpose(-1, -2) * inside.view(1, H, 1, CHUNK, CHUNK)) @ z
    if n > 1:
        sums = (y * _powers(g, CHUNK - 1 - i).view(1, H, 1, CHUNK, 1)).transpose(-1, -2) @ z
        c = torch.arange(n, device=x.device)
        apart = c[:, None] - 1 - c[None, :]
        carry = torch.where(apart >= 0, _powers(g, CHUNK * apart.clamp(min=0)), 0.0)
        before = (carry @ sums.reshape(B, H, n, D * D)).reshape(B, H, n, D, D)
        out = out + (x * _powers(g, i + 1).view(1, H, 1, CHUNK, 1)) @ before
    return out.reshape(B, H, n * CHUNK, D)[:, :, :N]


def _causal_reversed(x, y, z, g):
    return _causal(x.flip(2), y.flip(2), z.flip(2), g).flip(2)


def _plain_lengths(s, N):
    """(rows that count, their distance from the last one of the sequence), both (B, 1, N, 1), and the lengths."""
    B = s["q"].shape[0]
    lens = s["lens"].long() if s["lens"] is not None else torch.full((B,), N, device=s["q"].device)
    at = torch.arange(N, device=s["q"].device)
    return (at[None, :] < lens[:, None]).view(B, 1, N, 1), (lens[:, None] - 1 - at[None, :]).clamp(min=0), lens


def _plain_attention(s):
    c = s["case"]
    B, H, N, D = (c[n] for n in "BHND")
    g, scale, S0 = s["log_decay"], D ** -0.5, s["initial"]
    valid, left, lens = _plain_lengths(s, N)
    dt = s["q"].dtype
    q, k, v = (torch.where(valid, s[n].detach().float(), 0.0) for n in "qkv")
    since = _powers(g, torch.arange(N, device=q.device) + 1).view(1, H, N, 1)             # of the state before the first row
    until = _powers(g, left).transpose(0, 1).unsqueeze(-1)                                # (B, H, N, 1), to the state behind the last
    whole = _powers(g, lens).transpose(0, 1).view(B, H, 1, 1)
    out = _causal(q, k, v, g)
    if S0 is not None:
        S0 = S0.detach()
        out = out + since * (q @ S0)
    out = (out * scale).to(dt)
    final = (k * until).transpose(-1, -2) @ v
    if S0 is not None:
        final = final + whole * S0
    if c["kind"] == "prompt":
        return out, final
    d = torch.where(valid, s["d_out"].float(), 0.0)
    dq = _causal(d, v, k, g)
    dk = _causal_reversed(v, d, q, g)
    dv = _causal_reversed(k, q, d, g)
    if S0 is None:
        return (out, *((t * scale).to(dt) for t in (dq, dk, dv)))
    dS = s["d_final"]
    dq = (dq + since * (d @ S0.transpose(-1, -2))) * scale
    dk = torch.where(valid, dk * scale + until * (v @ dS.transpose(-1, -2)), 0.0)
    dv = torch.where(valid, dv * scale + until * (k @ dS), 0.0)
    dS0 = whole * dS + scale * ((q * since).transpose(-1, -2) @ d)
    return out, final, dq.to(dt), dk.to(dt), dv.to(dt), dS0


def _plain_decode(s):
    q, k, v, states, slots = s["q"].float(), s["k"].float(), s["v"].float(), s["states"], s["slots"]
    mul = torch.exp(s["log_decay"].double()).float().view(1, -1, 1, 1)
    old = states if slots is None else states[slots.clamp(min=0).long()]
    new = mul * old + k.unsqueeze(-1) * v.unsqueeze(-2)
    out = (q.unsqueeze(-1) * new).sum(-2) * q.shape[-1] ** -0.5
    if slots is None:
        states.copy_(new)
    else:
        out = torch.where((slots >= 0).view(-1, 1, 1), out, 0.0)
        taken = slots.view(1, -1) == torch.arange(states.shape[0], device=q.device).view(-1, 1)
        states.copy_(torch.where(taken.any(1).view(-1, 1, 1, 1), new[taken.int().argmax(1)], states))
    return out.to(s["q"].dtype), states


def _plain_norm(s):
    c = s["case"]
    rows, width, G = c["rows"], c["width"], c["groups"]
    x = s["x"].detach().float().view(rows, G, width // G)
    w, b = (s[n].detach().float().view(1, G, width // G) for n in ("weight", "bias"))
    mean = x.mean(-1, keepdim=True)
    off = x - mean
    r = torch.rsqrt((off * off).mean(-1, keepdim=True) + EPS)
    hat = off * r
    y = (hat * w + b).view(rows, width).to(s["x"].dtype)
    if c["kind"] == "norm":
        return y
    d = s["d_out"].float().view(rows, G, width // G)
    dh = d * w
    dx = r * (dh - dh.mean(-1, keepdim=True) - hat * (dh * hat).mean(-1, keepdim=True))
    pt = s["weight"].dtype
    return y, dx.view(rows, width).to(s["x"].dtype), (d * hat).sum(0).view(width).to(pt), d.sum(0).view(width).to(pt)


# ---- the framework's operators -------------------------------------------------------------------------------
def _own_attention(s):
    from flashnystrom_b200 import decay_attention
    c = s["case"]
    if c["kind"] == "prompt":
        return decay_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial"], seq_lens=s["lens"], return_state=True)
    if not c["state"]:
        out = decay_attention(s["q"], s["k"], s["v"], s["log_decay"], seq_lens=s["lens"])
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"]))
    out, final = decay_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial"], seq_lens=s["lens"], return_state=True)
    grads = torch.autograd.grad((out, final), (s["q"], s["k"], s["v"], s["initial"]), (s["d_out"], s["d_final"]))
    return (out.detach(), final.detach(), *grads)


def _own_decode(s):
    from flashnystrom_b200 import decay_attention_step
    return decay_attention_step(s["q"], s["k"], s["v"], s["states"], s["log_decay"], slots=s["slots"]), s["states"]


def _own_norm(s):
    from flashnystrom_b200 import layer_norm
    y = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, num_groups=s["case"]["groups"])
    if s["case"]["kind"] == "norm":
        return y
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["d_out"]))


def run(state):
    kind = state["case"]["kind"]
    if kind in ("prompt", "train"):
        return _own_attention(state) if own else _plain_attention(state)
    if kind == "decode":
        return _own_decode(state) if own else _plain_decode(state)
    return _own_norm(state) if own else _plain_norm(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    """Bytes: every input read once, every output written once.  Operations of the attention: those of the recurrence itself, a multiply
    and an add for each element of the state and each of its uses (two a row forward, five backward)."""
    e = BYTES[case["dtype"]]
    kind = case["kind"]
    if kind in ("prompt", "train"):
        B, H, N, D = (case[n] for n in "BHND")
        big, states = B * H * N * D * e, B * H * D * D * 4
        if kind == "prompt":
            return {"bytes": 4 * big + (2 if case["state"] else 1) * states, "flops": 4 * B * H * N * D * D}
        return {"bytes": 8 * big + (4 if case["state"] else 0) * states, "flops": 14 * B * H * N * D * D}
    if kind == "decode":
        B, H, D = case["B"], case["H"], case["D"]
        return {"bytes": B * H * (8 * D * D + 4 * D * e), "flops": 5 * B * H * D * D}
    n = case["rows"] * case["width"]
    if kind == "norm":
        return {"bytes": 2 * n * e, "flops": 8 * n}
    return {"bytes": 4 * n * e, "flops": 24 * n}


# ---- in 64 bits, from the definition -------------------------------------------------------------------------
def _exact_slice(q, k, v, g, scale, S0, d, dS):
    """One slice of its own length n, (n, D) each: every pair of rows."""
    n, D = q.shape
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    at = torch.arange(n, device=q.device, dtype=torch.float64)
    step = max(64, min(4096, (1 << 27) // max(1, n)))
    for a in range(0, n, step):
        b = min(n, a + step)
        apart = at[a:b, None] - at[None, :b]
        weight = torch.where(apart >= 0, torch.exp(g * apart.clamp(min=0)), 0.0) * scale
        scores = (q[a:b] @ k[:b].T) * weight
        out[a:b] = scores @ v[:b]
        if d is not None:
            dv[:b] += scores.T @ d[a:b]
            scores = (d[a:b] @ v[:b].T) * weight
            dq[a:b] = scores @ k[:b]
            dk[:b] += scores.T @ q[a:b]
    first, last = torch.exp(g * (at + 1))[:, None], torch.exp(g * (n - 1 - at))[:, None]
    final = (k * last).T @ v
    if S0 is not None:
        out += scale * first * (q @ S0)
        final += torch.exp(g * n) * S0
    dS0 = None
    if dS is not None:
        dq += scale * first * (d @ S0.T)
        dk += last * (v @ dS.T)
        dv += last * (k @ dS)
        dS0 = torch.exp(g * n) * dS + scale * (q * first).T @ d
    return out, final, dq, dk, dv, dS0


def _exact_attention(case, s):
    B, H, N, D = (case[n] for n in "BHND")
    scale = 1.0 / math.sqrt(D)
    train, state = case["kind"] == "train", case["state"]
    lens = s["lens"].tolist() if s["lens"] is not None else [N] * B
    big = [torch.zeros(B, H, N, D, device="cuda", dtype=torch.float64) for _ in range(4 if train else 1)]
    small = [torch.zeros(B, H, D, D, device="cuda", dtype=torch.float64) for _ in range(2)]
    with torch.no_grad():
        for b in range(B):
            n = lens[b]
            for h in range(H):
                q, k, v = (s[x][b, h, :n].double() for x in "qkv")
                out, final, dq, dk, dv, dS0 = _exact_slice(
                    q, k, v, s["log_decay"][h].double(), scale, s["initial"][b, h].double() if state else None,
                    s["d_out"][b, h, :n].double() if train else None, s["d_final"][b, h].double() if train and state else None)
                for to, t in zip(big, (out, dq, dk, dv)):
                    to[b, h, :n] = t
                small[0][b, h] = final
                if dS0 is not None:
                    small[1][b, h] = dS0
    if not train:
        return big[0], small[0]
    if not state:
        return tuple(big)
    return big[0], small[0], big[1], big[2], big[3], small[1]


def _exact_decode(case, s):
    slots = s["slots"].tolist() if s["slots"] is not None else list(range(case["B"]))
    states = s["states"].double()
    out = torch.zeros(case["B"], case["H"], case["D"], device="cuda", dtype=torch.float64)
    for i, slot in enumerate(slots):
        if slot >= 0:
            states[slot] *= torch.exp(s["log_decay"].double())[:, None, None]
            states[slot] += torch.einsum("hi,hj->hij", s["k"][i].double(), s["v"][i].double())
            out[i] = torch.einsum("hi,hij->hj", s["q"][i].double(), states[slot]) / math.sqrt(case["D"])
    return out, states


def _exact_norm(case, s):
    rows, width, G = case["rows"], case["width"], case["groups"]
    n = width // G
    outs = [torch.empty(rows, width, device="cuda", dtype=torch.float64) for _ in range(2)]
    dw, db = (torch.zeros(width, device="cuda", dtype=torch.float64) for _ in range(2))
    with torch.no_grad():
        w, b = s["weight"].double(), s["bias"].double()
        for i in range(G):
            cols = slice(i * n, (i + 1) * n)
            x = s["x"][:, cols].double()
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            sd = torch.sqrt(var + EPS)
            hat = (x - mean) / sd
            outs[0][:, cols] = hat * w[cols] + b[cols]
            if case["kind"] == "norm_train":
                d = s["d_out"][:, cols].double()
                dw[cols], db[cols] = torch.einsum("rc,rc->c", d, hat), torch.einsum("rc->c", d)
                u = d * w[cols]
                outs[1][:, cols] = (u - (u.sum(1, keepdim=True) + hat * torch.einsum("rc,rc->r", u, hat)[:, None]) / n) / sd
    return outs[0] if case["kind"] == "norm" else (outs[0], outs[1], dw, db)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("prompt", "train"):
        return _exact_attention(case, s)
    return _exact_decode(case, s) if case["kind"] == "decode" else _exact_norm(case, s)
