"""Causal attention with a decay against every pair of rows in float64: outputs, states and gradients, with bounds that are derived in
oracle/operators_oracle.py."""
import ctypes as C
import threading

import pytest
import torch

from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
INF = float("inf")


def _inputs(B, H, N, D, dtype, seed, split=False, state=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, d = (r(B, H, N, D).to(dtype).cuda() for _ in range(4))
    if split:
        q, k, v, d = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, d))
    s0, ds = (r(B, H, D, D).cuda() for _ in range(2)) if state else (None, None)
    log_decay = torch.log1p(-torch.exp2(-1.0 - 9.0 * torch.rand(H, generator=g))).cuda()
    return q, k, v, d, s0, ds, log_decay


def _check(q, k, v, d, s0, ds, log_decay, lens=None, scale=None, clean=None):
    """Forward and backward through the public call against the oracle.  clean: the same tensors with nothing odd in rows that do not count."""
    from flashnystrom_b200 import _C, decay_attention
    dtype, D = q.dtype, q.shape[-1]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([s0.detach().requires_grad_(True)] if s0 is not None else [])
    out, state = decay_attention(*leaves[:3], log_decay, scale=scale, initial_state=leaves[3] if s0 is not None else None, seq_lens=lens, return_state=True)
    grads = torch.autograd.grad((out, state) if ds is not None else out, leaves, (d, ds) if ds is not None else d)
    torch.cuda.synchronize()
    _C.check_device_status()
    cq, ck, cv, cd = (t.detach().double().requires_grad_(True) for t in (clean or (q, k, v, d)))
    cs = None if s0 is None else s0.double().requires_grad_(True)
    ref, ref_state = O.decay_attention(cq, ck, cv, log_decay, scale, cs, lens)
    top = (ref * cd.detach()).sum() + (0 if ds is None else (ref_state * ds.double()).sum())
    wanted = [cq, ck, cv] + ([cs] if cs is not None else [])
    refs = torch.autograd.grad(top, wanted)
    b = O.decay_bounds(cq.detach(), ck.detach(), cv.detach(), cd.detach(), log_decay, O.isqrt(D) if scale is None else scale,
                       None if cs is None else cs.detach(), None if ds is None else ds.double(), lens, dtype)
    O.within(out, ref, b[0], dtype)
    O.within(state, ref_state, b[1], torch.float32)
    for got, r, bound, t in zip(grads, refs, b[2:], (dtype, dtype, dtype, torch.float32)):
        assert got.dtype == t
        O.within(got, r, bound, t)
    return out, state, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,N,D,split,state", [
    (1, 1, 1, 16, False, True), (2, 3, 2, 64, True, False), (2, 3, 63, 32, True, True), (1, 2, 64, 64, False, True), (1, 2, 65, 128, True, True),
    (2, 2, 127, 64, False, False), (2, 2, 128, 128, True, True), (1, 3, 129, 16, True, True), (1, 2, 129, 64, False, True), (3, 2, 1000, 64, True, True),
    (1, 2, 1021, 128, False, True), (1, 1, 4099, 64, False, True), (1, 1, 4097, 128, True, False), (2, 1, 3001, 32, False, True), (5, 40, 200, 64, True, True)])
def test_forward_and_backward(cuda_device, dtype, B, H, N, D, split, state):
    out, _, grads = _check(*_inputs(B, H, N, D, dtype, N + D, split, state))
    if split and H > 1 and N > 1:
        assert all(t.transpose(1, 2).is_contiguous() for t in (out, *grads[:3])), "the order of memory of the inputs is kept"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("decay", [0.0, -INF, -1e-7, -0.5, -5.0, -200.0])
def test_decays(cuda_device, dtype, D, decay):
    """None at all, one that leaves a token to itself, and what underflows within a chunk."""
    q, k, v, d, s0, ds, log_decay = _inputs(1, 2, 333, D, dtype, 7)
    log_decay[:] = decay
    _check(q, k, v, d, s0, ds, log_decay)


def test_no_decay_over_a_long_sequence(cuda_device):
    """The state is multiplied chunk after chunk: a rounded factor would add up (float32, 20000 rows, slow decay)."""
    q, k, v, d, s0, ds, log_decay = _inputs(1, 1, 20000, 16, torch.float32, 3)
    log_decay[:] = -1.23e-5
    _check(q, k, v, d, s0, ds, log_decay)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,split", [(700, 64, True), (700, 128, False), (130, 32, True), (5000, 64, False)])
def test_padded_batch(cuda_device, dtype, N, D, split):
    """Lengths of zero, one, a chunk and its neighbours, all rows, and values out of range; NaN and infinities behind them."""
    lens = torch.tensor([0, 1, N, 127, 128, 129, 64, N - 1, -5, N + 100], dtype=torch.int32).clamp(max=N + 100)
    B = len(lens)
    q, k, v, d, s0, ds, log_decay = _inputs(B, 2, N, D, dtype, N, split)
    clean = tuple(t.clone() for t in (q, k, v, d))
    for i, n in enumerate(lens.tolist()):
        n = max(0, min(N, n))
        for t, bad in ((q, float("nan")), (k, INF), (v, float("nan")), (d, -INF)):
            t[i, :, n:] = bad
    out, state, grads = _check(q, k, v, d, s0, ds, log_decay, lens.cuda(), clean=clean)
    for i, n in enumerate(lens.tolist()):
        n = max(0, min(N, n))
        for t in (out, *grads[:3]):
            assert not t[i, :, n:].any(), "rows past the length are zeros"
    assert torch.equal(state[0], s0[0]) and torch.equal(grads[3][0], ds[0]), "an empty sequence hands its state through"


def _strided(kind, t):
    B, H, N, D = t.shape
    if kind == "fused":                   # q, k, v side by side in one projection
        room = torch.full((B, N, H, 3 * D), float("nan"), dtype=t.dtype, device=t.device)
        view = room[..., D:2 * D].permute(0, 2, 1, 3)
    elif kind == "odd_start":             # a pointer aligned to the type alone
        room = torch.empty(B * H * N * D + 1, dtype=t.dtype, device=t.device)
        view = room[1:].view(B, H, N, D)
    elif kind == "odd_rows":              # rows one element apart from a multiple of sixteen bytes
        view = torch.empty(B, H, N, D + 1, dtype=t.dtype, device=t.device)[..., :D]
    elif kind == "batch_inner":           # batch between rows and heads
        view = torch.empty(N, B, H, D, dtype=t.dtype, device=t.device).permute(1, 2, 0, 3)
    elif kind == "last_strided":          # the last dimension is not contiguous
        view = torch.empty(B, H, D, N, dtype=t.dtype, device=t.device).transpose(2, 3)
    view.copy_(t)
    return view


@pytest.mark.parametrize("kind", ["fused", "odd_start", "odd_rows", "batch_inner", "last_strided"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(cuda_device, kind, dtype):
    q, k, v, d, s0, ds, log_decay = _inputs(2, 3, 200, 64, dtype, 11)
    plain = _check(q, k, v, d, s0, ds, log_decay)
    other = _check(*(_strided(kind, t) for t in (q, k, v, d)), s0, ds, log_decay)
    if kind not in ("odd_start", "odd_rows"):       # (these may take another kernel)
        assert torch.equal(plain[0], other[0]) and torch.equal(plain[1], other[1])
    # one of them odd is enough
    _check(q, _strided(kind, k), v, d, s0, ds, log_decay)
    _check(q, k, v, _strided(kind, d), s0, ds, log_decay)


def test_broadcast_inputs(cuda_device):
    """Keys shared by the heads: the gradient of the shared tensor is the sum over them."""
    from flashnystrom_b200 import decay_attention
    q, k, v, d, _, _, log_decay = _inputs(2, 4, 150, 64, torch.float32, 5, state=False)
    shared = k[:, :1].detach().requires_grad_(True)
    out = decay_attention(q, shared.expand(-1, 4, -1, -1), v, log_decay)
    (g,) = torch.autograd.grad(out, shared, d)
    own = k[:, :1].expand(-1, 4, -1, -1).contiguous().requires_grad_(True)
    out2 = decay_attention(q, own, v, log_decay)
    (g2,) = torch.autograd.grad(out2, own, d)
    assert torch.equal(out, out2) and torch.allclose(g, g2.sum(1, keepdim=True), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_in_pieces(cuda_device, dtype, D):
    """A prompt in two calls and a few single tokens, each going on from the state before, against the whole sequence."""
    from flashnystrom_b200 import decay_attention, decay_attention_step
    q, k, v, _, s0, _, log_decay = _inputs(2, 3, 450, D, dtype, 9)
    ref, ref_state = O.decay_attention(q.double(), k.double(), v.double(), log_decay, None, s0.double())
    b = O.decay_bounds(q.double(), k.double(), v.double(), None, log_decay, O.isqrt(D), s0.double(), None, None, dtype)
    a, state = decay_attention(q[:, :, :300], k[:, :, :300], v[:, :, :300], log_decay, initial_state=s0, return_state=True)
    c, state = decay_attention(q[:, :, 300:440], k[:, :, 300:440], v[:, :, 300:440], log_decay, initial_state=state, return_state=True)
    tokens = [decay_attention_step(q[:, :, i], k[:, :, i], v[:, :, i], state, log_decay) for i in range(440, 450)]
    O.within(torch.cat([a, c, torch.stack(tokens, 2)], 2), ref, b[0], dtype)
    O.within(state, ref_state, 1.5 * b[1], torch.float32)


@pytest.mark.parametrize("scale", [1.0, -0.3, 1e-3, 100.0])
def test_scale(cuda_device, scale):
    for dtype in (torch.float32, torch.bfloat16):
        _check(*_inputs(1, 2, 300, 64, dtype, 21), scale=scale)


def test_gradients_against_differences(cuda_device):
    """The output is linear in each of q, k, v and the initial state: a central difference is the derivative, to float32 rounding."""
    from flashnystrom_b200 import decay_attention
    q, k, v, d, s0, ds, log_decay = _inputs(1, 2, 150, 32, torch.float32, 13)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]

    def f(*x):
        return decay_attention(*x[:3], log_decay, initial_state=x[3], return_state=True)
    grads = torch.autograd.grad(f(*leaves), leaves, (d, ds))
    for i, g in enumerate(grads):
        e = torch.randn_like(leaves[i])
        plus, minus = ([t.detach() if j != i else t.detach() + s * e for j, t in enumerate(leaves)] for s in (1, -1))
        (o1, s1), (o2, s2) = f(*plus), f(*minus)
        by_difference = (((o1.double() - o2.double()) * d).sum() + ((s1.double() - s2.double()) * ds).sum()) / 2
        mass = float((o1.abs().double() * d.abs()).sum() + (o2.abs().double() * d.abs()).sum() + ((s1.abs() + s2.abs()) * ds.abs()).double().sum())
        assert abs(float((g.double() * e).sum() - by_difference)) <= 2.0 ** -20 * mass


def test_only_what_is_wanted(cuda_device):
    from flashnystrom_b200 import decay_attention
    q, k, v, d, s0, ds, log_decay = _inputs(1, 2, 300, 64, torch.float16, 17)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
    out, state = decay_attention(*leaves[:3], log_decay, initial_state=leaves[3], return_state=True)
    full = torch.autograd.grad(out, leaves, d, retain_graph=True)
    for i, t in enumerate(leaves):
        args = [x.detach() if j != i else x for j, x in enumerate(leaves)]
        (g,) = torch.autograd.grad(decay_attention(*args[:3], log_decay, initial_state=args[3]), t, d)
        assert torch.equal(g, full[i])
    g = torch.autograd.grad(state, leaves, ds, allow_unused=True)         # the state alone
    assert g[0] is None or not g[0].any()
    assert bool(g[1].any()) and bool(g[2].any()) and bool(g[3].any())
    x = decay_attention(leaves[0], k, v, log_decay)
    (g,) = torch.autograd.grad(x, leaves[0], d, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), leaves[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_bits_again_and_on_another_stream(cuda_device, dtype, D):
    """Two calls, a call on a side stream while the first stream is busy, and two threads: the same bits."""
    from flashnystrom_b200 import decay_attention
    q, k, v, d, s0, ds, log_decay = _inputs(2, 3, 2000, D, dtype, 19)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, s0)]
        out, state = decay_attention(*leaves[:3], log_decay, initial_state=leaves[3], return_state=True)
        return [out.detach(), state.detach(), *torch.autograd.grad((out, state), leaves, (d, ds))]
    first = once()
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(10):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    results = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            results[i] = once()
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(first, results[i]))


def test_captured_and_replayed(cuda_device):
    """Two graphs of one pool replayed in turn with new inputs: outputs and gradients as eager calls give them."""
    from flashnystrom_b200 import decay_attention, decay_attention_step
    q, k, v, d, s0, ds, log_decay = _inputs(1, 4, 1500, 64, torch.bfloat16, 23)
    state = s0.clone()
    static = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out = decay_attention(*static, log_decay, initial_state=s0)
        return [out.detach(), *torch.autograd.grad(out, static, d)]

    def token():
        return decay_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], state, log_decay)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
            token()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = step()
    with torch.cuda.graph(g2, pool=g1.pool()):
        r2 = token()
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for t in static:
                t.copy_(torch.randn(t.shape, generator=gen))
        state.copy_(s0)
        g1.replay()
        got = [t.clone() for t in r1]
        g2.replay()
        token_got, state_got = r2.clone(), state.clone()
        state.copy_(s0)
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert torch.equal(token_got, token()) and torch.equal(state_got, state)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,D", [(1, 1, 16), (3, 5, 32), (37, 5, 64), (7, 2, 128), (300, 3, 128), (130, 8, 64)])
def test_step(cuda_device, dtype, B, H, D):
    from flashnystrom_b200 import decay_attention_step
    q, k, v, _, _, _, log_decay = _inputs(B, H, 1, D, dtype, B, state=False)
    q, k, v = (t[:, :, 0] for t in (q, k, v))
    g = torch.Generator().manual_seed(D)
    for pool in (0, B + 3):
        slots = None
        if pool:
            slots = torch.randperm(pool, generator=g)[:B].to(torch.int32)
            slots[::5] = -1
            if B > 4:
                slots[3], slots[4] = pool, 2 ** 31 - 1            # past the end: idle as well
        state = torch.randn(pool or B, H, D, D, generator=g).cuda()
        ref, ref_state = O.decay_step(q.double(), k.double(), v.double(), state.double(), log_decay, None, slots)
        mass, mass_state = O.decay_step(q.double().abs(), k.double().abs(), v.double().abs(), state.double().abs(), log_decay, None, slots)
        out = decay_attention_step(q, k, v, state, log_decay, slots=None if slots is None else slots.cuda())
        O.within(state, ref_state, 3 * 2.0 ** -24 * mass_state, torch.float32)
        O.within(out, ref, (D + 8) * 2.0 ** -24 * mass, dtype)
        if slots is not None:
            idle = (slots < 0) | (slots >= pool)
            assert not out[idle.cuda()].any()


@pytest.mark.parametrize("D", [32, 64, 128])
def test_step_rows_of_one_slot_follow_one_another(cuda_device, D):
    from flashnystrom_b200 import decay_attention_step
    B = 400
    q, k, v, _, _, _, log_decay = _inputs(B, 2, 1, D, torch.float32, 2, state=False)
    q, k, v = (t[:, :, 0] for t in (q, k, v))
    slots = torch.randint(-1, 60, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    slots[:5] = 7
    state = torch.randn(60, 2, D, D).cuda()
    ref, ref_state = O.decay_step(q.double(), k.double(), v.double(), state.double(), log_decay, None, slots)
    mass, mass_state = O.decay_step(q.double().abs(), k.double().abs(), v.double().abs(), state.double().abs(), log_decay, None, slots)
    again = state.clone()
    out = decay_attention_step(q, k, v, state, log_decay, slots=slots.cuda())
    O.within(state, ref_state, 20 * 3 * 2.0 ** -24 * mass_state, torch.float32)
    O.within(out, ref, (D + 80) * 2.0 ** -24 * mass, torch.float32)
    assert torch.equal(out, decay_attention_step(q, k, v, again, log_decay, slots=slots.cuda())) and torch.equal(state, again)


def test_step_strides_and_decays(cuda_device):
    from flashnystrom_b200 import decay_attention_step
    B, H, D = 6, 3, 64
    room = torch.randn(B, 3, H, D + 1, dtype=torch.float16).cuda()
    q, k, v = room[:, 0, :, :D], room[:, 1, :, 1:], room[:, 2, :, :D]
    state = torch.randn(B, H, D, D).cuda()
    log_decay = torch.tensor([0.0, -INF, -0.1]).cuda()
    ref, ref_state = O.decay_step(q.double(), k.double(), v.double(), state.double(), log_decay)
    state[:, 1] = float("nan")                 # -inf: nothing of the past
    before = state._version
    out = decay_attention_step(q, k, v, state, log_decay)
    assert state._version > before
    O.within(state, ref_state, 1e-5 * torch.ones_like(ref_state), torch.float32)
    O.within(out, ref, 1e-4 * torch.ones_like(ref), torch.float16)
    assert decay_attention_step(q[:0], k[:0], v[:0], state[:0], log_decay).shape == (0, H, D)


def test_empty(cuda_device):
    from flashnystrom_b200 import decay_attention
    q = torch.randn(2, 3, 0, 64, device="cuda", dtype=torch.float16)
    s0 = torch.randn(2, 3, 64, 64, device="cuda", requires_grad=True)
    out, state = decay_attention(q, q, q, torch.zeros(3, device="cuda"), initial_state=s0, return_state=True)
    assert out.shape == q.shape and torch.equal(state, s0)
    state.sum().backward()
    assert torch.equal(s0.grad, torch.ones_like(s0))
    out, state = decay_attention(q[:0], q[:0], q[:0], torch.zeros(3, device="cuda"), return_state=True)
    assert out.shape == (0, 3, 0, 64) and state.shape == (0, 3, 64, 64)
    leaves = [torch.zeros(2, 3, 0, 64, device="cuda", requires_grad=True) for _ in range(3)]
    grads = torch.autograd.grad(decay_attention(*leaves, torch.zeros(3, device="cuda")).sum(), leaves)
    assert all(g.shape == (2, 3, 0, 64) for g in grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** 64])
def test_scale_at_its_ends(cuda_device, dtype, scale):
    """(fp16 outputs would leave their range; those of the others and their sums, 2^64 times a few hundred, do not.)"""
    _check(*_inputs(1, 2, 700, 64, dtype, 23), scale=scale)


def test_c_abi_writes_nothing_but_its_rows(cuda_device):
    """Output rows inside a larger tensor: what lies between and behind them is left as it was."""
    from flashnystrom_b200 import _C, _lib
    lib = _lib.load()
    for D in (64, 128, 16):
        B, H, N = 2, 2, 200
        q, k, v, _, _, _, log_decay = _inputs(B, H, N, D, torch.bfloat16, 3, state=False)
        room = torch.full((B, H, N + 7, D + 64), 7.0, dtype=torch.bfloat16, device="cuda")
        out = room[:, :, :N, :D]
        shape = _lib.DecayShape(B, H, N, D, _lib.FNB_BF16, D ** -0.5, 0)
        rows = lambda t: _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))  # noqa: E731
        ws = torch.empty(lib.fnb_decay_workspace_bytes(C.byref(shape)), dtype=torch.uint8, device="cuda")
        seg = torch.empty(lib.fnb_decay_segment_floats(C.byref(shape)) + 1, device="cuda")
        args = _lib.DecayFwdArgs(shape, rows(q), rows(k), rows(v), rows(out), log_decay.data_ptr(), None, None, None, seg.data_ptr(), ws.data_ptr(),
                                 ws.numel(), 0, torch.cuda.current_stream().cuda_stream, _C._status(q.device).data_ptr())
        _lib.check(lib.fnb_decay_forward(C.byref(args)))
        ref, _ = O.decay_attention(q.double(), k.double(), v.double(), log_decay)
        b = O.decay_bounds(q.double(), k.double(), v.double(), None, log_decay, O.isqrt(D), None, None, None, torch.bfloat16)
        O.within(out, ref, b[0], torch.bfloat16)
        assert bool((room[:, :, N:] == 7).all()) and bool((room[:, :, :, D:] == 7).all())


def test_module(cuda_device):
    """The block forward in one call, in a padded batch, and token by token; its gradients against the same block in float64."""
    from flashnystrom_b200 import DecayAttention
    torch.manual_seed(0)
    m = DecayAttention(256, heads=4).cuda()
    x = torch.randn(2, 90, 256, device="cuda", requires_grad=True)
    y, state = m(x, return_state=True)
    d = torch.randn_like(y)
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(y, [x, *m.parameters()], d)
    p = {n: t.detach().double().requires_grad_(True) for n, t in m.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)
    q, k, v = ((x64 @ p[n + "_proj.weight"].T).view(2, 90, 4, 64).transpose(1, 2) for n in "qkv")
    o, ref_state = O.decay_attention(q, k, v, m.log_decay)
    o = O.layer_norm(o.transpose(1, 2).reshape(2, 90, 256), p["norm_weight"], p["norm_bias"], m.eps, 4)
    ref = o @ p["out_proj.weight"].T
    refs = torch.autograd.grad(ref, [x64, *p.values()], d.double())
    close = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert close(y, ref) <= 1e-5 and close(state, ref_state) <= 1e-5
    for n, a, b in zip(["x"] + names, grads, refs):
        assert close(a, b) <= 1e-4, n
    with torch.no_grad():
        s = m.new_state(2)
        tokens = torch.stack([m.step(x[:, i].contiguous(), s) for i in range(90)], 1)
        assert close(tokens, ref.detach()) <= 1e-5 and close(s, ref_state.detach()) <= 1e-5
        lens = torch.tensor([90, 37], dtype=torch.int32, device="cuda")
        z = m(x, seq_lens=lens)
        assert torch.equal(z[0], y[0]) and close(z[1, :37], ref[1, :37].detach()) <= 1e-5
    h = DecayAttention(256, heads=4).cuda().to(torch.bfloat16)
    assert h.log_decay.dtype == torch.float32 and h.q_proj.weight.dtype == torch.bfloat16
    h(torch.randn(1, 10, 256, device="cuda", dtype=torch.bfloat16)).sum().backward()
    assert all(t.grad is not None and bool(torch.isfinite(t.grad).all()) for t in h.parameters())


def test_compiled(cuda_device):
    """A compiler traces both operators without a break; the results are the eager ones."""
    from flashnystrom_b200 import decay_attention, layer_norm
    q, k, v, d, s0, ds, log_decay = _inputs(1, 2, 300, 64, torch.float32, 31)
    w = torch.randn(128, device="cuda")

    def f(q, k, v, s0, w):
        out, state = decay_attention(q, k, v, log_decay, initial_state=s0, return_state=True)
        return layer_norm(out.transpose(1, 2).reshape(1, 300, 128), w, None, num_groups=2), state

    def run(g):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0, w)]
        y, state = g(*leaves)
        return [y, state, *torch.autograd.grad((y, state), leaves, (torch.ones_like(y) * 0.5 + y.detach(), ds))]
    for a, b in zip(run(f), run(torch.compile(f, fullgraph=True, backend="aot_eager"))):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_compiled_step(cuda_device):
    from flashnystrom_b200 import decay_attention_step
    q, k, v, _, s0, _, log_decay = _inputs(3, 2, 1, 64, torch.float16, 33)
    q, k, v = (t[:, :, 0] for t in (q, k, v))
    a, b = s0.clone(), s0.clone()

    def f(state):
        return decay_attention_step(q, k, v, state, log_decay) * 2
    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(a), f(b)) and torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("N", [300, 6000])
def test_scores_and_states_past_the_range_of_fp16(cuda_device, D, N):
    """Scores of up to several hundred thousand and states of several million, with outputs of order one; the range is left in some tiles only."""
    q, k, v, d, s0, ds, log_decay = _inputs(1, 2, N, D, torch.float16, 41)
    q, k, v, d = (t.float() for t in (q, k, v, d))
    q, k, v, d = q * 100, k * 100, v * 1e-4, d * 1e-4                    # scores
    q[:, :, N // 2:] *= 1e-3
    _check(*(t.half() for t in (q, k, v, d)), s0 * 1e-6, ds * 1e-6, log_decay, scale=1.0)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(1, 2, N, D, generator=g).cuda() * 5 + 200 for _ in range(2))      # states: sums of one sign
    q, d = (torch.randn(1, 2, N, D, generator=g).cuda() * 1e-5 for _ in range(2))
    log_decay[:] = -1e-3
    _check(*(t.half() for t in (q, k, v, d)), s0 * 1e6, ds, log_decay)


@pytest.mark.parametrize("dtype", DTYPES)
def test_segments_of_odd_lengths(cuda_device, dtype):
    """Sequences that are split over many SMs: lengths that end in the first, a middle and the last segment, whole and partial chunks, from states and to them."""
    for N, D, lens in ((9000, 64, [9000, 1, 4500, 0, 8999, 128]), (7001, 128, [7001, 3000, 6999]), (5000, 16, [4999, 100])):
        q, k, v, d, s0, ds, log_decay = _inputs(len(lens), 1, N, D, dtype, N, split=True)
        _check(q, k, v, d, s0, ds, log_decay, torch.tensor(lens, dtype=torch.int32).cuda())
        _check(q, k, v, d, None, None, log_decay, torch.tensor(lens, dtype=torch.int32).cuda())


def test_calls_side_by_side(cuda_device):
    """Different shapes on two streams at once, each with workspaces of its own."""
    from flashnystrom_b200 import decay_attention
    sets = [_inputs(1, 4, 3000, 64, torch.bfloat16, 1), _inputs(2, 2, 2500, 128, torch.float16, 2)]
    alone = [decay_attention(s[0], s[1], s[2], s[6], initial_state=s[4], return_state=True) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        together = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                together.append(decay_attention(s[0], s[1], s[2], s[6], initial_state=s[4], return_state=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(alone, together) for a, b in zip(x, y))


def test_refusals(cuda_device):
    from flashnystrom_b200 import decay_attention, decay_attention_step
    q = torch.randn(2, 3, 20, 64, device="cuda", dtype=torch.float16)
    g = torch.zeros(3, device="cuda")
    s = torch.zeros(2, 3, 64, 64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    for message, call in [
            ("no CPU path", lambda: decay_attention(q.cpu(), q, q, g)), ("no CPU path", lambda: decay_attention(q, q, q, g.cpu())),
            ("dtypes must match", lambda: decay_attention(q, q.float(), q, g)), ("shapes must match", lambda: decay_attention(q, q[:, :2], q, g)),
            ("must be 4D", lambda: decay_attention(q[0], q[0], q[0], g)), ("one value a head", lambda: decay_attention(q, q, q, g[:2])),
            ("one value a head", lambda: decay_attention(q, q, q, g.half())), ("head_dim must be", lambda: decay_attention(*(q[..., :48],) * 3, g)),
            ("has no gradient", lambda: decay_attention(q, q, q, g.clone().requires_grad_(True))), ("scale must be", lambda: decay_attention(q, q, q, g, scale=0)),
            ("scale must be", lambda: decay_attention(q, q, q, g, scale=float("nan"))), ("must be float32", lambda: decay_attention(q, q, q, g, initial_state=s.half())),
            (r"\(B, H, D, D\)", lambda: decay_attention(q, q, q, g, initial_state=s[:1])), ("int32", lambda: decay_attention(q, q, q, g, seq_lens=lens.long())),
            ("one length a sequence", lambda: decay_attention(q, q, q, g, seq_lens=lens[:1])), ("Supported dtypes", lambda: decay_attention(*(q.double(),) * 3, g)),
            ("must be a CUDA tensor", lambda: decay_attention(q, q, q, g, seq_lens=lens.cpu()))]:
        with pytest.raises(RuntimeError, match=message):
            call()
    t = q[:, :, 0]
    for message, call in [
            ("no CPU path", lambda: decay_attention_step(t, t, t, s.cpu(), g)), ("must be 3D", lambda: decay_attention_step(q, q, q, s, g)),
            ("contiguous float32", lambda: decay_attention_step(t, t, t, s.transpose(2, 3), g)), ("contiguous float32", lambda: decay_attention_step(t, t, t, s.half(), g)),
            ("one entry for each row", lambda: decay_attention_step(t, t, t, s[:1], g)), ("int32", lambda: decay_attention_step(t, t, t, s, g, slots=lens.long())),
            ("has no gradient", lambda: decay_attention_step(t.clone().requires_grad_(True), t, t, s, g)), ("scale must be", lambda: decay_attention_step(t, t, t, s, g, scale=0.0)),
            ("head_dim must be", lambda: decay_attention_step(*(t[..., :48],) * 3, s[..., :48, :48].contiguous(), g))]:
        with pytest.raises(RuntimeError, match=message):
            call()
