"""Calls of the attention with a decay and of the layer norm at the edges of what their documentation allows."""
import ctypes as C

import pytest
import torch
import torch._dynamo.testing

from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu

INF = float("inf")


def _normal(*shape, seed=0, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * mul).to(dtype).cuda()


def _c_rows(t):
    from flashnystrom_b200 import _lib
    return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _c_call(q, k, v, d, log_decay, initial, final, d_final, d_initial, flags):
    """Forward and backward through the C ABI: (out, dq, dk, dv); the states are read and written where the caller says."""
    from flashnystrom_b200 import _C, _lib
    lib = _lib.load()
    B, H, N, D = q.shape
    shape = _lib.DecayShape(B, H, N, D, _C._DTYPES[q.dtype], D ** -0.5, flags)
    out, dq, dk, dv = (torch.full_like(q, float("nan")) for _ in range(4))
    ws = torch.empty(lib.fnb_decay_workspace_bytes(C.byref(shape)), dtype=torch.uint8, device="cuda")
    seg = torch.empty(lib.fnb_decay_segment_floats(C.byref(shape)) + 1, device="cuda")
    stream, status = torch.cuda.current_stream().cuda_stream, _C._status(q.device).data_ptr()
    entered = initial.clone()      # (the backward is handed what entered, wherever the forward's final state went)
    a = _lib.DecayFwdArgs(shape, *(_c_rows(t) for t in (q, k, v, out)), log_decay.data_ptr(), None, initial.data_ptr(), final.data_ptr(), seg.data_ptr(),
                          ws.data_ptr(), ws.numel(), 0, stream, status)
    _lib.check(lib.fnb_decay_forward(C.byref(a)))
    b = _lib.DecayBwdArgs(shape, *(_c_rows(t) for t in (q, k, v, d, dq, dk, dv)), log_decay.data_ptr(), None, entered.data_ptr(), d_final.data_ptr(),
                          d_initial.data_ptr(), seg.data_ptr(), ws.data_ptr(), ws.numel(), 0, stream, status)
    _lib.check(lib.fnb_decay_backward(C.byref(b)))
    torch.cuda.synchronize()
    return out, dq, dk, dv


@pytest.mark.parametrize("dtype,D,generic", [(torch.float16, 64, False), (torch.bfloat16, 128, False), (torch.float16, 64, True), (torch.float32, 32, False)])
@pytest.mark.parametrize("N", [1, 100, 5000])
def test_states_updated_where_they_lie(cuda_device, dtype, D, generic, N):
    """The final state in the initial state's memory, and its gradient likewise: one segment or many, the same bits as with buffers of their own."""
    from flashnystrom_b200 import _lib
    flags = _lib.FNB_FLAG_FORCE_GENERIC if generic else 0
    q, k, v, d = (_normal(1, 3, N, D, seed=i, dtype=dtype) for i in range(4))
    s0, ds = (_normal(1, 3, D, D, seed=i) for i in (5, 6))
    log_decay = torch.tensor([-0.1, -0.01, -1e-3], device="cuda")
    final, d_initial = torch.empty_like(s0), torch.empty_like(s0)
    apart = _c_call(q, k, v, d, log_decay, s0, final, ds, d_initial, flags)
    ref, _ = O.decay_attention(q.double(), k.double(), v.double(), log_decay, None, s0.double())
    O.within(apart[0], ref, O.decay_bounds(q.double(), k.double(), v.double(), None, log_decay, O.isqrt(D), s0.double(), None, None, dtype)[0], dtype)
    state, grad = s0.clone(), ds.clone()
    there = _c_call(q, k, v, d, log_decay, state, state, grad, grad, flags)
    assert all(torch.equal(a, b) for a, b in zip(apart, there))
    assert torch.equal(state, final) and torch.equal(grad, d_initial)


@pytest.mark.parametrize("decay", [-2.0 ** -12.1, -1.23e-5])
@pytest.mark.parametrize("rows", [1, 2048])
def test_many_tokens_with_a_slow_decay(cuda_device, decay, rows):
    """16384 tokens, one a call or 2048 that name the same state.  Each token rounds the state once, by at most half a step (2^-24, rms 2^-24 / sqrt 3 of it), in no
    direction: over the tokens that are remembered, 1 / (2 |g|) or all, that adds up as a random walk over the 4096 elements; four times its length is allowed.  A
    factor that is off by 2^-25 a token adds up in one direction instead: 5e-5 for the first of these decays."""
    from flashnystrom_b200 import decay_attention, decay_attention_step
    N, D = 16384, 64
    q, k, v = (_normal(1, 1, N, D, seed=i) for i in range(3))
    log_decay = torch.tensor([decay], device="cuda")
    state = torch.zeros(1, 1, D, D, device="cuda")
    t = lambda x: x[0, 0].view(N // rows, rows, 1, D)  # noqa: E731
    slots = torch.zeros(rows, dtype=torch.int32, device="cuda")
    for a, b, c in zip(t(q), t(k), t(v)):
        decay_attention_step(a, b, c, state, log_decay, slots=slots)
    w = torch.exp(log_decay.double() * torch.arange(N - 1, -1, -1, device="cuda").double()).unsqueeze(-1)
    ref = (k[0, 0].double() * w).T @ v[0, 0].double()
    off = lambda s: float((s[0, 0].double() - ref).norm() / ref.norm())  # noqa: E731
    room = 4 * 2.0 ** -24 / 3 ** 0.5 * min(N, 0.5 / abs(decay)) ** 0.5
    assert off(state) <= room
    _, whole = decay_attention(q, k, v, log_decay, return_state=True)
    assert off(whole) <= room


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bad", [INF, float("nan")])
def test_rows_behind_a_length_are_zeros_beside_rows_that_are_not_finite(cuda_device, dtype, D, bad):
    """An infinity or NaN in a row that counts, in the chunk in which its sequence ends, or in the state that enters it."""
    from flashnystrom_b200 import decay_attention
    N, lens = 300, [200, 130, 299, 70]
    log_decay = torch.tensor([-0.1, -0.01], device="cuda")
    for where in range(5):
        t = [_normal(4, 2, N, D, seed=i, dtype=dtype) for i in range(4)] + [_normal(4, 2, D, D, seed=5)]
        for b, n in enumerate(lens):
            if where < 4:
                t[where][b, :, n - 3, 1] = bad
            else:
                t[4][b, :, 1, 1] = bad
        leaves = [x.requires_grad_(True) for x in t[:3] + t[4:]]
        out = decay_attention(*leaves[:3], log_decay, initial_state=leaves[3], seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        grads = torch.autograd.grad(out, leaves, t[3])
        for b, n in enumerate(lens):
            for x in (out, *grads[:3]):
                assert not x[b, :, n:].any()
            assert where == 3 or not torch.isfinite(out[b]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D", [(3, 64), (300, 64), (300, 128), (700, 16), (5000, 64)])
def test_a_decay_to_nothing_takes_what_is_not_finite_with_it(cuda_device, dtype, N, D):
    """log_decay -inf: nothing of the state that enters is left, whatever it holds, as in the step; backwards the gradient of the final state reaches the
    last row alone."""
    from flashnystrom_b200 import decay_attention
    q, k, v, d = (_normal(1, 2, N, D, seed=i, dtype=dtype) for i in range(4))
    log_decay = torch.tensor([-INF, -300.0], device="cuda")
    s0, ds = _normal(1, 2, D, D, seed=4), _normal(1, 2, D, D, seed=5)
    s0[:, :, 0, 0], s0[:, :, 1, 1], ds[:, :, 2, 2] = float("nan"), INF, float("nan")
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]
    out, state = decay_attention(*leaves[:3], log_decay, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad((out, state), leaves, (d, ds))
    for t in (out, state, grads[0], grads[1][:, :, :max(0, N - 128)], grads[2][:, :, :max(0, N - 128)], grads[3]):
        assert torch.isfinite(t).all()
    ref, ref_state = O.decay_attention(q.detach().double(), k.detach().double(), v.detach().double(), log_decay)
    b = O.decay_bounds(q.detach().double(), k.detach().double(), v.detach().double(), None, log_decay, O.isqrt(D), None, None, None, dtype)
    O.within(out, ref, b[0], dtype)
    O.within(state, ref_state, b[1], torch.float32)


def _check_range(t, log_decay, s0=None, ds=None, scale=None, lens=None, final=True, in_range=True):
    """Outputs, states and gradients of fp16 calls within the roundings of values that are in range (no smallest step of fp16 but that of the result)."""
    from flashnystrom_b200 import _C, decay_attention
    leaves = [x.detach().requires_grad_(True) for x in t[:3]] + ([] if s0 is None else [s0.detach().requires_grad_(True)])
    out, state = decay_attention(*leaves[:3], log_decay, scale=scale, initial_state=None if s0 is None else leaves[3], seq_lens=lens, return_state=True)
    grads = torch.autograd.grad(out if ds is None else (out, state), leaves, t[3] if ds is None else (t[3], ds))
    torch.cuda.synchronize()
    _C.check_device_status()
    wide = [x.detach().double() for x in t]
    w0, ws = (None if x is None else x.double() for x in (s0, ds))
    asked = [x.clone().requires_grad_(True) for x in wide[:3]] + ([] if s0 is None else [w0.clone().requires_grad_(True)])
    ref, ref_state = O.decay_attention(*asked[:3], log_decay, scale, None if s0 is None else asked[3], lens)
    refs = torch.autograd.grad((ref * wide[3]).sum() + (0 if ds is None else (ref_state * ws).sum()), asked)
    bounds = O.decay_bounds(*wide, log_decay, O.isqrt(t[0].shape[-1]) if scale is None else scale, w0, ws, lens, t[0].dtype, in_range=in_range)
    O.within(out, ref, bounds[0], t[0].dtype)
    if final:
        O.within(state, ref_state, bounds[1], torch.float32)
    for g, r, b in zip(grads, refs, bounds[2:]):
        O.within(g, r, b, g.dtype)


# magnitudes of q, k, v and the gradient, and the scale (None: D^-1/2)
SMALL = [(1.0, 1.0, 1.0, 1e-5, None), (1.0, 1.0, 2.0 ** 12, 1.0, 2.0 ** -24), (1e-3, 1e-3, 2.0 ** 12, 1e-3, None), (1.0, 1e-4, 1.0, 1.0, 100.0), (30.0, 30.0, 1e-4, 0.3, None)]


@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("size", SMALL)
def test_small_scores_in_fp16(cuda_device, D, size):
    """Scores far below fp16's normal numbers, one chunk: their products are as exact as those of any others."""
    t = [_normal(2, 3, 120, D, seed=i, mul=m).half() for i, m in enumerate(size[:4])]
    t[0][:, :, 5:50:3] *= 1e-2      # (rows of their own magnitude)
    _check_range(t, torch.tensor([-0.2, -0.01, 0.0], device="cuda"), scale=size[4], final=False)


@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("size", [2.0 ** -22, 2.0 ** -40, 2.0 ** 40])
def test_states_of_any_size_in_fp16(cuda_device, D, size):
    """States that enter a chunk, and their gradients, far below fp16's numbers and far above, brought back by the scale."""
    scale = 2.0 ** -10 / size
    t = [_normal(2, 3, 120, D, seed=i, mul=m).half() for i, m in enumerate((1.0, 2.0 ** -10, 2.0 ** -10, 1.0))]
    t[0], t[3] = (x if size < 1 else x * 2.0 ** -6 for x in (t[0], t[3]))
    s0, ds = (_normal(2, 3, D, D, seed=i, mul=m) for i, m in ((4, size), (5, size * scale)))
    if size < 2.0 ** -30:      # (pairs would leave the range with so large a scale)
        t[1], t[2] = t[1] * 0, t[2] * 0
    _check_range(t, torch.tensor([-0.2, -0.01, 0.0], device="cuda"), s0, ds, scale=scale, final=False)


@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("size", SMALL)
@pytest.mark.parametrize("padded", [False, True])
def test_small_keys_over_chunks_in_fp16(cuda_device, D, size, padded):
    """The same over three chunks of sequences of one segment (there are more slices than SMs): what reaches a row from the chunks before it goes through the state.
    Chunks of their own magnitudes."""
    t = [_normal(50, 3, 300, D, seed=i, mul=m).half() for i, m in enumerate(size[:4])]
    for x in t:
        x[:, :, 128:256] *= 0.125
    lens = None
    if padded:
        lens = torch.tensor([300, 299, 257, 130, 1] * 10, dtype=torch.int32, device="cuda")
    scale = size[4] if size[4] is None else min(size[4], 10.0)      # (times 100 the gradient of k, scale sqrt(D rows), would leave the range)
    _check_range(t, torch.tensor([-0.2, -0.01, 0.0], device="cuda"), scale=scale, lens=lens, final=False)


@pytest.mark.parametrize("D", [64, 128, 16])
@pytest.mark.parametrize("N", [100, 700, 5000])
@pytest.mark.parametrize("size", [1e-5, 3e-4, 0.02, 0.5])
def test_small_keys_in_sums_in_fp16(cuda_device, D, N, size):
    """States that are handed out, of a sequence and of its segments, and their gradients: the sums of small keys (and queries, backwards) have FP32's bits."""
    t = [_normal(1, 2, N, D, seed=i, mul=m).half() for i, m in enumerate((size, size, 1.0, 1.0))]
    _check_range(t, torch.tensor([-0.02, -1e-3], device="cuda"), _normal(1, 2, D, D, seed=7, mul=size), _normal(1, 2, D, D, seed=8, mul=size), scale=1 / size)


@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("N,lens", [(300, None), (1500, None), (6000, None), (1100, [1100, 1000, 513, 77])])
def test_keys_whose_size_changes_in_fp16(cuda_device, D, N, lens):
    """Rows that grow and shrink by many powers of two from block to block, zeros among them: sums begin small and meet what their factor is too large for, in
    either direction of time."""
    B = 1 if lens is None else len(lens)
    t = [_normal(B, 2, N, D, seed=i).half() for i in range(4)]
    sizes = torch.tensor([1e-5, 0.0, 1e-3, 1e-2, 0.1, 1.0, 20.0, 3.0, 1e-4, 0.05, 5.0, 1e-6, 1e-2], dtype=torch.float16, device="cuda")
    at = torch.arange(N, device="cuda")
    for x, rows in ((t[0], 45), (t[1], 32)):
        x *= sizes[at // rows % len(sizes)].view(1, 1, N, 1)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    _check_range(t, torch.tensor([-0.02, -1e-3], device="cuda"), _normal(B, 2, D, D, seed=7), _normal(B, 2, D, D, seed=8), lens=lens)
    again = [_call_state(t, lens) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*again))


def _call_state(t, lens):
    from flashnystrom_b200 import decay_attention
    return decay_attention(*t[:3], torch.tensor([-0.02, -1e-3], device="cuda"), seq_lens=lens, return_state=True)


def _three():
    """The three calls, each of one tensor, with what they are called on."""
    from flashnystrom_b200 import decay_attention, decay_attention_step, layer_norm
    q, k, v = (_normal(1, 2, 100, 64, seed=i, dtype=torch.float16) for i in range(3))
    log_decay, state, x = torch.tensor([-0.1, -0.01], device="cuda"), _normal(1, 2, 64, 64, seed=4), _normal(5, 64, seed=5)
    t = lambda a: a[:, :, 0].contiguous()  # noqa: E731
    kt, vt = t(k), t(v)
    return {"attention": (lambda a: decay_attention(a, k, v, log_decay), q), "step": (lambda a: decay_attention_step(a, kt, vt, state, log_decay), t(q)),
            "norm": (layer_norm, x)}, state


@pytest.mark.parametrize("name", ["attention", "step", "norm"])
def test_traced_and_recorded(cuda_device, name):
    """A trace, a mode that records operators and a subclass see the whole call: an operator that writes its result, and the state that a step writes."""
    from torch.utils._python_dispatch import TorchDispatchMode
    calls, state = _three()
    f, x = calls[name]
    before = state.clone()
    want = f(x)
    after = state.clone()
    state.copy_(before)
    traced = torch.jit.trace(f, (x,), check_trace=False)
    state.copy_(before)
    assert torch.equal(traced(x), want) and torch.equal(state, after)
    assert torch.equal(traced(-x) if name != "step" else want, f(-x) if name != "step" else want)

    class Recorder(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))
    state.copy_(before)
    with Recorder() as recorder:
        got = f(x)
    assert torch.equal(got, want) and torch.equal(state, after)
    assert any(s.startswith("flashnystrom_b200.") for s in recorder.seen), recorder.seen

    class Sub(torch.Tensor):
        pass
    state.copy_(before)
    assert torch.equal(f(x.as_subclass(Sub)).as_subclass(torch.Tensor), want) and torch.equal(state, after)


@pytest.mark.parametrize("name", ["attention", "step", "norm"])
def test_fake_tensors(cuda_device, name):
    """Tensors without memory, under their mode and outside of it: the call gives one like its result, and touches nothing."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    calls, state = _three()
    f, x = calls[name]
    want = f(x)
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    fake, before = mode.from_tensor(x), state.clone()
    with mode:
        got = f(fake)
    assert got.shape == want.shape and got.dtype == want.dtype and got.device == want.device and got.stride() == want.stride()
    if name != "step":      # (the state of the step is not one of these: it has to be under the mode)
        got = f(fake)
        assert got.shape == want.shape
    torch.cuda.synchronize()
    assert torch.equal(state, before)


@pytest.mark.parametrize("name", ["attention", "step", "norm"])
def test_tangents_are_refused(cuda_device, name):
    """A forward-mode derivative is an error, not zero; outside of one the call is as before."""
    from torch.autograd import forward_ad
    calls, state = _three()
    f, x = calls[name]
    with forward_ad.dual_level():
        f(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


def test_negative_views(cuda_device):
    """Tensors whose negative bit is set hold the opposite of what they are: read as what they are, in every place that takes one."""
    from flashnystrom_b200 import decay_attention, decay_attention_step, layer_norm
    neg = torch._neg_view
    q, k, v, d = (_normal(1, 2, 200, 64, seed=i) for i in range(4))
    s0, ds = _normal(1, 2, 64, 64, seed=5), _normal(1, 2, 64, 64, seed=6)
    log_decay = torch.tensor([-0.1, -0.01], device="cuda")

    def run(q, k, v, g, s0, d, ds):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, s0)]
        out, state = decay_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
        return [out, state, *torch.autograd.grad((out, state), leaves, (d, ds))]
    plain = run(-q, -k, -v, log_decay, -s0, -d, -ds)
    views = run(neg(q), neg(k), neg(v), neg(-log_decay), neg(s0), neg(d), neg(ds))
    assert all(torch.equal(a, b) for a, b in zip(plain, views))
    t = lambda a: a[:, :, 0]  # noqa: E731
    a, b = s0.clone(), s0.clone()
    assert torch.equal(decay_attention_step(t(-q), t(-k), t(-v), a, log_decay), decay_attention_step(neg(t(q)), neg(t(k)), neg(t(v)), b, neg(-log_decay))) and torch.equal(a, b)
    with pytest.raises(RuntimeError, match="negative view"):
        decay_attention_step(t(q), t(k), t(v), neg(a), log_decay)
    x, w, bias, dy = _normal(7, 64, seed=1), _normal(64, seed=2), _normal(64, seed=3), _normal(7, 64, seed=4)

    def norm(*p):
        leaves = [t.detach().requires_grad_(True) for t in p[:3]]
        y = layer_norm(*leaves)
        return [y, *torch.autograd.grad(y, leaves, p[3])]
    assert all(torch.equal(a, b) for a, b in zip(norm(-x, -w, -bias, -dy), norm(neg(x), neg(w), neg(bias), neg(dy))))


@pytest.mark.parametrize("shape", [(2, 3, 0, 64), (0, 3, 10, 64)])
def test_empty_calls_compiled(cuda_device, shape):
    """Nothing to attend to or to normalise: a compiled call gives what the eager one does, its gradients too."""
    from flashnystrom_b200 import decay_attention, layer_norm
    log_decay = torch.zeros(3, device="cuda")

    def f(q, s0):
        return decay_attention(q, q, q, log_decay, initial_state=s0, return_state=True)

    def g(x, w, b):
        return layer_norm(x, w, b)
    for fn, sizes in ((f, (shape, (shape[0], 3, 64, 64))), (g, ((0, 5, 48), (48,), (48,)))):
        torch._dynamo.reset()
        results = []
        for call in (fn, torch.compile(fn, fullgraph=True, backend="aot_eager")):
            leaves = [_normal(*s, seed=1).requires_grad_(True) for s in sizes]
            out = call(*leaves)
            out = out if isinstance(out, tuple) else (out,)
            results.append([*out, *torch.autograd.grad(sum(o.sum() for o in out), leaves)])
        for a, b in zip(*results):
            assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("split,state", [(True, False), (False, True)])
def test_compiled_calls_are_the_eager_ones(cuda_device, dtype, split, state):
    """Bits, order of memory and gradients of a compiled call, over lengths that it was not compiled for: one compilation serves them all."""
    from flashnystrom_b200 import decay_attention, layer_norm
    log_decay = torch.tensor([-0.1, -0.01], device="cuda")
    torch._dynamo.reset()
    counter = torch._dynamo.testing.CompileCounterWithBackend("aot_eager")

    def f(q, k, v, s0):
        return decay_attention(q, k, v, log_decay, initial_state=s0, return_state=state)
    compiled = torch.compile(f, fullgraph=True, backend=counter, dynamic=True)
    for N in (300, 130, 4097, 700):
        def make(seed):
            t = _normal(2, N, 2, 64, seed=seed, dtype=dtype).transpose(1, 2)
            return t if split else t.contiguous()
        d, ds, results = make(5), _normal(2, 2, 64, 64, seed=6), []
        for call in (f, compiled):
            leaves = [make(i).requires_grad_(True) for i in range(3)]
            s0 = _normal(2, 2, 64, 64, seed=7).requires_grad_(True) if state else None
            r = call(*leaves, s0)
            leaves += [s0] if state else []
            results.append([*(r if state else (r,)), *torch.autograd.grad(r, leaves, (d, ds) if state else d)])
        for a, b in zip(*results):
            assert torch.equal(a, b) and a.stride() == b.stride()
    assert counter.frame_count == 1
    x, w, b = _normal(30, 96, seed=1, dtype=dtype), _normal(96, seed=2), _normal(96, seed=3)
    for wanted in ((True, True, True), (False, True, False), (True, False, True), (False, False, False)):
        results = []
        for call in (layer_norm, torch.compile(lambda *a: layer_norm(*a), fullgraph=True, backend="aot_eager")):
            leaves = [t.clone().requires_grad_(q) for t, q in zip((x, w, b), wanted)]
            y = call(*leaves)
            results.append([y, *torch.autograd.grad(y, [t for t in leaves if t.requires_grad], x)] if any(wanted) else [y])
        assert all(torch.equal(p, q) for p, q in zip(*results))
    with torch.no_grad():
        assert torch.equal(torch.compile(lambda *a: layer_norm(*a), fullgraph=True, backend="aot_eager")(x, w, b), layer_norm(x, w, b))


def test_registered_operators(cuda_device):
    """Their schemas, fake results (sizes, strides, types) and autograd formulas against real calls."""
    ops = torch.ops.flashnystrom_b200
    log_decay, s0 = torch.tensor([-0.1, -0.01], device="cuda"), _normal(1, 2, 64, 64, seed=4)
    for split in (False, True):
        q, k, v = (_normal(1, 200, 2, 64, seed=i, dtype=torch.float32).transpose(1, 2) for i in range(3))
        if not split:
            q, k, v = (t.contiguous() for t in (q, k, v))
        for want_state, bounded in ((True, False), (False, True)):
            torch.library.opcheck(ops.decay_fwd.default, (q, k, v, log_decay, 0.125, s0, None, want_state, bounded), test_utils=("test_schema", "test_faketensor"))
        segments = ops.decay_fwd(q, k, v, log_decay, 0.125, s0, None)[2]
        for d_state, want_initial in ((None, False), (s0, True)):
            torch.library.opcheck(ops.decay_bwd.default, (v, d_state, q, k, v, log_decay, 0.125, s0, None, segments, want_initial), test_utils=("test_schema", "test_faketensor"))
    t = lambda a: a[:, :, 0].contiguous()  # noqa: E731
    torch.library.opcheck(ops.decay_step.default, (t(q), t(k), t(v), s0.clone(), log_decay, 0.125, None), test_utils=("test_schema", "test_faketensor"))
    x, w = _normal(7, 96, seed=1), _normal(96, seed=2)
    for keep in (True, False):
        torch.library.opcheck(ops.norm_fwd.default, (x, w, None, 1e-5, 3, keep), test_utils=("test_schema", "test_faketensor"))
    _, mean, rstd = ops.norm_fwd(x, w, None, 1e-5, 3)
    for want in ((True, True, True), (False, True, False)):
        torch.library.opcheck(ops.norm_bwd.default, (x, x, w, mean, rstd, 1e-5, 3, True, *want), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e-4, 0.3, 1.0])
@pytest.mark.parametrize("B,N", [(1, 700), (1, 4000), (160, 300)])
def test_growing_decays_in_fp16(cuda_device, D, size, B, N):
    """log_decay above 0 is the caller's affair, and not refused: weights above 1 leave no type's range that the result and its terms keep to.  (Growth of e^0.8 over
    4000 rows, e^3 over 300.)"""
    t = [_normal(B, 2, N, D, seed=i, mul=m).half() for i, m in enumerate((1.0, size, 1.0, 0.1))]
    _check_range(t, torch.tensor([0.01 if N == 300 else 2e-4, 1e-4], device="cuda"), scale=0.01, in_range=False)
