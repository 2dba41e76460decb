"""Argument checks of the causal attention with a decay and of the layer norm that come before any device is touched, and the plain
restatements that the GPU tests compare with, against torch's own differentiation."""
import ctypes as C

import pytest
import torch

from flashnystrom_b200 import DecayAttention, LayerNorm, _lib, decay_attention, decay_attention_step, default_log_decay, layer_norm
from oracle import operators_oracle as O


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _shape(B=1, H=2, N=100, D=64, dtype=_lib.FNB_F16, scale=0.125, flags=0):
    return _lib.DecayShape(B, H, N, D, dtype, scale, flags)


@pytest.mark.parametrize("kw,message", [
    (dict(B=0), "must be positive"), (dict(H=0), "must be positive"), (dict(N=0), "must be positive"), (dict(D=48), "head_dim must be"), (dict(D=256), "head_dim must be"),
    (dict(dtype=7), "Supported dtypes"), (dict(scale=0.0), "scale must be"), (dict(scale=float("inf")), "scale must be"), (dict(scale=1e-20), "scale must be"), (dict(scale=-1e20), "scale must be"), (dict(flags=4), "unknown flags"),
    (dict(B=300, H=300), "exceeds 65535"), (dict(N=2 ** 31), "exceeds 2"), (dict(B=2 ** 40, H=2 ** 40), "exceeds 65535")])
def test_decay_shapes(lib, kw, message):
    s = _shape(**kw)
    assert lib.fnb_check_decay_shape(C.byref(s)) == -1 and message in _lib.last_error()
    assert lib.fnb_decay_workspace_bytes(C.byref(s)) == 0 and lib.fnb_decay_segment_floats(C.byref(s)) == 0


def test_decay_sizes(lib):
    small, large = _shape(N=1), _shape(H=16, N=65536)
    assert lib.fnb_decay_segment_floats(C.byref(small)) == 0          # one run of rows: nothing between
    n = lib.fnb_decay_segment_floats(C.byref(large))
    assert n > 0 and n % (16 * 64 * 64) == 0 and n <= 65536 // 128 * 16 * 64 * 64
    assert lib.fnb_decay_workspace_bytes(C.byref(large)) % 256 == 0
    assert lib.fnb_check_decay_shape(None) == -1


def test_decay_pointers(lib):
    assert lib.fnb_decay_forward(None) == -1 and lib.fnb_decay_backward(None) == -1 and lib.fnb_decay_step(None) == -1
    a = _lib.DecayFwdArgs()
    a.shape = _shape()
    assert lib.fnb_decay_forward(C.byref(a)) == -1 and "q must not be NULL" in _lib.last_error()
    rows = _lib.Rows(64, 0, 0, 64)
    a.q = a.k = a.v = a.out = rows
    a.out = _lib.Rows(65, 0, 0, 64)
    assert lib.fnb_decay_forward(C.byref(a)) == -1 and "out is not aligned" in _lib.last_error()
    a.out = _lib.Rows(64, 0, -64, 64)
    assert lib.fnb_decay_forward(C.byref(a)) == -1 and "negative stride" in _lib.last_error()
    s = _lib.DecayStepArgs(3, 2, 2, 64, _lib.FNB_F32, 1.0, rows, rows, rows, rows, 64, 64, None, 0, None)
    assert lib.fnb_decay_step(C.byref(s)) == -1 and "2 states for 3 rows" in _lib.last_error()
    s = _lib.DecayStepArgs(3, 2, 3, 64, _lib.FNB_F32, 1.0, rows, rows, rows, rows, 64, 72, None, 0, None)
    assert lib.fnb_decay_step(C.byref(s)) == -1 and "16-byte aligned" in _lib.last_error()
    s = _lib.DecayStepArgs(3, 2, 3, 64, _lib.FNB_F32, 1.0, rows, rows, rows, rows, None, 64, None, 0, None)
    assert lib.fnb_decay_step(C.byref(s)) == -1 and "must not be NULL" in _lib.last_error()
    s = _lib.DecayStepArgs(65535, 65535, 65535, 64, _lib.FNB_F32, 1.0, rows, rows, rows, rows, 64, 64, 64, 0, None)
    assert lib.fnb_decay_step(C.byref(s)) == -1 and "exceeds 2^31" in _lib.last_error()
    s = _lib.DecayStepArgs(2 ** 33, 2, 3, 64, _lib.FNB_F32, 1.0, rows, rows, rows, rows, 64, 64, 64, 0, None)
    assert lib.fnb_decay_step(C.byref(s)) == -1 and "exceeds 65535" in _lib.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(rows=0), "must be positive"), (dict(cols=0), "must be positive"), (dict(groups=3), "multiple of groups"), (dict(groups=0), "multiple of groups"), (dict(cols=16400), "at most 16384"),
    (dict(dtype=9), "Supported dtypes"), (dict(param_dtype=2), "weight and bias must be"), (dict(eps=-1.0), "eps must be"), (dict(eps=float("nan")), "eps must be")])
def test_norm_shapes(lib, kw, message):
    d = dict(rows=10, cols=64, groups=1, dtype=_lib.FNB_F16, param_dtype=_lib.FNB_F32, eps=1e-5)
    d.update(kw)
    s = _lib.NormShape(*(d[n] for n in ("rows", "cols", "groups", "dtype", "param_dtype", "eps")))
    assert lib.fnb_check_norm_shape(C.byref(s)) == -1 and message in _lib.last_error()
    assert lib.fnb_norm_workspace_bytes(C.byref(s)) == 0


def test_norm_pointers(lib):
    s = _lib.NormShape(10, 64, 1, _lib.FNB_F16, _lib.FNB_F32, 1e-5)
    assert lib.fnb_norm_workspace_bytes(C.byref(s)) >= 2 * 64 * 4
    assert lib.fnb_norm_forward(None) == -1 and lib.fnb_norm_backward(None) == -1
    a = _lib.NormFwdArgs(s, None, 64, 64, 64, None, None, None, None, 0, None)
    assert lib.fnb_norm_forward(C.byref(a)) == -1 and "must not be NULL" in _lib.last_error()
    a = _lib.NormFwdArgs(s, 65, 64, 64, 64, None, None, None, None, 0, None)
    assert lib.fnb_norm_forward(C.byref(a)) == -1 and "not aligned" in _lib.last_error()
    b = _lib.NormBwdArgs(s, 64, 64, 64, 64, 64, 64, None, None, 64, 64, 64, None, 0, 0, None)
    assert lib.fnb_norm_backward(C.byref(b)) == -1 and "must not be NULL" in _lib.last_error()


def test_python_refuses_cpu_tensors():
    q = torch.zeros(1, 1, 8, 16)
    g = torch.zeros(1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        decay_attention(q, q, q, g)
    with pytest.raises(RuntimeError, match="no CPU path"):
        decay_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], torch.zeros(1, 1, 16, 16), g)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(q)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        layer_norm(3)


def test_modules_on_the_host():
    m = DecayAttention(256, heads=4)
    assert sorted(n for n, _ in m.named_parameters()) == ["k_proj.weight", "norm_bias", "norm_weight", "out_proj.weight", "q_proj.weight", "v_proj.weight"]
    assert "log_decay" in m.state_dict() and bool((m.log_decay < 0).all()) and m.new_state(3).shape == (3, 4, 64, 64)
    assert m.half().log_decay.dtype == torch.float32 and torch.equal(m.log_decay, default_log_decay(4))
    assert m.double().log_decay.dtype == torch.float32
    assert default_log_decay(1).shape == (1,)
    for bad in (dict(dim=250, heads=4), dict(dim=192, heads=4), dict(dim=256, heads=4, log_decay=[0.0, 0.1, -1.0, -1.0]), dict(dim=256, heads=4, log_decay=[-1.0])):
        with pytest.raises(ValueError):
            DecayAttention(**bad)
    with pytest.raises(ValueError):
        LayerNorm(64, num_groups=3)
    assert LayerNorm(64, bias=False).bias is None and LayerNorm(64, elementwise_affine=False).weight is None


def test_oracle_is_the_recurrence():
    """Every pair of rows at once is the recurrence token by token, at lengths of its own and from a state."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 3, 20, 16, generator=g, dtype=torch.float64) for _ in range(3))
    s0 = torch.randn(2, 3, 16, 16, generator=g, dtype=torch.float64)
    decay = torch.tensor([0.0, -0.3, -float("inf")])
    lens = [20, 7]
    out, state = O.decay_attention(q, k, v, decay, None, s0, lens)
    for b in range(2):
        s = s0[b:b + 1].clone()
        for t in range(lens[b]):
            o, s = O.decay_step(q[b:b + 1, :, t], k[b:b + 1, :, t], v[b:b + 1, :, t], s, decay)
            assert torch.allclose(o[0], out[b, :, t])
        assert torch.allclose(s[0], state[b]) and not out[b, :, lens[b]:].any()


def test_oracle_of_the_norm():
    x = torch.randn(5, 48, dtype=torch.float64)
    w, b = torch.randn(48, dtype=torch.float64), torch.randn(48, dtype=torch.float64)
    assert torch.allclose(O.layer_norm(x, w, b), torch.nn.functional.layer_norm(x, (48,), w, b))
    assert torch.allclose(O.layer_norm(x, w, b, num_groups=3), torch.nn.functional.group_norm(x, 3, w, b))
