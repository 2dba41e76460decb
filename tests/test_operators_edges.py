"""Sizes and refusals of the attention with a decay and of the layer norm that no device is needed for."""
import ctypes as C
import random

import pytest
import torch

from flashnystrom_b200 import DecayAttention, _lib, _ops


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_bound_of_the_states_at_the_cuts(lib):
    """What a traced call sets aside for the states at the cuts is enough for every length: the split never has more segments than the bound allows."""
    r = random.Random(1)
    for _ in range(3000):
        B, H, N, D = r.randint(1, 40), r.randint(1, 40), int(2 ** r.uniform(0, 20)), r.choice([16, 32, 64, 128])
        for code, dtype in ((_lib.FNB_F32, torch.float32), (_lib.FNB_F16, torch.float16), (_lib.FNB_BF16, torch.bfloat16)):
            s = _lib.DecayShape(B, H, N, D, code, 0.125, 0)
            # (the SM count without a device is that of a B200)
            assert lib.fnb_decay_segment_floats(C.byref(s)) <= _ops._segment_bound(B, H, N, D, dtype, 148)


@pytest.mark.parametrize("where", ["log_decay", "seq_lens", "initial_state", "final_state", "segment_states", "d_final_state", "d_initial_state", "slots"])
def test_words_off_their_alignment(lib, where):
    """A float or int32 array that begins between words is refused before any device is touched."""
    rows, shape = _lib.Rows(64, 0, 0, 64), _lib.DecayShape(1, 2, 100, 64, _lib.FNB_F16, 0.125, 0)
    for args, call in ((_lib.DecayFwdArgs(), lib.fnb_decay_forward), (_lib.DecayBwdArgs(), lib.fnb_decay_backward), (_lib.DecayStepArgs(), lib.fnb_decay_step)):
        names = [n for n, _ in args._fields_]
        if where not in names:
            continue
        for n in names:
            if n in ("q", "k", "v", "out", "d_out", "dq", "dk", "dv"):
                setattr(args, n, rows)
        if "shape" in names:
            args.shape = shape
        else:
            args.batch, args.heads, args.num_states, args.head_dim, args.dtype, args.scale, args.states = 1, 2, 1, 64, _lib.FNB_F16, 0.125, 64
        args.log_decay = 64
        setattr(args, where, 66)
        assert call(C.byref(args)) == -1 and "not aligned to its type" in _lib.last_error()


def test_module_without_memory():
    """Built on the meta device, given memory, then a checkpoint's values."""
    whole = DecayAttention(128, heads=2)
    with torch.device("meta"):
        m = DecayAttention(128, heads=2)
    assert m.log_decay.is_meta and m.q_proj.weight.is_meta
    m.to_empty(device="cpu").load_state_dict(whole.state_dict())
    assert torch.equal(m.log_decay, whole.log_decay) and m.log_decay.dtype == torch.float32
