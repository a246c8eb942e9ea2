"""CPU: what the recurrent-policy operators refuse, by their Python front end and behind the C ABI, without a launch."""
import ctypes as C

import pytest
import torch

from omniisaacgymenvs_amd import _lib
from omniisaacgymenvs_amd.utils.rlgames.memory_ops import decay_attention, decay_attention_step, layer_norm


def _seq(n=2, t=5, h=4, hk=2, dk=8, dv=6, dtype=torch.float32):
    return (torch.zeros(n, t, h, dk, dtype=dtype), torch.zeros(n, t, hk, dk, dtype=dtype), torch.zeros(n, t, hk, dv, dtype=dtype),
            torch.ones(h))


def _step(n=2, h=4, hk=2, dk=8, dv=6):
    return torch.zeros(n, h, dk), torch.zeros(n, hk, dk), torch.zeros(n, hk, dv), torch.ones(h), torch.zeros(n, h, dk, dv)


@pytest.mark.parametrize("args, match", [
    ((torch.zeros(3, 4),), "no CPU fallback"),
    ((None,), "must be a tensor"),
    ((torch.zeros(3, 4, dtype=torch.float64),), "float64"),
    ((torch.zeros(3, 4, dtype=torch.int64),), "int64"),
    ((torch.zeros(()),), "last axis"),
    ((torch.zeros(3, 0),), "last axis"),
    ((torch.zeros(1, 16385),), "16384"),
    ((torch.zeros(3, 4), torch.zeros(5)), "weight has shape"),
    ((torch.zeros(3, 4), torch.zeros(4), torch.zeros(1, 4)), "bias has shape"),
    ((torch.zeros(3, 4), torch.zeros(4, dtype=torch.float16)), "expected torch.float32"),
    ((torch.zeros(3, 4, dtype=torch.float16), torch.zeros(4), torch.zeros(4, dtype=torch.float16)), "one type"),
    ((torch.zeros(3, 4), 1.0), "weight must be a tensor"),
    ((torch.zeros(3, 4), None, None, -1.0), "eps"),
    ((torch.zeros(3, 4), None, None, float("nan")), "eps"),
])
def test_layer_norm_refuses(args, match):
    with pytest.raises(_lib.OigeError, match=match):
        layer_norm(*args)


def _change(args, **kw):
    names = ("q", "k", "v", "decay", "state")
    return [kw.get(n, a) for n, a in zip(names, args)]


@pytest.mark.parametrize("change, kw, match", [
    ({}, {}, "no CPU fallback"),
    ({"q": torch.zeros(2, 5, 8)}, {}, "axes"),
    ({"k": torch.zeros(2, 5, 8)}, {}, "axes"),
    ({"q": torch.zeros(2, 5, 4, 8, dtype=torch.float64)}, {}, "float64"),
    ({"v": torch.zeros(2, 5, 2, 6, dtype=torch.float16)}, {}, "q is torch.float32"),
    ({"k": torch.zeros(2, 4, 2, 8)}, {}, "shape"),
    ({"k": torch.zeros(2, 5, 3, 8), "v": torch.zeros(2, 5, 3, 6)}, {}, "4 heads over 3"),
    ({"v": torch.zeros(2, 5, 4, 6)}, {}, "do not match"),
    ({"k": torch.zeros(2, 5, 2, 7)}, {}, "do not match"),
    ({"v": torch.zeros(2, 5, 2, 129)}, {}, "head size 129"),
    ({"v": torch.zeros(2, 5, 2, 0)}, {}, "head size 0"),
    ({"decay": torch.ones(3)}, {}, "decay must be"),
    ({"decay": torch.ones(4, dtype=torch.float64)}, {}, "decay must be"),
    ({"decay": torch.ones(4, requires_grad=True)}, {}, "constant"),
    ({"decay": 0.9}, {}, "decay must be a tensor"),
    ({}, {"state": torch.zeros(2, 4, 8, 7)}, "state must be"),
    ({}, {"state": torch.zeros(2, 4, 8, 6, dtype=torch.bfloat16)}, "state must be"),
    ({}, {"resets": torch.zeros(2, 4, dtype=torch.bool)}, "resets has shape"),
    ({}, {"resets": torch.zeros(2, 5)}, "resets is torch.float32"),
    ({}, {"lengths": torch.zeros(3, dtype=torch.int64)}, "lengths must be"),
    ({}, {"lengths": torch.zeros(2)}, "lengths must be"),
    ({}, {"scale": float("inf")}, "scale"),
])
def test_decay_attention_refuses(change, kw, match):
    with pytest.raises(_lib.OigeError, match=match):
        decay_attention(*_change(_seq(), **change), **kw)


@pytest.mark.parametrize("change, kw, match", [
    ({}, {}, "no CPU fallback"),
    ({"q": torch.zeros(2, 1, 4, 8)}, {}, "axes"),
    ({"state": None}, {}, "state must be a tensor"),
    ({"state": torch.zeros(2, 4, 6, 8).transpose(2, 3)}, {}, "contiguous"),
    ({"state": torch.zeros(2, 2, 8, 6)}, {}, "state must be"),
    ({"k": torch.zeros(3, 2, 8)}, {}, "shape"),
    ({"q": torch.zeros(2, 4, 8, requires_grad=True)}, {}, "no gradient"),
    ({}, {"resets": torch.zeros(3, dtype=torch.int64)}, "resets has shape"),
    ({}, {"resets": torch.zeros(2, dtype=torch.int32)}, "resets is torch.int32"),
])
def test_decay_attention_step_refuses(change, kw, match):
    with pytest.raises(_lib.OigeError, match=match):
        decay_attention_step(*_change(_step(), **change), **kw)


def _fail(rc, match):
    assert rc < 0 and match in _lib.load().oige_last_error().decode()


def test_abi_layer_norm_refuses():
    lib = _lib.load()
    io = _lib.LayerNormIo()
    _fail(lib.oige_layer_norm_forward(C.byref(io), None), "dtype")
    io.dtype, io.weight_dtype, io.rows, io.width = _lib.BF16, _lib.F16, 4, 8
    _fail(lib.oige_layer_norm_forward(C.byref(io), None), "activations' type")
    io.weight_dtype = _lib.F32
    _fail(lib.oige_layer_norm_forward(C.byref(io), None), "null x")
    io.x = 16
    _fail(lib.oige_layer_norm_forward(C.byref(io), None), "null y")
    io.y, io.mean = 16, 16
    _fail(lib.oige_layer_norm_forward(C.byref(io), None), "together")
    for width in (0, 16385, -1):
        io.width = width
        _fail(lib.oige_layer_norm_forward(C.byref(io), None), "width")
        _fail(lib.oige_layer_norm_workspace_floats(4, width), "width")
    io.width = 8
    _fail(lib.oige_layer_norm_backward(C.byref(io), None), "null dy")
    io.dy = io.rstd = 16
    _fail(lib.oige_layer_norm_backward(C.byref(io), None), "no gradient")
    io.dweight = 16
    _fail(lib.oige_layer_norm_backward(C.byref(io), None), "workspace")
    io.workspace, io.workspace_floats = 16, lib.oige_layer_norm_workspace_floats(4, 8) - 1
    _fail(lib.oige_layer_norm_backward(C.byref(io), None), "too small")


def test_abi_decay_attention_refuses():
    lib = _lib.load()
    io = _lib.DecayAttentionIo()
    calls = (lib.oige_decay_attention_forward, lib.oige_decay_attention_backward)

    def both(match):
        for fn in calls:
            _fail(fn(C.byref(io), None), match)

    both("dtype")
    io.dtype, io.num_envs, io.num_tokens = _lib.F32, -1, 4
    both("sequences")
    io.num_envs, io.heads, io.kv_heads = 2, 4, 3
    both("key / value heads")
    io.kv_heads, io.key_dim, io.value_dim = 2, 8, 129
    both("head sizes")
    io.value_dim = 8
    both("null decay")
    io.decay, io.resets, io.resets_bytes = 16, 16, 4
    both("resets")
    io.resets_bytes, io.lengths, io.lengths_bytes = 8, 16, 1
    both("lengths")
    io.lengths_bytes = 4
    both("null q")
    for name in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(io, name, 16)
    io.num_tokens = 4096  # few sequences, many tokens: cut over time, needs scratch
    for fn, back in zip(calls, (0, 1)):
        need = lib.oige_decay_attention_workspace_floats(C.byref(io), back)
        assert need > 0
        io.workspace, io.workspace_floats = 16, need - 1
        _fail(fn(C.byref(io), None), "workspace")
        io.workspace, io.workspace_floats = 20, need
        _fail(fn(C.byref(io), None), "16-byte aligned")
    io.num_tokens = 0
    _fail(calls[0](C.byref(io), None), "no tokens")
    _fail(calls[1](C.byref(io), None), "no tokens")


def test_abi_decay_attention_refuses_states_in_place():
    lib = _lib.load()
    io = _lib.DecayAttentionIo()
    io.dtype, io.num_envs, io.num_tokens, io.heads, io.kv_heads, io.key_dim, io.value_dim = _lib.F32, 2, 4, 1, 1, 8, 8
    for name in ("q", "k", "v", "o", "decay", "d_o", "dq", "dk", "dv"):
        setattr(io, name, 16)
    io.state_in = io.state_out = 32
    _fail(lib.oige_decay_attention_forward(C.byref(io), None), "state_out must not be state_in")
    io.d_state_in = 32
    _fail(lib.oige_decay_attention_backward(C.byref(io), None), "d_state_in must be neither")
    io.state_in, io.d_state_out = 48, 32
    _fail(lib.oige_decay_attention_backward(C.byref(io), None), "d_state_in must be neither")


def test_abi_decay_attention_step_refuses():
    lib = _lib.load()
    io = _lib.DecayAttentionStepIo()
    fn = lib.oige_decay_attention_step
    _fail(fn(C.byref(io), None), "dtype")
    io.dtype, io.num_envs = _lib.F16, -1
    _fail(fn(C.byref(io), None), "sequences")
    io.num_envs, io.heads, io.kv_heads = 2, 4, 0
    _fail(fn(C.byref(io), None), "key / value heads")
    io.kv_heads, io.key_dim, io.value_dim = 4, 0, 8
    _fail(fn(C.byref(io), None), "head sizes")
    io.key_dim, io.resets, io.resets_bytes = 8, 16, 2
    _fail(fn(C.byref(io), None), "resets")
    io.resets_bytes = 1
    _fail(fn(C.byref(io), None), "null decay")
    io.decay = 16
    _fail(fn(C.byref(io), None), "null q")


def test_packed_argument_blocks_match_the_structures():
    from omniisaacgymenvs_amd.utils.rlgames import memory_ops as m

    for struct, pack in ((_lib.LayerNormIo, m._pack_norm), (_lib.DecayAttentionIo, m._pack_attention), (_lib.DecayAttentionStepIo, m._pack_step)):
        count = sum(kind._length_ if issubclass(kind, C.Array) else 1 for _, kind in struct._fields_)
        block = pack(*range(1, count + 1))
        assert len(block) == C.sizeof(struct)
        got = []
        for name, _ in struct._fields_:
            v = getattr(struct.from_buffer_copy(block), name)
            got += list(v) if isinstance(v, C.Array) else [v]
        assert [int(x) for x in got] == list(range(1, count + 1))


def test_policy_refuses():
    from omniisaacgymenvs_amd.scripts import random_policy
    from omniisaacgymenvs_amd.utils.rlgames.memory_policy import MemoryPolicy

    with pytest.raises(ValueError, match="not a multiple"):
        MemoryPolicy(10, 2, width=30, heads=4)
    with pytest.raises(ValueError, match="uniform or memory"):
        random_policy.run({}, frames=1, policy="lstm")
    with pytest.raises(SystemExit):
        random_policy.main(["task=Ant", "--policy", "lstm"])
    policy = MemoryPolicy(10, 2, width=32, heads=4, layers=2)
    assert policy.initial_state(5).shape == (2, 5, 4, 8, 8)
    with pytest.raises(_lib.OigeError, match="no CPU fallback"):
        policy.step(torch.zeros(5, 10), policy.initial_state(5))
    with pytest.raises(_lib.OigeError, match="no CPU fallback"):
        policy(torch.zeros(5, 3, 10))
