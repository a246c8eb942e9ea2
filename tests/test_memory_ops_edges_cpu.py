"""CPU: calls of the recurrent-policy operators that tests/test_memory_ops_cpu.py does not make, without a launch."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from omniisaacgymenvs_amd import _lib
from omniisaacgymenvs_amd.utils.rlgames.memory_ops import decay_attention, decay_attention_step, layer_norm


def _calls():
    """name, function, its tensor arguments."""
    q, k, v, decay, state = torch.ones(2, 5, 4, 8), torch.ones(2, 5, 2, 8), torch.ones(2, 5, 2, 6), torch.ones(4), torch.ones(2, 4, 8, 6)
    return [("layer_norm", layer_norm, [torch.ones(3, 4), torch.ones(4), torch.zeros(4)]),
            ("decay_attention", decay_attention, [q, k, v, decay, state]),
            ("decay_attention_step", decay_attention_step, [q[:, 0], k[:, 0], v[:, 0], decay, state])]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(which, requires_grad):
    name, fn, args = _calls()[which]
    for i in range(len(args)):
        with forward_ad.dual_level():
            dual = list(args)
            dual[i] = forward_ad.make_dual(args[i].clone().requires_grad_(requires_grad), torch.ones_like(args[i]))
            with pytest.raises(_lib.OigeError, match=f"{name}: .* has a tangent"):
                fn(*dual)
            with pytest.raises(_lib.OigeError, match="no CPU fallback"):  # none of the arguments has one: refused for another reason
                fn(*args)
    with pytest.raises(_lib.OigeError, match="has a tangent"):
        torch.func.jvp(lambda x: fn(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))


@pytest.mark.parametrize("which", [0, 1, 2])
def test_traces_are_refused(which):
    name, fn, args = _calls()[which]
    with pytest.raises(_lib.OigeError, match=f"{name}: cannot be traced"):
        torch.jit.trace(fn, tuple(args), check_trace=False)
    with pytest.raises(_lib.OigeError, match=f"{name}: cannot be traced"):
        make_fx(lambda *a: fn(*a))(*args)


def test_abi_layer_norm_backward_without_rows():
    """An empty dx has no address: with no parameter's gradient asked for there is nothing to do."""
    lib = _lib.load()
    io = _lib.LayerNormIo()
    io.dtype = io.weight_dtype = _lib.F32
    io.rows, io.width = 0, 8
    assert lib.oige_layer_norm_backward(C.byref(io), None) == 0
    io.rows = 1
    assert lib.oige_layer_norm_backward(C.byref(io), None) < 0


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16().float(), lambda m: m.to("meta", torch.float16)])
def test_policy_keeps_decays_and_states_in_32_bits(cast):
    from omniisaacgymenvs_amd.utils.rlgames.memory_policy import MemoryPolicy

    want = MemoryPolicy(10, 2, width=32, heads=4, layers=2).blocks[1].decay.clone()
    policy = cast(MemoryPolicy(10, 2, width=32, heads=4, layers=2))
    for block in policy.blocks:
        assert block.decay.dtype == torch.float32 and block.decay.device == policy.mu.weight.device
        assert block.decay.is_meta or torch.equal(block.decay, want)
    torch.set_default_dtype(torch.float64)
    try:
        state = policy.initial_state(3)
    finally:
        torch.set_default_dtype(torch.float32)
    assert state.dtype == torch.float32 and state.device == policy.mu.weight.device and state.shape == (2, 3, 4, 8, 8)


@pytest.mark.parametrize("kw, match", [({"width": 1024, "heads": 4}, "1 to 128 wide"), ({"width": 129, "heads": 1}, "1 to 128 wide"),
                                       ({"width": 128 * 129, "heads": 129}, "all of them 16384"), ({"width": 32, "heads": 0}, "not a multiple"),
                                       ({"width": 0, "heads": 4}, "not a multiple"), ({"layers": 0}, "0 layers")])
def test_policy_refuses_what_no_call_would_take(kw, match):
    from omniisaacgymenvs_amd.utils.rlgames.memory_policy import MemoryPolicy

    with pytest.raises(ValueError, match=match):
        MemoryPolicy(10, 2, **kw)
    MemoryPolicy(10, 2, width=128, heads=1)
