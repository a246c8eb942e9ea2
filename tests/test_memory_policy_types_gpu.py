"""-m gpu: utils/rlgames/memory_policy.py in half precision, cast and under autocast."""
import pytest
import torch

from omniisaacgymenvs_amd.utils.rlgames.memory_ops import decay_attention, decay_attention_step, layer_norm
from omniisaacgymenvs_amd.utils.rlgames.memory_policy import MemoryPolicy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _policy():
    torch.manual_seed(3)
    return MemoryPolicy(60, 8, width=64, heads=4, layers=1).to(DEV)


def _inputs(dtype):
    g = torch.Generator(device=DEV).manual_seed(4)
    obs = torch.randn(16, 12, 60, generator=g, device=DEV).to(dtype)
    return obs, torch.rand(16, 12, generator=g, device=DEV) < 0.1, torch.randn(1, 16, 4, 16, 16, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cast_policy_is_its_operators_with_decays_in_32_bits(dtype):
    net = _policy()
    decay = net.blocks[0].decay.clone()
    net = net.to(dtype)
    obs, resets, state = _inputs(dtype)
    b = net.blocks[0]

    def read(x):
        x = layer_norm(x, net.norm.weight, net.norm.bias)
        return torch.tanh(net.mu(x)), net.value(x).squeeze(-1)

    def heads(x):
        return b.qkv(layer_norm(x, b.norm.weight, b.norm.bias)).unflatten(-1, (3, 4, 16)).unbind(-3)

    got = net(obs, state, resets)
    x = net.encoder(obs)
    o, behind = decay_attention(*heads(x), decay, state[0], resets)
    for mine, want in zip(got, (*read(x + b.out(o.flatten(-2))), behind[None])):
        assert torch.equal(mine, want)
    assert got[0].dtype == dtype and got[2].dtype == torch.float32
    params = list(net.parameters())
    grads = torch.autograd.grad((got[0].float().sum() + got[1].float().sum(), got[2].sum()), params)
    assert all(g.dtype == dtype and g.isfinite().all() and g.any() for g in grads)
    mine, want = state.clone(), state.clone()
    with torch.no_grad():
        mu, value = net.step(obs[:, 0], mine, resets[:, 0])
        x = net.encoder(obs[:, 0])
        x = x + b.out(decay_attention_step(*heads(x), decay, want[0], resets[:, 0]).flatten(-2))
        assert torch.equal(mu, read(x)[0]) and torch.equal(value, read(x)[1]) and torch.equal(mine, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_policy_under_autocast(dtype):
    """Against the same policy in 32 bits.  Projections and memory in the narrow type: weights, inputs and results of six stages are
    rounded, four roundings a stage of half a step of the largest magnitude each."""
    net = _policy()
    obs, resets, state = _inputs(torch.float32)
    want = net(obs, state, resets)
    params = list(net.parameters())
    with torch.autocast("cuda", dtype):
        got = net(obs, state, resets)
        stepped = state.clone()
        mu, value = net.step(obs[:, 0], stepped, resets[:, 0])
    tol = 6 * 4 * torch.finfo(dtype).eps / 2
    for a, b in zip((*got, mu, value), (*want, want[0][:, 0], want[1][:, 0])):
        assert (a.float() - b).abs().max() <= tol * b.abs().max()
    assert got[2].dtype == stepped.dtype == torch.float32
    grads = torch.autograd.grad((got[0].float().sum() + got[1].float().sum(), got[2].sum()), params)
    assert all(g.dtype == torch.float32 and g.isfinite().all() and g.any() for g in grads)
