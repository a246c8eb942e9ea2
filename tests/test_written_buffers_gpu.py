"""-m gpu: a backward pass that saved a task's buffer raises once an env step has written it (the kernels write through raw pointers,
which torch's version counters do not see by themselves)."""
import pytest
import torch

from helpers import make_task
from omniisaacgymenvs_amd.utils.rlgames.memory_ops import decay_attention, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WRITTEN = "modified by an inplace operation"


def _graphs(task, env_obs=None):
    """One result per saved buffer, with the leaf it is differentiated in and the gradient of a copy."""
    n = task.num_envs
    obs = task.obs_buf if env_obs is None else env_obs
    w = torch.ones(obs.shape[1], device=DEV, requires_grad=True)
    q = torch.randn(n, 1, 2, 8, device=DEV, requires_grad=True)
    state, decay = torch.randn(n, 2, 8, 8, device=DEV), torch.full((2,), 0.5, device=DEV)
    return {"obs": (lambda x: layer_norm(x, w).square().sum(), obs, w),
            "reset": (lambda x: decay_attention(q, q, q, decay, state, resets=x[:, None])[0].square().sum(), task.reset_buf, q)}


def _check(task, step, env_obs=None):
    graphs = _graphs(task, env_obs)
    for name, (f, x, leaf) in graphs.items():  # before the step both are differentiable, and twice
        want, = torch.autograd.grad(f(x.clone()), leaf)
        assert torch.equal(torch.autograd.grad(f(x), leaf)[0], want), name
    held = {name: (f(x), f(x.clone()), leaf) for name, (f, x, leaf) in graphs.items()}
    step()
    for name, (live, copied, leaf) in held.items():
        with pytest.raises(RuntimeError, match=WRITTEN):
            torch.autograd.grad(live, leaf)
        torch.autograd.grad(copied, leaf)


@pytest.mark.parametrize("name", ["Ant", "Cartpole", "ShadowHand", "AnymalTerrain", "Anymal", "Quadcopter", "BallBalance", "Ingenuity", "Crazyflie",
                                  "FrankaCabinet", "TomoDJnewhandCabinet"])
def test_a_step_invalidates_what_was_saved_of_its_buffers(name):
    env, task = make_task(name, 64)
    env.reset()
    actions = torch.zeros(64, task.num_actions, device=DEV)
    _check(task, lambda: env.step(actions))
    version = task.reset_buf._version
    task.pre_physics_step(actions)  # flags are cleared here (AnymalTerrain: in the post kernel)
    assert name == "AnymalTerrain" or task.reset_buf._version > version
    _check(task, task.post_physics_step)


@pytest.mark.parametrize("name", ["Ant", "AnymalTerrain", "ShadowHand"])
def test_replayed_steps_too(name):
    env, task = make_task(name, 64)
    env.reset()
    actions = torch.zeros(64, task.num_actions, device=DEV)
    task.set_reset_scatter("device")
    env.capture_step(actions)
    env.replay_step()
    out = env.replay_step()
    _check(task, env.replay_step, env_obs=out[0]["obs"])


def test_the_counts_of_the_flags_stay_valid_behind_a_step():
    """The next pre_physics_step still skips its recount."""
    env, task = make_task("Ant", 64)
    env.reset()
    env.step(torch.zeros(64, task.num_actions, device=DEV))
    assert task._counts_valid(task.reset_buf)
    task.reset_buf[3] = 1
    assert not task._counts_valid(task.reset_buf)


def test_noise_invalidates_observations_and_their_clamped_copy():
    from omniisaacgymenvs_amd.utils.domain_randomization import noise_hip

    n, w = 64, 12
    obs, out = torch.randn(n, w, device=DEV), torch.empty(n, w, device=DEV)
    before = obs._version, out._version
    term = {"operation": "additive", "distribution": "gaussian", "distribution_parameters": [0.0, 0.1], "frequency_interval": 1}
    noise_hip.apply(obs, torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV),
                    torch.zeros(n, w, device=DEV), {"on_interval": term}, noise_hip.NoiseState(n, DEV), 1, 0, 0, clamped_out=out, clip=5.0)
    assert obs._version > before[0] and out._version > before[1]
