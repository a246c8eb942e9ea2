"""-m gpu: the recurrent-policy operators (utils/rlgames/memory_ops.py) against their formulas in 64 bits (tests/memory_cases.py).
Every tolerance is a running error bound of a 32-bit evaluation plus half a step of the stored type."""
import gc
import math

import pytest
import torch

from memory_cases import assert_within, attention, attention_bounds, norm, rounding
from omniisaacgymenvs_amd import _lib
from omniisaacgymenvs_amd.utils.rlgames.memory_ops import decay_attention, decay_attention_step, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
inf, nan = math.inf, math.nan


def _cpu(x):
    return None if x is None else x.detach().cpu()


# ------------------------------------------------------------------------------------------------ layer norm
def _check_norm(x, weight, bias, dy, eps=1e-5):
    rows = (-1, x.shape[-1])
    leaves = [p for p in (x, weight, bias) if p is not None]
    for p in leaves:
        p.requires_grad_(True)
    y = layer_norm(x, weight, bias, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, weight, bias, eps), y)  # kept statistics change nothing
    want, bound = norm(_cpu(x).reshape(rows), _cpu(weight), _cpu(bias), eps, _cpu(dy).reshape(rows))
    got = {"y": y.detach().reshape(rows), "dx": grads[0].reshape(rows)}
    rest = list(grads[1:])
    if weight is not None:
        got["dw"] = rest.pop(0)
    if bias is not None:
        got["db"] = rest.pop(0)
    for name, g in got.items():
        assert_within(g, want[name], bound[name] + rounding(want[name], g.dtype), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, width", [
    (1, 1), (3, 2), (1, 256), (5, 7), (200, 60), (777, 64), (300, 87), (129, 187), (1025, 211), (64, 512), (33, 513), (70, 1000), (40, 1024),
    (9, 1025), (21, 2048), (6, 2056), (5, 4096), (3, 4100), (2, 8191), (3, 16384), (2, 16383), (5000, 8), (2500, 33)])
def test_layer_norm_widths(rows, width, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows * 31 + width)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = (r(rows, width) * (0.5 + torch.rand(rows, 1, generator=g, device=DEV)) + r(rows, 1)).to(dtype)
    _check_norm(x, (1 + 0.3 * r(width)).to(dtype), (0.3 * r(width)).to(dtype), r(rows, width).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["both", "weight", "bias", "none"])
def test_layer_norm_parameters_in_32_bits_or_absent(dtype, which):
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    w = 1 + r(96) if which in ("both", "weight") else None
    b = r(96) if which in ("both", "bias") else None
    _check_norm(r(50, 96).to(dtype), w, b, r(50, 96).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["columns", "odd start", "time first", "expanded rows", "strided last", "vector"])
def test_layer_norm_layouts(dtype, layout):
    g = torch.Generator(device=DEV).manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    x = {"columns": lambda: r(40, 160)[:, 32:96], "odd start": lambda: r(40, 161)[:, 1:65], "time first": lambda: r(6, 10, 64).transpose(0, 1),
         "expanded rows": lambda: r(1, 64).expand(9, 64), "strided last": lambda: r(9, 128)[:, ::2], "vector": lambda: r(64)}[layout]()
    dy = r(*x.shape) if layout != "time first" else r(1, 1, 64).expand(10, 6, 64)
    _check_norm(x.detach(), r(128)[::2], r(64), dy)


def test_layer_norm_hard_rows():
    """Constant rows, rows far from zero, tiny and huge ones; a row that is not finite keeps that to itself."""
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(8, 200, generator=g, device=DEV)
    x[0] = 3.0
    x[1] = 0.0
    x[2] += 1000.0
    x[3] *= 1e-6
    x[4] *= 1e8
    _check_norm(x, torch.ones(200, device=DEV), torch.zeros(200, device=DEV), torch.randn(8, 200, generator=g, device=DEV))
    clean = layer_norm(x.detach())
    for width in (200, 8):  # one row per wave, rows that share a wave
        x = torch.randn(64, width, generator=g, device=DEV)
        clean = layer_norm(x)
        bad = x.clone()
        bad[5, 3], bad[9, 0] = inf, nan
        y = layer_norm(bad)
        assert y[5].isnan().any() and y[9].isnan().all()
        keep = [i for i in range(64) if i not in (5, 9)]
        assert torch.equal(y[keep], clean[keep])


def test_layer_norm_no_rows():
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    w, b = torch.ones(32, device=DEV, requires_grad=True), torch.zeros(32, device=DEV, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 32, device=DEV))
    assert y.shape == dx.shape == (0, 32) and not dw.any() and not db.any()


def test_layer_norm_offsets_beyond_32_bits():
    rows, width = (1 << 31) // 512 + 77, 512
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    x[:1000].normal_()
    x[-1000:].normal_()
    x[1000:-1000] = 1
    y = layer_norm(x)
    assert torch.equal(y[-1000:], layer_norm(x[-1000:].clone())) and torch.equal(y[:1000], layer_norm(x[:1000].clone()))


@pytest.mark.parametrize("rows", [4, 3000])
def test_layer_norm_gradient_against_differences(rows):
    """Central differences of the 64-bit formula along random directions; the kernel's gradients are 32-bit."""
    g = torch.Generator(device=DEV).manual_seed(8)
    x, dy = torch.randn(rows, 40, generator=g, device=DEV), torch.randn(rows, 40, generator=g, device=DEV)
    w, b = torch.randn(40, generator=g, device=DEV), torch.randn(40, generator=g, device=DEV)
    leaves = [p.requires_grad_(True) for p in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    f = lambda *p: (norm(p[0], p[1], p[2], 1e-5)[0]["y"] * _cpu(dy).double()).sum()
    base = [_cpu(p).double() for p in leaves]
    for i, gr in enumerate(grads):
        d = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        h = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        slope = float((f(*up) - f(*down)) / (2 * h))
        mine = float((gr.double().cpu() * d).sum())
        mass = float((gr.double().cpu() * d).abs().sum())
        # differences: h^2 of curvature; the gradients' own 32-bit sums: rows + width roundings of each term at most
        assert abs(slope - mine) <= (rows + 60) * 2.0 ** -24 * mass * 4 + 1e-6 * mass, (i, slope, mine)


# ------------------------------------------------------------------------------------------------ decay attention
def _attention_inputs(n, t, h, hk, dk, dv, dtype, seed, state=True, resets=0.0, ragged=False, time_first=False, decay=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    tok = (lambda heads, d: r(t, n, heads, d).to(dtype).transpose(0, 1)) if time_first else (lambda heads, d: r(n, t, heads, d).to(dtype))
    kw = {"q": tok(h, dk), "k": tok(hk, dk), "v": tok(hk, dv)}
    kw["decay"] = 1 - 2.0 ** -(1 + 6 * torch.arange(h, device=DEV) / max(h - 1, 1)) if decay is None else torch.tensor(decay, device=DEV)
    kw["state"] = r(n, h, dk, dv) if state else None
    kw["resets"] = torch.rand(n, t, generator=g, device=DEV) < resets if resets else None
    kw["lengths"] = torch.randint(0, t + 1, (n,), generator=g, device=DEV) if ragged else None
    return kw, tok(h, dv), r(n, h, dk, dv)


def _check_attention(kw, d_o, d_state, forward_only=False):
    dtype = kw["q"].dtype
    leaves = [kw[x] for x in ("q", "k", "v", "state") if kw[x] is not None]
    if not forward_only:
        for x in leaves:
            x.requires_grad_(True)
    o, state = decay_attention(**kw)
    assert o.dtype == dtype and state.dtype == torch.float32
    got = {"o": o.detach(), "state": state.detach()}
    cpu = {key: _cpu(x) for key, x in kw.items()}
    extra = {}
    if not forward_only:
        grads = torch.autograd.grad((o, state), leaves, (d_o, d_state))
        got.update(zip(("dq", "dk", "dv", "d_state_in"), grads))
        extra = {"d_o": _cpu(d_o), "d_state": _cpu(d_state)}
    want = attention(**cpu, **extra)
    bound = attention_bounds(want, **cpu, **extra, dtype=dtype)
    for name, x in got.items():
        assert x.shape == want[name].shape, name
        assert_within(x, want[name], bound[name], name)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, t, h, hk, dk, dv", [
    (1, 1, 1, 1, 1, 1), (3, 1, 2, 2, 16, 16), (2, 2, 1, 1, 64, 64), (2, 15, 3, 1, 8, 24), (2, 16, 4, 4, 64, 64), (2, 17, 2, 2, 32, 48),
    (1, 33, 6, 2, 40, 72), (3, 48, 2, 2, 128, 128), (1, 70, 2, 1, 100, 36), (2, 100, 1, 1, 17, 33), (1, 130, 2, 2, 64, 128),
    (2, 300, 2, 1, 128, 16), (1, 1000, 1, 1, 16, 20), (300, 20, 4, 4, 16, 32), (1, 64, 2, 2, 127, 113), (2, 40, 5, 5, 24, 64),
    (1, 144, 1, 1, 3, 128)])
def test_decay_attention_shapes(n, t, h, hk, dk, dv, dtype):
    kw, d_o, d_state = _attention_inputs(n, t, h, hk, dk, dv, dtype, seed=t * 7 + dk)
    _check_attention(kw, d_o, d_state)


@pytest.mark.parametrize("resets, ragged, state, time_first", [
    (0.1, False, True, True), (0.02, True, False, False), (0.0, True, True, True), (0.9, True, True, False), (1.0, False, True, False)])
@pytest.mark.parametrize("t", [16, 61, 400])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_attention_episodes_and_lengths(t, resets, ragged, state, time_first, dtype):
    kw, d_o, d_state = _attention_inputs(5, t, 2, 1, 32, 24, dtype, 3 * t, state, resets, ragged, time_first)
    got = _check_attention(kw, d_o, d_state)
    if time_first:  # results lie in memory as the rollout does
        assert got["o"].transpose(0, 1).is_contiguous() and got["dk"].transpose(0, 1).is_contiguous()


@pytest.mark.parametrize("flags", [torch.bool, torch.uint8, torch.int64])
@pytest.mark.parametrize("lengths", [torch.int32, torch.int64])
def test_decay_attention_flag_types(flags, lengths):
    kw, d_o, d_state = _attention_inputs(4, 50, 2, 2, 16, 16, torch.float32, 11, resets=0.1, ragged=True)
    a = decay_attention(**kw)
    kw["resets"] = kw["resets"].to(flags) if flags is torch.bool else kw["resets"].to(flags) * 3  # any non-zero value is a flag
    kw["lengths"] = kw["lengths"].to(lengths)
    b = decay_attention(**kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decay_attention_lengths_are_clamped_and_empty_sequences_pass_the_state_on():
    kw, d_o, d_state = _attention_inputs(4, 200, 2, 2, 16, 16, torch.float32, 12)
    kw["lengths"] = torch.tensor([-5, 0, 1000, 200], device=DEV)
    got = _check_attention(kw, d_o, d_state)
    assert torch.equal(got["state"][:2], kw["state"][:2]) and not got["o"][:2].any()
    assert torch.equal(got["d_state_in"][:2], d_state[:2]) and not got["dv"][:2].any()
    kw, _, d_state = _attention_inputs(2, 0, 2, 1, 16, 8, torch.float32, 13)
    o, state = decay_attention(**{**kw, "state": kw["state"].requires_grad_(True), "q": kw["q"].requires_grad_(True)})
    dq, ds = torch.autograd.grad(state, (kw["q"], kw["state"]), d_state, allow_unused=True)
    assert o.shape == (2, 0, 2, 8) and torch.equal(state, kw["state"]) and torch.equal(ds, d_state) and dq.shape == (2, 0, 2, 16)
    kw, _, _ = _attention_inputs(0, 5, 2, 1, 16, 8, torch.float32, 13)
    o, state = decay_attention(**kw)
    assert o.shape == (0, 5, 2, 8) and state.shape == (0, 2, 16, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, t, h, hk, dk, dv", [
    (256, 37, 4, 2, 64, 64), (512, 20, 2, 2, 32, 64), (512, 35, 2, 1, 24, 56), (1024, 18, 1, 1, 16, 30), (1024, 34, 1, 1, 40, 32),
    (1, 6300, 2, 2, 128, 120), (4, 1500, 16, 16, 32, 64)])
def test_decay_attention_wide_slices_of_many_sequences(n, t, h, hk, dk, dv, dtype):
    """Enough sequences, or tokens, for up to 64 columns of the state to a wave."""
    kw, d_o, d_state = _attention_inputs(n, t, h, hk, dk, dv, dtype, 21, resets=0.04, ragged=n > 1)
    _check_attention(kw, d_o, d_state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, t, h, hk, dk, dv", [(5, 7, 6, 3, 20, 12), (9, 1, 10, 5, 8, 128), (2, 50, 14, 2, 7, 9), (3, 70, 4, 1, 4, 6)])
def test_decay_attention_shared_heads(n, t, h, hk, dk, dv, dtype):
    """Sums over query heads whose rows end inside a workgroup's."""
    kw, d_o, d_state = _attention_inputs(n, t, h, hk, dk, dv, dtype, 22, resets=0.1)
    _check_attention(kw, d_o, d_state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, t, h, hk, dk, dv", [
    (1024, 34, 1, 1, 33, 61), (512, 19, 2, 1, 17, 47), (1, 6300, 2, 2, 101, 67), (3, 40, 2, 1, 2, 1), (3, 40, 2, 2, 1, 2), (2, 300, 1, 1, 65, 33),
    (2, 33, 1, 1, 127, 17)])
def test_decay_attention_odd_heads(n, t, h, hk, dk, dv, dtype):
    """Rows on no boundary, heads whose last columns are held twice; what lies around the results is left alone."""
    kw, d_o, d_state = _attention_inputs(n, t, h, hk, dk, dv, dtype, 23, resets=0.04, ragged=n > 1)
    _check_attention(kw, d_o, d_state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk, dv", [(19, 35), (100, 101)])
def test_decay_attention_odd_heads_with_values_that_are_not_finite(dk, dv, dtype):
    kw, _, _ = _attention_inputs(2, 70, 2, 2, dk, dv, dtype, 24)
    kw["resets"] = torch.zeros(2, 70, dtype=torch.bool, device=DEV)
    kw["resets"][0, 50] = True
    for name, column in (("q", 0), ("q", dk - 1), ("k", dk - 1), ("v", dv - 1), ("v", dv - 2)):
        bad = dict(kw)
        bad[name] = kw[name].clone()
        bad[name][0, 40, 0, column] = inf
        o, state = decay_attention(**bad)
        hit = torch.zeros_like(o, dtype=torch.bool)
        seen = slice(40, 41) if name == "q" else slice(40, 50)
        hit[0, seen, 0, column if name == "v" else slice(None)] = True
        assert o[~hit].isfinite().all() and state.isfinite().all() and not o[0, 40, 0, column if name == "v" else 0].isfinite().all()


@pytest.mark.parametrize("decay", [0.0, 1.0, 1.01, 1e-30, 0.5])
def test_decay_attention_extreme_decays(decay):
    kw, d_o, d_state = _attention_inputs(2, 150, 1, 1, 16, 16, torch.float32, 14, resets=0.02, decay=[decay])
    _check_attention(kw, d_o, d_state)


def test_decay_attention_long_memory_keeps_its_scale():
    """decay^16 rounded once would be off by up to 2^-25 per block of 16 tokens, 2e-5 after 800 of them."""
    kw, d_o, d_state = _attention_inputs(1, 12800, 1, 1, 4, 4, torch.float32, 15, decay=[1 - 2.0 ** -14])
    kw["k"], kw["v"] = torch.ones_like(kw["k"]), torch.ones_like(kw["v"])
    _, state = decay_attention(**kw)
    want = attention(**{key: _cpu(x) for key, x in kw.items()})["state"]
    # sums of positive terms: every block of 16 adds 5 roundings at most, damped by what later blocks keep
    assert ((state.double().cpu() - want).abs() / want).max() <= 12800 / 16 * 5 * 2.0 ** -24 / 8


@pytest.mark.parametrize("t", [40, 300])
@pytest.mark.parametrize("layout", ["shared by stride", "columns", "odd start", "strided last", "transposed state"])
def test_decay_attention_layouts(layout, t):
    kw, d_o, d_state = _attention_inputs(3, t, 4, 4, 24, 16, torch.bfloat16, 16)
    if layout == "shared by stride":
        kw["k"], kw["v"] = kw["k"][:, :, :1].expand(3, t, 4, 24), kw["v"][:1].expand(3, t, 4, 16)
        d_o = d_o[:, :1].expand(3, t, 4, 16)
    elif layout == "columns":
        qkv = torch.randn(3, t, 4, 64, device=DEV).bfloat16()
        kw["q"], kw["k"], kw["v"] = qkv[..., :24], qkv[..., 24:48], qkv[..., 48:]
    elif layout == "odd start":
        qkv = torch.randn(3, t, 4, 65, device=DEV).bfloat16()
        kw["q"], kw["k"], kw["v"] = qkv[..., 1:25], qkv[..., 25:49], qkv[..., 49:]
    elif layout == "strided last":
        kw["v"] = torch.randn(3, t, 4, 32, device=DEV).bfloat16()[..., ::2]
        d_o = d_o[..., :1].expand(3, t, 4, 16)
    else:
        kw["state"], d_state = torch.randn(3, 4, 16, 24, device=DEV).transpose(2, 3), torch.randn(3, 4, 16, 24, device=DEV).transpose(2, 3)
    kw = {key: x.detach() if x is not None else None for key, x in kw.items()}
    _check_attention(kw, d_o, d_state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [inf, -inf, nan])
@pytest.mark.parametrize("t", [30, 400])
def test_decay_attention_not_finite_values_reach_only_who_sees_them(dtype, value, t):
    """Rows in front of the value, later episodes, other sequences, and what lies behind a sequence's end."""
    kw, d_o, d_state = _attention_inputs(2, t, 2, 2, 32, 32, dtype, 17, resets=0.0)
    kw["resets"] = torch.zeros(2, t, dtype=torch.bool, device=DEV)
    kw["resets"][0, t - 9] = True
    kw["lengths"] = torch.tensor([t, t - 5], device=DEV)
    clean, clean_state = decay_attention(**kw)
    at = t - 13
    for name in ("q", "k", "v"):
        bad = dict(kw)
        bad[name] = kw[name].clone()
        bad[name][0, at] = value           # sequence 0: behind it a reset
        bad[name][1, t - 5:] = value       # sequence 1: behind its end
        o, state = decay_attention(**bad)
        assert not o[0, at].isfinite().all()
        seen = slice(at, t - 9) if name != "q" else slice(at, at + 1)
        same = torch.ones(2, t, dtype=torch.bool, device=DEV)
        same[0, seen] = False
        assert o[same].isfinite().all() and state.isfinite().all()
        # a block that is summed again adds its products in another order: 16 more roundings of terms at most
        cpu = {key: _cpu(x) for key, x in kw.items()}
        bound = attention_bounds({"o": _cpu(clean).double()}, **cpu, dtype=dtype)["o"]
        mask = same.cpu()
        assert_within(o.cpu()[mask], _cpu(clean).double()[mask], 2 * bound[mask], name)
        assert torch.equal(state, clean_state)
    # backward: a gradient that is not finite in one token
    for x in (kw["q"], kw["k"], kw["v"]):
        x.requires_grad_(True)
    o, state = decay_attention(**kw)
    d_o = d_o.clone()
    d_o[0, at] = value
    d_o[1, t - 5:] = value
    dq, dk, dv = torch.autograd.grad((o, state), (kw["q"], kw["k"], kw["v"]), (d_o, d_state))
    assert dq[0, :at].isfinite().all() and dq[0, at + 1:].isfinite().all() and dq[1].isfinite().all()
    for x in (dk, dv):
        assert x[0, at + 1:].isfinite().all() and x[1].isfinite().all() and not x[0, at].isfinite().all()


def test_decay_attention_gradient_against_differences():
    """The result is linear in q, k, v and the initial state each: a central difference of the forward pass is exact but for rounding."""
    kw, d_o, d_state = _attention_inputs(2, 150, 4, 2, 16, 24, torch.float32, 18, resets=0.03, ragged=True)
    leaves = [kw[x].requires_grad_(True) for x in ("q", "k", "v", "state")]
    grads = torch.autograd.grad(decay_attention(**kw), leaves, (d_o, d_state))
    f = lambda **c: sum((a.double() * b.double()).sum() for a, b in zip(decay_attention(**{**kw, **c}), (d_o, d_state)))
    with torch.no_grad():
        for name, gr in zip(("q", "k", "v", "state"), grads):
            d = torch.randn_like(kw[name])
            slope = float((f(**{name: kw[name] + d}) - f(**{name: kw[name] - d})) / 2)
            mine = float((gr.double() * d.double()).sum())
            masses = [float((a.double() * b.double()).abs().sum()) for a, b in zip(decay_attention(**{**kw, name: kw[name].abs() + d.abs()}), (d_o, d_state))]
            assert abs(slope - mine) <= (16 + 24 + 300 + 34) * 2.0 ** -24 * 4 * sum(masses), (name, slope, mine)


def test_decay_attention_partial_gradients():
    """Gradients of the result alone, of the state alone, and without a wanted state."""
    kw, d_o, d_state = _attention_inputs(2, 40, 2, 2, 16, 16, torch.float32, 19)
    q, k, v, s = (kw[x].requires_grad_(True) for x in ("q", "k", "v", "state"))
    both = torch.autograd.grad(decay_attention(**kw), (q, k, v, s), (d_o, d_state))
    only_o = torch.autograd.grad(decay_attention(**kw)[0], (q, k, v, s), d_o)
    o, none = decay_attention(**kw, return_state=False)
    assert none is None
    for a, b in zip(torch.autograd.grad(o, (q, k, v, s), d_o), only_o):
        assert torch.equal(a, b)
    only_s = torch.autograd.grad(decay_attention(**kw)[1], (k, v, s), d_state)
    for i, (a, b) in enumerate(zip(only_s, (both[1] - only_o[1], both[2] - only_o[2], both[3] - only_o[3]))):
        assert torch.allclose(a, b, rtol=0, atol=1e-4 * float(b.abs().max())), i  # a difference of two sums of ~1e2 terms
    assert not torch.autograd.grad(decay_attention(**kw)[1], q, d_state)[0].any()
    kw["k"] = kw["k"].detach()
    got = torch.autograd.grad(decay_attention(**kw), (q, v), (d_o, d_state))
    assert torch.equal(got[0], both[0]) and torch.equal(got[1], both[2])
    with pytest.raises(RuntimeError):  # differentiable once
        x = torch.autograd.grad(decay_attention(**kw)[0].sum(), q, create_graph=True)[0]
        torch.autograd.grad(x.sum(), q)


def test_decay_attention_in_pieces_equals_the_whole():
    """A sequence taken in three calls, the state handed on, and in single steps."""
    kw, _, _ = _attention_inputs(3, 90, 2, 2, 32, 48, torch.float32, 20, resets=0.05)
    o, state = decay_attention(**kw)
    cpu = {key: _cpu(x) for key, x in kw.items()}
    want = attention(**cpu)
    bound = attention_bounds(want, **cpu, dtype=torch.float32)
    s, parts = kw["state"], []
    for a, b in ((0, 1), (1, 50), (50, 90)):
        part, s = decay_attention(kw["q"][:, a:b], kw["k"][:, a:b], kw["v"][:, a:b], kw["decay"], s, kw["resets"][:, a:b])
        parts.append(part)
    assert_within(torch.cat(parts, 1), want["o"], bound["o"], "pieces")
    assert_within(s, want["state"], bound["state"], "pieces' state")
    s = kw["state"].clone()
    steps = torch.stack([decay_attention_step(kw["q"][:, i], kw["k"][:, i], kw["v"][:, i], kw["decay"], s, kw["resets"][:, i]) for i in range(90)], 1)
    assert_within(steps, want["o"], bound["o"], "steps")
    assert_within(s, want["state"], bound["state"], "steps' state")


@pytest.mark.parametrize("n, t, h, d, dtype", [(3, 70000, 64, 128, torch.bfloat16)])
def test_decay_attention_offsets_beyond_32_bits(n, t, h, d, dtype):
    """More than 2^31 elements in a tensor: the last sequence's last tokens against a call on those tokens alone, started from a state
    that the decay of 1/2 has long made independent of what came before."""
    q, k, v = (torch.zeros(n, t, h, d, dtype=dtype, device=DEV) for _ in range(3))
    assert q.numel() > 3 << 29 and (n - 1) * t * h * d + (t - 1) * h * d > 1 << 30
    tail = 300
    for x in (q, k, v):
        x[-1, -tail:].normal_()
        x[0, :tail].normal_()
    decay = torch.full((h,), 0.5, device=DEV)
    o, state = decay_attention(q, k, v, decay)
    for part, got in (((slice(-1, None), slice(-tail, None)), o[-1:, -tail:]), ((slice(0, 1), slice(0, tail)), o[:1, :tail])):
        cut = {"q": q[part][:, :, -2:], "k": k[part][:, :, -2:], "v": v[part][:, :, -2:], "decay": decay[-2:]}
        cpu = {key: _cpu(x) for key, x in cut.items()}
        want = attention(**cpu)
        assert_within(got[:, :, -2:], want["o"], attention_bounds(want, **cpu, dtype=dtype)["o"], "o")
    assert not o[1].any() and not state[1].any()


# ------------------------------------------------------------------------------------------------ one step
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, h, hk, dk, dv", [(1, 1, 1, 1, 1), (1, 4, 4, 64, 64), (5, 3, 1, 8, 12), (70, 4, 2, 64, 64), (33, 2, 2, 128, 128),
                                              (3, 6, 2, 40, 72), (9, 1, 1, 127, 113), (2, 2, 1, 128, 1), (4, 3, 3, 1, 128), (1000, 2, 2, 16, 16), (7, 2, 2, 17, 100)])
@pytest.mark.parametrize("flags", [None, torch.int64, torch.bool])
def test_decay_attention_step(n, h, hk, dk, dv, dtype, flags):
    kw, _, _ = _attention_inputs(n, 1, h, hk, dk, dv, dtype, n + dk, resets=0.3)
    resets = kw["resets"][:, 0].to(flags) if flags else None
    state = kw["state"].clone()
    state0 = state.clone()
    if flags:
        state[resets.bool()] = nan  # what a finished episode left is not read into anything
    o = decay_attention_step(kw["q"][:, 0], kw["k"][:, 0], kw["v"][:, 0], kw["decay"], state, resets)
    cpu = {key: _cpu(x) for key, x in kw.items()}
    cpu["state"], cpu["resets"] = _cpu(state0), _cpu(kw["resets"]) if flags else None
    want = attention(**cpu)
    bound = attention_bounds(want, **cpu, dtype=dtype)
    assert o.shape == (n, h, dv) and o.dtype == dtype
    assert_within(o, want["o"][:, 0], bound["o"][:, 0], "o")
    assert_within(state, want["state"], bound["state"], "state")


def test_decay_attention_step_layouts():
    """Columns of one projection (odd starts), flags taken from a wider table, a state on no 16-byte boundary."""
    g = torch.Generator(device=DEV).manual_seed(22)
    n, h, dk, dv = 6, 2, 20, 36
    qkv = torch.randn(n, h, 2 * dk + dv + 1, generator=g, device=DEV)
    flags = torch.randint(0, 2, (n, 3), generator=g, device=DEV)
    store = torch.randn(n * h * dk * dv + 1, generator=g, device=DEV)
    state = store[1:].view(n, h, dk, dv)
    state0 = state.clone()
    decay = torch.rand(h, generator=g, device=DEV)
    q, k, v = qkv[..., 1:dk + 1], qkv[..., dk + 1:2 * dk + 1], qkv[..., 2 * dk + 1:]
    o = decay_attention_step(q, k, v, decay, state, flags[:, 1], scale=0.7)
    cpu = {"q": _cpu(q)[:, None], "k": _cpu(k)[:, None], "v": _cpu(v)[:, None], "decay": _cpu(decay), "state": _cpu(state0),
           "resets": _cpu(flags[:, 1:2]), "scale": 0.7}
    want = attention(**cpu)
    bound = attention_bounds(want, **cpu, dtype=torch.float32)
    assert_within(o, want["o"][:, 0], bound["o"][:, 0], "o")
    assert_within(state, want["state"], bound["state"], "state")
    assert decay_attention_step(q[:0], k[:0], v[:0], decay, state[:0]).shape == (0, h, dv)


def test_decay_attention_step_offsets_beyond_32_bits():
    n, h, d = 33000, 16, 64
    state = torch.zeros(n, h, d, d, device=DEV)
    assert state.numel() > 1 << 31
    q, k, v = (torch.randn(n, h, d, device=DEV) for _ in range(3))
    state[-1] = 1.0
    decay = torch.full((h,), 0.5, device=DEV)
    o = decay_attention_step(q, k, v, decay, state)
    small = torch.cat([torch.zeros_like(state[:1]), torch.ones_like(state[:1])])
    pick = [0, n - 1]
    assert torch.equal(o[pick], decay_attention_step(q[pick], k[pick], v[pick], decay, small)) and torch.equal(state[pick], small)


def test_step_invalidates_graphs_that_saved_the_state():
    kw, d_o, _ = _attention_inputs(2, 4, 1, 1, 8, 8, torch.float32, 23)
    q = kw["q"].requires_grad_(True)
    o, _ = decay_attention(**kw)
    with torch.no_grad():
        decay_attention_step(kw["q"][:, 0], kw["k"][:, 0], kw["v"][:, 0], kw["decay"], kw["state"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, q, d_o)
    with torch.inference_mode():
        decay_attention_step(kw["q"][:, 0], kw["k"][:, 0], kw["v"][:, 0], kw["decay"], torch.zeros(2, 1, 8, 8, device=DEV))


# ------------------------------------------------------------------------------------------------ streams, graphs, repetition
def _everything(kw, d_o, d_state, x, w, b, dx):
    """A policy's block forward and backward, and a step, on fresh leaves."""
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    mem = [kw[n].detach().requires_grad_(True) for n in ("q", "k", "v", "state")]
    o, s = decay_attention(*mem[:3], kw["decay"], mem[3], kw["resets"], kw["lengths"])
    grads = torch.autograd.grad(y, leaves, dx) + torch.autograd.grad((o, s), mem, (d_o, d_state))
    state = kw["state"].detach().clone()
    with torch.no_grad():
        step = decay_attention_step(kw["q"][:, 0], kw["k"][:, 0], kw["v"][:, 0], kw["decay"], state, kw["resets"][:, 0])
    return [t.detach() for t in (y, o, s, *grads, step, state)]


def _everything_inputs(seed, n=4, t=300, h=4, hk=2, dtype=torch.bfloat16):
    kw, d_o, d_state = _attention_inputs(n, t, h, hk, 32, 64, dtype, seed, resets=0.02, ragged=True)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    return kw, d_o, d_state, r(500, 87), r(87), r(87), r(500, 87)


def test_repeated_calls_and_other_streams_agree_bit_for_bit():
    args = _everything_inputs(30)
    want = _everything(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _everything(*args)
    again = _everything(*args)  # both streams at once
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(want, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_graphs_replay():
    """Forward, backward and a step in one graph; two graphs, replayed in turns with eager work between, new inputs each time."""
    sets = [_everything_inputs(40), _everything_inputs(41, n=2, t=40)]
    graphs, outs = [], []
    for args in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _everything(*args)
        torch.cuda.current_stream().wait_stream(side)
        gc.collect()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(_everything(*args))
        graphs.append(graph)
    for turn in range(3):
        for args, graph, out in zip(sets, graphs, outs):
            with torch.no_grad():
                args[0]["q"].normal_()
                args[0]["v"].mul_(-1)
                args[3].normal_()
            want = _everything(*args)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, out):
                assert torch.equal(a, b), turn
