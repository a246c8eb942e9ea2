"""ctypes front end of csrc/layer_norm.hip and csrc/decay_attention.hip: the operators of a policy with a memory.

``layer_norm``            layer norm over the last axis, differentiable
``decay_attention``       linear attention with one decay per head over whole sequences, differentiable
``decay_attention_step``  the same recurrence for one token per env, the state updated in place

They work on what the tasks hand out: ``resets`` is a task's ``reset_buf`` as it is (int64, or AnymalTerrain's bool), a rollout
may be stored time first (pass ``x.transpose(0, 1)``: only the last axis has to be contiguous, and results come back in the same
order in memory).  fp32, fp16 and bf16; every sum, statistic and state is fp32.  Calls are asynchronous launches on torch's
current stream of the tensors' device, allocate through torch and never synchronise, so they can be captured into a graph.
Derivatives are reverse-mode, once; forward-mode tangents and traces (torch.jit.trace, make_fx) are refused.
What a call saved for its backward pass and an env step has written since (``obs_buf``, ``reset_buf``, the clamped observations) makes
that pass raise: a rollout that is trained on is a copy.
A backward pass inside a capture needs leaves no eager graph of which is alive: torch ties a leaf's gradient accumulation to
the stream it was first used on (``detach().requires_grad_()`` inside the capture gives fresh leaves).
No torch/CPU fallback: tensors must live on a ROCm device.
"""
from __future__ import annotations

import ctypes as C
from struct import Struct as _Struct
from typing import Callable, Optional, Tuple

import torch
from torch.autograd import forward_ad

from ... import _lib

MAX_HEAD_DIM = 128
MAX_WIDTH = 16384


_TYPES = _lib.ELEM_TYPES
_FLAGS = (torch.bool, torch.uint8, torch.int64)
_error = _lib.OigeError
_LARGEST = torch.finfo(torch.float32).max  # of eps and scale, which the kernels take in 32 bits


def _packer(struct) -> Callable[..., bytes]:
    """The fields of an argument block, in order, as its bytes: one pack instead of a ctypes store per field."""
    fmt, at = "<", 0
    codes = {C.c_void_p: "Q", C.c_int64: "q", C.c_int32: "i", C.c_float: "f"}
    for name, kind in struct._fields_:
        count = 1
        if issubclass(kind, C.Array):
            kind, count = kind._type_, kind._length_
        offset = getattr(struct, name).offset
        fmt += f"{offset - at}x" * (offset > at) + f"{count}{codes[kind]}"
        at = offset + getattr(struct, name).size
    fmt += f"{C.sizeof(struct) - at}x" * (C.sizeof(struct) > at)
    return _Struct(fmt).pack


_pack_norm, _pack_attention, _pack_step = _packer(_lib.LayerNormIo), _packer(_lib.DecayAttentionIo), _packer(_lib.DecayAttentionStepIo)


def _ptr(t: Optional[torch.Tensor]) -> int:
    if t is None:
        return 0
    p = t.data_ptr()
    if not p and t.numel():  # a wrapper or fake tensor would pass for an argument that was left out
        raise _error(f"a {type(t).__name__} of shape {tuple(t.shape)} has no memory a kernel could read")
    return p


def _last_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _needs_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _tensors(what: str, required, optional=()) -> None:
    for name, t in required:
        if not isinstance(t, torch.Tensor):
            raise _error(f"{what}: {name} must be a tensor, got {type(t).__name__}")
    for name, t in optional:
        if t is not None and not isinstance(t, torch.Tensor):
            raise _error(f"{what}: {name} must be a tensor, got {type(t).__name__}")
    # A launch is no torch operation: a trace would record the empty result alone, and a tangent would be lost without a word
    if torch._C._is_tracing() or (torch._C._len_torch_dispatch_stack() and _recording()):
        raise _error(f"{what}: cannot be traced (capture the call into a graph instead)")
    if forward_ad._current_level >= 0:
        for name, t in (*required, *optional):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise _error(f"{what}: {name} has a tangent; there is no forward-mode derivative")


def _recording() -> bool:
    from torch.fx.experimental.proxy_tensor import get_proxy_mode

    return get_proxy_mode() is not None


def _on_device(what: str, device: torch.device, named) -> None:
    if device.type != "cuda":
        raise _error(f"{what}: tensors are on {device}; liboige_hip kernels need ROCm device tensors (no CPU fallback)")
    for name, t in named:
        if t is not None and t.device != device:
            raise _error(f"{what}: {name} is on {t.device}, the other tensors on {device}")


def _call(fn: str, block: bytes, device: torch.device) -> None:
    lib = _lib.load()
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = getattr(lib, fn)(block, _lib.current_stream(device))
    else:
        rc = getattr(lib, fn)(block, _lib.current_stream(device))
    if rc:
        _lib.check(rc, fn)


# ------------------------------------------------------------------------------------------------ layer norm
def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """(rows, width) with a contiguous last axis: a view wherever the leading axes collapse into one stride."""
    return _last_contiguous(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))


def _norm_forward(x, weight, bias, eps, keep):
    x2 = _rows_of(x)
    rows, width = x2.shape
    dtype = x2.dtype
    y = torch.empty(x.shape, dtype=dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    at = _ptr(stats)
    param = weight if weight is not None else bias
    _call("oige_layer_norm_forward", _pack_norm(
        x2.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), at, at and at + 4 * rows, 0, 0, 0, 0, 0,
        0, rows, x2.stride(0) if rows > 1 else width, 0, width, _TYPES[dtype], _TYPES[dtype if param is None else param.dtype], eps), x.device)
    return y, x2, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, x2, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, bias, stats)
        ctx.eps, ctx.shape = eps, x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, bias, stats = ctx.saved_tensors
        needs = ctx.needs_input_grad
        device, dtype = x2.device, x2.dtype
        rows, width = x2.shape
        dy2 = _rows_of(dy)
        dx = torch.empty((rows, width), dtype=dtype, device=device) if needs[0] else None
        dw = torch.empty(width, dtype=weight.dtype, device=device) if needs[1] else None
        db = torch.empty(width, dtype=bias.dtype, device=device) if needs[2] else None
        ws, size = None, 0
        if rows and (needs[1] or needs[2]):
            size = _lib.load().oige_layer_norm_workspace_floats(rows, width)
            ws = torch.empty(size, dtype=torch.float32, device=device)
        param = weight if weight is not None else bias
        at = stats.data_ptr()
        _call("oige_layer_norm_backward", _pack_norm(
            x2.data_ptr(), _ptr(weight), _ptr(bias), 0, at, at + 4 * rows, dy2.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
            size, rows, x2.stride(0) if rows > 1 else width, dy2.stride(0) if rows > 1 else width, width,
            _TYPES[dtype], _TYPES[dtype if param is None else param.dtype], ctx.eps), device)
        return (dx.view(ctx.shape) if needs[0] else None), dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis (1 to 16384 wide) of ``x`` (..., width).

    ``weight`` and ``bias`` are (width,) of x's type or both fp32 (either may be None); the result has x's shape and type and is
    contiguous.  Differentiable once in x, weight and bias; the parameters' gradients are sums in a fixed order."""
    _tensors("layer_norm", (("x", x),), (("weight", weight), ("bias", bias)))
    dtype = x.dtype
    if dtype not in _TYPES:
        raise _error(f"layer_norm: x is {dtype}; float32, float16 and bfloat16 are supported")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise _error(f"layer_norm: x of shape {tuple(x.shape)} needs a last axis of 1 to {MAX_WIDTH}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            if p.dtype is not dtype and p.dtype is not torch.float32:
                raise _error(f"layer_norm: {name} is {p.dtype}, expected {dtype} or torch.float32")
            if p.dim() != 1 or p.shape[0] != x.shape[-1]:
                raise _error(f"layer_norm: {name} has shape {tuple(p.shape)}, expected {(x.shape[-1],)}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise _error(f"layer_norm: weight is {weight.dtype} and bias {bias.dtype}; they need one type")
    eps = float(eps)
    if not 0 <= eps <= _LARGEST:
        raise _error(f"layer_norm: eps = {eps}")
    _on_device("layer_norm", x.device, (("weight", weight), ("bias", bias)))
    weight = None if weight is None else _last_contiguous(weight)
    bias = None if bias is None else _last_contiguous(bias)
    if _needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ------------------------------------------------------------------------------------------------ decay attention
def _like(x: torch.Tensor, heads: int, d: int) -> torch.Tensor:
    """(N, T, heads, d), in memory in x's order of the first two axes (a rollout stored time first stays so)."""
    n, t = x.shape[:2]
    if n > 1 and t > 1 and x.stride(0) < x.stride(1):
        return torch.empty((t, n, heads, d), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((n, t, heads, d), dtype=x.dtype, device=x.device)


def _check_heads(what, q, k, v, decay, state, resets, lead):
    """Shapes and types of the tensors both forms share; ``lead`` = the number of axes in front of (heads, d)."""
    dtype = q.dtype
    if dtype not in _TYPES:
        raise _error(f"{what}: q is {dtype}; float32, float16 and bfloat16 are supported")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != lead + 2:
            raise _error(f"{what}: {name} has {t.dim()} axes, expected {('N', 'T')[:lead] + ('heads', 'd')}")
        if t.dtype is not dtype:
            raise _error(f"{what}: {name} is {t.dtype}, q is {dtype}")
        if not 1 <= t.shape[-1] <= MAX_HEAD_DIM:
            raise _error(f"{what}: head size {t.shape[-1]} of {name} (1 to {MAX_HEAD_DIM})")
    qs, ks, vs = q.shape, k.shape, v.shape
    for name, shape in (("k", ks), ("v", vs)):
        if shape[:lead] != qs[:lead]:
            raise _error(f"{what}: {name} has shape {tuple(shape)}, q {tuple(qs)}")
    h, hk = qs[lead], ks[lead]
    if vs[lead] != hk or ks[-1] != qs[-1]:
        raise _error(f"{what}: q {tuple(qs)}, k {tuple(ks)}, v {tuple(vs)} do not match")
    if h < 1 or hk < 1 or h % hk:
        raise _error(f"{what}: {h} heads over {hk} key / value heads")
    if decay.dtype is not torch.float32 or decay.dim() != 1 or decay.shape[0] != h:
        raise _error(f"{what}: decay must be float32 of shape {(h,)}, got {decay.dtype} {tuple(decay.shape)}")
    if decay.requires_grad:
        raise _error(f"{what}: decay is a constant of the head, it has no gradient")
    if state is not None and (state.dtype is not torch.float32 or state.shape != (qs[0], h, qs[-1], vs[-1])):
        raise _error(f"{what}: state must be float32 of shape {(qs[0], h, qs[-1], vs[-1])}, got {state.dtype} {tuple(state.shape)}")
    if resets is not None:
        if resets.dtype not in _FLAGS:
            raise _error(f"{what}: resets is {resets.dtype}; bool, uint8 and int64 are supported")
        if resets.shape != qs[:lead]:
            raise _error(f"{what}: resets has shape {tuple(resets.shape)}, expected {tuple(qs[:lead])}")


_NO3, _NO2 = (0, 0, 0), (0, 0)
_workspace_floats: dict = {}  # by sizes, type and direction, which is all that the size depends on


def _attention(fn, q, k, v, decay, state, resets, lengths, scale, o=None, state_out=None, d_o=None, d_state=None, dq=None, dk=None, dv=None,
               d_state_in=None):
    """Fill the argument block, give the call its workspace and make it."""
    n, t, h, key_dim = q.shape
    stride = lambda x: _NO3 if x is None else x.stride()[:3]

    def block(ws, size):
        return _pack_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(o), decay.data_ptr(), _ptr(state), _ptr(state_out), _ptr(resets), _ptr(lengths),
            _ptr(d_o), _ptr(d_state), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(d_state_in), ws, size,
            *stride(q), *stride(k), *stride(v), *stride(o), *stride(d_o), *stride(dq), *stride(dk), *stride(dv),
            *(_NO2 if resets is None else resets.stride()), n, t, h, v.shape[2], key_dim, v.shape[3], _TYPES[q.dtype],
            0 if resets is None else resets.element_size(), 0 if lengths is None else lengths.element_size(), scale)

    key = (n, t, h, v.shape[2], key_dim, v.shape[3], q.dtype, o is None)
    size = _workspace_floats.get(key)
    if size is None:
        size = _lib.load().oige_decay_attention_workspace_floats(block(0, 0), o is None)
        if size < 0:
            _lib.check(int(size), "oige_decay_attention_workspace_floats")
        if len(_workspace_floats) >= 1024:
            _workspace_floats.clear()
        _workspace_floats[key] = size
    ws = torch.empty(size, dtype=torch.float32, device=q.device) if size else None
    _call(fn, block(_ptr(ws), size), q.device)


def _attention_forward(q, k, v, state, decay, resets, lengths, scale, return_state):
    n, t, h, dk = q.shape
    dv = v.shape[3]
    o = _like(q, h, dv)
    state_out = torch.empty((n, h, dk, dv), dtype=torch.float32, device=q.device) if return_state else None
    if n and (t or return_state):
        _attention("oige_decay_attention_forward", q, k, v, decay, state, resets, lengths, scale, o=o, state_out=state_out)
    return o, state_out


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, decay, resets, lengths, scale, return_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, state, decay, resets, lengths)
        ctx.scale = scale
        return _attention_forward(q, k, v, state, decay, resets, lengths, scale, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_state):
        q, k, v, state, decay, resets, lengths = ctx.saved_tensors
        n, t, h, dk = q.shape
        hk, dv = v.shape[2:]
        d_o = q.new_zeros((n, t, h, dv)) if d_o is None else _last_contiguous(d_o)
        d_state = None if d_state is None else d_state.contiguous()
        dq, dk_, dv_ = _like(q, h, dk), _like(k, hk, dk), _like(v, hk, dv)
        ds = torch.empty_like(state) if ctx.needs_input_grad[3] else None
        if n and (t or ds is not None):
            _attention("oige_decay_attention_backward", q, k, v, decay, state, resets, lengths, ctx.scale, d_o=d_o, d_state=d_state, dq=dq,
                       dk=dk_, dv=dv_, d_state_in=ds)
        return dq, dk_, dv_, ds, None, None, None, None, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: Optional[torch.Tensor] = None,
                    resets: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    return_state: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Linear attention with one decay per head over sequences of tokens:

        S_t = a_t S_{t-1} + k_t v_t^T        a_t = decay[h], 0 where ``resets[n, t]`` is set
        o_t = scale * S_t^T q_t

    q (N, T, heads, key_dim); k (N, T, kv_heads, key_dim) and v (N, T, kv_heads, value_dim) with kv_heads dividing heads (query
    head h reads key / value head h // (heads / kv_heads)); head sizes 1 to 128.  decay (heads,) float32, a constant.
    ``state`` (N, heads, key_dim, value_dim) float32 is S before the first token (None: zeros).  A reset clears the state before
    its token is taken in: the flag belongs to the first token of an episode.  ``lengths`` (N,) int32 / int64 ends sequence n
    before token lengths[n] (clamped to 0 .. T); rows behind the end are zero in the result and in the gradients and may hold
    anything.  ``scale`` defaults to key_dim ** -0.5.  An infinite or NaN value makes the results that depend on it NaN or
    infinite, and no others.

    Returns ``(o, state)``: o (N, T, heads, value_dim) of q's type, and S behind every sequence's last token (None with
    ``return_state=False``).  Differentiable once in q, k, v and state; the backward pass recomputes the states."""
    what = "decay_attention"
    _tensors(what, (("q", q), ("k", k), ("v", v), ("decay", decay)), (("state", state), ("resets", resets), ("lengths", lengths)))
    _check_heads(what, q, k, v, decay, state, resets, 2)
    if lengths is not None and (lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != q.shape[:1]):
        raise _error(f"{what}: lengths must be int32 or int64 of shape {(q.shape[0],)}, got {lengths.dtype} {tuple(lengths.shape)}")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _LARGEST:
        raise _error(f"{what}: scale = {scale}")
    _on_device(what, q.device, (("k", k), ("v", v), ("decay", decay), ("state", state), ("resets", resets), ("lengths", lengths)))
    args = (_last_contiguous(q), _last_contiguous(k), _last_contiguous(v), None if state is None else state.contiguous(), decay.contiguous(),
            resets, None if lengths is None else lengths.contiguous(), scale, bool(return_state))
    return _DecayAttention.apply(*args) if _needs_grad(q, k, v, state) else _attention_forward(*args)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
                         resets: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """One token of ``decay_attention`` per env: updates ``state`` (N, heads, key_dim, value_dim; float32, contiguous) in place and
    returns o (N, heads, value_dim).  q (N, heads, key_dim), k (N, kv_heads, key_dim), v (N, kv_heads, value_dim); ``resets`` (N,)
    is a task's ``reset_buf`` as it is after ``env.step``: flagged envs start from an empty state.  Not differentiable."""
    what = "decay_attention_step"
    _tensors(what, (("q", q), ("k", k), ("v", v), ("decay", decay), ("state", state)), (("resets", resets),))
    _check_heads(what, q, k, v, decay, state, resets, 1)
    if not state.is_contiguous():
        raise _error(f"{what}: state is updated in place and must be contiguous")
    if _needs_grad(q, k, v, state):
        raise _error(f"{what}: updates the state in place and has no gradient; use decay_attention, or torch.no_grad()")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _LARGEST:
        raise _error(f"{what}: scale = {scale}")
    device = q.device
    _on_device(what, device, (("k", k), ("v", v), ("decay", decay), ("state", state), ("resets", resets)))
    q, k, v, decay = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v), decay.contiguous()
    n, h, dk = q.shape
    hk, dv = v.shape[1:]
    o = torch.empty((n, h, dv), dtype=q.dtype, device=device)
    if n:
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        _call("oige_decay_attention_step", _pack_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), state.data_ptr(), decay.data_ptr(), _ptr(resets),
            qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], 0 if resets is None else resets.stride(0), n, h, hk, dk, dv, _TYPES[q.dtype],
            0 if resets is None else resets.element_size(), scale, 0), device)
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)  # a graph that saved the state must not be run backward any more
    return o
