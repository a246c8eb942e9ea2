"""ctypes front end of csrc/layer_norm.hip and csrc/decay_attention.hip: the operators of a policy with a memory.

``layer_norm``            layer norm over the last axis, differentiable
``decay_attention``       linear attention with one decay per head over whole sequences, differentiable
``decay_attention_step``  the same recurrence for one token per env, the state updated in place

They work on what the tasks hand out: ``resets`` is a task's ``reset_buf`` as it is (int64, or AnymalTerrain's bool), a rollout
may be stored time first (pass ``x.transpose(0, 1)``: only the last axis has to be contiguous, and results come back in the same
order in memory).  fp32, fp16 and bf16; every sum, statistic and state is fp32.  Calls are asynchronous launches on torch's
current stream of the tensors' device, allocate through torch and never synchronise, so they can be captured into a graph.
A backward pass inside a capture needs leaves no eager graph of which is alive: torch ties a leaf's gradient accumulation to
the stream it was first used on (``detach().requires_grad_()`` inside the capture gives fresh leaves).
No torch/CPU fallback: tensors must live on a ROCm device.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from ... import _lib

MAX_HEAD_DIM = 128
MAX_WIDTH = 16384


def _require(cond: bool, message: str) -> None:
    if not cond:
        raise _lib.OigeError(message)


def _tensors(what: str, required, optional=()) -> None:
    for (name, t), needed in [(x, True) for x in required] + [(x, False) for x in optional]:
        _require(isinstance(t, torch.Tensor) or (t is None and not needed), f"{what}: {name} must be a tensor, got {type(t).__name__}")


def _on_device(what: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        _require(t.device.type == "cuda", f"{what}: {name} is on {t.device}; liboige_hip kernels need a ROCm device tensor (no CPU fallback)")
        _require(t.device == device, f"{what}: {name} is on {t.device}, the other tensors on {device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _last_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _call(fn: str, io: C.Structure, device: torch.device) -> None:
    lib = _lib.load()
    if device.index is not None and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = getattr(lib, fn)(C.byref(io), _lib.current_stream(device))
    else:
        rc = getattr(lib, fn)(C.byref(io), _lib.current_stream(device))
    _lib.check(rc, fn)


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_io(x2: torch.Tensor, weight, bias, eps: float) -> _lib.LayerNormIo:
    io = _lib.LayerNormIo()
    io.x, io.weight, io.bias = x2.data_ptr(), _ptr(weight), _ptr(bias)
    io.rows, io.width = x2.shape
    io.x_row_stride = x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]
    io.dtype = _lib.ELEM_TYPES[x2.dtype]
    param = weight if weight is not None else bias
    io.weight_dtype = _lib.ELEM_TYPES[param.dtype] if param is not None else io.dtype
    io.eps = eps
    return io


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """(rows, width) with a contiguous last axis: a view wherever the leading axes collapse into one stride."""
    return _last_contiguous(x.reshape(-1, x.shape[-1]))


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows_of(x)
        keep = any(ctx.needs_input_grad)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        io = _norm_io(x2, weight, bias, eps)
        io.y = y.data_ptr()
        stats = torch.empty((2, x2.shape[0]), dtype=torch.float32, device=x.device) if keep else None
        if keep:
            io.mean, io.rstd = stats.data_ptr(), stats.data_ptr() + 4 * x2.shape[0]
        _call("oige_layer_norm_forward", io, x.device)
        if keep:
            ctx.save_for_backward(x2, weight, bias, stats)
            ctx.eps, ctx.shape = eps, x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, bias, stats = ctx.saved_tensors
        dx, dw, db = _layer_norm_backward(x2, weight, bias, stats, dy, ctx.eps, ctx.needs_input_grad)
        return (dx.view(ctx.shape) if dx is not None else None), dw, db, None


def _layer_norm_backward(x2, weight, bias, stats, dy, eps, needs):
    dy2 = _rows_of(dy)
    rows, width = x2.shape
    io = _norm_io(x2, weight, bias, eps)
    io.mean, io.rstd = stats.data_ptr(), stats.data_ptr() + 4 * rows
    io.dy, io.dy_row_stride = dy2.data_ptr(), dy2.stride(0) if rows > 1 else width
    dx = torch.empty((rows, width), dtype=x2.dtype, device=x2.device) if needs[0] else None
    dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if weight is not None and needs[1] else None
    db = torch.empty_like(bias, memory_format=torch.contiguous_format) if bias is not None and needs[2] else None
    io.dx, io.dweight, io.dbias = _ptr(dx), _ptr(dw), _ptr(db)
    ws = None
    if (dw is not None or db is not None) and rows:
        size = _lib.load().oige_layer_norm_workspace_floats(rows, width)
        ws = torch.empty(size, dtype=torch.float32, device=x2.device)
        io.workspace, io.workspace_floats = ws.data_ptr(), size
    if io.dx or io.dweight or io.dbias:
        _call("oige_layer_norm_backward", io, x2.device)
    return dx, dw, db


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis (1 to 16384 wide) of ``x`` (..., width).

    ``weight`` and ``bias`` are (width,) of x's type or both fp32 (either may be None); the result has x's shape and type and is
    contiguous.  Differentiable once in x, weight and bias; the parameters' gradients are sums in a fixed order."""
    _tensors("layer_norm", (("x", x),), (("weight", weight), ("bias", bias)))
    _require(x.dtype in _lib.ELEM_TYPES, f"layer_norm: x is {x.dtype}; float32, float16 and bfloat16 are supported")
    _require(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_WIDTH, f"layer_norm: x of shape {tuple(x.shape)} needs a last axis of 1 to {MAX_WIDTH}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _require(p.dtype in (x.dtype, torch.float32), f"layer_norm: {name} is {p.dtype}, expected {x.dtype} or float32")
            _require(tuple(p.shape) == (x.shape[-1],), f"layer_norm: {name} has shape {tuple(p.shape)}, expected {(x.shape[-1],)}")
    if weight is not None and bias is not None:
        _require(weight.dtype == bias.dtype, f"layer_norm: weight is {weight.dtype} and bias {bias.dtype}; they need one type")
    _require(math.isfinite(eps) and eps >= 0, f"layer_norm: eps = {eps}")
    _on_device("layer_norm", x.device, x=x, weight=weight, bias=bias)
    return _LayerNorm.apply(x, None if weight is None else _last_contiguous(weight), None if bias is None else _last_contiguous(bias), float(eps))


# ------------------------------------------------------------------------------------------------ decay attention
def _like(x: torch.Tensor, heads: int, d: int, dtype=None) -> torch.Tensor:
    """(N, T, heads, d), in memory in x's order of the first two axes (a rollout stored time first stays so)."""
    n, t = x.shape[:2]
    if n > 1 and t > 1 and x.stride(0) < x.stride(1):
        return torch.empty((t, n, heads, d), dtype=dtype or x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((n, t, heads, d), dtype=dtype or x.dtype, device=x.device)


def _check_flags(what, resets, shape):
    if resets is None:
        return
    _require(resets.dtype in (torch.bool, torch.uint8, torch.int64), f"{what}: resets is {resets.dtype}; bool, uint8 and int64 are supported")
    _require(tuple(resets.shape) == shape, f"{what}: resets has shape {tuple(resets.shape)}, expected {shape}")


def _check_heads(what, q, k, v, decay, state, lead):
    """Shapes and types of the tensors both forms share; ``lead`` = the axes in front of (heads, d)."""
    _require(q.dtype in _lib.ELEM_TYPES, f"{what}: q is {q.dtype}; float32, float16 and bfloat16 are supported")
    nl = len(lead)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _require(t.dim() == nl + 2, f"{what}: {name} has {t.dim()} axes, expected {lead + ('heads', 'd')}")
        _require(t.dtype == q.dtype, f"{what}: {name} is {t.dtype}, q is {q.dtype}")
        _require(t.shape[:nl] == q.shape[:nl], f"{what}: {name} has shape {tuple(t.shape)}, q {tuple(q.shape)}")
        _require(1 <= t.shape[-1] <= MAX_HEAD_DIM, f"{what}: head size {t.shape[-1]} of {name} (1 to {MAX_HEAD_DIM})")
    h, hk = q.shape[nl], k.shape[nl]
    _require(v.shape[nl] == hk and k.shape[-1] == q.shape[-1], f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match")
    _require(h >= 1 and hk >= 1 and h % hk == 0, f"{what}: {h} heads over {hk} key / value heads")
    _require(decay.dtype == torch.float32 and tuple(decay.shape) == (h,), f"{what}: decay must be float32 of shape {(h,)}, got {decay.dtype} {tuple(decay.shape)}")
    _require(not decay.requires_grad, f"{what}: decay is a constant of the head, it has no gradient")
    if state is not None:
        want = (q.shape[0], h, q.shape[-1], v.shape[-1])
        _require(state.dtype == torch.float32 and tuple(state.shape) == want,
                 f"{what}: state must be float32 of shape {want}, got {state.dtype} {tuple(state.shape)}")


def _attention_io(q, k, v, decay, state, resets, lengths, scale) -> _lib.DecayAttentionIo:
    io = _lib.DecayAttentionIo()
    io.q, io.k, io.v, io.decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr()
    io.q_stride[:], io.k_stride[:], io.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    io.state_in = _ptr(state)
    if resets is not None:
        io.resets, io.resets_bytes, io.resets_stride[:] = resets.data_ptr(), resets.element_size(), resets.stride()
    if lengths is not None:
        io.lengths, io.lengths_bytes = lengths.data_ptr(), lengths.element_size()
    io.num_envs, io.num_tokens, io.heads, io.key_dim = q.shape
    io.kv_heads, io.value_dim = v.shape[2], v.shape[3]
    io.dtype, io.scale = _lib.ELEM_TYPES[q.dtype], scale
    return io


def _workspace(io: _lib.DecayAttentionIo, backward: bool, device) -> Optional[torch.Tensor]:
    size = _lib.load().oige_decay_attention_workspace_floats(C.byref(io), int(backward))
    if size < 0:
        _lib.check(int(size), "oige_decay_attention_workspace_floats")
    if size == 0:
        return None
    ws = torch.empty(size, dtype=torch.float32, device=device)
    io.workspace, io.workspace_floats = ws.data_ptr(), size
    return ws


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, decay, resets, lengths, scale, return_state):
        ctx.set_materialize_grads(False)
        n, t, h, dk = q.shape
        dv = v.shape[3]
        io = _attention_io(q, k, v, decay, state, resets, lengths, scale)
        o = _like(q, h, dv)
        io.o, io.o_stride[:] = o.data_ptr(), o.stride()[:3]
        state_out = torch.empty((n, h, dk, dv), dtype=torch.float32, device=q.device) if return_state else None
        io.state_out = _ptr(state_out)
        if n and (t or return_state):
            ws = _workspace(io, False, q.device)  # noqa: F841 (kept alive over the launch)
            _call("oige_decay_attention_forward", io, q.device)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(q, k, v, state, decay, resets, lengths)
            ctx.scale = scale
        return o, state_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_state):
        q, k, v, state, decay, resets, lengths = ctx.saved_tensors
        return (*_decay_attention_backward(q, k, v, decay, state, resets, lengths, ctx.scale, d_o, d_state,
                                           state is not None and ctx.needs_input_grad[3]), None, None, None, None, None)


def _decay_attention_backward(q, k, v, decay, state, resets, lengths, scale, d_o, d_state, state_grad):
    n, t, h, dk = q.shape
    hk, dv = v.shape[2:]
    d_o = q.new_zeros((n, t, h, dv)) if d_o is None else _last_contiguous(d_o)
    d_state = None if d_state is None else d_state.contiguous()
    io = _attention_io(q, k, v, decay, state, resets, lengths, scale)
    io.d_o, io.d_o_stride[:], io.d_state_out = d_o.data_ptr(), d_o.stride()[:3], _ptr(d_state)
    dq, dk_, dv_ = _like(q, h, dk), _like(k, hk, dk), _like(v, hk, dv)
    io.dq, io.dk, io.dv = dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr()
    io.dq_stride[:], io.dk_stride[:], io.dv_stride[:] = dq.stride()[:3], dk_.stride()[:3], dv_.stride()[:3]
    ds = torch.empty_like(state) if state_grad else None
    io.d_state_in = _ptr(ds)
    if n and (t or state_grad):
        ws = _workspace(io, True, q.device)  # noqa: F841
        _call("oige_decay_attention_backward", io, q.device)
    return dq, dk_, dv_, ds


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
    anything.  ``scale`` defaults to key_dim ** -0.5.

    Returns ``(o, state)``: o (N, T, heads, value_dim) of q's type, and S behind every sequence's last token (None with
    ``return_state=False``).  Differentiable once in q, k, v and state; the backward pass recomputes the states."""
    what = "decay_attention"
    _tensors(what, (("q", q), ("k", k), ("v", v), ("decay", decay)), (("state", state), ("resets", resets), ("lengths", lengths)))
    _require(q.dim() == 4, f"{what}: q has {q.dim()} axes, expected (N, T, heads, key_dim)")
    _check_heads(what, q, k, v, decay, state, ("N", "T"))
    _check_flags(what, resets, tuple(q.shape[:2]))
    if lengths is not None:
        _require(lengths.dtype in (torch.int32, torch.int64) and tuple(lengths.shape) == (q.shape[0],),
                 f"{what}: lengths must be int32 or int64 of shape {(q.shape[0],)}, got {lengths.dtype} {tuple(lengths.shape)}")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    _require(math.isfinite(scale), f"{what}: scale = {scale}")
    _on_device(what, q.device, q=q, k=k, v=v, decay=decay, state=state, resets=resets, lengths=lengths)
    return _DecayAttention.apply(_last_contiguous(q), _last_contiguous(k), _last_contiguous(v), None if state is None else state.contiguous(),
                                 decay.contiguous(), resets, None if lengths is None else lengths.contiguous(), scale, bool(return_state))


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
                         resets: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """One token of ``decay_attention`` per env: updates ``state`` (N, heads, key_dim, value_dim; float32, contiguous) in place and
    returns o (N, heads, value_dim).  q (N, heads, key_dim), k (N, kv_heads, key_dim), v (N, kv_heads, value_dim); ``resets`` (N,)
    is a task's ``reset_buf`` as it is after ``env.step``: flagged envs start from an empty state.  Not differentiable."""
    what = "decay_attention_step"
    _tensors(what, (("q", q), ("k", k), ("v", v), ("decay", decay), ("state", state)), (("resets", resets),))
    _require(q.dim() == 3, f"{what}: q has {q.dim()} axes, expected (N, heads, key_dim)")
    _check_heads(what, q, k, v, decay, state, ("N",))
    _check_flags(what, resets, (q.shape[0],))
    _require(state.is_contiguous(), f"{what}: state is updated in place and must be contiguous")
    _require(not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)),
             f"{what}: updates the state in place and has no gradient; use decay_attention, or torch.no_grad()")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    _require(math.isfinite(scale), f"{what}: scale = {scale}")
    _on_device(what, q.device, q=q, k=k, v=v, decay=decay, state=state, resets=resets)
    q, k, v, decay = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v), decay.contiguous()
    n, h, dk = q.shape
    o = torch.empty((n, h, v.shape[2]), dtype=q.dtype, device=q.device)
    io = _lib.DecayAttentionStepIo()
    io.q, io.k, io.v, io.o, io.state, io.decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), state.data_ptr(), decay.data_ptr()
    io.q_stride[:], io.k_stride[:], io.v_stride[:] = q.stride()[:2], k.stride()[:2], v.stride()[:2]
    if resets is not None:
        io.resets, io.resets_bytes, io.resets_stride = resets.data_ptr(), resets.element_size(), resets.stride(0)
    io.num_envs, io.heads, io.kv_heads, io.key_dim, io.value_dim = n, h, k.shape[1], dk, v.shape[2]
    io.dtype, io.scale = _lib.ELEM_TYPES[q.dtype], scale
    if n:
        _call("oige_decay_attention_step", io, q.device)
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)  # a graph that saved the state must not be run backward any more
    return o
