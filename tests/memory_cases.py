"""The recurrent-policy operators' formulas in 64 bits, token by token, with the running error bound of a 32-bit evaluation.

Every result is a sum of products; a 32-bit evaluation in any order, with at most ``depth`` roundings on the way of a term, is off
by at most depth * 2^-24 times the sum of the terms' absolute values (to first order), and the store rounds once more, by half a
step of the type.  ``mass`` below is that sum of absolute values: the same recurrence on |q|, |k|, |v|.
"""
import torch

U32 = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SUBNORMAL = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def assert_within(got, want, bound, name):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~(err <= bound) & ~(got.isnan() & want.isnan()) & ~((got == want) & want.isinf())
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst "
                           f"{float((err / bound.clamp(min=1e-300))[bad].max()):.3g} x its bound at {bad.nonzero()[0].tolist()}")


def rounding(want, dtype):
    return HALF_STEP[dtype] * want.abs() + SUBNORMAL[dtype]


# ------------------------------------------------------------------------------------------------ decay attention
def attention(q, k, v, decay, state=None, resets=None, lengths=None, scale=None, d_o=None, d_state=None):
    """All on the CPU in float64: dict of o, state and (with d_o) dq, dk, dv, d_state_in."""
    q, k, v = q.double(), k.double(), v.double()
    n, t, h, dk = q.shape
    hk, dv = v.shape[2:]
    rep = h // hk
    k, v = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    a = decay.double()[None, :, None, None]
    scale = dk ** -0.5 if scale is None else scale
    length = torch.full((n,), t) if lengths is None else lengths.clamp(0, t)
    s = torch.zeros(n, h, dk, dv, dtype=torch.float64) if state is None else state.double().clone()
    o, dq = torch.zeros(n, t, h, dv, dtype=torch.float64), torch.zeros_like(q)

    def decayed(x, i):
        x = x * a
        return x if resets is None else torch.where(resets[:, i].bool()[:, None, None, None], torch.zeros_like(x), x)

    for i in range(t):
        live = (i < length)[:, None, None]
        new = decayed(s, i) + k[:, i, :, :, None] * v[:, i, :, None, :]
        s = torch.where(live[..., None], new, s)
        o[:, i] = torch.where(live, scale * (q[:, i, :, :, None] * s).sum(-2), 0.0)
        if d_o is not None:
            dq[:, i] = torch.where(live, scale * (s * d_o[:, i].double()[:, :, None, :]).sum(-1), 0.0)
    out = {"o": o, "state": s}
    if d_o is None:
        return out
    g = torch.zeros_like(s) if d_state is None else d_state.double().clone()
    dk_, dv_ = torch.zeros_like(k), torch.zeros_like(v)
    for i in range(t - 1, -1, -1):
        live = (i < length)[:, None, None]
        new = g + scale * q[:, i, :, :, None] * d_o[:, i].double()[:, :, None, :]
        dk_[:, i] = torch.where(live, (new * v[:, i, :, None, :]).sum(-1), 0.0)
        dv_[:, i] = torch.where(live, (new * k[:, i, :, :, None]).sum(-2), 0.0)
        g = torch.where(live[..., None], decayed(new, i), g)
    out.update(dq=dq, dk=dk_.view(n, t, hk, rep, dk).sum(3), dv=dv_.view(n, t, hk, rep, dv).sum(3), d_state_in=g)
    return out


def attention_bounds(want, q, k, v, decay, state=None, resets=None, lengths=None, scale=None, d_o=None, d_state=None, dtype=None):
    def mag(x):
        return None if x is None else x.double().abs()

    t, h, dk = q.shape[1:]
    rep, dv = h // v.shape[2], v.shape[3]
    scale = dk ** -0.5 if scale is None else scale
    mass = attention(mag(q), mag(k), mag(v), mag(decay), mag(state), resets, lengths, abs(scale), mag(d_o), mag(d_state))
    # a term passes at most one head size of additions on either side, one addition and one decay per token (or block of
    # tokens) and a handful of weights; shared heads are added up once more
    depth = dk + dv + 2 * t + rep + 32
    out = {}
    for name, w in want.items():
        stored = torch.float32 if name in ("state", "d_state_in") else dtype
        out[name] = depth * U32 * mass[name] + rounding(w, stored)
    return out


# ------------------------------------------------------------------------------------------------ layer norm
def norm(x, weight, bias, eps, dy=None):
    """(rows, width) on the CPU in float64: results and bounds of y and (with dy) dx, dw, db, before the stores' rounding."""
    x = x.double()
    rows, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(d, dtype=torch.float64) if bias is None else bias.double()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xhat = xc * rstd
    u = U32 * (d + 16)
    # the mean is off by u mean|x|, which shifts every centred value; the scale by a relative u (the shift's share of the variance
    # is of second order: kept for rows whose variance is nothing but that)
    shift = u * x.abs().mean(-1, keepdim=True) + U32 * x.abs()
    wobble = u + 0.5 * (shift.amax(-1, keepdim=True) * rstd) ** 2
    e_xhat = rstd * shift + xhat.abs() * wobble
    want = {"y": xhat * w + b}
    bound = {"y": e_xhat * w.abs() + 4 * U32 * ((xhat * w).abs() + b.abs())}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        mgx = (g * xhat).mean(-1, keepdim=True)
        inner = g - g.mean(-1, keepdim=True) - xhat * mgx
        want["dx"] = rstd * inner
        mass = g.abs() + g.abs().mean(-1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(-1, keepdim=True)
        bound["dx"] = rstd * (u * mass + e_xhat * mgx.abs() + xhat.abs() * (g.abs() * e_xhat).mean(-1, keepdim=True) + wobble * inner.abs())
        want["dw"], want["db"] = (dy * xhat).sum(0), dy.sum(0)
        bound["dw"] = (rows + 16) * U32 * (dy * xhat).abs().sum(0) + (dy.abs() * e_xhat).sum(0)
        bound["db"] = (rows + 16) * U32 * dy.abs().sum(0)
    return want, bound
