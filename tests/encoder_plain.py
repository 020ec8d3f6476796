"""The embedding encoder's operators in 64 bits, from their definitions (test infrastructure), with the error that 32-bit
arithmetic and one rounding of the result can make, element by element.

U is half a step of fp32. A result of type t is off by at most half a step of t, eps(t) / 2 relative to it, plus what the
32-bit arithmetic before that rounding is off; TINY covers results below the type's normal range (half a subnormal step)."""
import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def rows8(x):
    """(q, scale) of fp32 rows: an fp32 product with the neighbour of 1/127 and an IEEE fp32 quotient, so these are the
    operator's values bit for bit."""
    x = x.float().cpu()
    amax = x.abs().amax(dim=-1)
    bad = ~torch.isfinite(x).all(dim=-1)
    scale = (amax * torch.tensor(1 / 127, dtype=torch.float32)).masked_fill(bad, float("nan"))
    div = torch.where(scale > 0, scale, torch.tensor(float("inf")))
    q = torch.clamp(torch.round(x / div[..., None]), -127, 127)
    q = torch.where(bad[..., None], torch.zeros(()), q)
    return q.to(torch.int8), scale


def linear(q, sx, w, sw, bias, act, out_dtype):
    """(y, tolerance). The sum is exact; fp32 sees it converted (U), the product of the scales (U), their product (U), the
    sum with the bias (U): 4 U of |sum * scales| + |bias|. GELU: its slope is below 1.13, erf is off by less than 4 steps of
    fp32 (8 U) of a value up to 1, and three more roundings follow, of values up to |y|: 12 U |y|."""
    acc = q.double().cpu() @ w.double().cpu().t()
    y = acc * (sx.double().cpu()[..., None] * sw.double().cpu())
    size = y.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        size = size + bias.double().cpu().abs()
    tol = 4 * U * size
    if act == "gelu":
        tol = 1.13 * tol + 12 * U * y.abs()
        y = 0.5 * y * torch.special.erfc(-y / math.sqrt(2.0))
    return y, tol * (1 + 2 ** -6) + HALF_STEP[out_dtype] * y.abs() + TINY[out_dtype]


def _norm(v, err, kind, w, b, eps):
    """(normalised, error bound) of rows v known to `err` (per row). A 32-bit sum of n values, in whatever order, is off by
    at most n U of the sum of magnitudes; the rows here are summed by at least 64 lanes: (n / 64 + 16) U covers it."""
    n = v.shape[-1]
    c = (n / 64 + 16) * U
    big = v.abs().amax(-1, keepdim=True)
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(big)
    d = v - mean
    e_d = 2 * err + (c + 2 * U) * big                              # of a centred value
    var = (d * d).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    # sqrt(var) is a norm: it moves by at most the largest error of an element, and c relative
    e_r = r * (e_d * r + c + 4 * U)
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    o = d * r * w
    e = w.abs() * (e_d * r + d.abs() * e_r) + 3 * U * o.abs()
    if b is not None:
        o = o + b.double().cpu()
        e = e + U * o.abs()
    return o, e


def block_norm(y, x, rs, gate, per, post, pw, pb, nxt, nw, nb, eps):
    """{"stream": (value, error), "normed": ...} before the rounding to the result's type."""
    u = y.double().cpu()
    e = torch.zeros_like(u)
    if post != "none":
        u, e = _norm(u, torch.zeros_like(u[..., :1]), post, pw, pb, eps)
    if gate is not None:
        g = gate.double().cpu()[torch.arange(u.shape[0]) // per]
        u, e = u * g, e * g.abs() + U * (u * g).abs()
    if x is not None:
        xs = rs * x.double().cpu()
        e = e + U * xs.abs() + U * (u + xs).abs()
        u = u + xs
    out = {"stream": (u, e)}
    if nxt != "none":
        out["normed"] = _norm(u, e.amax(-1, keepdim=True), nxt, nw, nb, eps)
    return out


def within(got, want, err, dtype):
    """|got - want| <= err + one rounding to dtype, everywhere; NaN and infinities at the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    tol = err * (1 + 2 ** -6) + HALF_STEP[dtype] * want.abs() + TINY[dtype]
    off = (got - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or off.max() <= 0, f"off by {off.max():.3g} beyond the tolerance"


def attention(q, k, v, there, scale):
    """(out, error before the result's rounding) of q (queries, heads, d), k, v (keys, kv_heads, d), there (keys) bool.

    A score is off by (d + 4) U of sum |q k| scale; a weight exp(score - m) by that, by U |score - m| and by 8 U of its
    own; the sums of n terms by n U; a 16-bit type's weights are rounded once (half a step). All of it weighs on
    sum p |v|, twice for the part that the denominator shares."""
    t = q.dtype
    q, k, v = q.double().cpu(), k.double().cpu()[there.cpu()], v.double().cpu()[there.cpu()]
    n, group = k.shape[0], q.shape[1] // k.shape[1]
    if n == 0:
        z = torch.zeros_like(q)
        return z, z
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    size = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()) * abs(scale)
    p = torch.softmax(s, -1)
    o = torch.einsum("hqk,khd->qhd", p, v)
    far = (s.amax(-1, keepdim=True) - s)
    each = (q.shape[-1] + 4) * U * size + U * far + 8 * U + n * U
    w = torch.einsum("hqk,khd->qhd", p * each, v.abs()) + torch.einsum("hqk->qh", p * each)[..., None] * \
        torch.einsum("hqk,khd->qhd", p, v.abs())
    if t != torch.float32:
        w = w + HALF_STEP[t] * torch.einsum("hqk,khd->qhd", p, v.abs())
    return o, w + 4 * U * o.abs()
