"""Plain float64 forms of the operators over serialised points (window attention, rotary positions, RMS norm), on the CPU, and the
elementwise bounds of what the kernels' roundings can add up to.  u(t) is half a step of type t relative to the value."""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def visible(N, S, i0, length, left, right, sinks):
    """(N, S) truth values: row r stands at position i0 + r."""
    i, j = i0 + torch.arange(N)[:, None], torch.arange(S)[None]
    ok = (j < length) & (i < length) & (i >= 0)
    if right is not None:
        ok &= j <= i + right
    if left is not None:
        ok &= (j >= i - left) | (j < sinks)
    return ok


def attention(q, k, v, left, right, sinks, lengths, scale=None, step=False, dout=None, dtype=torch.float32):
    """q (B, N, H, D), k / v (B, S, G, D) of any type.  Returns {name: (value, bound)} for out and, with dout, dq, dk, dv.

    Bounds.  Scores: a product of D terms accumulated in fp32 is off by (D + 8) u32 sum |q||k|, the operands of the matrix cores add
    `prod` of the same sum where they are rounded pieces (half gradients: two bf16 pieces, 2^-16); exp2 of the fp32 difference, the
    sum and its reciprocal add a relative (S + 32) u32 and the rounding of c m - c s, 2 u32 |s|max.  Together p is off by
    es = 2 ds + (S + 32) u32 relative.  p enters its product rounded by `w`: u(bf16), u(half), or u32 for exact fp32 pieces.
    out: u |o| + (w + es) sum p |v|.  delta = dout . out inherits out's error.  dS = p (dP - delta) the same way, then its products."""
    B, N, H, D = q.shape
    S, G = k.shape[1:3]
    f = [t.detach().cpu().double() for t in (q, k, v)]
    q, k, v = f[0], f[1].repeat_interleave(H // G, 2), f[2].repeat_interleave(H // G, 2)
    scale = 1 / math.sqrt(D) if scale is None else scale
    lens = [S] * B if lengths is None else [max(0, min(S, int(x))) for x in lengths]
    ok = torch.stack([visible(N, S, n - N if step else 0, n, left, right, sinks) for n in lens])[:, None]
    zero = torch.zeros((), dtype=torch.float64)
    mm = lambda s, a, b: torch.einsum(s, a, b)  # noqa: E731
    clean = lambda t, rows: torch.where(rows, t, zero)  # noqa: E731
    krow = torch.stack([torch.arange(S) < n for n in lens])[:, :, None, None]
    k, v = clean(k, krow), clean(v, krow)
    if not step:
        q = clean(q, krow)
    s = scale * mm("bihd,bjhd->bhij", q, k)
    sabs = scale * mm("bihd,bjhd->bhij", q.abs(), k.abs())
    any_ = ok.any(-1, keepdim=True)
    p = torch.where(any_ & ok, torch.softmax(torch.where(ok, s, torch.where(any_, -math.inf, 0.0)), -1), zero)
    o = mm("bhij,bjhd->bihd", p, v)
    uo, w = u(dtype), U32 * 4 if dtype == torch.float32 else u(dtype)
    smax = float(torch.where(ok, sabs, zero).max()) if ok.any() else 0.0
    es = 2 * (D + 8) * U32 * smax + (S + 32) * U32 + 2 * U32 * smax
    A = mm("bhij,bjhd->bihd", p, v.abs())
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0          # half a step of half's subnormals
    got = {"out": (o, uo * o.abs() + (w + es) * A + tiny)}
    if dout is None:
        return got
    g = clean(dout.detach().cpu().double(), krow)
    prod = 2.0 ** -15 if dtype == torch.float16 else U32 * 8
    wg = {torch.float32: U32 * 4, torch.bfloat16: u(torch.bfloat16), torch.float16: 2.0 ** -15}[dtype]
    eg = es + 2 * prod * smax
    delta = (g * o).sum(-1).permute(0, 2, 1)[..., None]
    derr = (g.abs() * (got["out"][1] + (D + 8) * U32 * o.abs())).sum(-1).permute(0, 2, 1)[..., None]
    dp = mm("bihd,bjhd->bhij", g, v)
    dperr = (prod + (D + 8) * U32) * mm("bihd,bjhd->bhij", g.abs(), v.abs())
    ds = p * (dp - delta)
    dserr = (wg + eg) * ds.abs() + p * (derr + dperr)
    fold = lambda t: t.view(B, S, G, H // G, D).sum(3)  # noqa: E731
    acc = (S + 32) * U32
    dq, eq = scale * mm("bhij,bjhd->bihd", ds, k), scale * mm("bhij,bjhd->bihd", dserr + (acc + prod) * ds.abs(), k.abs())
    dk, ek = scale * fold(mm("bhij,bihd->bjhd", ds, q)), scale * fold(mm("bhij,bihd->bjhd", dserr + (acc * (H // G) + prod) * ds.abs(), q.abs()))
    dv, ev = fold(mm("bhij,bihd->bjhd", p, g)), (wg + eg + prod + acc * (H // G)) * fold(mm("bhij,bihd->bjhd", p, g.abs()))
    for name, x, e in (("dq", dq, eq), ("dk", dk, ek), ("dv", dv, ev)):
        got[name] = (x, uo * x.abs() + e + tiny)
    return got


def rotary(x, positions, freqs, magnitude, layout, sign=1.0, dtype=torch.float32):
    """(value, bound): products and polynomials of sine and cosine in fp32, a few u32 each, then one rounding."""
    x, pos, f = x.detach().cpu().double(), positions.detach().cpu().double(), freqs.cpu().double()
    if pos.dim() == 1:
        pos = pos.expand(x.shape[0], -1)
    if pos.dim() == 2:
        pos = pos[..., None]
    y, bound, P = x.clone(), torch.zeros_like(x), f.numel()
    for a in range(pos.shape[2]):
        ang = sign * pos[:, :, a, None] * f
        c, s = (torch.cos(ang) * magnitude)[:, :, None], (torch.sin(ang) * magnitude)[:, :, None]
        i = torch.arange(P) * (1 if layout == "half" else 2) + 2 * P * a
        j = i + (P if layout == "half" else 1)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        e = 12 * U32 * magnitude * (x[..., i].abs() + x[..., j].abs())
        bound[..., i], bound[..., j] = e, e
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    rot = bound > 0
    return y, torch.where(rot, bound + u(dtype) * y.abs() + tiny, torch.zeros(()).double())


def rms(x, w, eps, residual, dy=None, ds=None):
    """{name: (value, bound)}.  A lane adds at most 64 squares, the group 8 more times: the sum is off by 72 u32 relative, its root by
    half of that; the products add a few."""
    t = x.dtype
    xs = x.detach().cpu()
    s = xs.double() if residual is None else (xs.double() + residual.detach().cpu().double()).to(residual.dtype).double()
    w = w.detach().cpu().double()
    C = s.shape[-1]
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = s * rstd
    y = n * w
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    got = {"stream": (s, torch.zeros_like(s)), "y": (y, (u(t) + 48 * U32) * y.abs() + tiny)}
    if dy is None:
        return got
    dy = dy.detach().cpu().double()
    g = dy * w
    c = (g * n).mean(-1, keepdim=True)
    dx = rstd * (g - n * c) + (0 if ds is None else ds.detach().cpu().double())
    e = 160 * U32 * (rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + dx.abs())
    rows = s.reshape(-1, C).shape[0]
    got["dx"] = (dx, u(t) * dx.abs() + e + tiny)
    got["dr"] = (dx, (u(residual.dtype) if residual is not None else u(t)) * dx.abs() + e + tiny)
    dw = (dy * n).reshape(-1, C).sum(0)
    got["dw"] = (dw, (rows + 64) * U32 * (dy * n).abs().reshape(-1, C).sum(0))
    return got


def check(name, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - value).abs() - bound
    at = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or float(over.max()) <= 0, \
        f"{name}: {float(got.flatten()[at])} for {float(value.flatten()[at])}, bound {float(bound.flatten()[at])} (element {at} of {over.numel()}, {int((over > 0).sum())} over)"
