"""Float64 formulas of the token-side operators (CPU) with a bound on what the kernels may differ from them by.

Every bound is arithmetic: u = 2^-24 is half a step of float32 arithmetic, h = torch.finfo(dtype).eps / 2 half a step of a
result's type. A sum of n terms in any order of depth d is off by at most d u sum |terms|; the kernels' sums over a row have
depth at most 16 (a thread) + 10 (lanes, waves) and their sums over rows at most rows / 256 + 96. Each formula's value is
accompanied by the same formula over absolute values, which the count of roundings multiplies.
"""

import torch

U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the subnormal numbers of a type (what rounding can lose next to zero)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(got, want, tol, what):
    """|got - want| <= tol everywhere, NaN and infinities in the same places."""
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} for {tuple(want.shape)}"
    same = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), same), f"{what}: not finite in other places than the formula"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    if not same.any():
        return
    off, tol = (got - want).abs()[same], tol.expand_as(want)[same]
    worst = (off / tol.clamp_min(1e-300)).max()
    assert bool((off <= tol).all()), f"{what}: off by {float(worst):.3g} times the bound (largest difference {float(off.max()):.3g})"


# ------------------------------------------------------------------------------------------------ layer norm
def norm_parts(x, eps):
    x = x.double().cpu()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    # a centred value is off by 28 u of the row's largest: xh by that times rstd and, through rstd, by as much of itself
    delta = 64 * U * (1 + x.abs().amax(-1, keepdim=True) * rstd)
    return (x - mean) * rstd, rstd, delta


def _rows(t, like):
    return torch.zeros_like(like) if t is None else t.double().cpu()


def norm_forward(x, w, b, eps):
    xh, _, delta = norm_parts(x, eps)
    w = 1.0 if w is None else w.double().cpu()
    b = 0.0 if b is None else b.double().cpu()
    y = xh * w + b
    w = torch.as_tensor(w)
    return y, delta * w.abs() * (1 + xh.abs()) + 4 * U * (torch.as_tensor(b).abs() + (xh * w).abs()) + half_step(x.dtype) * y.abs() + tiny(x.dtype)


def _along(t, xh, rstd):
    """P(t) and P over absolute values."""
    v = rstd * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
    a = rstd * (t.abs() + t.abs().mean(-1, keepdim=True) + (1 + xh.abs()) * (t.abs() * (1 + xh.abs())).mean(-1, keepdim=True))
    return v, a


def norm_backward(x, w, g, eps, param):
    xh, rstd, delta = norm_parts(x, eps)
    D = x.shape[-1]
    g = g.double().cpu()
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu()
    dx, ax = _along(g * w, xh, rstd)
    rows = max(1, x.numel() // D)
    depth = (96 + rows / 256) * U
    flat = lambda t: t.reshape(-1, D)  # noqa: E731
    dw, db = flat(g * xh).sum(0), flat(g).sum(0)
    tw = depth * flat((g * xh).abs()).sum(0) + flat(g.abs() * (1 + xh.abs()) * delta).sum(0) + half_step(param) * dw.abs() + tiny(param)
    tb = depth * flat(g.abs()).sum(0) + half_step(param) * db.abs() + tiny(param)
    return (dx, 2 * delta * ax + half_step(x.dtype) * dx.abs() + tiny(x.dtype)), (dw, tw), (db, tb)


def norm_second(x, w, g, u, a, c, eps, param):
    """Gradients of <u, dx> + <a, dw> + <c, db> with respect to x, w, g."""
    xh, rstd, delta = norm_parts(x, eps)
    D = x.shape[-1]
    g = g.double().cpu()
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu()
    u, a, c = _rows(u, xh), _rows(a, w), _rows(c, w)
    gw = g * w
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    one = 1 + xh.abs()
    pu, apu = _along(u, xh, rstd)
    dx, adx = _along(gw, xh, rstd)
    hh = a * g - rstd * (u * mean(gw * xh) + gw * mean(u * xh))
    ahh = (a * g).abs() + rstd * (u.abs() * mean(gw.abs() * one) + gw.abs() * mean(u.abs() * one))
    ph = _along(hh, xh, rstd)[0]
    aph = rstd * (ahh + mean(ahh) + one * mean(ahh * one))
    gx = ph - rstd * xh * mean(u * dx)
    agx = aph + rstd * one * mean(u.abs() * adx)
    gg = w * pu + a * xh + c
    agg = w.abs() * apu + a.abs() * one + c.abs()
    flat = lambda t: t.reshape(-1, D)  # noqa: E731
    gwt, agwt = flat(g * pu).sum(0), flat(g.abs() * apu)
    rows = max(1, x.numel() // D)
    dt = x.dtype
    tw = (2 * flat(delta.expand_as(xh)) * agwt).sum(0) + (96 + rows / 256) * U * agwt.sum(0) + half_step(param) * gwt.abs() + tiny(param)
    return ((gx, 4 * delta * agx + half_step(dt) * gx.abs() + tiny(dt)), (gwt, tw), (gg, 2 * delta * agg + half_step(dt) * gg.abs() + tiny(dt)))


# ------------------------------------------------------------------------------------------------ embedding
def embed_forward(ids, w, scale):
    y = w.double().cpu()[ids.cpu().long()] * scale
    return y, (half_step(w.dtype) + 2 * U) * y.abs() + tiny(w.dtype)


def embed_backward(ids, g, V, scale, padding):
    D, dt = g.shape[-1], g.dtype
    ids, g = ids.reshape(-1).cpu().long(), g.double().cpu().reshape(-1, D)
    live = (ids >= 0) & (ids < V) & (ids != padding)
    dw = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids[live], g[live]) * scale
    aw = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids[live], g[live].abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, ids[live], torch.ones(int(live.sum()), dtype=torch.float64))
    # a row of n tokens is summed in some order of depth at most n, and multiplied and rounded once
    return dw, (n + 2).unsqueeze(1) * U * aw + half_step(dt) * dw.abs() + tiny(dt)


# ------------------------------------------------------------------------------------------------ linear cross entropy
def linear_ce(x, w, b, t, ignore, reduction, g=None):
    """{name: (value, bound)} of loss and, for the loss's gradient g, dx, dw, db."""
    dt = x.dtype
    V, D = w.shape
    x, w = x.detach().double().cpu().reshape(-1, D), w.detach().double().cpu()
    t = t.cpu().reshape(-1).long()
    bias = torch.zeros(V, dtype=torch.float64) if b is None else b.detach().double().cpu()
    good = (t != ignore) & (t >= 0) & (t < V)
    bad = (t != ignore) & ~good
    xk = torch.where(good.unsqueeze(1), x, 0.0)
    z = xk @ w.t() + bias
    # products of 16-bit values are exact in float32; those of float32 values lose at most 12 u in their two float16 planes
    # (each operand's rest 2^-22, and the product of the second planes 2^-22); a sum over k has at most D roundings
    # a bias of minus infinity is exact: its classes have nothing to be off by
    dz_ = (D + 16) * U * (xk.abs() @ w.abs().t() + torch.where(torch.isfinite(bias), bias.abs(), 0.0))
    top = z.amax(1, keepdim=True)
    dzm = dz_.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    ti = torch.where(good, t, 0).unsqueeze(1)
    # the exponent's argument is rounded three times and exp2 once; a total of V terms has depth at most V / 16 + 64
    arg = torch.where(torch.isfinite(z), 4 * U * (top - z) + 4 * U, 0.0)
    rel = 2 * dzm + arg + (2 * (e * arg).sum(1, keepdim=True) / total + (V / 16 + 64) * U)
    each = (torch.log(total) - (z.gather(1, ti) - top)).squeeze(1)
    teach = (2 * dzm + (p * arg).sum(1, keepdim=True) + (V / 16 + 72) * U + 4 * U * (torch.log(total) + (top - z.gather(1, ti)))).squeeze(1)
    each, teach = torch.where(good, each, 0.0), torch.where(good, teach, 0.0)
    each = torch.where(bad, float("nan"), each)
    n = good.sum().double()
    N = x.shape[0]
    if reduction == "none":
        out = {"loss": (each, teach)}
    else:
        k = n if reduction == "mean" else torch.tensor(1.0, dtype=torch.float64)
        s = each.sum()
        out = {"loss": (s / k, (teach.sum() + (N / 1024 + 32) * U * each.nan_to_num().abs().sum()) / k + 2 * U * (s / k).abs())}
    if g is None:
        return out
    g = g.double().cpu().reshape(-1).expand(N)
    up = torch.where(good, g, 0.0) / (n if reduction == "mean" and n > 0 else 1.0)
    onehot = torch.zeros_like(p).scatter_(1, ti, 1.0)
    d = (p - onehot) * up.unsqueeze(1)
    # dz's own error, its rounding to 16 bits as an operand (float32: three planes, 2^-23), and float16's subnormals
    h = half_step(dt) if dt != torch.float32 else 2.0**-23
    ad = (p * rel + (p - onehot).abs() * (h + 8 * U)) * up.abs().unsqueeze(1) + onehot * 2 * U * up.abs().unsqueeze(1)
    if dt == torch.float16:
        ad = ad + 2.0**-39 * up.abs().max()
    ad = torch.where(good.unsqueeze(1), ad, 0.0)
    step = lambda v: half_step(dt) * v.abs() + tiny(dt)  # noqa: E731
    dx, dw, db = d @ w, d.t() @ xk, d.sum(0)
    dx = torch.where(bad.unsqueeze(1), float("nan"), dx)
    out["dx"] = (dx, ad @ w.abs() + (V + 16) * U * (d.abs() @ w.abs()) + step(dx.nan_to_num()))
    out["dw"] = (dw, ad.t() @ xk.abs() + (N + 16) * U * (d.abs().t() @ xk.abs()) + step(dw))
    out["db"] = (db, ad.sum(0) + (N + 16) * U * d.abs().sum(0) + step(db))
    return out
