"""The operators over feature rows in 64 bits, with a bound on how far an evaluation in 32-bit sums and one rounding to
the tensors' type may lie from them.

Bounds are worst cases, element by element.  u is half a step of the type (finfo.eps / 2), e = 2^-24 that of float32.
A sum of n products in float32, in any order, is within n e of the sum of the products' magnitudes (to first order;
what is doubled below covers the rest), and what a 16-bit type rounds below its smallest normal number is within half
its smallest subnormal one."""
import math

import torch

E = 2.0 ** -24
F = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2 if dtype != torch.float32 else 2.0 ** -126


def rounded(value, error, dtype):
    """Bound after one rounding to `dtype` of something within `error` of `value`."""
    return error + half_step(dtype) * (value.abs() + error) + tiny(dtype)


def activation(z, act):
    """-> value, derivative, largest |derivative| anywhere, largest |second derivative| anywhere"""
    if act == "none":
        return z, torch.ones_like(z), 1.0, 0.0
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(F), 1.0, 0.0
    if act == "gelu":
        phi, pdf = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * phi, phi + z * pdf, 1.13, 0.8
    s = torch.sigmoid(z)
    if act == "silu":
        return z * s, s * (1 + z * (1 - s)), 1.1, 0.5
    return s, s * (1 - s), 0.25, 0.1


def linear(x, weight, bias, act, residual, dy):
    """-> {name: (value, bound)} for y, dx, dweight, dbias (and dresidual)"""
    dtype = x.dtype
    u = half_step(dtype)
    x, w = x.to(F).reshape(-1, x.shape[-1]), weight.to(F)
    k, n, rows = w.shape[1], w.shape[0], x.shape[0]
    b = torch.zeros(n, dtype=F, device=w.device) if bias is None else bias.to(F)
    z = x @ w.t() + b
    dz_err = 2 * (k + 2) * E * (x.abs() @ w.abs().t() + b.abs())
    value, slope, steep, bend = activation(z, act)
    # the activation's own evaluation: the float32 functions in it are good to a few units in the last place, their
    # arguments (z / sqrt 2, z^2 / 2) to two, which the exponential turns into two |argument| of its value
    act_err = 0.0 if act in ("none", "relu") else 16 * E * (1 + z.abs())
    y, err = value, steep * dz_err + act_err
    if residual is not None:
        r = residual.to(F).reshape(-1, n)
        y = y + r
        err = err + E * (value.abs() + r.abs())
    out = {"y": (y, rounded(y, err, dtype))}
    if dy is None:
        return out
    g = dy.to(F).reshape(-1, n)
    dz = g * slope
    slope_err = bend * dz_err + act_err
    if act != "none" and dtype != torch.float32:  # the derivative travels in half precision
        slope_err = slope_err + 2.0 ** -11 * slope.abs() + 2.0 ** -25
    exact_dz_err = g.abs() * slope_err + E * dz.abs()
    stored = exact_dz_err if act == "none" or dtype == torch.float32 else rounded(dz, exact_dz_err, dtype)
    dx = dz @ w
    out["dx"] = (dx, rounded(dx, stored @ w.abs() + 2 * (n + 2) * E * ((dz.abs() + stored) @ w.abs()), dtype))
    dw = dz.t() @ x
    out["dweight"] = (dw, rounded(dw, stored.t() @ x.abs() + 2 * (rows + 2) * E * ((dz.abs() + stored).t() @ x.abs()), dtype))
    db = dz.sum(0)
    out["dbias"] = (db, rounded(db, exact_dz_err.sum(0) + 2 * (rows + 2) * E * dz.abs().sum(0), dtype))
    out["dresidual"] = (g, torch.zeros_like(g))
    return out


def layer_norm(x, weight, bias, eps, dy):
    dtype, wtype = x.dtype, (weight if weight is not None else bias if bias is not None else x).dtype
    x = x.to(F).reshape(-1, x.shape[-1])
    rows, d = x.shape
    w = torch.ones(d, dtype=F, device=x.device) if weight is None else weight.to(F)
    b = torch.zeros(d, dtype=F, device=x.device) if bias is None else bias.to(F)
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    u = c * r
    # the mean is off by at most (d + 2) e mean|x|, every centred value by that and its own rounding
    mean_err = 2 * (d + 2) * E * x.abs().mean(1, keepdim=True)
    c_err = mean_err + E * (c.abs() + mean_err)
    var_err = 2 * (d + 4) * E * (var + eps) + 2 * (c.abs() * c_err).mean(1, keepdim=True) + (c_err ** 2).mean(1, keepdim=True)
    r_rel = var_err / (2 * (var + eps)) * 1.5 + 4 * E  # d r / r = -d var / (2 (var + eps)), to second order
    u_err = c_err * r + u.abs() * (r_rel + 2 * E) + c_err * r * r_rel
    y = u * w + b
    out = {"y": (y, rounded(y, u_err * w.abs() + 3 * E * ((u * w).abs() + b.abs()), dtype))}
    if dy is None:
        return out
    dy = dy.to(F).reshape(-1, d)
    g = dy * w
    mg, mgu = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
    dx = r * (g - mg - u * mgu)
    mg_err = 2 * (d + 3) * E * g.abs().mean(1, keepdim=True)
    mgu_err = 2 * (d + 4) * E * (g * u).abs().mean(1, keepdim=True) + (g.abs() * u_err).mean(1, keepdim=True)
    inner = 2 * E * g.abs() + mg_err + u_err * mgu.abs() + u.abs() * mgu_err + u_err * mgu_err + \
        4 * E * (g.abs() + mg.abs() + (u * mgu).abs())
    dx_err = r * inner * (1 + r_rel) + (r_rel + 2 * E) * r * (g.abs() + mg.abs() + (u * mgu).abs())
    out["dx"] = (dx, rounded(dx, dx_err, dtype))
    dw, db = (dy * u).sum(0), dy.sum(0)
    out["dweight"] = (dw, rounded(dw, (dy.abs() * u_err).sum(0) + 2 * (rows + 2) * E * (dy * u).abs().sum(0), wtype))
    out["dbias"] = (db, rounded(db, 2 * (rows + 2) * E * dy.abs().sum(0), wtype))
    return out


def kept(numel, p, seed, offset):
    """The mask as the definition has it, element by element in Python's whole numbers."""
    word = 0xFFFFFFFF
    threshold = int(math.floor(p * 65536 + 0.5))
    mask, halves = [], []
    for i in range(numel):
        if i % 8 == 0:
            block = i // 8
            a, b, c, d = block & word, block >> 32, offset & word, (offset >> 32) & word
            k0, k1 = seed & word, (seed >> 32) & word
            for _ in range(7):
                l, h = a * 0xD2511F53, c * 0xCD9E8D57
                a, b, c, d = (h >> 32) ^ b ^ k0, h & word, (l >> 32) ^ d ^ k1, l & word
                k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
            halves = [w >> s & 0xFFFF for w in (a, b, c, d) for s in (0, 16)]
        mask.append(halves[i % 8] >= threshold)
    return torch.tensor(mask, dtype=torch.bool)


def dropout(x, mask, p, residual, dy):
    threshold = int(math.floor(p * 65536 + 0.5))
    scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    dtype = x.dtype

    def one(t, r):
        v = torch.where(mask, t.to(F) * scale, 0.0)
        err = 2 * E * v.abs()
        if r is not None:
            v = v + r.to(F)
            err = err + E * v.abs()
        return v, rounded(v, err, dtype)

    out = {"y": one(x, residual)}
    if dy is not None:
        out["dx"] = one(dy, None)
        out["dresidual"] = (dy.to(F), torch.zeros_like(dy, dtype=F))
    return out


def assert_within(got, want, what):
    """`want` as (value, bound); the largest excess is named."""
    value, bound = want
    diff = (got.detach().to(F).reshape(value.shape) - value).abs()
    bad = ~(diff <= bound)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%s: %d of %d elements out of bounds, first at %s: got %r, want %r, bound %.3e" % (
            what, int(bad.sum()), bad.numel(), at, got.detach().reshape(value.shape)[tuple(at)].item(),
            value[tuple(at)].item(), bound[tuple(at)].item()))
