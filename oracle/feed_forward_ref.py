"""Float64 forms of the feed-forward operators (nerfool_amd/gnt/feed_forward.py) with bounds on how far a computation in `dtype` may be from
them.  Bounds are worst cases, element by element, made of: half a step (finfo.eps / 2 of the value) for each rounding to the tensors' type; for a
sum of K products in float32 (K + 8) 2^-23 times the sum of the magnitudes (twice the classical K 2^-24, for a matrix core that cuts off
instead of rounding; a float32 operand in three parts makes six products of each, the dropped ones below 2^-24: 6 K instead of K); 16 units of
2^-24 for an activation."""
import math

import torch

U = 2.0 ** -24
LIPSCHITZ = {'silu': (1.1, 0.5), 'gelu': (1.13, 0.8), 'relu': (1.0, 0.0)}      # max |act'|, max |act''|


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_step(dtype):
    """half the spacing of the subnormal values: what a rounding can lose of a tiny value (float32 products may flush: the least normal number)"""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def rounded(value, bound, dtype, scale=1.0):
    """value +- bound, rounded to dtype, as held times `scale`"""
    return bound + half_step(dtype) * (value.abs() + bound) + floor_step(dtype) / scale


def act(name, g):
    if name == 'silu':
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == 'gelu':
        c = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).to(g.dtype)


def norm(x, weight, residual, eps, dy=None, dh=None, dtype=torch.float32, lost=None):
    """-> {name: (value, bound)}; lost: what the h that the backward pass reads is off by, relative (None: a rounding to dtype); sums over a row are trees of at most 64 links plus the row's 16-byte vectors a thread"""
    x, r = x.double(), None if residual is None else residual.double()
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    h = x if r is None else x + r
    n = x.shape[1]
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    xhat = h * rstd
    y = xhat * w
    k = (96 + n // 256) * U
    got = {'h': (h, rounded(h, U * h.abs(), dtype)), 'y': (y, rounded(y, k * y.abs(), dtype))}
    if dy is None:
        return got
    dy = dy.double()
    if lost is None:
        lost = half_step(dtype) if r is not None else 0.0
    g = dy * w
    mean = (g * xhat).mean(1, keepdim=True)
    mean_abs = (g * xhat).abs().mean(1, keepdim=True)
    dx = rstd * (g - xhat * mean)
    b = rstd * (k * (g.abs() + xhat.abs() * mean_abs) + lost * xhat.abs() * (mean.abs() + mean_abs) * (1 + lost))
    if dh is not None:
        dx = dx + dh.double()
        b = b + 4 * U * (dh.double().abs() + dx.abs())
    got['dx'] = (dx, rounded(dx, b, dtype))
    s = (dy * xhat).abs().sum(0)
    got['dweight'] = ((dy * xhat).sum(0), rounded((dy * xhat).sum(0), ((x.shape[0] + 96) * U + k + lost) * s, dtype))
    return got


def _product(a, ea, b, eb, parts):
    """(value, bound) of a @ b for operands known to ea, eb"""
    k = (6 * a.shape[1] if parts else a.shape[1]) + 8
    mag = a.abs() @ b.abs()
    bound = k * 2.0 ** -23 * mag
    for p, q in ((ea, b.abs()), (a.abs(), eb), (ea, eb)):
        if p is not None and q is not None:
            bound = bound + p @ q
    return a @ b, bound


def gated(x, w_gate, w_up, w_down, name, dy=None, dtype=torch.float32, sides=False, scale=1.0):
    """-> {name: (value, bound)}; sides: relu's side of zero has to be the exact sum's, also where that is below what a float32 sum is off by;
    scale: dg and du have to be held times at least that"""
    parts = dtype == torch.float32
    x, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    l1, l2 = LIPSCHITZ[name]
    g, eg = _product(x, None, wg.t(), None, parts)
    u, eu = _product(x, None, wu.t(), None, parts)
    a, slope = act(name, g)
    ea = l1 * eg + 16 * U * (a.abs() + U)
    h = a * u
    eh = rounded(h, ea * u.abs() + (a.abs() + ea) * eu + 2 * U * h.abs(), dtype)
    out, eo = _product(h, eh, wd.t(), None, parts)
    got = {'out': (out, rounded(out, eo, dtype))}
    if dy is None:
        return got
    dy = dy.double()
    dh, edh = _product(dy, None, wd, None, parts)
    es = l2 * eg + 16 * U * (1 + g.abs()) + ((g.abs() <= eg).double() if name == 'relu' and not sides else 0)
    dg, du = dh * u * slope, dh * a
    edg = edh * (u.abs() + eu) * (slope.abs() + es) + dh.abs() * (eu * (slope.abs() + es) + u.abs() * es) + 4 * U * dg.abs()
    edu = edh * (a.abs() + ea) + dh.abs() * ea + 4 * U * du.abs()
    edg, edu = rounded(dg, edg, dtype, scale), rounded(du, edu, dtype, scale)
    v1, b1 = _product(torch.cat([dg, du], 1), torch.cat([edg, edu], 1), torch.cat([wg, wu], 0), None, parts)
    got['dx'] = (v1, rounded(v1, b1, dtype))
    for key, (d, e), other in (('dw_gate', (dg, edg), x), ('dw_up', (du, edu), x)):
        v, b = _product(d.t(), e.t(), other, None, parts)
        got[key] = (v, rounded(v, b, dtype))
    v, b = _product(dy.t(), None, h, eh, parts)
    got['dw_down'] = (v, rounded(v, b, dtype))
    return got


def to_8bit(v):
    """float64 [rows, n] -> (e4m3 values, 2^e per block of 32)"""
    rows, n = v.shape
    full = torch.nn.functional.pad(v, (0, -n % 32)).reshape(rows, -1, 32)
    top = full.abs().amax(2, keepdim=True)
    e = torch.full_like(top, -127.0)
    for k in range(-127, 121):          # the least e that is enough
        e = torch.where((top > 448 * 2.0 ** (k - 1)) & (top <= 448 * 2.0 ** k) & (k > -127), torch.full_like(e, float(k)), e)
    z = full / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(z / step) * step).reshape(rows, -1)[:, :n], torch.exp2(e[:, :, 0])
