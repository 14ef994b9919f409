"""Norm and rotation of the rows of a head in float64, and how far a kernel may be off.

y = x / sqrt(mean x^2 + eps) w, the first R columns turned by (cos, sin) of their row; u is half a step of the element type
relative to the value, v = 2^-24 the same of float32.

* r = 1 / sqrt(mean + eps): a sum of D squares in float32, in any order at most D roundings of each (32 in the order of the kernels: up to 16
  in a lane and 6 between lanes; D <= 256), half of that in the root, 2 v for the root itself: c v with c = 24.
* z_a = y_a c - y_b s: y is off by (c + 2) v of itself, the products and the sum by 2 v more: 32 v (|y_a c| + |y_b s|), and u |z|.
* gradient, g the gradient of z turned back (off by 3 v of the sizes of its terms, G): dx = r (g w - x^ m), m = mean(g w x^) (off by
  64 v of its terms' mean with G for g, for the sum is like that of r):  96 v r (G |w| + |x^| mean(G |w| |x^|)), and u |dx|.
* dw: the sum over n rows of g x^, in float32: (32 + n) v sum G |x^|, and u_w |dw|."""
import torch


def turn(x, c, s, R, interleaved):
    """The first R columns of [..., D] turned; c, s [..., R / 2]."""
    out = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a], x[..., b]
    out[..., a], out[..., b] = xa * c - xb * s, xb * c + xa * s
    return out


def sizes(x, c, s, R, interleaved):
    """The sum of the sizes of the terms of turn."""
    out = x.abs().clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a].abs(), x[..., b].abs()
    out[..., a], out[..., b] = xa * c.abs() + xb * s.abs(), xb * c.abs() + xa * s.abs()
    return out


def angles(pos, cos, sin):
    """Rows of the table for the positions (any shape); 1 and 0 outside it."""
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = torch.where(ok, pos, 0)
    one = lambda x, v: torch.where(ok[..., None], x.double()[at], torch.full((), v, dtype=torch.float64, device=x.device))
    return one(cos, 1.0), one(sin, 0.0)


def forward(x, w, c, s, R, interleaved, eps, norm=True):
    x = x.double()
    y = x
    if norm:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double()
    return turn(y, c, s, R, interleaved)


def bounds(x, w, c, s, R, interleaved, eps, dtype, norm=True, dz=None, w_dtype=torch.float32):
    """(bound of z) or (bound of z, of dx, of dw)."""
    v = 2.0 ** -24
    u = torch.finfo(dtype).eps / 2
    x = x.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    xh = x * r
    ww = torch.ones_like(x[0, 0, 0]) if w is None else w.double()
    z = forward(x, w, c, s, R, interleaved, eps, norm)
    bz = u * z.abs() + 32 * v * sizes(xh * ww, c, s, R, interleaved)
    if dz is None:
        return bz
    dz = dz.double()
    g, G = turn(dz, c, -s, R, interleaved), sizes(dz, c, s, R, interleaved)
    gw, Gw = g * ww, G * ww.abs()
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True)) if norm else gw
    bx = u * dx.abs() + 96 * v * r * (Gw + (xh.abs() * (Gw * xh.abs()).mean(-1, keepdim=True) if norm else 0.0))
    n = x.numel() // x.shape[-1]
    dw = (g * xh).flatten(0, -2).sum(0)
    bw = torch.finfo(w_dtype).eps / 2 * dw.abs() + (32 + n) * v * (G * xh.abs()).flatten(0, -2).sum(0)
    return bz, bx, bw
