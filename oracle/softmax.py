"""Softmax attention in float64, one pair of tokens at a time in the formulas, and how far a kernel may be off.

The bounds follow from the roundings that the kernels make, worst case, element by element.  u is half a step of the element
type relative to the value (``torch.finfo(t).eps / 2``), w the same of float32.

* score: a sum of K products in float32, (K + 8) w scale sum_d |q_d k_d|; the cap's tanh and the bias a few w of their size;
  the scale to the base 2 a w of the score.  The exponential turns an absolute error of the score into a relative one of p, and so
  does the sum: twice the largest of the row, and (n + 16) w for n terms of the sum and the exponentials themselves: ``rel``.
  The tanh of a cap is off by 16 w, of itself where the cap is above 1024 (CAP_NEAR of the kernels), else of 1.
* o: the products take p rounded to the element type (u), o is rounded once: u |o| + (u + rel + n w) sum_j p |v|.
* dv: the same with do in place of v, summed over rows (and heads).
* delta = do . o from o to 2^-15 (2-byte elements: o and what its rounding left, in 2^-8 of the last place): sum_d |do_d| err(o_d)
  with that in place of the u |o|, and V w sum |do o|;  dp: V w sum_d |do_d v_d|.
* ds = p (dp - delta) (1 - tanh^2), rounded to the element type: (u + rel) |ds| + p (err(dp) + err(delta)); the factor of the cap has
  an absolute error of 8 w.
* dq, dk: u |dq| + scale sum err(ds) |k| + n w scale sum |ds k|.
Products of the element type are exact in float32; w n covers the order of the sums."""
import math

import torch


def _rel(u_sum, smax, K, n, cap):
    w = 2.0 ** -24
    return 2 * ((K + 8) * w * u_sum + (6 * smax + 16 * (cap if cap <= 1024 else smax)) * w) + (n + 16) * w


def head(q, k, v, scale, causal=True, cap=0.0, slope=0.0, prefix=0, do=None, dtype=torch.float64, low=True):
    """One head of one sequence: q [n, K], k [m, K], v [m, V], the last of the n queries at the last of the m keys.
    Returns o and its bound; with do also (dq, dk, dv) and their bounds (to be rounded and summed by the caller: the bounds
    leave out the final rounding of dk and dv).  low=False: delta from o as it is rounded."""
    w = 2.0 ** -24
    u = 2.0 ** -24 if dtype in (torch.float32, torch.float64) else torch.finfo(dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    n, m, K, V = q.shape[0], k.shape[0], q.shape[1], v.shape[1]
    i, j = torch.arange(m - n, m, device=q.device)[:, None], torch.arange(m, device=q.device)[None, :]
    ok = (j <= i) | (j < prefix) if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
    x = scale * (q @ k.T)
    th = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    s = (cap * th if cap else x) - slope * (i - j).abs()
    s = torch.where(ok, s, -math.inf)
    p = torch.softmax(s, 1)
    p = torch.where(ok, p, torch.zeros_like(p))
    sums = torch.where(ok, abs(scale) * (q.abs() @ k.abs().T), torch.zeros_like(x)).amax(1, keepdim=True)
    smax = torch.where(ok, s.abs() + slope * (i - j).abs(), torch.zeros_like(x)).amax(1, keepdim=True)
    rel = _rel(sums, smax, K, m, cap)
    o = p @ v
    err_o = u * o.abs() + (u + rel + m * w) * (p @ v.abs())
    if do is None:
        return o, err_o
    do = do.double()
    dp, delta = do @ v.T, (do * o).sum(1, keepdim=True)
    err_dp = V * w * (do.abs() @ v.abs().T)
    err_delta = (do.abs() * (err_o - (u - min(u, 2.0 ** -15) if low else 0.0) * o.abs())).sum(1, keepdim=True) + V * w * (do * o).abs().sum(1, keepdim=True)
    fac = 1 - th * th
    ds = p * (dp - delta) * fac
    err_ds = (u + rel) * ds.abs() + p * (err_dp + err_delta) + (8 * w * p * (dp - delta).abs() if cap else 0.0)
    dq, dk, dv = scale * (ds @ k), scale * (ds.T @ q), p.T @ do
    tot = m * w
    err_dq = u * dq.abs() + abs(scale) * (err_ds @ k.abs()) + tot * abs(scale) * (ds.abs() @ k.abs())
    err_dk = abs(scale) * (err_ds.T @ q.abs()) + tot * abs(scale) * (ds.abs().T @ q.abs())
    err_dv = (p * (u + rel + tot)).T @ do.abs()
    return o, err_o, (dq, dk, dv), (err_dq, err_dk, err_dv)


def attn(q, k, v, scale=None, causal=True, softcap=0.0, slopes=None, prefix_lens=None, cu=None, do=None, low=True):
    """[B, T, H, D], in the type the kernel is given.  Returns {name: (value, bound)} for o and, with do, dq, dk, dv."""
    B, T, HQ, K = q.shape
    HKV, G = k.shape[2], q.shape[2] // k.shape[2]
    scale = K ** -0.5 if scale is None else scale
    z = lambda x, c=None: torch.zeros(*x.shape[:3], c or x.shape[3], dtype=torch.float64, device=x.device)
    out = {"o": (z(q, v.shape[3]), z(q, v.shape[3]))}
    if do is not None:
        out.update(dq=(z(q), z(q)), dk=(z(k), z(k)), dv=(z(v), z(v)))
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, cu[n], cu[n + 1]) for n in range(len(cu) - 1)]
    for n, (b, t0, t1) in enumerate(spans):
        if t1 == t0:
            continue
        for h in range(HQ):
            at, kv = (b, slice(t0, t1), h), (b, slice(t0, t1), h // G)
            prefix = 0 if prefix_lens is None else min(max(int(prefix_lens[n]), 0), t1 - t0)
            r = head(q[at], k[kv], v[kv], scale, causal, softcap, 0.0 if slopes is None else float(slopes[h]), prefix,
                     None if do is None else do[at], q.dtype, low)
            out["o"][0][at], out["o"][1][at] = r[0], r[1]
            if do is not None:
                for name, where, x, e in zip(("dq", "dk", "dv"), (at, kv, kv), r[2], r[3]):
                    out[name][0][where] += x
                    out[name][1][where] += e
    if do is not None:
        u = torch.finfo(q.dtype).eps / 2
        for name in ("dk", "dv"):
            out[name][1].add_(out[name][0].abs() * (u + T * G * 2.0 ** -24))
    return out


def check(got, want, what=""):
    """got: tensor; want: (value, bound).  The float64 sums of the oracle are exact beside the bounds."""
    ref, bound = want
    x = got.detach().to(ref.device).double()
    assert x.shape == ref.shape, (what, x.shape, ref.shape)
    assert torch.isfinite(x).all(), f"{what}: not finite"
    off = (x - ref).abs() - bound - 1e-30
    worst = int(off.argmax())
    assert off.max() <= 0, (f"{what}: off by {(x - ref).abs().flatten()[worst]:.3e} where {bound.flatten()[worst]:.3e} is allowed "
                            f"(element {worst} of {tuple(x.shape)}, {int((off > 0).sum())} beyond)")
