"""Attention with shaped scores or a shared prefix from its definition in 64 bits, and how far the kernels may be from it."""
import math

import torch

D = 128
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative


def rand(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def reference(q, k, v, first, scale, cap=0.0, slopes=None, window=0, begin=None, end=None, prefix=None):
    """q [S, B, Hq, D]; k, v [B, Hkv, rows, D]; first: own row of each sequence's first query; begin, end: per sequence a
    list over own rows, or None; prefix: (k, v) [Hkv, rows, D] or None.  Returns out and lse in 64 bits and the bound on
    the error of either: every operand rounded half a step once, sums and scores with the errors of 32-bit arithmetic."""
    s, b, hq, _ = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    half, u = HALF[q.dtype], 2.0 ** -24
    out = torch.zeros((s, b, hq, D), dtype=torch.float64, device=q.device)
    lse = torch.full((s, b, hq), -math.inf, dtype=torch.float64, device=q.device)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    n_prefix = 0 if prefix is None else prefix[0].shape[1]
    for i in range(b):
        for t in range(s):
            own = first[i] + t
            p = n_prefix + own
            lo = 0 if begin is None else int(begin[i][own])
            hi = p + 1 if end is None else min(int(end[i][own]), k.shape[2])
            if window:
                lo = max(lo, p + 1 - window)
            if lo >= hi:
                continue
            n = hi - lo
            j = torch.arange(lo, hi, device=q.device, dtype=torch.float64)
            for h in range(hkv):
                if n_prefix:
                    kk, vv = (torch.cat([a[h, lo:hi], c[i, h, max(0, lo - n_prefix):hi - n_prefix]]).double()
                              for a, c in ((prefix[0], k), (prefix[1], v)))
                else:
                    kk, vv = k[i, h, lo:hi].double(), v[i, h, lo:hi].double()
                rows = slice(h * group, (h + 1) * group)
                qq = q[t, i, rows].double()
                x = qq @ kk.T * scale
                err = (D + 4) * u * float((qq.abs() @ kk.abs().T).max()) * abs(scale)
                if cap:
                    x = cap * torch.tanh(x / cap)
                    err += 16 * u * cap
                if slopes is not None:
                    far = slopes[rows].double()[:, None] * (p - j).abs()
                    x = x - far
                    err += 4 * u * float(far.abs().max())
                err += 4 * u * float(x.abs().max())
                total = torch.logsumexp(x, dim=-1)
                w = torch.exp(x - total[:, None])
                y, size = w @ vv, w @ vv.abs()
                out[t, i, rows], lse[t, i, rows] = y, total
                tol = half * (y.abs() + (1 + 2 * half) * size) + (2 * err + (n + 8) * u) * size
                if q.dtype == torch.float16:   # weights below 2^-14 of the row's reference, and results, have absolute steps
                    tol = tol + n * 2.0 ** -25 * vv.abs().max() + 2.0 ** -25
                out_tol[t, i, rows] = tol
                lse_tol[t, i, rows] = err + (n + 8) * u + 4 * u * total.abs()
    return out, lse, out_tol, lse_tol


def check(got, got_lse, want, what=""):
    out, lse, out_tol, lse_tol = want
    err = (got.double() - out).abs()
    assert not torch.isnan(got).any(), f"{what}: NaN in the output"
    worst = float((err / out_tol.clamp_min(1e-30)).max())
    assert (err <= out_tol).all(), f"{what}: {worst:.2f} of the bound"
    if got_lse is not None:
        seen = lse > -math.inf
        assert torch.equal(got_lse.double()[~seen], lse[~seen]), f"{what}: lse of rows that see nothing"
        off = (got_lse.double() - lse).abs()[seen]
        assert (off <= lse_tol[seen]).all(), f"{what}: lse off by {float(off.max()):.2e}"
    return worst
