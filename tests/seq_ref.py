"""Float64 definitions of layer norm, dropout and dot-product attention, with bounds on how far a kernel that
works in fp32 (and stores fp32 or bf16) may be from them.

The bounds follow from the arithmetic: a sum of n terms taken in fp32 is off by at most K * U * sum |terms| with K
the longest chain of roundings a term goes through (far below n for a sum over lanes and tiles), a stored value by
half a step of its type on top.  U = 2^-24 is half a step of fp32.
"""
import math

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, bound, what):
    """|got - want| <= bound element by element; both finite in the same places."""
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    both = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), both), f"{what}: finite in other places"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    bad = both & ~((got - want).abs() <= bound)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[i]:.9g} want {want[i]:.9g} "
                             f"bound {bound[i]:.3g}")


# ---- layer norm ----------------------------------------------------------------------------------------

def layer_norm(x, weights, eps, dy=None, skip=None):
    """{y, mean, rstd[, dx, dw]} and the same keys' bounds for fp32 results, in float64."""
    x = x.double().cpu()
    w = torch.stack([torch.ones(x.shape[1]), torch.zeros(x.shape[1])], 1).double() if weights is None else weights.double().cpu()
    n, c = x.shape
    k = c / 256 + 64  # longest chain: the elements of one lane (a row is shared by 16 lanes up to 256 elements), then the lanes
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = d * rstd
    e_mean = k * U * x.abs().mean(1, keepdim=True)
    e_d = e_mean + U * d.abs()
    # d(var) = mean 2 d e_d + k U var; rstd is half as sensitive, relative to var + eps
    rel_rstd = ((d.abs() * e_d).mean(1, keepdim=True) + e_mean ** 2 + k * U * var) / (var + eps) + 4 * U
    e_xhat = rstd * e_d + xhat.abs() * (rel_rstd + 2 * U)
    val = {"y": xhat * w[:, 0] + w[:, 1], "mean": mean, "rstd": rstd}
    bnd = {"y": w[:, 0].abs() * e_xhat + 3 * U * ((xhat * w[:, 0]).abs() + w[:, 1].abs()), "mean": e_mean + U * mean.abs(),
           "rstd": rstd * rel_rstd}
    if dy is not None:
        dy = dy.double().cpu()
        g = dy * w[:, 0]
        m0, m1 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
        dx = rstd * (g - m0 - xhat * m1)
        size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
        by_xhat = rstd * (e_xhat * m1.abs() + xhat.abs() * (g.abs() * e_xhat).mean(1, keepdim=True))
        val["dx"], bnd["dx"] = dx, by_xhat + size * (rel_rstd + (k + 8) * U)
        if skip is not None:
            val["dx"] = dx + skip.double().cpu()
            bnd["dx"] = bnd["dx"] + U * (dx.abs() + skip.double().cpu().abs())
        chain = n / 512 + 64  # rows of one workgroup's group, the groups of a workgroup
        val["dw"] = torch.stack([(dy * xhat).sum(0), dy.sum(0)], 1)
        bnd["dw"] = torch.stack([(dy.abs() * e_xhat).sum(0) + chain * U * (dy * xhat).abs().sum(0), chain * U * dy.abs().sum(0)], 1)
    return val, bnd


# ---- dropout -------------------------------------------------------------------------------------------

def philox4x32_10(counter, key):
    """counter [n, 4], key (2,) of 32-bit words -> [n, 4] (Salmon, Moraes, Dror, Shaw 2011), numpy uint64."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    m = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1)


def dropout_numbers(n, seed, offset, first=0):
    """The 32-bit numbers of the elements [first, first + n); first is a multiple of 8."""
    blocks = np.arange(first // 8, first // 8 + (n + 7) // 8, dtype=np.uint64)
    out = 0
    for f in (0, 1):
        ctr = np.stack([blocks & np.uint64(0xFFFFFFFF), (blocks >> np.uint64(32)) + np.uint64(f << 31),
                        np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)], 1)
        words = philox4x32_10(ctr, (seed & 0xFFFFFFFF, seed >> 32))
        halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)
        out = out * np.uint64(65536) + halves if f else halves
    return out[:n]


def dropout_kept(rows, channels, p, seed, offset):
    return torch.from_numpy(dropout_numbers(rows * channels, seed, offset) >= np.uint64(round(p * 2 ** 32))).reshape(rows, channels)


# ---- attention -----------------------------------------------------------------------------------------

def attention(q, k, v, lens_q, lens_k, hq, hk, d, scale, causal, dtype, dout=None):
    """Values and bounds {out, lse[, dq, dk, dv]} for packed q [tq, hq*d], k, v [tk, hk*d] in float64."""
    q, k, v = (t.double().cpu().reshape(t.shape[0], -1, d) for t in (q, k, v))
    tq, tk = q.shape[0], k.shape[0]
    step = half_step(torch.bfloat16) if dtype == torch.bfloat16 else 0.0   # of weights rounded for a product
    store = half_step(dtype)
    val = {"out": torch.zeros(tq, hq, d).double(), "lse": torch.zeros(tq, hq).double()}
    if dout is not None:
        dout = dout.double().cpu().reshape(tq, hq, d)
        val.update(dq=torch.zeros(tq, hq, d).double(), dk=torch.zeros(tk, hk, d).double(), dv=torch.zeros(tk, hk, d).double())
    bnd = {n: torch.zeros_like(t) for n, t in val.items()}
    bq = bk = 0
    for nq, nk in zip(lens_q, lens_k):
        rq, rk = slice(bq, bq + nq), slice(bk, bk + nk)
        bq, bk = bq + nq, bk + nk
        if nq == 0:
            continue
        seen = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            seen = seen.tril(nk - nq)
        some = seen.any(1)
        for h in range(hq):
            kv = h // (hq // hk)
            qh, kh, vh = q[rq, h], k[rk, kv], v[rk, kv]

            def dot(a, b):  # a @ b with what is hidden kept out, whatever it holds
                return torch.where(seen, a @ b, 0.0)

            s = dot(qh, kh.T) * scale
            lse = torch.where(some, torch.logsumexp(s.masked_fill(~seen, -math.inf), 1), torch.tensor(-math.inf).double())
            p = torch.where(seen, torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
            fin = lambda t: torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731  for the bounds only

            def mix(w, x):  # sum over keys of w x, only over seen keys
                if torch.isfinite(x).all() and torch.isfinite(w).all():
                    return w @ x
                return torch.stack([sum((w[i, j] * x[j] for j in range(nk) if seen[i, j]), torch.zeros(d).double()) for i in range(nq)])

            out = mix(p, vh)
            # a score is off by (d/16 + 8) roundings of its terms, its exponent by a few roundings of |s| and |lse|: relative error of a weight
            e_w = (d / 16 + 8) * U * scale * fin(dot(qh.abs(), kh.abs().T)) + 8 * U * (s.abs() + fin(lse).abs()[:, None] + 12.0)
            e_w = fin(e_w)
            chain = (nk / 32 + 64) * U
            e_row = fin((p * e_w).sum(1, keepdim=True))  # of the sum of weights
            e_out = fin((p * (e_w + e_row + step + chain)) @ fin(vh).abs())
            val["out"][rq, h], bnd["out"][rq, h] = out, e_out + store * fin(out).abs()
            val["lse"][rq, h] = lse
            bnd["lse"][rq, h] = e_row[:, 0] + chain + 4 * U * (fin(lse).abs() + 1)
            if dout is None:
                continue
            do = dout[rq, h]
            delta = torch.where(some, (do * out).sum(1), 0.0)[:, None]
            dp = dot(do, vh.T)
            ds = torch.where(seen, p * (dp - delta), 0.0)
            e_p = e_w + e_row + chain + 8 * U * fin(lse).abs()[:, None]
            e_delta = (fin(do).abs() * (e_out + store * fin(out).abs())).sum(1, keepdim=True) + (d / 8 + 8) * U * fin(do * out).abs().sum(1, keepdim=True)
            e_dp = (d / 16 + 8) * U * fin(dot(do.abs(), vh.abs().T))
            e_ds = fin(p * (e_dp + e_delta) + ds.abs() * (e_p + step + 4 * U))
            # the delta of a weight's own error acts on dP - delta as a whole
            chain_q = (nq / 32 + 64) * U
            seen_t = seen.T

            def mix_t(w, x):  # sum over queries
                if torch.isfinite(x).all() and torch.isfinite(w).all():
                    return w.T @ x
                return torch.stack([sum((w[i, j] * x[i] for i in range(nq) if seen_t[j, i]), torch.zeros(d).double()) for j in range(nk)])

            dq = mix(ds, kh) * scale
            val["dq"][rq, h], bnd["dq"][rq, h] = dq, scale * ((e_ds + chain * fin(ds).abs()) @ fin(kh).abs()) + (store + U) * fin(dq).abs()
            if nk:
                val["dk"][rk, kv] += mix_t(ds, qh) * scale
                bnd["dk"][rk, kv] += scale * ((e_ds + chain_q * fin(ds).abs()).T @ fin(qh).abs())
                val["dv"][rk, kv] += mix_t(p, do)
                bnd["dv"][rk, kv] += fin(p * (e_p + step + chain_q)).T @ fin(do).abs()
    if dout is not None:
        for n in ("dk", "dv"):
            bnd[n] = bnd[n] + (store + (hq // hk) * 2 * U) * torch.nan_to_num(val[n], nan=0.0, posinf=0.0, neginf=0.0).abs()
    flat = lambda t: t if t.dim() == 2 else t.reshape(t.shape[0], -1)  # noqa: E731
    # an absolute floor for what underflows: the smallest normal number of fp32, some thousands of them added
    return {n: flat(t) for n, t in val.items()}, {n: flat(t) + 1e-34 for n, t in bnd.items()}
