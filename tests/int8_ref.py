"""Serving in 8 bits by plain numpy: the quantizer's f32 steps as include/hy_int8.h gives them, and
what they are applied to in 64 bits."""
import numpy as np

import paged_ref as R
from paged_ref import F32, Pool

f32 = np.float32


def scale(big):
    """d and 1 / d of groups whose largest magnitudes are given (f32 arrays)."""
    big = np.asarray(big, f32)
    with np.errstate(all="ignore"):
        d = big / f32(127)
        d = np.where(~np.isfinite(big), f32(np.nan), np.where(d < f32(2.0 ** -126), f32(0), d)).astype(f32)
        inv = np.where(d > 0, f32(1) / d, f32(0)).astype(f32)
    return d, inv


def largest(x, axis):
    """Largest magnitude, NaN if there is one."""
    with np.errstate(invalid="ignore"):
        return np.abs(x).max(axis=axis)  # max hands NaN on


def codes(x, inv):
    """Codes of f32 values, inv 1 / d (0: all 0)."""
    with np.errstate(all="ignore"):
        q = np.rint((x.astype(f32) * inv).astype(f32))
        return np.where(inv == 0, 0, q).astype(np.int8)


def quantize(x):
    """Codes and scales of the rows of x."""
    d, inv = scale(largest(x.astype(f32), -1))
    return codes(x, inv[..., None]), d


def gemm(xq, xs, wq, ws, resid=None):
    """hy_gemm_i8, each rounding as the header gives them (sums below 2^53 are exact in 64-bit floats)."""
    acc = (xq.astype(np.float64) @ wq.astype(np.float64).T).astype(f32)
    with np.errstate(all="ignore"):
        y = (acc * xs[:, None]).astype(f32) * ws
        return y if resid is None else y + resid


class PoolI8:
    """A pool of codes k, v (shapes as paged_ref.Pool) with scales ks, vs [page][kv head][block], every
    position's code and every scale `fill`."""

    def __init__(self, n_pages, page, nkv, hd, block, order="head", fill=0, scale_fill=1.0):
        self.n_pages, self.page, self.nkv, self.hd, self.block, self.order = n_pages, page, nkv, hd, block, order
        shape = (n_pages, nkv, page, hd) if order == "head" else (n_pages, page, nkv, hd)
        self.k, self.v = np.full(shape, fill, np.int8), np.full(shape, fill, np.int8)
        self.ks = np.full((n_pages, nkv, page // block), scale_fill, f32)
        self.vs = self.ks.copy()

    def strides(self):
        return Pool.strides(self)

    def values(self):
        """A paged_ref.Pool of what is held, in 64 bits."""
        p = Pool(self.n_pages, self.page, self.nkv, self.hd, F32, self.order)
        with np.errstate(all="ignore"):
            for name, a, s in (("k", self.k, self.ks), ("v", self.v, self.vs)):
                s = np.repeat(s, self.block, axis=2).astype(np.float64)  # [page][kv head][position]
                s = np.where(np.isinf(s), np.nan, s)
                s = s[..., None] if self.order == "head" else s.transpose(0, 2, 1)[..., None]
                setattr(p, name, a.astype(np.float64) * s)
        return p

    def write(self, y, slots, which):
        """Rows y [n][nkv][hd] f32 of one run after another at their slots, into "k" or "v"."""
        a, sc = getattr(self, which), getattr(self, which + "s")
        i = 0
        while i < len(slots):
            n, s = 1, int(slots[i])
            while i + n < len(slots) and slots[i + n] == s + n and (s + n) % self.block:
                n += 1
            p, at = divmod(s, self.page)
            b, off = divmod(at, self.block)
            for g in range(self.nkv):
                rows = y[i:i + n, g].astype(f32)
                old = f32(0) if off == 0 else sc[p, g, b]
                d, inv = scale(largest(rows, (0, 1)))
                grows = not (old >= d or np.isnan(old))
                if not grows:
                    d = old
                    inv = f32(1) / old if old >= f32(2.0 ** -126) and np.isfinite(old) else f32(0)
                for o in range(self.block):
                    cell = (p, g, b * self.block + o) if self.order == "head" else (p, b * self.block + o, g)
                    if off <= o < off + n:
                        a[cell] = codes(rows[o - off], inv)
                    elif off == 0:
                        a[cell] = 0
                    elif grows:
                        a[cell] = codes(a[cell], f32(old / d) if d > 0 else f32(0))
                if grows or off == 0:
                    sc[p, g, b] = d
            i += n


def small_products(q, pool, q_start, kv_len, table, scale, seen=None):
    """What an output may be off because a weight times its value's scale is far below the row's largest, [rows]
    [nh].  Such products are taken to 2^-31 of the largest, M = max_j p_j vs_j, whatever they are (a code of 0 where
    the weight lies leaves nothing else in an output): with codes up to 127, n keys add n 127 2^-31 M."""
    p = PoolI8(pool.n_pages, pool.page, pool.nkv, 1, pool.block, "head", fill=1)
    p.vs = pool.vs
    T, nh, hd = q.shape
    out = np.zeros((T, nh))
    vals, ones = pool.values(), p.values()
    cap = table.shape[1] * pool.page
    for r in range(len(kv_len)):
        kv = min(max(kv_len[r], 0), cap)
        js = np.array([j for j in range(kv) if 0 <= table[r, j // pool.page] < pool.n_pages], np.int64)
        if not len(js):
            continue
        pg, at = table[r, js // pool.page], js % pool.page
        k = np.stack([vals.at(vals.k, a, b) for a, b in zip(pg, at)])
        sv = ones.v[pg, :, at, 0]
        for t in range(q_start[r], q_start[r + 1]):
            end = min(kv - (q_start[r + 1] - t) + 1 if seen is None else seen[t], kv)
            vis = js < end
            if not vis.any():
                continue
            for h in range(nh):
                g = h // (nh // pool.nkv)
                s = k[vis, g] @ q[t, h].astype(np.float64) * scale
                e = np.exp(s - s.max())
                out[t, h] = vis.sum() * 127 * 2.0 ** -31 * (e / e.sum() * sv[vis, g]).max()
    return out


def check_attention(got, q, pool, q_start, kv_len, table, scale, seen=None, sentinel=-3.0):
    """As the paged attention's check: element by element, then normwise."""
    values = pool.values()
    want, dot, pv = R.attention(q, values, q_start, kv_len, table, scale, seen)
    nobody = np.isnan(want).all(axis=(1, 2))
    assert (got[nobody] == sentinel).all()
    live = ~nobody
    assert np.isfinite(got[live]).all()
    off = np.abs(got - want)
    bound = R.attention_bound(dot, pv, pool.hd, max(1, int(np.max(kv_len, initial=0))))
    if not (off[live] <= bound[live]).all():
        bound = bound + small_products(q, pool, q_start, kv_len, table, scale, seen)[..., None]
    assert (off[live] <= bound[live]).all(), float((off[live] / np.maximum(bound[live], 1e-300)).max())
    ref = want[live]
    if np.linalg.norm(ref):
        S = dot[live].max()
        tol = 2 * R.EPS32 * (2 * (np.sqrt(pool.hd) + 4) * max(S, 1.0) + 8)
        assert np.linalg.norm(off[live]) <= tol * np.linalg.norm(ref)
    return want
