"""Paged serving in 64 bits by plain numpy loops, and the inputs its tests share."""
import numpy as np

F32, F16, BF16 = 0, 1, 30
EPS32 = 2.0 ** -24                                   # half a step of 1.0
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def to_bf16(x):
    """f32 -> bf16 bits (uint16), to nearest, ties to even; NaN stays NaN."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def encode(x, wtype):
    """f32 values in a cache type's storage (bf16 as uint16)."""
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float32) if wtype == F32 else np.asarray(x, np.float32).astype(np.float16) \
            if wtype == F16 else to_bf16(x)


def decode(a, wtype):
    """Stored values as float64."""
    if wtype == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


class Pool:
    """A pool of pages as numpy storage k, v [n_pages][nkv][page][hd], or [n_pages][page][nkv][hd]
    for order "token"; every position filled with `fill` until written."""

    def __init__(self, n_pages, page, nkv, hd, wtype, order="head", fill=0.0):
        self.n_pages, self.page, self.nkv, self.hd, self.wtype, self.order = n_pages, page, nkv, hd, wtype, order
        shape = (n_pages, nkv, page, hd) if order == "head" else (n_pages, page, nkv, hd)
        self.k = encode(np.full(shape, fill, np.float32), wtype)
        self.v = self.k.copy()

    def strides(self):
        if self.order == "head":
            return (self.nkv * self.page * self.hd, self.page * self.hd, self.hd)
        return (self.nkv * self.page * self.hd, self.hd, self.nkv * self.hd)

    def at(self, a, p, i):
        """Storage of page p, position i of a (self.k or self.v): [nkv][hd]."""
        return a[p, :, i] if self.order == "head" else a[p, i]

    def put(self, a, p, i, x):
        if self.order == "head":
            a[p, :, i] = x
        else:
            a[p, i] = x


def attention(q, pool, q_start, kv_len, table, scale, seen=None, n_pages=None):
    """out [rows][nh][hd] float64 (NaN rows where a row belongs to nobody), the largest
    absolute score sum per row and head, and sum p |v|."""
    T, nh, hd = q.shape
    G = nh // pool.nkv
    n_pages = pool.n_pages if n_pages is None else n_pages
    out = np.full((T, nh, hd), np.nan)
    dot = np.zeros((T, nh))
    pv = np.zeros((T, nh, hd))
    cap = table.shape[1] * pool.page
    for r in range(len(kv_len)):
        kv, s0, s1 = min(max(kv_len[r], 0), cap), q_start[r], q_start[r + 1]
        keys = [(j, table[r, j // pool.page], j % pool.page) for j in range(kv)]
        keys = [(j, p, i) for j, p, i in keys if 0 <= p < n_pages]
        js = np.array([j for j, _, _ in keys], np.int64)
        if keys:
            k = np.stack([decode(pool.at(pool.k, p, i), pool.wtype) for _, p, i in keys])
            v = np.stack([decode(pool.at(pool.v, p, i), pool.wtype) for _, p, i in keys])
        for t in range(s0, s1):
            end = min(kv - (s1 - t) + 1 if seen is None else seen[t], kv)
            vis = js < end
            for h in range(nh):
                if not vis.any():
                    out[t, h] = 0.0
                    continue
                kk, vv = k[vis, h // G], v[vis, h // G]
                x = q[t, h].astype(np.float64)
                s = kk @ x * scale
                dot[t, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ vv
                pv[t, h] = p @ np.abs(vv)
    return out, dot, pv


def attention_bound(dot, pv, hd, keys):
    """How far an f32 evaluation may be off: a score is a sum of hd products, each and every
    partial sum rounded (or cut) once, (hd + 4) half steps of the sum of magnitudes with
    the operands' scaling and 22-bit operand pieces (4 half steps) among them; an error d of
    the scores changes p by 2 d relative; sums over the keys add one half step per key, the
    exponential and the division 8 more."""
    d = (hd + 8) * 2 * EPS32 * dot
    return (2 * d + (keys + 16) * 2 * EPS32)[..., None] * pv


def softmax64(x):
    w = np.exp(x - x.max())
    return w / w.sum()


def plan(cached, new, held, table, free, n_free, n_rows, page, n_pages):
    """hy_paged_plan request by request."""
    R, max_pages = table.shape
    table, free = table.copy(), free.copy()
    n = min(max(int(n_free), 0), n_pages)
    q_start, status, want = [0], [], []
    at = 0
    for r in range(R):
        c, a, h = int(cached[r]), int(new[r]), int(held[r])
        w = -(-(c + a) // page)
        st = 3 if c < 0 or a < 0 or at + a > n_rows or h < 0 or h > max_pages else 2 if w > max_pages else 0
        status.append(st)
        want.append(w)
        at += a if 0 <= a <= n_rows else 0
        q_start.append(min(at, n_rows))
    for r in range(R):
        if status[r] == 0:
            for k in range(want[r], held[r]):
                if n < n_pages:
                    free[n] = table[r, k]
                    n += 1
    held_out, gone = np.array(held), False
    for r in range(R):
        if status[r]:
            continue
        need = max(0, want[r] - int(held[r]))
        gone = gone or need > n
        if need and gone:
            status[r] = 1
            continue
        for k in range(need):
            n -= 1
            table[r, held[r] + k] = free[n]
        held_out[r] = want[r]
    pos, slot = np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int32)
    for r in range(R):
        for i in range(q_start[r + 1] - q_start[r] if status[r] == 0 else 0):
            p = int(cached[r]) + i
            pg = int(table[r, p // page])
            pos[q_start[r] + i] = p
            if 0 <= pg < n_pages:
                slot[q_start[r] + i] = pg * page + p % page
    kv = [int(c) + int(a) if s == 0 else 0 for c, a, s in zip(cached, new, status)]
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(table=table, held_out=i32(held_out), free=free, n_free_out=i32([n]), q_start=i32(q_start),
                kv_len=i32(kv), positions=pos, slots=slot, status=i32(status))


def verify(logits, draft, ids, q_start, temp, u_accept, u_sample, max_new):
    """hy_verify_drafts token by token.  Also the smallest distance of a decision from its
    border, relative (decisions nearer than a 64-bit sum's error prove nothing)."""
    R, V = len(q_start) - 1, logits.shape[1]
    accepted, tokens, margin = [], np.full((R, max_new), -1, np.int32), np.inf
    for r in range(R):
        rows = range(q_start[r], q_start[r + 1])
        if len(rows) == 0 or len(rows) > max_new:
            accepted.append(-1)
            continue
        n = 0
        for row in rows:
            l = logits[row].astype(np.float64)
            if np.isnan(l).any() or (l == np.inf).any() or (l == -np.inf).all():
                break
            x = int(ids[row + 1]) if row + 1 < q_start[r + 1] else None
            t = 1.0 if temp is None else float(temp[r])
            if not t > 0:
                tok = int(np.argmax(l))
                tokens[r, n] = tok
                if tok == x:
                    n += 1
                    continue
                break
            p = softmax64(l / t)
            rest = p
            if x is not None:
                q = np.zeros(V) if draft is None else draft[row].astype(np.float64)
                if draft is None and 0 <= x < V:
                    q[x] = 1.0
                if 0 <= x < V:
                    a, b = float(u_accept[row]) * q[x], p[x]
                    if a > 0 and b > 0:  # a zero decides exactly
                        margin = min(margin, abs(a - b) / b)
                    if a < b:
                        tokens[r, n] = x
                        n += 1
                        continue
                rest = np.where(p > q, p - q, 0.0) if draft is not None else np.where(q > 0, 0.0, p)
                if not rest.sum() > 0:
                    rest = p
            cdf = np.cumsum(rest)
            thr = float(u_sample[r]) * cdf[-1]
            over = np.nonzero(cdf > thr)[0]
            tokens[r, n] = over[0] if len(over) else np.nonzero(rest > 0)[0][-1]
            margin = min(margin, np.abs(cdf - thr).min() / cdf[-1])
            break
        accepted.append(n)
    return np.array(accepted, np.int32), tokens, margin
