"""Paged serving on the GPU against plain numpy in 64 bits (paged_ref.py): tables and slots,
the write of the cache, attention of ragged batches, the verification of drafts, and the
step that uses them together through the attention layer and the backbone."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from paged_ref import BF16, EPS32, F16, F32, Pool

pytestmark = pytest.mark.gpu


def dev(gpu, a, dtype=None):
    return gpu.Buf.from_array(np.ascontiguousarray(a, dtype))


# ------------------------------------------------------------------ tables and slots

class PlanBufs:
    """Device arrays of one hy_paged_plan call."""

    def __init__(self, gpu, cached, new, held, table, free, n_free, n_rows, page, n_pages):
        self.gpu, self.n_rows, self.page, self.n_pages = gpu, n_rows, page, n_pages
        self.R, self.max_pages = table.shape
        i32 = np.int32
        self.cached, self.new, self.held = dev(gpu, cached, i32), dev(gpu, new, i32), dev(gpu, held, i32)
        self.table, self.free, self.n_free = dev(gpu, table, i32), dev(gpu, free, i32), dev(gpu, [n_free], i32)
        self.held_out, self.n_free_out = dev(gpu, np.full(self.R, 77, i32)), dev(gpu, [77], i32)
        self.q_start, self.kv_len = dev(gpu, np.full(self.R + 1, 77, i32)), dev(gpu, np.full(self.R, 77, i32))
        self.status = dev(gpu, np.full(self.R, 77, i32))
        self.positions, self.slots = dev(gpu, np.full(n_rows, 77, i32)), dev(gpu, np.full(n_rows, 77, i32))

    def run(self, stream=None, in_place=False):
        self.gpu.paged_plan(self.cached, self.new, self.R, self.n_rows, self.page, self.max_pages, self.n_pages,
                            self.table, self.held, self.held if in_place else self.held_out, self.free, self.n_free,
                            self.n_free if in_place else self.n_free_out, self.q_start, self.kv_len, self.positions,
                            self.slots, self.status, stream)

    def check(self, want, in_place=False):
        for name, w in want.items():
            src = {"held_out": "held", "n_free_out": "n_free"}.get(name, name) if in_place else name
            np.testing.assert_array_equal(getattr(self, src).numpy(), w, err_msg=name)


def random_plan(rng, n_req, max_new, page, max_pages, spare, pad=0, hostile=False):
    cap = max_pages * page
    cached = rng.integers(0, cap, n_req)
    new = rng.integers(0, max_new + 1, n_req)
    ended = rng.random(n_req) < 0.15
    cached[ended] = new[ended] = 0
    new = np.minimum(new, cap - cached)
    held = np.minimum(-(-cached // page) + rng.integers(0, 3, n_req) * (rng.random(n_req) < 0.4), max_pages)
    held[ended] = rng.integers(0, max_pages + 1, ended.sum())
    total = int(held.sum())
    n_pages = total + spare
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n_req, max_pages), -7, np.int32)
    at = 0
    for r in range(n_req):
        table[r, :held[r]] = perm[at:at + held[r]]
        at += held[r]
    free = np.full(n_pages, -9, np.int32)
    free[:spare] = perm[total:]
    n_rows = int(new.sum()) + pad
    if hostile:  # lengths out of range, too long, pages that do not exist
        for r in range(0, n_req, 3):
            what = r % 5
            if what == 0:
                cached[r] = -1 - rng.integers(0, 5)
            elif what == 1:
                new[r] = -3
            elif what == 2:
                cached[r] = cap + 1
            elif what == 3:
                held[r] = max_pages + 2
            else:
                cached[r] = 2 ** 31 - 1
        table[rng.random(table.shape) < 0.1] = n_pages + 5
    return cached, new, held, table, free, spare, max(n_rows, 1), page, n_pages


@pytest.mark.parametrize("n_req,max_new,page,max_pages,spare,pad", [
    (1, 1, 16, 1, 3, 0), (1, 0, 8, 4, 0, 2), (8, 1, 16, 130, 20, 0), (5, 700, 16, 60, 200, 9), (63, 6, 8, 40, 30, 0),
    (64, 300, 32, 16, 5, 1), (65, 5, 4096, 3, 9, 0), (1000, 3, 16, 33, 100, 50), (4096, 4, 8, 9, 4000, 3),
    (17, 2000, 64, 70, 300, 17), (3000, 1, 128, 5, 0, 0), (40, 9, 8, 30, 2, 0)])
def test_plan(gpu, n_req, max_new, page, max_pages, spare, pad):
    rng = np.random.default_rng(n_req * 1000 + max_new)
    args = random_plan(rng, n_req, max_new, page, max_pages, spare, pad)
    want = R.plan(*args)
    b = PlanBufs(gpu, *args)
    b.run()
    b.check(want)
    b.run()  # the same inputs again: the same outputs
    b.check(want)
    c = PlanBufs(gpu, *args)
    c.run(in_place=True)
    c.check(want, in_place=True)


@pytest.mark.parametrize("n_req,n_rows", [(7, None), (200, None), (31, 5), (2000, 100)])
def test_plan_hostile_lengths(gpu, n_req, n_rows):
    """Requests with lengths out of range, too many rows, pages that do not exist: refused or
    without a slot, the others served."""
    rng = np.random.default_rng(n_req)
    args = list(random_plan(rng, n_req, 5, 16, 12, 50, 2, hostile=True))
    if n_rows is not None:
        args[6] = n_rows
    want = R.plan(*args)
    assert {0, 3} <= set(want["status"].tolist())
    b = PlanBufs(gpu, *args)
    b.run()
    b.check(want)


def test_plan_stack_counts_out_of_range(gpu):
    rng = np.random.default_rng(3)
    for n_free in (-5, 10 ** 6):
        args = list(random_plan(rng, 9, 4, 16, 12, 50))
        args[5] = n_free
        args[4] = np.arange(args[8], dtype=np.int32)
        b = PlanBufs(gpu, *args)
        b.run()
        b.check(R.plan(*args))


def test_plan_over_many_steps(gpu):
    """A server's life: requests grow, end and start; no page is ever in two places."""
    rng = np.random.default_rng(11)
    n_req, page, max_pages, n_pages = 24, 8, 20, 160
    held, table = np.zeros(n_req, np.int32), np.zeros((n_req, max_pages), np.int32)
    free, n_free, cached = rng.permutation(n_pages).astype(np.int32), n_pages, np.zeros(n_req, np.int64)
    for _ in range(25):
        new = rng.integers(0, 20, n_req)
        over = cached + new > page * max_pages
        cached[over | (rng.random(n_req) < 0.1)] = 0
        back = np.minimum(cached, rng.integers(0, 4, n_req))  # drafts that were not taken
        cached -= back
        args = (cached, new, held, table, free, n_free, int(new.sum()), page, n_pages)
        want = R.plan(*args)
        b = PlanBufs(gpu, *args)
        b.run()
        b.check(want)
        held, table, free, n_free = want["held_out"], want["table"], want["free"], int(want["n_free_out"][0])
        cached = np.where(want["status"] == 0, cached + new, cached)
        pages = [table[r, k] for r in range(n_req) for k in range(held[r])] + free[:n_free].tolist()
        assert sorted(pages) == list(range(n_pages))


# ------------------------------------------------------------------ the write of the cache

def upload(gpu, pool):
    return dev(gpu, pool.k), dev(gpu, pool.v)


def cache_of(gpu, pool, kb, vb, **kw):
    return gpu.PagedCache(kb, vb, pool.wtype, pool.n_pages, pool.page, pool.nkv, pool.hd,
                          pool.strides() if pool.order == "token" else (0, 0, 0), **kw)


def append_ref(qkv, nh, nkv, hd, positions, theta, cos, sin, qn, kn, eps):
    x = qkv.astype(np.float64).reshape(len(qkv), nh + 2 * nkv, hd)
    if cos is not None:
        c, s = cos[positions, ::2].astype(np.float64), sin[positions, ::2].astype(np.float64)
    elif theta:
        ang = positions[:, None].astype(np.float64) * float(np.float32(theta)) ** (-2.0 * np.arange(hd // 2) / hd)
        c, s = np.cos(ang), np.sin(ang)
    else:
        c, s = np.ones((len(qkv), hd // 2)), np.zeros((len(qkv), hd // 2))
    y = x[:, :nh + nkv].copy()
    y[..., ::2] = x[:, :nh + nkv, ::2] * c[:, None] - x[:, :nh + nkv, 1::2] * s[:, None]
    y[..., 1::2] = x[:, :nh + nkv, ::2] * s[:, None] + x[:, :nh + nkv, 1::2] * c[:, None]
    rms = 1.0 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    # the turn's own magnitude: what its f32 rounding is relative to
    mag = np.repeat(np.hypot(x[:, :nh + nkv, ::2], x[:, :nh + nkv, 1::2]), 2, axis=-1) * rms
    y = y * rms
    one = np.ones(hd)
    wq, wk = one if qn is None else qn.astype(np.float64), one if kn is None else kn.astype(np.float64)
    return y[:, :nh] * wq, y[:, nh:] * wk, x[:, nh + nkv:], mag[:, :nh] * np.abs(wq), mag[:, nh:] * np.abs(wk)


# f32 steps: sine and cosine off by 2 half steps and by the f32 angle's (|angle| <= pi:
# 4 half steps); a product each, their sum, rms (sum of hd squares in a tree, mean, eps, root,
# quotient: 16), two products: 32 half steps of the pair's magnitude
APPEND_TOL = 32 * EPS32


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,hd,page,mode,order,T,pad", [
    (32, 8, 128, 16, "theta", "head", 5, 0), (32, 8, 128, 64, "table", "head", 77, 3), (16, 4, 64, 8, "theta", "token", 33, 2),
    (5, 5, 64, 16, "none", "head", 9, 0), (20, 4, 128, 32, "theta", "token", 1, 4), (6, 1, 128, 4096, "table", "token", 300, 0)])
def test_append(gpu, wtype, nh, nkv, hd, page, mode, order, T, pad):
    rng = np.random.default_rng(T * 7 + wtype)
    n_rows = T + pad
    qkv = rng.standard_normal((n_rows, (nh + 2 * nkv) * hd)).astype(np.float32) * 3
    qkv[T:] = np.nan  # rows of nobody
    n_pages = (T + 40) // page + 2
    slots = np.full(n_rows, -1, np.int32)
    slots[:T] = rng.choice(n_pages * page, T, replace=False)
    if T > 8:
        slots[3] = n_pages * page + 5  # outside the pool: skipped
    positions = np.zeros(n_rows, np.int32)
    positions[:T] = rng.integers(0, 200000 if mode == "theta" else 500, T)
    n_pos, cos, sin = 0, None, None
    if mode == "table":
        n_pos = 500
        ang = rng.random((n_pos, hd // 2)) * 6
        cos = np.repeat(np.cos(ang), 2, axis=1).astype(np.float32)
        sin = np.repeat(np.sin(ang), 2, axis=1).astype(np.float32)
    if mode == "table" and T > 8:
        positions[5] = 500  # outside the tables: skipped
    qn = None if mode == "none" else (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    kn = None if mode == "none" else (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    pool = Pool(n_pages, page, nkv, hd, wtype, order, fill=7.0)
    kb, vb = upload(gpu, pool)
    q0 = np.full((n_rows, nh, hd), 5.0, np.float32)
    qb = dev(gpu, q0)
    opt = lambda a: None if a is None else dev(gpu, a)  # noqa: E731
    gpu.rope_qknorm_paged(dev(gpu, qkv), n_rows, nh, cache_of(gpu, pool, kb, vb), dev(gpu, positions),
                          dev(gpu, slots), 10000.0 if mode != "none" else 0.0, opt(cos), opt(sin), n_pos, opt(qn),
                          opt(kn), 1e-5, qb)
    live = [t for t in range(T) if 0 <= slots[t] < n_pages * page and not (mode == "table" and positions[t] >= n_pos)]
    assert len(live) >= T - 2
    q, k, v, qm, km = append_ref(qkv[live], nh, nkv, hd, positions[live], 1e4 if mode == "theta" else 0, cos, sin, qn,
                                 kn, 1e-5)
    got_q = qb.numpy()
    assert (np.abs(got_q[live] - q) <= APPEND_TOL * qm).all()
    dead = np.setdiff1d(np.arange(n_rows), live)
    np.testing.assert_array_equal(got_q[dead], q0[dead])
    gk, gv = kb.numpy(), vb.numpy()
    tiny = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}[wtype]
    untouched = np.ones((n_pages, page), bool)
    for i, t in enumerate(live):
        p, o = divmod(int(slots[t]), page)
        untouched[p, o] = False
        step = R.HALF_STEP[wtype]
        assert (np.abs(R.decode(pool.at(gk, p, o), wtype) - k[i]) <= APPEND_TOL * km[i] + step * np.abs(k[i]) * 1.01 + tiny).all()
        np.testing.assert_array_equal(pool.at(gv, p, o), R.encode(v[i].astype(np.float32), wtype))
    for p, o in np.argwhere(untouched):
        np.testing.assert_array_equal(pool.at(gk, p, o), pool.at(pool.k, p, o))
        np.testing.assert_array_equal(pool.at(gv, p, o), pool.at(pool.v, p, o))


# ------------------------------------------------------------------ attention

def make_batch(rng, lens, page, nkv, hd, wtype, order="head", extra_pages=2, k_std=1.0, fill=0.0):
    """lens: (kv, new) per request.  A pool whose used positions are random and whose other
    ones hold `fill`, tables over it, row starts."""
    need = [-(-max(kv, 0) // page) for kv, _ in lens]
    n_pages = sum(need) + extra_pages
    pool = Pool(n_pages, page, nkv, hd, wtype, order, fill)
    perm = rng.permutation(n_pages)
    width = max(max(need), 1)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
        for j in range(max(lens[r][0], 0)):
            p, i = table[r, j // page], j % page
            pool.put(pool.k, p, i, R.encode(rng.standard_normal((nkv, hd)).astype(np.float32) * k_std, wtype))
            pool.put(pool.v, p, i, R.encode(rng.standard_normal((nkv, hd)).astype(np.float32), wtype))
    q_start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
    kv_len = np.array([kv for kv, _ in lens], np.int32)
    return pool, table, q_start, kv_len


class Ws:
    """A workspace for one PagedBatch, filled with NaN."""

    def __init__(self, gpu, nh, cache, batch):
        self.n = gpu.paged_attention_ws(nh, cache, batch)
        self.b = dev(gpu, np.full(self.n // 4 + 1, np.nan, np.float32))


def attend(gpu, q, pool, q_start, kv_len, table, scale, seen=None, max_new=None, sentinel=-3.0, stream=None):
    n_rows, nh, hd = q.shape
    kb, vb = upload(gpu, pool)
    cache = cache_of(gpu, pool, kb, vb)
    new = int(np.diff(q_start).max())
    bufs = [dev(gpu, a, np.int32) for a in (q_start, kv_len, table)]
    batch = gpu.PagedBatch(len(kv_len), n_rows, table.shape[1], new if max_new is None else max_new, *bufs,
                           seen=None if seen is None else dev(gpu, seen, np.int32))
    out = dev(gpu, np.full(q.shape, sentinel, np.float32))
    ws = Ws(gpu, nh, cache, batch)
    gpu.paged_attention(dev(gpu, q), nh, cache, batch, scale, out, ws.b, ws.n, stream)
    return out.numpy()


def check_attention(got, q, pool, q_start, kv_len, table, scale, seen=None, sentinel=-3.0):
    want, dot, pv = R.attention(q, pool, q_start, kv_len, table, scale, seen)
    nobody = np.isnan(want).all(axis=(1, 2))
    assert (got[nobody] == sentinel).all()
    live = ~nobody
    assert np.isfinite(got[live]).all()
    bound = R.attention_bound(dot, pv, pool.hd, max(1, int(np.max(kv_len, initial=0))))
    off = np.abs(got - want)
    assert (off[live] <= bound[live]).all(), float((off[live] / np.maximum(bound[live], 1e-300)).max())
    # the roundings are independent: normwise an f32 evaluation stays near its own precision.
    # Scores of magnitude up to S carry (sqrt(hd) + 4) half steps of S, the output 8 more.
    ref = want[live]
    if np.linalg.norm(ref):
        S = dot[live].max()
        tol = 2 * EPS32 * (2 * (np.sqrt(pool.hd) + 4) * max(S, 1.0) + 8)
        assert np.linalg.norm(off[live]) <= tol * np.linalg.norm(ref)
    return want


LENS = {
    "one": [(1, 1)],
    "short": [(5, 1), (1, 1), (17, 1), (33, 1), (64, 1)],
    "decode": [(1000, 1), (3, 1), (777, 1), (64, 1), (1, 1), (2049, 1), (512, 1)],
    "draft": [(300, 5), (41, 3), (9, 9), (128, 6), (2, 2), (1025, 7)],
    "empty": [(0, 0), (40, 2), (0, 3), (10, 0), (7, 7), (0, 0)],
    "chunk": [(200, 130), (64, 64), (333, 77), (31, 31)],
    "mixed": [(500, 1), (260, 200), (90, 4), (150, 150), (1, 1), (700, 33)],
    "fewer": [(3, 9), (20, 45)],  # fewer keys than rows: the first rows see nothing
}


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", LENS)
def test_attention_lengths(gpu, wtype, lens):
    rng = np.random.default_rng(wtype + len(lens))
    nh, nkv, hd, page = 8, 2, 128, 16
    pool, table, q_start, kv_len = make_batch(rng, LENS[lens], page, nkv, hd, wtype)
    pad = 3 if lens != "one" else 0
    q = rng.standard_normal((q_start[-1] + pad, nh, hd)).astype(np.float32) * 2
    args = (q, pool, q_start, kv_len, table, hd ** -0.5)
    check_attention(attend(gpu, *args), *args)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,hd,page,order", [
    (4, 1, 64, 8, "head"), (16, 4, 64, 32, "token"), (8, 8, 128, 16, "token"), (10, 2, 128, 64, "head"),
    (32, 1, 128, 8, "head"), (48, 2, 64, 16, "token"), (3, 1, 64, 4096, "head"), (14, 2, 128, 128, "token"),
    (16, 8, 128, 256, "head")])
def test_attention_layouts(gpu, wtype, nh, nkv, hd, page, order):
    rng = np.random.default_rng(nh * hd + page)
    for lens in ([(150, 1), (35, 1), (8, 1)], [(90, 3), (33, 2), (160, 20)], [(140, 100), (5, 1)]):
        pool, table, q_start, kv_len = make_batch(rng, lens, page, nkv, hd, wtype, order, fill=50.0)
        q = rng.standard_normal((q_start[-1], nh, hd)).astype(np.float32)
        args = (q, pool, q_start, kv_len, table, hd ** -0.5)
        check_attention(attend(gpu, *args), *args)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_max_new_only_chooses(gpu, wtype):
    """Whatever bound is given: the same sums within rounding."""
    rng = np.random.default_rng(5)
    pool, table, q_start, kv_len = make_batch(rng, [(300, 90), (200, 1), (60, 8)], 16, 2, 128, wtype)
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    for max_new in (0, 1, 8, 90, 2 ** 31):
        check_attention(attend(gpu, *args, max_new=max_new), *args)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_seen(gpu, wtype):
    """Spans that see past themselves, rows that see nothing (or less than nothing), bounds past
    the keys."""
    rng = np.random.default_rng(6)
    lens = [(200, 120), (50, 4), (130, 1), (64, 40)]
    pool, table, q_start, kv_len = make_batch(rng, lens, 16, 2, 128, wtype)
    n = int(q_start[-1])
    q = rng.standard_normal((n + 2, 8, 128)).astype(np.float32)
    seen = rng.integers(0, 220, n + 2).astype(np.int32)
    seen[:64] = 144            # an image's span
    seen[70:75] = (0, -4, 2 ** 31 - 1, 1, -2 ** 31)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    want = check_attention(attend(gpu, *args, seen=seen), *args, seen)
    assert (want[70:72] == 0).all() and (want[74] == 0).all()
    seen[:] = 0                # nothing at all
    assert (attend(gpu, *args, seen=seen)[:n] == 0).all()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("trash", [np.inf, np.nan, -np.inf, 3e38])
def test_attention_unseen_keys_do_not_matter(gpu, wtype, trash):
    """Unused positions, and keys that only later rows see, may hold anything; rows that do see
    a NaN key are NaN, and only they."""
    rng = np.random.default_rng(7)
    lens = [(100, 60), (37, 1), (90, 5)]
    for order in ("head", "token"):
        pool, table, q_start, kv_len = make_batch(rng, lens, 16, 2, 128, wtype, order, fill=trash)
        q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
        args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
        check_attention(attend(gpu, *args), *args)
    # a key in the middle of request 0's chunk: rows before it must not notice
    j = 75
    pool.put(pool.k, table[0, j // 16], j % 16, R.encode(np.full((2, 128), trash, np.float32), wtype))
    pool.put(pool.v, table[0, j // 16], j % 16, R.encode(np.full((2, 128), trash, np.float32), wtype))
    got = attend(gpu, *args)
    first = j - 40             # the first row that sees key j (row i sees keys 0 .. 40 + i)
    lo = [(75, 35), (37, 1), (90, 5)]
    keep = np.r_[0:first, 60:66]
    sub_start = np.array([0, first, first + 1, first + 6], np.int32)
    sub = (q[keep], pool, sub_start, np.array([kv for kv, _ in lo], np.int32), table, 128 ** -0.5)
    check_attention(got[keep], *sub)
    if np.isnan(trash):
        assert np.isnan(got[first:60]).all()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_magnitudes(gpu, wtype):
    """Large and tiny keys and values, keys of very different size side by side, scores far
    apart, ties."""
    rng = np.random.default_rng(8)
    for k_scale, v_scale, q_scale in ((1e-3, 1e-4, 1.0), (30.0, 1e3, 0.05), (1.0, 1.0, 40.0), (0.0, 1.0, 1.0)):
        lens = [(150, 1), (100, 40), (70, 6)]
        pool, table, q_start, kv_len = make_batch(rng, lens, 16, 2, 128, wtype)
        pool.k = R.encode(R.decode(pool.k, wtype).astype(np.float32) * np.float32(k_scale), wtype)
        pool.v = R.encode(R.decode(pool.v, wtype).astype(np.float32) * np.float32(v_scale), wtype)
        q = (rng.standard_normal((q_start[-1], 8, 128)) * q_scale).astype(np.float32)
        args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
        check_attention(attend(gpu, *args), *args)
    # sizes of neighbouring keys a factor 1e4 apart
    pool, table, q_start, kv_len = make_batch(rng, [(200, 50), (90, 2)], 16, 2, 128, wtype)
    f = np.float32(10.0) ** rng.integers(-2, 3, (pool.n_pages, 1, 16, 1)).astype(np.float32)
    pool.v = R.encode(R.decode(pool.v, wtype).astype(np.float32) * f, wtype)
    pool.k = R.encode(R.decode(pool.k, wtype).astype(np.float32) * f, wtype)
    q = (rng.standard_normal((q_start[-1], 8, 128)) * 0.05).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    check_attention(attend(gpu, *args), *args)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_bad_pages(gpu, wtype):
    """Positions whose page does not exist hold no key."""
    rng = np.random.default_rng(9)
    pool, table, q_start, kv_len = make_batch(rng, [(150, 1), (100, 40), (70, 6), (40, 2)], 16, 2, 128, wtype)
    table[0, 2] = -1
    table[1, 5] = pool.n_pages
    table[1, 0] = 2 ** 31 - 1
    table[2, :] = -2 ** 31
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    want = check_attention(attend(gpu, *args), *args)
    assert (want[41:47] == 0).all()


def test_attention_length_past_the_table(gpu):
    """kv_len beyond the table's reach ends there; q_start beyond the rows too."""
    rng = np.random.default_rng(10)
    pool, table, q_start, kv_len = make_batch(rng, [(64, 3), (64, 2)], 16, 2, 64, F16)
    kv_len[:] = (10 ** 9, -5)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    seen = np.array([64, 60, 10 ** 9, 3, 4], np.int32)
    args = (q, pool, q_start, kv_len, table, 0.125)
    check_attention(attend(gpu, *args, seen=seen), *args, seen)
    got = attend(gpu, q, pool, np.array([0, 3, 2 ** 31 - 1], np.int32), np.array([64, 64], np.int32), table, 0.125,
                 seen=seen)
    check_attention(got, q, pool, q_start, np.array([64, 64], np.int32), table, 0.125, seen)


def test_attention_many_requests(gpu):
    rng = np.random.default_rng(12)
    lens = [(int(rng.integers(0, 40)), 1) for _ in range(4096)]
    pool, table, q_start, kv_len = make_batch(rng, lens, 8, 1, 64, BF16)
    q = rng.standard_normal((q_start[-1], 4, 64)).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 0.125)
    check_attention(attend(gpu, *args), *args)


@pytest.mark.parametrize("wtype,lens", [(F32, [(9000, 1), (20, 1)]), (F16, [(20000, 3)]), (BF16, [(5000, 70)])])
def test_attention_long(gpu, wtype, lens):
    rng = np.random.default_rng(13)
    pool, table, q_start, kv_len = make_batch(rng, lens, 64, 1, 128, wtype)
    q = rng.standard_normal((q_start[-1], 4, 128)).astype(np.float32) * 2
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    check_attention(attend(gpu, *args), *args)


def test_offsets_past_32_bits(gpu):
    """Pages 2^32 elements apart: write and attention reach them."""
    rng = np.random.default_rng(14)
    hd, page, stride = 64, 16, 1 << 32
    kb, vb = gpu.Buf(2 * (stride + page * hd)), gpu.Buf(2 * (stride + page * hd))
    cache = gpu.PagedCache(kb, vb, F16, 2, page, 1, hd, (stride, hd, hd))
    T, nh = 32, 4
    qkv = rng.standard_normal((T, (nh + 2) * hd)).astype(np.float32)
    slots, pos = np.arange(T, dtype=np.int32), np.arange(T, dtype=np.int32)
    qb = gpu.Buf.empty((T, nh, hd))
    gpu.rope_qknorm_paged(dev(gpu, qkv), T, nh, cache, dev(gpu, pos), dev(gpu, slots), 1e4, None, None, 0, None, None,
                          1e-5, qb)
    small = Pool(2, page, 1, hd, F16)
    skb, svb = upload(gpu, small)
    sq = gpu.Buf.empty((T, nh, hd))
    small_cache = cache_of(gpu, small, skb, svb)
    gpu.rope_qknorm_paged(dev(gpu, qkv), T, nh, small_cache, dev(gpu, pos), dev(gpu, slots), 1e4, None, None, 0, None,
                          None, 1e-5, sq)
    for new in (T, 1):
        arrays = [dev(gpu, a, np.int32) for a in ([0, new], [T], [[1, 0]])]
        outs = []
        for c in (cache, small_cache):
            batch = gpu.PagedBatch(1, T, 2, new, *arrays)
            out, ws = dev(gpu, np.zeros((T, nh, hd), np.float32)), Ws(gpu, nh, c, batch)
            gpu.paged_attention(qb, nh, c, batch, 0.125, out, ws.b, ws.n)
            outs.append(out.numpy())
        assert np.abs(outs[0]).max() > 0.1
        np.testing.assert_array_equal(outs[0], outs[1])


def test_attention_same_result_each_time(gpu):
    rng = np.random.default_rng(15)
    pool, table, q_start, kv_len = make_batch(rng, [(900, 1), (500, 60), (40, 3)], 16, 2, 128, F32)
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    first = attend(gpu, q, pool, q_start, kv_len, table, 0.1)
    for _ in range(3):
        np.testing.assert_array_equal(attend(gpu, q, pool, q_start, kv_len, table, 0.1), first)


# ------------------------------------------------------------------ verification

class VerifyBufs:
    def __init__(self, gpu, logits, draft, ids, q_start, temp, ua, us, max_new):
        self.gpu, self.max_new = gpu, max_new
        self.R, (self.n_rows, self.V) = len(q_start) - 1, logits.shape
        f = lambda a: None if a is None else dev(gpu, a, np.float32)  # noqa: E731
        self.logits, self.draft, self.temp, self.ua, self.us = f(logits), f(draft), f(temp), f(ua), f(us)
        self.ids, self.q_start = dev(gpu, ids, np.int32), dev(gpu, q_start, np.int32)
        self.accepted, self.tokens = dev(gpu, np.full(self.R, 77, np.int32)), dev(gpu, np.full((self.R, max_new), 77, np.int32))
        self.n = gpu.verify_drafts_ws(self.R, self.n_rows, self.V)
        self.ws = dev(gpu, np.full(self.n // 4 + 1, np.nan, np.float32))

    def run(self, stream=None):
        self.gpu.verify_drafts(self.logits, self.draft, self.ids, self.q_start, self.R, self.n_rows, self.max_new,
                               self.V, self.temp, self.ua, self.us, self.accepted, self.tokens, self.ws, self.n,
                               stream)

    def result(self):
        return self.accepted.numpy(), self.tokens.numpy()


def drafts(rng, news, V, probs, spread=3.0, pad=0):
    n = sum(news) + pad
    logits = (rng.standard_normal((n, V)) * spread).astype(np.float32)
    d = np.exp(logits.astype(np.float64) * 0.8 + rng.standard_normal((n, V)) * 0.4)
    d = (d / d.sum(1, keepdims=True)).astype(np.float32)
    ids = np.zeros(n, np.int32)
    for i in range(1, n):
        ids[i] = rng.choice(V, p=d[i - 1].astype(np.float64) / d[i - 1].astype(np.float64).sum()) if probs \
            else int(np.argmax(logits[i - 1])) if rng.random() < 0.7 else rng.integers(0, V)
    q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return logits, d if probs else None, ids, q_start, rng.random(n).astype(np.float32), \
        rng.random(len(news)).astype(np.float32)


def check_verify(gpu, logits, draft, ids, q_start, temp, ua, us, max_new):
    acc, tok, margin = R.verify(logits, draft, ids, q_start, temp, ua, us, max_new)
    # 64-bit sums of V terms in another order differ by V 2^-53 of the whole at most, the
    # weights' exponentials by 1e-14: decisions have to be farther from their borders
    assert margin > 2e-14 + logits.shape[1] * 2.0 ** -52
    b = VerifyBufs(gpu, logits, draft, ids, q_start, temp, ua, us, max_new)
    b.run()
    got = b.result()
    np.testing.assert_array_equal(got[0], acc)
    np.testing.assert_array_equal(got[1], tok)
    return acc, tok


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 8191, 32003, 133120])
@pytest.mark.parametrize("probs", [False, True])
def test_verify(gpu, V, probs):
    rng = np.random.default_rng(V + probs)
    news = [5, 1, 3, 8, 2, 6] if V < 100000 else [4, 1, 3]
    logits, d, ids, q_start, ua, us = drafts(rng, news, V, probs, pad=2)
    temp = (0.5 + rng.random(len(news))).astype(np.float32)
    temp[2] = 0.0
    check_verify(gpu, logits, d, ids, q_start, temp, ua, us, 8)
    check_verify(gpu, logits, d, ids, q_start, None, ua, us, 9)


def test_verify_flat_distribution(gpu):
    """Many tokens of the same small weight: the drawn index shows any error of the sums."""
    rng = np.random.default_rng(21)
    V, n = 133120, 24
    logits = np.zeros((n, V), np.float32)
    logits[8:] = rng.standard_normal((n - 8, V)) * 0.01
    us = rng.random(n).astype(np.float32)
    acc, tok = check_verify(gpu, logits, None, np.zeros(n, np.int32), np.arange(n + 1, dtype=np.int32), None,
                            rng.random(n).astype(np.float32), us, 1)
    assert (acc == 0).all()
    np.testing.assert_allclose(tok[:8, 0], np.floor(us[:8] * np.float64(V)), atol=1)


def test_verify_greedy_ties_and_negative_temperature(gpu):
    V = 777
    logits = np.zeros((6, V), np.float32)
    logits[0, [700, 5, 300]] = 2.0     # ties: 5
    logits[1, 776] = 1.0
    ids = np.array([0, 5, 776, 0, 300, 0], np.int32)
    logits[3, [300, 40]] = 9.0         # tie: 40, and the draft says 300
    acc, tok, _ = R.verify(logits, None, ids, [0, 3, 6], [0.0, -1.0], np.zeros(6), np.zeros(2), 3)
    b = VerifyBufs(gpu, logits, None, ids, [0, 3, 6], [0.0, -1.0], np.zeros(6), np.zeros(2), 3)
    b.run()
    got = b.result()
    np.testing.assert_array_equal(got[0], acc)
    np.testing.assert_array_equal(got[1], tok)
    assert acc.tolist() == [2, 0] and tok.tolist() == [[5, 776, 0], [40, -1, -1]]
    b = VerifyBufs(gpu, logits, None, ids, [0, 3, 6], [np.nan, 0.0], np.zeros(6), np.zeros(2), 3)
    b.run()
    np.testing.assert_array_equal(b.result()[1], tok)


def test_verify_masked_and_broken_rows(gpu):
    """-inf logits are never drawn; rows without a distribution end their request with -1;
    requests without rows or with too many give -1."""
    rng = np.random.default_rng(22)
    V = 5000
    logits, d, ids, _, ua, us = drafts(rng, [24], V, True)
    logits[:, 100:] = -np.inf
    ids[:] = rng.integers(0, 100, 24)
    logits[3, 50] = np.nan
    logits[6, :] = -np.inf
    logits[9, 7] = np.inf
    logits[12, :] = -np.inf
    logits[12, 4321] = -1e30                       # one token left
    q_start = np.array([0, 3, 6, 6, 9, 12, 14, 22, 24], np.int32)
    us = rng.random(8).astype(np.float32)
    ids[13] = 4321
    for temp in (None, np.full(8, 0.7, np.float32), np.zeros(8, np.float32), np.full(8, np.inf, np.float32)):
        if temp is not None and np.isinf(temp).all():
            continue_rows = np.array([0, 3], np.int32)  # the flat limit over what is not masked
            lg = logits[:3]
            b = VerifyBufs(gpu, lg, d[:3], ids[:3], continue_rows, temp[:1], ua[:3], us[:1], 3)
            b.run()
            a, t = b.result()
            assert 0 <= a[0] <= 2 and (t[0, :a[0] + 1] >= 0).all() and (t[0, :a[0] + 1] < 100).all()
            continue
        acc, tok, _ = R.verify(logits, d, ids, q_start, temp, ua, us, 6)
        b = VerifyBufs(gpu, logits, d, ids, q_start, temp, ua, us, 6)
        b.run()
        np.testing.assert_array_equal(b.result()[0], acc)
        np.testing.assert_array_equal(b.result()[1], tok)
        assert acc[2] == -1 and acc[6] == -1 and acc[1] == 0 and tok[1, 0] == -1


def test_verify_drafts_outside_the_vocabulary_and_equal_distributions(gpu):
    rng = np.random.default_rng(23)
    V = 600
    logits, d, ids, q_start, ua, us = drafts(rng, [3, 3, 3], V, True)
    ids[1], ids[4] = V, -1
    check_verify(gpu, logits, d, ids, q_start, None, ua, us, 3)
    # p is 0 wherever the draft may go, and equals q elsewhere: nothing is left, p is drawn from
    logits[:] = np.log(np.float32(1 / 512))
    logits[:, 512:] = -np.inf
    d = np.zeros((9, V), np.float32)
    d[:, :512] = 1 / 512
    ids[:] = 550
    check_verify(gpu, logits, d, ids, q_start, None, ua, us, 3)


def test_verify_u_at_its_ends(gpu):
    rng = np.random.default_rng(24)
    V = 3001
    logits, d, ids, q_start, ua, us = drafts(rng, [4, 4], V, True)
    top = np.float32(1) - np.float32(2.0 ** -24)
    for a, s in ((0.0, 0.0), (top, top), (0.0, top), (top, 0.0)):
        ua[:], us[:] = a, s
        acc, tok, _ = R.verify(logits, d, ids, q_start, None, ua, us, 4)
        b = VerifyBufs(gpu, logits, d, ids, q_start, None, ua, us, 4)
        b.run()
        np.testing.assert_array_equal(b.result()[0], acc)
        np.testing.assert_array_equal(b.result()[1], tok)


# ------------------------------------------------------------------ streams and graphs

def test_two_streams_at_once(gpu):
    """Calls that overlap, each with a workspace of its own."""
    rng = np.random.default_rng(30)
    jobs = []
    for i in range(4):
        lens = [(700 + 50 * i, 1), (300, 40 if i % 2 else 2), (90, 3)]
        pool, table, q_start, kv_len = make_batch(rng, lens, 16, 2, 128, (F32, F16, BF16, F32)[i])
        q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
        kb, vb = upload(gpu, pool)
        cache = cache_of(gpu, pool, kb, vb)
        batch = gpu.PagedBatch(3, len(q), table.shape[1], int(np.diff(q_start).max()),
                               *[dev(gpu, a, np.int32) for a in (q_start, kv_len, table)])
        jobs.append(dict(st=gpu.Stream(), args=(q, pool, q_start, kv_len, table, 0.1), q=dev(gpu, q), cache=cache,
                         batch=batch, out=dev(gpu, np.full(q.shape, -3.0, np.float32)), ws=Ws(gpu, 8, cache, batch)))
    gpu.sync()
    for _ in range(5):
        for j in jobs:
            gpu.paged_attention(j["q"], 8, j["cache"], j["batch"], 0.1, j["out"], j["ws"].b, j["ws"].n, j["st"].h)
    for j in jobs:
        j["st"].synchronize()
    for j in jobs:
        check_attention(j["out"].numpy(), *j["args"])
        j["st"].close()


def test_captured_step(gpu):
    """Tables, write, attention and verification in one graph, replayed with other contents
    and with eager work between: every replay equals the eager calls."""
    rng = np.random.default_rng(31)
    n_req, nh, nkv, hd, page, max_pages, V = 5, 8, 2, 64, 16, 12, 1500
    n_rows, n_pages = 40, 70
    cached = np.array([30, 0, 77, 5, 100])
    news = np.array([5, 20, 1, 3, 7])
    held = -(-cached // page)
    table = np.zeros((n_req, max_pages), np.int32)
    perm = rng.permutation(n_pages)
    at = 0
    for r in range(n_req):
        table[r, :held[r]] = perm[at:at + held[r]]
        at += held[r]
    free = np.zeros(n_pages, np.int32)
    free[:n_pages - at] = perm[at:]

    class Step:
        def __init__(self):
            self.plan = PlanBufs(gpu, cached, news, held, table, free, n_pages - at, n_rows, page, n_pages)
            self.pool = Pool(n_pages, page, nkv, hd, BF16)
            self.kb, self.vb = upload(gpu, self.pool)
            self.qkv = dev(gpu, np.zeros((n_rows, (nh + 2 * nkv) * hd), np.float32))
            self.q, self.out = dev(gpu, np.zeros((n_rows, nh, hd), np.float32)), dev(gpu, np.zeros((n_rows, nh, hd), np.float32))
            p = self.plan
            self.cache = cache_of(gpu, self.pool, self.kb, self.vb)
            self.batch = gpu.PagedBatch(n_req, n_rows, max_pages, 20, p.q_start, p.kv_len, p.table, p.positions, p.slots)
            self.ws = Ws(gpu, nh, self.cache, self.batch)
            self.ver = VerifyBufs(gpu, np.zeros((n_rows, V), np.float32), None, np.zeros(n_rows), np.zeros(n_req + 1),
                                  None, np.full(n_rows, 0.5), np.full(n_req, 0.5), 20)

        def fill(self, seed):
            g = np.random.default_rng(seed)
            put = lambda b, a: gpu.check(gpu.lib().hy_memcpy_h2d(b.ptr, a.ctypes.data, a.nbytes))  # noqa: E731
            put(self.qkv, g.standard_normal((n_rows, (nh + 2 * nkv) * hd)).astype(np.float32))
            logits = (g.standard_normal((n_rows, V)) * 4).astype(np.float32)
            put(self.ver.logits, logits)
            ids = np.zeros(n_rows, np.int32)
            ids[1:] = np.where(g.random(n_rows - 1) < 0.6, logits[:-1].argmax(1), 3)
            put(self.ver.ids, ids)
            put(self.ver.ua, g.random(n_rows).astype(np.float32))
            put(self.ver.us, g.random(n_req).astype(np.float32))

        def run(self, st):
            p = self.plan
            p.run(st)
            gpu.rope_qknorm_paged(self.qkv, n_rows, nh, self.cache, p.positions, p.slots, 1e4, None, None, 0, None, None,
                                  1e-5, self.q, st)
            gpu.paged_attention(self.q, nh, self.cache, self.batch, 0.125, self.out, self.ws.b, self.ws.n, st)
            v = self.ver
            gpu.verify_drafts(v.logits, None, v.ids, p.q_start, n_req, n_rows, 20, V, None, v.ua, v.us, v.accepted,
                              v.tokens, v.ws, v.n, st)

        def results(self):
            return [b.numpy() for b in (self.plan.slots, self.kb, self.vb, self.out, self.ver.accepted, self.ver.tokens)]

    st, a, b = gpu.Stream(), Step(), Step()
    g = gpu.Graph(st, lambda: a.run(st.h))
    try:
        for rep in range(4):
            a.fill(100 + rep)
            b.fill(100 + rep)
            b.run(st.h)
            st.synchronize()
            g.launch()
            st.synchronize()
            for x, y in zip(a.results(), b.results()):
                np.testing.assert_array_equal(x, y)
            assert (a.results()[3][:36] != 0).any()
    finally:
        g.close()
        st.close()


# ------------------------------------------------------------------ the step as a whole

def paged_step(gpu, cached, news, held, table, free, n_free, page, n_pages):
    """The plan of a step and its batch."""
    p = PlanBufs(gpu, cached, news, held, table, free, n_free, int(sum(news)), page, n_pages)
    p.run(in_place=True)
    assert (p.status.numpy() == 0).all()
    batch = gpu.PagedBatch(p.R, p.n_rows, p.max_pages, int(max(news)), p.q_start, p.kv_len, p.table, p.positions, p.slots)
    return p, batch


@pytest.mark.parametrize("wtype", [F32, BF16])
def test_attention_layer_in_chunks_equals_one_prompt(gpu, wtype):
    """hy_attn_forward over a whole prompt and hy_attn_forward_paged over its pieces, two requests
    side by side.  f32: as far apart as two f32 evaluations with sums of hidden = 512 and
    hd = 128 terms may be; bf16: keys and values rounded by 2^-9 relative."""
    H, nh, nkv, hd, T, page = 512, 8, 2, 128, 75, 16
    att = gpu.Attn(H, nh, nkv, hd, 128)
    att.synth(0, seed=5, std=0.05)
    rng = np.random.default_rng(40)
    xs = [rng.standard_normal((T, H)).astype(np.float32) for _ in range(2)]
    want = [att.run(x) for x in xs]
    n_pages, max_pages = 16, 6
    pool = Pool(n_pages, page, nkv, hd, wtype)
    kb, vb = upload(gpu, pool)
    cache = cache_of(gpu, pool, kb, vb)
    held, table = np.zeros(2, np.int32), np.zeros((2, max_pages), np.int32)
    free, n_free, cached = rng.permutation(n_pages).astype(np.int32), n_pages, np.zeros(2, np.int64)
    got = [[], []]
    for news in ([40, 3], [1, 30], [33, 1], [1, 41]):
        p, batch = paged_step(gpu, cached, news, held, table, free, n_free, page, n_pages)
        x = np.concatenate([xs[r][cached[r]:cached[r] + news[r]] for r in range(2)])
        out = gpu.Buf.empty(x.shape)
        ws = Ws(gpu, nh, cache, batch)
        att.forward_paged(dev(gpu, x), cache, batch, out, ws.b, ws.n)
        o = out.numpy()
        got[0].append(o[:news[0]])
        got[1].append(o[news[0]:])
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        cached = cached + news
    att.close()
    for g, w in zip(got, want):
        g = np.concatenate(g)
        assert g.shape == w.shape
        # the 1D path forms its angles in f32: positions below 75 carry 75 half steps of error
        tol = 2e-5 if wtype == F32 else 2.0 ** -8
        assert np.linalg.norm(g - w) <= tol * np.linalg.norm(w)


def test_layer_refusals(gpu):
    att = gpu.Attn(256, 8, 2, 64, 16)
    att.synth(0, seed=5, std=0.05)
    pool = Pool(4, 16, 2, 64, F16)
    kb, vb = upload(gpu, pool)
    i32 = lambda n: dev(gpu, np.zeros(n, np.int32))  # noqa: E731
    x, out = gpu.Buf.empty((16, 256)), gpu.Buf.empty((16, 256))

    def call(cache=None, batch=None, ws_off=0, layer=0, **kw):
        c = cache or cache_of(gpu, pool, kb, vb)
        b = batch or gpu.PagedBatch(1, 8, 4, 8, i32(2), i32(1), i32(4), i32(8), i32(8))
        n = 1 << 28
        ws = gpu.Buf(n)
        att.forward_paged(x, c, b, out, ws, n * (1 - ws_off), layer=layer, **kw)

    call()
    bad = cache_of(gpu, pool, kb, vb)
    bad.n_kv_heads = 4
    with pytest.raises(gpu.HyError):
        call(cache=bad)
    with pytest.raises(gpu.HyError):
        call(batch=gpu.PagedBatch(1, 17, 4, 8, i32(2), i32(1), i32(4), i32(17), i32(17)))
    with pytest.raises(gpu.HyError):
        call(batch=gpu.PagedBatch(1, 8, 4, 8, i32(2), i32(1), i32(4)))
    with pytest.raises(gpu.HyError):
        call(ws_off=1)
    with pytest.raises(gpu.HyError):
        call(layer=1)
    with pytest.raises(gpu.HyError):
        call(cache=cache_of(gpu, pool, kb, vb, layer_stride=4))
    with pytest.raises(gpu.HyError):
        call(cos=x, n_pos=3)
    att.close()


def greedy_model(gpu):
    H, I, E, K, nh, nkv, hd, V, L = 256, 128, 8, 2, 8, 2, 64, 500, 2
    m = gpu.Model(H, I, E, K, gpu.F32, nh, nkv, hd, V, L, 128)
    m.synth_globals(seed=3, std=0.5)
    for l in range(L):
        m.attn.synth(l, seed=7 + l, std=0.08)
        m.moe.synth(l, seed=9 + l, std=0.05)
    return m, nh, nkv, hd, V, L


def test_speculative_decoding_equals_greedy_decoding(gpu):
    """The loop of a server: plan, backbone over the paged cache, verification, next lengths.  A
    drafter that guesses from the known continuation, with mistakes, does not change what
    is generated; the greedy continuation comes from hy_model_forward on whole sequences."""
    m, nh, nkv, hd, V, L = greedy_model(gpu)
    rng = np.random.default_rng(50)
    prompts = [rng.integers(0, V, n).tolist() for n in (9, 23, 1)]
    steps = 20
    want = []
    for p in prompts:
        seq = list(p)
        for _ in range(steps):
            lb = gpu.Buf.empty((len(seq), V))
            m.forward(dev(gpu, seq, np.int32), len(seq), lb)
            last = np.sort(lb.numpy()[-1])
            assert last[-1] - last[-2] > 1e-4 * abs(last[-1])  # no near tie decides
            seq.append(int(np.argmax(lb.numpy()[-1])))
        want.append(seq[len(p):])
    page, n_pages, max_pages = 8, 40, 8
    pool = Pool(n_pages * L, page, nkv, hd, F32)
    kb, vb = upload(gpu, pool)
    cache = gpu.PagedCache(kb, vb, F32, n_pages, page, nkv, hd, layer_stride=n_pages * nkv * page * hd)
    n = len(prompts)
    held, table = np.zeros(n, np.int32), np.zeros((n, max_pages), np.int32)
    free, n_free, cached = rng.permutation(n_pages).astype(np.int32), n_pages, np.zeros(n, np.int64)
    done = [[] for _ in prompts]
    todo = [list(p) for p in prompts]  # rows to run next: the prompt, then the last token and drafts
    first, accepted_in_all = True, 0
    while min(len(d) for d in done) < steps:
        news = [len(t) for t in todo]
        p, batch = paged_step(gpu, cached, news, held, table, free, n_free, page, n_pages)
        ids = np.concatenate(todo).astype(np.int32)
        logits = gpu.Buf.empty((len(ids), V))
        ws = Ws(gpu, nh, cache, batch)
        m.forward_paged(dev(gpu, ids), cache, batch, logits, ws.b, ws.n)
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        if first:  # the prompts' own tokens are no drafts: the last row's prediction alone
            q_start, rows = np.arange(n + 1), np.cumsum(news) - 1
            vb_ = VerifyBufs(gpu, logits.numpy()[rows], None, np.zeros(n), q_start, np.zeros(n), np.zeros(n),
                             np.zeros(n), 1)
            vb_.run()
        else:
            vb_ = VerifyBufs(gpu, logits.numpy(), None, ids, p.q_start.numpy(), np.zeros(n), np.zeros(len(ids)),
                             np.zeros(n), max(news))
            vb_.run()
        acc, tok = vb_.result()
        for r in range(n):
            cached[r] += news[r] if first else acc[r] + 1
            done[r] += tok[r, :acc[r] + 1].tolist()
            accepted_in_all += int(acc[r])
            known = want[r][len(done[r]):len(done[r]) + int(rng.integers(0, 5))]
            drafts_ = [t if rng.random() < 0.8 else (t + 1) % V for t in known]
            todo[r] = [done[r][-1]] + drafts_ if len(done[r]) < steps else [done[r][-1]]
        first = False
        if max(cached) + 6 > page * max_pages:
            break
    m.close()
    assert accepted_in_all > 10
    for d, w in zip(done, want):
        assert d[:steps] == w[:len(d)][:steps]


# ------------------------------------------------------------------ the ends of the ranges

def test_append_of_more_waves_than_one_grid_dimension_holds(gpu):
    """2^20 rows of 253 heads: 2^32 threads.  Only a few rows have a slot, so little is touched."""
    T, nh, nkv, hd, page = 1 << 20, 252, 1, 64, 16
    row = (nh + 2 * nkv) * hd
    qkv, qb = gpu.Buf(4 * T * row), gpu.Buf(4 * T * nh * hd)
    rng = np.random.default_rng(60)
    live = np.array([0, 1, 77777, T // 2, T - 2, T - 1])
    x = rng.standard_normal((len(live), row)).astype(np.float32)
    slots, pos = np.full(T, -1, np.int32), np.zeros(T, np.int32)
    slots[live], pos[live] = np.arange(len(live)) + 3, live
    put = lambda at, a: gpu.check(gpu.lib().hy_memcpy_h2d(at, a.ctypes.data, a.nbytes))  # noqa: E731
    for i, t in enumerate(live):
        put(qkv.ptr + 4 * int(t) * row, np.ascontiguousarray(x[i]))
    pool = Pool(2, page, nkv, hd, F32, fill=7.0)
    kb, vb = upload(gpu, pool)
    gpu.rope_qknorm_paged(qkv, T, nh, cache_of(gpu, pool, kb, vb), dev(gpu, pos), dev(gpu, slots), 1e4, None, None, 0,
                          None, None, 1e-5, qb)
    gpu.sync()
    q, k, v, qm, km = append_ref(x, nh, nkv, hd, pos[live], 1e4, None, None, None, None, 1e-5)
    got, gk, gv = np.empty((nh, hd), np.float32), kb.numpy(), vb.numpy()
    for i, t in enumerate(live):
        gpu.check(gpu.lib().hy_memcpy_d2h(got.ctypes.data, qb.ptr + 4 * int(t) * nh * hd, got.nbytes))
        assert (np.abs(got - q[i]) <= APPEND_TOL * qm[i]).all()
        p, o = divmod(int(slots[t]), page)
        assert (np.abs(pool.at(gk, p, o) - k[i]) <= APPEND_TOL * km[i] + EPS32 * np.abs(k[i])).all()
        np.testing.assert_array_equal(pool.at(gv, p, o), v[i].astype(np.float32))
    qkv.free()
    qb.free()


def test_model_of_a_padded_batch(gpu):
    """Rows behind the last sequence and rows of a request that got no pages change nothing for
    the others, whatever their ids."""
    m, nh, nkv, hd, V, L = greedy_model(gpu)
    rng = np.random.default_rng(61)
    page, n_pages, max_pages = 8, 6, 8
    news = [9, 23, 30, 1]                     # 2 + 3 + (4: refused) + 1 pages of 6

    def run(news, pad):
        pool = Pool(n_pages * L, page, nkv, hd, F32, fill=np.nan)
        kb, vb = upload(gpu, pool)
        cache = gpu.PagedCache(kb, vb, F32, n_pages, page, nkv, hd, layer_stride=n_pages * nkv * page * hd)
        n = len(news)
        p = PlanBufs(gpu, np.zeros(n), news, np.zeros(n), np.zeros((n, max_pages)), np.arange(n_pages), n_pages,
                     sum(news) + pad, page, n_pages)
        p.run()
        batch = gpu.PagedBatch(n, p.n_rows, max_pages, max(news), p.q_start, p.kv_len, p.table, p.positions, p.slots)
        ids = np.full(p.n_rows, -5, np.int32)
        at = 0
        for new, seq in zip(news, (seqs[0], seqs[1], seqs[2], seqs[3])):
            ids[at:at + new] = seq[:new]
            at += new
        if pad:
            ids[at:] = 2 ** 31 - 1
        logits = gpu.Buf.empty((p.n_rows, V))
        ws = Ws(gpu, nh, cache, batch)
        m.forward_paged(dev(gpu, ids), cache, batch, logits, ws.b, ws.n)
        return p.status.numpy().tolist(), logits.numpy(), p

    seqs = [rng.integers(0, V, 40) for _ in range(4)]
    st, got, p = run(news, 7)
    # the request that lacks pages, and those that lack them behind it
    assert st == [0, 0, 1, 1]
    for r in range(2):
        lb = gpu.Buf.empty((news[r], V))
        m.forward(dev(gpu, seqs[r][:news[r]], np.int32), news[r], lb)
        want = lb.numpy()
        g = got[sum(news[:r]):sum(news[:r + 1])]
        assert np.isfinite(g).all()
        # two f32 evaluations of two layers, as far apart as the layer test's, and their
        # experts' products
        assert np.linalg.norm(g - want) <= 1e-4 * np.linalg.norm(want)
    m.close()


def test_model_refuses_before_it_writes(gpu):
    """A layer without experts: refused with the cache as it was."""
    H, I, E, K, nh, nkv, hd, V, L = 256, 128, 8, 2, 8, 2, 64, 500, 2
    m = gpu.Model(H, I, E, K, gpu.F32, nh, nkv, hd, V, L, 64)
    m.synth_globals(seed=3, std=0.5)
    for l in range(L):
        m.attn.synth(l, seed=7 + l, std=0.08)
    m.moe.synth(0, seed=9, std=0.05)
    pool = Pool(4 * L, 16, nkv, hd, F16, fill=3.0)
    kb, vb = upload(gpu, pool)
    cache = gpu.PagedCache(kb, vb, F16, 4, 16, nkv, hd, layer_stride=4 * nkv * 16 * hd)
    i32 = lambda *a: dev(gpu, np.array(a, np.int32))  # noqa: E731
    batch = gpu.PagedBatch(1, 2, 4, 2, i32(0, 2), i32(2), i32(0, 1, 2, 3), i32(0, 1), i32(0, 1))
    ws = Ws(gpu, nh, cache, batch)
    logits = dev(gpu, np.full((2, V), 8.0, np.float32))
    call = lambda w, n: m.forward_paged(i32(4, 5), cache, batch, logits, w, n)  # noqa: E731
    with pytest.raises(gpu.HyError):
        call(ws.b, ws.n)
    m.moe.synth(1, seed=10, std=0.05)
    with pytest.raises(gpu.HyError):
        call(ws.b, ws.n - 1)

    class Odd:
        ptr = ws.b.ptr + 4
    with pytest.raises(gpu.HyError):
        call(Odd, ws.n)
    gpu.sync()
    np.testing.assert_array_equal(kb.numpy(), pool.k)
    np.testing.assert_array_equal(vb.numpy(), pool.v)
    assert (logits.numpy() == 8.0).all()
    call(ws.b, ws.n)
    assert np.isfinite(logits.numpy()).all() and (kb.numpy() != pool.k).any()
    m.close()


def test_attention_unwritten_page_ends_take_no_longer_path(gpu):
    """What lies behind a request's last key in its page may be anything, infinities and NaN among
    it: the sums are the same bits as over zeros there."""
    rng = np.random.default_rng(62)
    for wtype in (F32, F16, BF16):
        outs = []
        pool, table, q_start, kv_len = make_batch(rng, [(700, 1), (37, 1), (90, 3), (200, 1)], 64, 2, 128, wtype)
        q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
        used = np.zeros((pool.n_pages, 64), bool)
        for r, kv in enumerate(kv_len):
            for j in range(kv):
                used[table[r, j // 64], j % 64] = True
        for fill in (0.0, np.nan, np.inf):
            for p, i in np.argwhere(~used):
                for a in (pool.k, pool.v):
                    pool.put(a, p, i, R.encode(np.full((2, 128), fill, np.float32), wtype))
            outs.append(attend(gpu, q, pool, q_start, kv_len, table, 0.1))
        np.testing.assert_array_equal(outs[0], outs[1])
        np.testing.assert_array_equal(outs[0], outs[2])


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,page,order,trash", [(8, 2, 8, "head", 0.0), (10, 2, 64, "token", np.nan),
                                                     (16, 1, 32, "head", np.inf)])
def test_attention_long_chunks_of_small_heads(gpu, wtype, nh, nkv, page, order, trash):
    """More rows than the streams take for head_dim 64, beside requests of few rows."""
    rng = np.random.default_rng(63 + nh)
    n = 2100 // (nh // nkv) + 5
    lens = [(n + 61, n), (40, 1), (90, 3), (0, 0), (200, 33)]
    pool, table, q_start, kv_len = make_batch(rng, lens, page, nkv, 64, wtype, order, fill=trash)
    q = rng.standard_normal((q_start[-1] + 2, nh, 64)).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 0.125)
    check_attention(attend(gpu, *args), *args)
    seen = np.minimum(rng.integers(0, n + 90, q_start[-1] + 2), np.repeat(kv_len, np.diff(q_start)).max()).astype(np.int32)
    seen[5:40] = 0
    check_attention(attend(gpu, *args, seen=seen), *args, seen)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_rows_around_the_streams_limits(gpu, wtype, hd):
    """Row counts on both sides of every choice of kernel and tile: the same sums within rounding."""
    rng = np.random.default_rng(64)
    nh, nkv = 8, 2
    for news in ((4, 4, 4), (5, 1, 3), (8, 8, 2), (9, 8, 2), (16, 2, 2), (17, 16, 1), (32, 31, 2), (33, 9, 8), (64, 20, 1),
                 (65, 64, 3), (128, 7, 1), (129, 8, 9)):
        lens = [(n + int(rng.integers(0, 80)), n) for n in news]
        for part in (lens, lens[:2], lens[:1]):
            pool, table, q_start, kv_len = make_batch(rng, part, 16, nkv, hd, wtype)
            q = rng.standard_normal((q_start[-1], nh, hd)).astype(np.float32)
            args = (q, pool, q_start, kv_len, table, hd ** -0.5)
            check_attention(attend(gpu, *args), *args)


def test_model_refuses_layers_that_share_a_pool(gpu):
    m, nh, nkv, hd, V, L = greedy_model(gpu)
    pool = Pool(4, 16, nkv, hd, F32, fill=3.0)
    kb, vb = upload(gpu, pool)
    i32 = lambda *a: dev(gpu, np.array(a, np.int32))  # noqa: E731
    cache = cache_of(gpu, pool, kb, vb)
    batch = gpu.PagedBatch(1, 2, 4, 2, i32(0, 2), i32(2), i32(0, 1, 2, 3), i32(0, 1), i32(0, 1))
    ws, logits = Ws(gpu, nh, cache, batch), gpu.Buf.empty((2, V))
    with pytest.raises(gpu.HyError):
        m.forward_paged(i32(4, 5), cache, batch, logits, ws.b, ws.n)
    gpu.sync()
    np.testing.assert_array_equal(kb.numpy(), pool.k)
    m.close()
