"""Serving in 8 bits on the GPU (include/hy_int8.h) against plain numpy (int8_ref.py): products with
token and channel scales bit for bit, the quantizing write of a paged cache code for code, and attention
over it against 64 bits."""
import numpy as np
import pytest

import int8_ref as Q
import paged_ref as R
from int8_ref import PoolI8
from test_paged_gpu import APPEND_TOL, LENS, append_ref, dev

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ products

class GemmBufs:
    def __init__(self, gpu, linear, x, xs, w, ws, resid, fill=-3.0):
        T, K, N = x.shape[0], x.shape[1], w.shape[0]
        self.gpu, self.linear, self.sizes = gpu, linear, (T, K, N)
        self.x, self.xs, self.w, self.ws = dev(gpu, x), None if linear else dev(gpu, xs), dev(gpu, w), dev(gpu, ws)
        self.resid = None if resid is None else dev(gpu, resid)
        # 64 floats behind the last row: nothing of theirs is written
        self.out = dev(gpu, np.full(T * N + 64, fill, np.float32))
        self.n = (gpu.linear_i8_ws if linear else gpu.gemm_i8_ws)(T, K, N)
        self.wsp = dev(gpu, np.full(self.n // 4 + 1, np.nan, np.float32))

    def run(self, stream=None):
        a = (self.x, self.w) if self.linear else (self.x, self.xs, self.w)
        f = self.gpu.linear_i8 if self.linear else self.gpu.gemm_i8
        f(*a, self.ws, self.resid, *self.sizes, self.out, self.wsp, self.n, stream)

    def result(self, fill=-3.0):
        T, _, N = self.sizes
        got = self.out.numpy()
        assert (got[T * N:] == fill).all()
        return got[:T * N].reshape(T, N)


def same_bits(a, b):
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
    np.testing.assert_array_equal(np.where(np.isnan(a), 0, a), np.where(np.isnan(b), 0, b))


SHAPES = [(1, 16, 1), (1, 4096, 6144), (2, 272, 33), (3, 48, 513), (5, 1040, 100), (16, 4096, 1000), (17, 144, 4096),
          (31, 2048, 65), (33, 4096, 257), (64, 1024, 512), (65, 2064, 130), (100, 32, 31), (128, 4096, 4096),
          (129, 528, 255), (200, 8192, 96), (256, 256, 256), (300, 4096, 1000), (511, 1008, 385), (700, 64, 2000),
          (1025, 512, 300), (16, 16, 20000), (4096, 16, 5), (1, 131056, 40), (40, 131056, 9), (5, 272, 33000),
          # tiles of 128 and of 256, with and without a last round of halves; reductions that end inside a stage
          (1100, 400, 4200), (1000, 144, 6100), (2500, 272, 6144), (4100, 144, 4200), (4096, 80, 6145),
          (3000, 2064, 11000)]


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_gemm(gpu, T, K, N):
    rng = np.random.default_rng(T * 31 + K + N)
    x, w = rng.integers(-128, 128, (T, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    xs, ws = np.exp(rng.standard_normal(T)).astype(np.float32), np.exp(rng.standard_normal(N)).astype(np.float32)
    for resid in (None, rng.standard_normal((T, N)).astype(np.float32) * 1000):
        b = GemmBufs(gpu, False, x, xs, w, ws, resid)
        b.run()
        same_bits(b.result(), Q.gemm(x, xs, w, ws, resid))


# tiles of 64 x 128; one row of tiles over weights of more than 256 MB, with a reduction that ends inside a stage
@pytest.mark.parametrize("T,K,N", [(500, 272, 6100), (700, 2064, 4096), (20, 65520, 4200), (50, 65520, 4200),
                                   (32, 65536, 4097), (64, 65536, 4097)])
def test_gemm_wide_and_long(gpu, T, K, N):
    test_gemm(gpu, T, K, N)


@pytest.mark.parametrize("T,K,N", [(1, 4096, 300), (2, 64, 7), (3, 4112, 64), (8, 6160, 40), (17, 4096, 100),
                                   (70, 2048, 129), (300, 1024, 256), (600, 272, 70), (2, 131056, 8)])
def test_linear(gpu, T, K, N):
    rng = np.random.default_rng(T + K + N)
    x = (rng.standard_normal((T, K)) * np.exp(rng.standard_normal((1, K)))).astype(np.float32)
    w, ws = Q.quantize(rng.standard_normal((N, K)).astype(np.float32) * 0.02)
    resid = rng.standard_normal((T, N)).astype(np.float32) if T % 2 else None
    b = GemmBufs(gpu, True, x, None, w, ws, resid)
    b.run()
    xq, xs = Q.quantize(x)
    same_bits(b.result(), Q.gemm(xq, xs, w, ws, resid))


def test_largest_sums(gpu):
    """Codes of -128 alone, the widest rows: the sum stays below 2^31."""
    K = 131056
    x, w = np.full((3, K), -128, np.int8), np.full((70, K), -128, np.int8)
    w[1::2] = 127
    one = np.ones(70, np.float32)
    b = GemmBufs(gpu, False, x, one[:3], w, one, None)
    b.run()
    same_bits(b.result(), Q.gemm(x, one[:3], w, one))


@pytest.mark.parametrize("rows,cols", [(1, 16), (7, 48), (300, 4096), (33, 4112), (2, 8208), (5, 131056), (3000, 16)])
def test_quantize_rows(gpu, rows, cols):
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(3 * rng.standard_normal((rows, 1)))).astype(np.float32)
    x[rng.random((rows, cols)) < 0.01] *= 30
    x[0, :] = 0.0
    if rows > 2:
        # halfway between codes: a row of multiples of half a step, the largest 127 steps
        x[1] = np.float32(0.25) * rng.integers(-127, 128, cols).astype(np.float32)
        x[1, 0] = np.float32(63.5)
        x[2] = rng.standard_normal(cols) * 2.0 ** -120   # a scale near the smallest
    if rows > 6:
        x[3, 5], x[4, 0], x[5, cols - 1] = np.nan, np.inf, -np.inf
        x[6] = rng.standard_normal(cols) * 2.0 ** -127   # below it
    c, s = dev(gpu, np.full((rows, cols), 99, np.int8)), dev(gpu, np.full(rows, 7.0, np.float32))
    gpu.quantize_rows_i8(dev(gpu, x), rows, cols, c, s)
    wc, wd = Q.quantize(x)
    np.testing.assert_array_equal(c.numpy(), wc)
    same_bits(s.numpy(), wd)


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_linear_broken_tokens_stay_alone(gpu, T):
    """A token with an infinity or NaN is NaN, the others' outputs are the same bits as without it."""
    rng = np.random.default_rng(T)
    K, N = 512, 200
    x = rng.standard_normal((T, K)).astype(np.float32)
    w, ws = Q.quantize(rng.standard_normal((N, K)).astype(np.float32))
    ws[3], w[3] = np.nan, 0            # a channel too
    clean = GemmBufs(gpu, True, x, None, w, ws, None)
    clean.run()
    x[T // 2, 7] = np.inf
    x[0, 500] = np.nan
    b = GemmBufs(gpu, True, x, None, w, ws, None)
    b.run()
    got, want = b.result(), clean.result().copy()
    want[[0, T // 2]] = np.nan
    same_bits(got, want)
    assert np.isnan(got[:, 3]).all() and (T < 2 or np.isfinite(np.delete(got, 3, 1)[1 if T // 2 != 1 else 2]).all())


@pytest.mark.parametrize("T,N", [(4, 4096), (60, 700), (520, 512)])
def test_gemm_onto_its_residual(gpu, T, N):
    rng = np.random.default_rng(T)
    K = 1024
    x, w = rng.integers(-127, 128, (T, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    xs, ws = rng.random(T).astype(np.float32), rng.random(N).astype(np.float32)
    r = rng.standard_normal((T, N)).astype(np.float32) * 100
    b = GemmBufs(gpu, False, x, xs, w, ws, None)
    b.resid = b.out = dev(gpu, np.concatenate([r.ravel(), np.full(64, -3.0, np.float32)]))
    b.run()
    same_bits(b.result(), Q.gemm(x, xs, w, ws, r))


def test_gemm_unaligned_outputs(gpu):
    """out, resid and the scales lie anywhere in memory."""
    rng = np.random.default_rng(3)

    class At:
        def __init__(self, b, off):
            self.b, self.ptr = b, b.ptr + off
    for T, K, N in ((2, 256, 128), (40, 256, 128), (300, 512, 384)):
        x, w = rng.integers(-127, 128, (T, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
        xs, ws = rng.random(T).astype(np.float32), rng.random(N).astype(np.float32)
        r = rng.standard_normal((T, N)).astype(np.float32)
        pad = lambda a: np.concatenate([np.zeros(1, np.float32), a.ravel()])  # noqa: E731
        b = GemmBufs(gpu, False, x, xs, w, ws, r)
        out = dev(gpu, np.zeros(T * N + 3, np.float32))
        gpu.gemm_i8(b.x, At(dev(gpu, pad(xs)), 4), b.w, At(dev(gpu, pad(ws)), 4), At(dev(gpu, pad(r)), 4), T, K, N,
                    At(out, 8), b.wsp, b.n)
        got = out.numpy()
        assert (got[:2] == 0).all() and got[-1] == 0
        same_bits(got[2:-1].reshape(T, N), Q.gemm(x, xs, w, ws, r))


# ------------------------------------------------------------------ the write of the cache

def upload(gpu, p):
    return [dev(gpu, a) for a in (p.k, p.ks, p.v, p.vs)]


def cache_of(gpu, p, bufs, n_pages=None):
    k, ks, v, vs = bufs
    pool = gpu.PagedCache(k, v, gpu.I8, p.n_pages if n_pages is None else n_pages, p.page, p.nkv, p.hd, p.strides())
    return gpu.PagedCacheI8(pool, ks, vs, p.block)


def download(p, bufs):
    q = PoolI8(p.n_pages, p.page, p.nkv, p.hd, p.block, p.order)
    q.k, q.ks, q.v, q.vs = (b.numpy() for b in bufs)
    return q


def same_pool(got, want):
    for name in ("ks", "vs"):
        same_bits(getattr(got, name), getattr(want, name))
    for name in ("k", "v"):
        np.testing.assert_array_equal(getattr(got, name), getattr(want, name))


def append(gpu, p, bufs, qkv, positions, slots, nh, theta=1e4, cos=None, sin=None, qn=None, kn=None, stream=None,
           n_pages=None):
    n = len(slots)
    q = dev(gpu, np.full((n, nh, p.hd), 5.0, np.float32))
    opt = lambda a: None if a is None else dev(gpu, a)  # noqa: E731
    gpu.rope_qknorm_paged_i8(dev(gpu, qkv), n, nh, cache_of(gpu, p, bufs, n_pages), dev(gpu, positions, np.int32),
                             dev(gpu, slots, np.int32), theta, opt(cos), opt(sin), 0 if cos is None else len(cos),
                             opt(qn), opt(kn), 1e-5, q, stream)
    return q.numpy()


def runs_of(rng, lens, page, n_pages):
    """Rows of requests (cached, new), each in pages of its own: positions and slots."""
    perm, at = rng.permutation(n_pages), 0
    pos, slots = [], []
    for ctx, new in lens:
        first = ctx // page
        for i in range(ctx, ctx + new):
            pos.append(i)
            slots.append(perm[at + i // page - first] * page + i % page)
        at += -(-(ctx + new) // page) - first if new else 0
    return np.array(pos, np.int32), np.array(slots, np.int32)


def random_pool(rng, n_pages, page, nkv, hd, block, order="head"):
    p = PoolI8(n_pages, page, nkv, hd, block, order)
    p.k, p.v = (rng.integers(-127, 128, p.k.shape).astype(np.int8) for _ in range(2))
    p.ks, p.vs = (np.exp(rng.standard_normal(p.ks.shape) - 4).astype(np.float32) for _ in range(2))
    return p


@pytest.mark.parametrize("nh,nkv,hd,page,block,order,mode,lens", [
    (32, 8, 128, 16, 16, "head", "theta", [(100, 5)]),
    (8, 2, 128, 64, 16, "head", "table", [(3, 77), (0, 40)]),
    (16, 4, 64, 8, 8, "token", "theta", [(0, 1), (5, 1), (8, 1), (100000, 33)]),
    (5, 5, 64, 128, 64, "head", "none", [(70, 130), (0, 64), (64, 1)]),
    (20, 4, 128, 32, 8, "token", "theta", [(i, 1) for i in range(24)]),
    (6, 1, 128, 4096, 4096, "token", "table", [(200, 300)]),
    (6, 1, 64, 512, 512, "head", "theta", [(0, 513), (17, 18)]),
    (12, 3, 128, 256, 128, "head", "theta", [(120, 17), (1000, 16), (255, 2)]),
    (4, 4, 64, 16, 16, "head", "theta", [(i % 16, 1 + i % 3) for i in range(700)])])  # more rows than one per wave
def test_append(gpu, nh, nkv, hd, page, block, order, mode, lens):
    rng = np.random.default_rng(page + block + nh)
    n_pages = sum(-(-(c + n) // page) - c // page for c, n in lens) + 2
    pos, slots = runs_of(rng, lens, page, n_pages)
    T, pad = len(pos), 3
    qkv = rng.standard_normal((T + pad, (nh + 2 * nkv) * hd)).astype(np.float32)
    qkv *= np.exp(rng.standard_normal((T + pad, 1))).astype(np.float32)
    qkv[T:] = np.nan  # rows of nobody
    cos = sin = None
    if mode == "table":
        ang = rng.random((500, hd // 2)) * 6
        cos, sin = (np.repeat(f(ang), 2, axis=1).astype(np.float32) for f in (np.cos, np.sin))
    qn, kn = (None if mode == "none" else (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    theta = 0.0 if mode == "none" else 1e4
    p = random_pool(rng, n_pages, page, nkv, hd, block, order)
    bufs = upload(gpu, p)
    full = lambda a, f: np.concatenate([a, np.full(pad, f, np.int32)])  # noqa: E731
    got_q = append(gpu, p, bufs, qkv, full(pos, 0), full(slots, -1), nh, theta, cos, sin, qn, kn)
    q, k, v, qm, _ = append_ref(qkv[:T], nh, nkv, hd, pos, theta if cos is None else 0, cos, sin, qn, kn, 1e-5)
    assert (np.abs(got_q[:T] - q) <= APPEND_TOL * qm).all()
    assert (got_q[T:] == 5.0).all()
    p.write(k.astype(np.float32), slots, "k")
    p.write(v.astype(np.float32), slots, "v")
    same_pool(download(p, bufs), p)


def test_append_skipped_rows_end_runs(gpu):
    """Rows without a slot, with one outside the pool or a position outside the tables are skipped; what
    stands on both sides of them are runs of their own."""
    rng = np.random.default_rng(5)
    nh, nkv, hd, page, block = 4, 2, 64, 32, 16
    p = random_pool(rng, 3, page, nkv, hd, block)
    slots = np.r_[32:48, 64:72, 0:6].astype(np.int32)   # a whole block, half of one, a start
    pos = np.arange(len(slots), dtype=np.int32)
    slots[3] = -1                      # positions 0..2 begin the block anew, 4.. come behind
    slots[18] = 3 * page + 4           # outside the pool
    pos[25] = 100                      # outside the tables
    ang = rng.random((60, hd // 2))
    cos, sin = (np.repeat(f(ang), 2, axis=1).astype(np.float32) for f in (np.cos, np.sin))
    qkv = rng.standard_normal((len(slots), (nh + 2 * nkv) * hd)).astype(np.float32)
    # two runs of one call in one block would race: each block here has one run that is kept apart
    keep = [i for i in range(len(slots)) if i not in (3, 18, 25)]
    keep_call = [i for i in keep if not 4 <= i < 16 and not 19 <= i < 24 and not 26 <= i]
    s2 = slots.copy()
    s2[[i for i in range(len(slots)) if i not in keep_call]] = -1
    s2[18], pos2 = slots[18], pos.copy()
    bufs = upload(gpu, p)
    got = append(gpu, p, bufs, qkv, pos2, s2, nh, 0.0, cos, sin)
    q, k, v, qm, _ = append_ref(qkv[keep_call], nh, nkv, hd, pos[keep_call], 0, cos, sin, None, None, 1e-5)
    assert (np.abs(got[keep_call] - q) <= APPEND_TOL * qm).all()
    dead = [i for i in range(len(slots)) if i not in keep_call]
    assert (got[dead] == 5.0).all()
    for which, y in (("k", k), ("v", v)):
        p.write(y.astype(np.float32), slots[keep_call], which)
    same_pool(download(p, bufs), p)


def test_append_one_by_one_and_drafts_again(gpu):
    """A block filled token by token grows its scale as the reference's; drafts that are written again keep
    it; beginning anew gives it back."""
    rng = np.random.default_rng(6)
    nh, nkv, hd, page, block = 8, 2, 128, 16, 16
    p = random_pool(rng, 4, page, nkv, hd, block)
    bufs = upload(gpu, p)
    qkv = (rng.standard_normal((40, (nh + 2 * nkv) * hd)) * np.linspace(0.2, 3, 40)[:, None]).astype(np.float32)
    steps = [(i, i + 1) for i in range(20)] + [(20, 26), (22, 27), (21, 23), (16, 18), (18, 32)]
    for a, b in steps:
        at = np.arange(a, b)
        table = np.array([2, 0])
        slots, pos = (table[at // page] * page + at % page).astype(np.int32), at.astype(np.int32)
        append(gpu, p, bufs, qkv[a:b], pos, slots, nh)
        _, k, v, _, _ = append_ref(qkv[a:b], nh, nkv, hd, pos, 1e4, None, None, None, None, 1e-5)
        p.write(k.astype(np.float32), slots, "k")
        p.write(v.astype(np.float32), slots, "v")
        same_pool(download(p, bufs), p)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_extremes(gpu, hd):
    """Zeros, values whose scale would be too small, infinities and NaN: the block's scale says so, its
    neighbours and other heads keep theirs."""
    rng = np.random.default_rng(7)
    nh, nkv, page, block = 2, 2, 32, 8
    p = random_pool(rng, 6, page, nkv, hd, block)
    lens = [(0, 8), (8, 8), (3, 5), (20, 4), (2, 3), (5, 2)]
    # one request per page
    slots = np.concatenate([r * page + np.arange(c, c + n) for r, (c, n) in enumerate(lens)]).astype(np.int32)
    pos = np.zeros(len(slots), np.int32)
    x = rng.standard_normal((len(slots), nh + 2 * nkv, hd)).astype(np.float32)
    x[0:8, 2:] = 0.0                       # K: 0 / sqrt(eps) = 0, V: 0
    x[8:16, 4] = 1e-44                     # V head 0: too small
    x[16, 5, 3] = np.inf                   # V head 1, behind held tokens
    x[22, 4, hd - 1] = np.nan              # V head 0
    x[25, 2, 0] = -np.inf                  # K head 0: the norm makes it NaN
    x[28, 5] = 3e38                        # V head 1: the largest
    p.vs[5, 0, 0] = np.nan                 # a block that is NaN already stays so
    p.ks[5, 1, 0] = 0.0                    # a block of zeros grows
    p.k[5, 1] = 0
    qkv = x.reshape(len(slots), -1)
    bufs = upload(gpu, p)
    append(gpu, p, bufs, qkv, pos, slots, nh, 0.0)
    with np.errstate(all="ignore"):
        _, k, v, _, _ = append_ref(qkv, nh, nkv, hd, pos, 0, None, None, None, None, 1e-5)
        p.write(k.astype(np.float32), slots, "k")
        p.write(v.astype(np.float32), slots, "v")
    assert np.isnan(p.vs[2, 1, 0]) and np.isnan(p.vs[3, 0, 2]) and np.isnan(p.vs[5, 0, 0]) and p.vs[1, 0, 1] == 0
    same_pool(download(p, bufs), p)


def test_append_out_of_order_stays_in_its_blocks(gpu):
    """Rows that break the order (the same slot twice, backwards): blocks that they do not name are
    untouched."""
    rng = np.random.default_rng(8)
    p = random_pool(rng, 4, 16, 2, 64, 8)
    bufs = upload(gpu, p)
    slots = np.array([5, 4, 3, 3, 3, 40, 40, 41, 33, 32], np.int32)
    qkv = rng.standard_normal((10, (2 + 4) * 64)).astype(np.float32)
    append(gpu, p, bufs, qkv, np.zeros(10, np.int32), slots, 2)
    got = download(p, bufs)
    named = {0, 5, 4}  # blocks of 8 positions
    for b in range(8):
        if b not in named:
            pg, o = divmod(b, 2)
            for a in ("k", "v"):
                np.testing.assert_array_equal(getattr(got, a)[pg, :, 8 * o:8 * o + 8], getattr(p, a)[pg, :, 8 * o:8 * o + 8])
                np.testing.assert_array_equal(getattr(got, a + "s")[pg, :, o], getattr(p, a + "s")[pg, :, o])


# ------------------------------------------------------------------ attention

def make_batch(rng, lens, page, nkv, hd, block, order="head", extra_pages=2, v_spread=1.0, trash=None):
    """lens: (kv, new) per request.  A pool of random codes and scales of differing size; with `trash`, blocks
    that no request has keys in hold that scale."""
    need = [-(-max(kv, 0) // page) for kv, _ in lens]
    p = random_pool(rng, sum(need) + extra_pages, page, nkv, hd, block, order)
    p.ks = (np.exp(0.3 * rng.standard_normal(p.ks.shape)) / 60).astype(np.float32)
    p.vs = (np.exp(v_spread * rng.standard_normal(p.vs.shape)) / 60).astype(np.float32)
    perm = rng.permutation(p.n_pages)
    table = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    used, at = np.zeros((p.n_pages, page // block), bool), 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
        for b in range(-(-max(lens[r][0], 0) // block)):
            used[table[r, b * block // page], b % (page // block)] = True
    if trash is not None:
        for s in (p.ks, p.vs):
            s[np.broadcast_to(~used[:, None], s.shape)] = trash
    q_start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
    return p, table, q_start, np.array([kv for kv, _ in lens], np.int32)


class Ws:
    """A workspace for one PagedBatch, filled with NaN."""

    def __init__(self, gpu, nh, cache, batch):
        self.n = gpu.paged_attention_i8_ws(nh, cache, batch)
        self.b = dev(gpu, np.full(self.n // 4 + 1, np.nan, np.float32))


def attend(gpu, q, p, q_start, kv_len, table, scale, seen=None, max_new=None, sentinel=-3.0, stream=None):
    cache = cache_of(gpu, p, upload(gpu, p))
    bufs = [dev(gpu, a, np.int32) for a in (q_start, kv_len, table)]
    batch = gpu.PagedBatch(len(kv_len), q.shape[0], table.shape[1],
                           int(np.diff(q_start).max()) if max_new is None else max_new, *bufs,
                           seen=None if seen is None else dev(gpu, seen, np.int32))
    out, ws = dev(gpu, np.full(q.shape, sentinel, np.float32)), Ws(gpu, q.shape[1], cache, batch)
    gpu.paged_attention_i8(dev(gpu, q), q.shape[1], cache, batch, scale, out, ws.b, ws.n, stream)
    return out.numpy()


check = Q.check_attention


@pytest.mark.parametrize("block", [8, 16])
@pytest.mark.parametrize("lens", LENS)
def test_attention_lengths(gpu, lens, block):
    rng = np.random.default_rng(len(lens))
    p, table, q_start, kv_len = make_batch(rng, LENS[lens], 16, 2, 128, block)
    pad = 3 if lens != "one" else 0
    q = rng.standard_normal((q_start[-1] + pad, 8, 128)).astype(np.float32) * 2
    args = (q, p, q_start, kv_len, table, 128 ** -0.5)
    check(attend(gpu, *args), *args)


@pytest.mark.parametrize("nh,nkv,hd,page,block,order", [
    (4, 1, 64, 8, 8, "head"), (16, 4, 64, 32, 16, "token"), (8, 8, 128, 16, 16, "token"), (10, 2, 128, 64, 32, "head"),
    (32, 1, 128, 8, 8, "head"), (48, 2, 64, 16, 8, "token"), (3, 1, 64, 4096, 64, "head"),
    (14, 2, 128, 128, 128, "token"), (16, 8, 128, 256, 8, "head"), (8, 2, 128, 4096, 4096, "head")])
def test_attention_layouts(gpu, nh, nkv, hd, page, block, order):
    rng = np.random.default_rng(nh * hd + page)
    for lens in ([(150, 1), (35, 1), (8, 1)], [(90, 3), (33, 2), (160, 20)], [(140, 100), (5, 1)]):
        args = make_batch(rng, lens, page, nkv, hd, block, order)
        q = rng.standard_normal((args[2][-1], nh, hd)).astype(np.float32)
        args = (q, args[0], args[2], args[3], args[1], hd ** -0.5)
        check(attend(gpu, *args), *args)


def test_attention_max_new_only_chooses(gpu):
    rng = np.random.default_rng(5)
    p, table, q_start, kv_len = make_batch(rng, [(300, 90), (200, 1), (60, 8)], 16, 2, 128, 16)
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    args = (q, p, q_start, kv_len, table, 128 ** -0.5)
    for max_new in (0, 1, 8, 90, 2 ** 31):
        check(attend(gpu, *args, max_new=max_new), *args)


def test_attention_seen(gpu):
    """Spans that see past themselves, rows that see nothing (or less than nothing), bounds past
    the keys."""
    rng = np.random.default_rng(6)
    p, table, q_start, kv_len = make_batch(rng, [(200, 120), (50, 4), (130, 1), (64, 40)], 16, 2, 128, 8)
    n = int(q_start[-1])
    q = rng.standard_normal((n + 2, 8, 128)).astype(np.float32)
    seen = rng.integers(0, 220, n + 2).astype(np.int32)
    seen[:64] = 144            # an image's span
    seen[70:75] = (0, -4, 2 ** 31 - 1, 1, -2 ** 31)
    args = (q, p, q_start, kv_len, table, 128 ** -0.5)
    want = check(attend(gpu, *args, seen=seen), *args, seen)
    assert (want[70:72] == 0).all() and (want[74] == 0).all()
    seen[:] = 0                # nothing at all
    assert (attend(gpu, *args, seen=seen)[:n] == 0).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("trash", [np.inf, np.nan, 3e38])
def test_attention_unseen_scales_do_not_matter(gpu, hd, trash):
    """Scales of blocks without keys may be anything; a block that only later rows see makes them, and only
    them, NaN where it is NaN or infinite."""
    rng = np.random.default_rng(7)
    for order, lens in (("head", [(100, 60), (37, 1), (90, 5)]), ("token", [(100, 24), (37, 1), (90, 5)])):
        p, table, q_start, kv_len = make_batch(rng, lens, 16, 2, hd, 8, order, trash=trash)
        q = rng.standard_normal((q_start[-1], 8, hd)).astype(np.float32)
        args = (q, p, q_start, kv_len, table, hd ** -0.5)
        check(attend(gpu, *args), *args)
        if trash == 3e38:
            continue
        n0 = lens[0][1]
        j = 80                     # a block in the middle of request 0's rows
        for which in ("ks", "vs"):
            p2 = PoolI8(p.n_pages, p.page, p.nkv, p.hd, p.block, p.order)
            p2.k, p2.v, p2.ks, p2.vs = p.k, p.v, p.ks.copy(), p.vs.copy()
            getattr(p2, which)[table[0, j // 16], :, (j % 16) // 8] = trash
            got = attend(gpu, q, p2, *args[2:])
            first = max(j - (100 - n0), 0)      # the first row that sees key j
            assert np.isnan(got[first:n0]).all()
            keep = np.r_[0:first, n0:len(q)]
            sub_start = np.array([0, first, first + 1, first + 6], np.int32)
            sub_len = np.array([100 - n0 + first, 37, 90], np.int32)
            if first == 0:
                keep, sub_start, sub_len, t2 = np.r_[n0:len(q)], sub_start[1:], sub_len[1:], table[1:]
            else:
                t2 = table
            check(got[keep], q[keep], p, sub_start, sub_len, t2, hd ** -0.5)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_magnitudes(gpu, hd):
    """Scales of differing size, blocks of zeros, scores far apart, ties."""
    rng = np.random.default_rng(8)
    for k_scale, v_scale, q_scale in ((1e-3, 1e-4, 1.0), (30.0, 1e3, 0.05), (1.0, 1.0, 40.0), (0.0, 1.0, 1.0),
                                      (1.0, 0.0, 1.0), (1.0, 2.0 ** -50, 1.0), (1.0, 2.0 ** 33, 1.0),
                                      (2.0 ** 40, 1.0, 2.0 ** -40)):
        p, table, q_start, kv_len = make_batch(rng, [(150, 1), (100, 40), (70, 6)], 16, 2, hd, 16, v_spread=0.3)
        p.ks, p.vs = p.ks * np.float32(k_scale), p.vs * np.float32(v_scale)
        q = (rng.standard_normal((q_start[-1], 8, hd)) * q_scale).astype(np.float32)
        args = (q, p, q_start, kv_len, table, hd ** -0.5)
        check(attend(gpu, *args), *args)
    # neighbouring blocks' scales a factor 1e8 apart, some zero
    p, table, q_start, kv_len = make_batch(rng, [(200, 50), (90, 2), (40, 1)], 16, 2, hd, 8)
    for name in ("ks", "vs"):
        f = np.float32(10.0) ** rng.integers(-4, 5, p.ks.shape).astype(np.float32)
        f[rng.random(f.shape) < 0.1] = 0
        setattr(p, name, (getattr(p, name) * f).astype(np.float32))
    q = (rng.standard_normal((q_start[-1], 8, hd)) * 1e-4).astype(np.float32)
    args = (q, p, q_start, kv_len, table, hd ** -0.5)
    check(attend(gpu, *args), *args)


def test_attention_small_weights_on_large_values(gpu):
    """A row whose weight lies almost whole on keys of small values, beside keys of large ones that it hardly
    sees, and the other way round."""
    rng = np.random.default_rng(81)
    for new in (1, 6, 90):
        p, table, q_start, kv_len = make_batch(rng, [(160, new)], 16, 2, 128, 16)
        p.vs[table[0, ::2]] *= np.float32(2.0 ** 20)
        p.vs[table[0, 1::2]] *= np.float32(2.0 ** -20)
        p.ks[table[0, ::2]] *= np.float32(1e-3)
        q = (rng.standard_normal((q_start[-1], 8, 128)) * 8).astype(np.float32)
        args = (q, p, q_start, kv_len, table, 128 ** -0.5)
        check(attend(gpu, *args), *args)


def test_attention_bad_pages(gpu):
    """Positions whose page does not exist hold no key."""
    rng = np.random.default_rng(9)
    p, table, q_start, kv_len = make_batch(rng, [(150, 1), (100, 40), (70, 6), (40, 2)], 16, 2, 128, 8)
    table[0, 2] = -1
    table[1, 5] = p.n_pages
    table[1, 0] = 2 ** 31 - 1
    table[2, :] = -2 ** 31
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    args = (q, p, q_start, kv_len, table, 128 ** -0.5)
    want = check(attend(gpu, *args), *args)
    assert (want[41:47] == 0).all()


def test_attention_length_past_the_table(gpu):
    rng = np.random.default_rng(10)
    p, table, q_start, kv_len = make_batch(rng, [(64, 3), (64, 2)], 16, 2, 64, 16)
    kv_len[:] = (10 ** 9, -5)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    seen = np.array([64, 60, 10 ** 9, 3, 4], np.int32)
    args = (q, p, q_start, kv_len, table, 0.125)
    check(attend(gpu, *args, seen=seen), *args, seen)


def test_attention_many_requests(gpu):
    rng = np.random.default_rng(12)
    lens = [(int(rng.integers(0, 40)), 1) for _ in range(4096)]
    p, table, q_start, kv_len = make_batch(rng, lens, 8, 1, 64, 8)
    q = rng.standard_normal((q_start[-1], 4, 64)).astype(np.float32)
    args = (q, p, q_start, kv_len, table, 0.125)
    check(attend(gpu, *args), *args)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_req,new,kv", [(1, 1, 3000), (1, 4, 4000), (1, 6, 2500), (3, 4, 1500), (32, 1, 300), (33, 1, 300),
                                          (32, 4, 200), (33, 4, 200), (32, 6, 150), (33, 6, 150), (1, 24, 900), (2, 32, 700),
                                          (1, 64, 5000), (1, 130, 3000), (2, 96, 1200), (7, 33, 300)])
def test_attention_pieces_and_workers(gpu, hd, n_req, new, kv):
    """Few and many items (request x kv head x rows) for the streams' workers, and items in many pieces."""
    rng = np.random.default_rng(n_req * 1000 + new)
    lens = [(kv + int(rng.integers(0, 60)), new) for _ in range(n_req)]
    p, table, q_start, kv_len = make_batch(rng, lens, 16, 8, hd, 16)
    q = rng.standard_normal((q_start[-1], 32, hd)).astype(np.float32)
    args = (q, p, q_start, kv_len, table, hd ** -0.5)
    check(attend(gpu, *args), *args)


@pytest.mark.parametrize("lens,block", [([(9000, 1), (20, 1)], 64), ([(20000, 3)], 16), ([(5000, 70)], 32)])
def test_attention_long(gpu, lens, block):
    rng = np.random.default_rng(13)
    p, table, q_start, kv_len = make_batch(rng, lens, 64, 1, 128, block)
    q = rng.standard_normal((q_start[-1], 4, 128)).astype(np.float32) * 2
    args = (q, p, q_start, kv_len, table, 128 ** -0.5)
    check(attend(gpu, *args), *args)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_rows_around_the_choices(gpu, hd):
    """Row counts on both sides of every choice of kernel and tile."""
    rng = np.random.default_rng(64)
    for news in ((4, 4, 4), (5, 1, 3), (8, 8, 2), (9, 8, 2), (16, 2, 2), (17, 16, 1), (32, 31, 2), (33, 9, 8), (64, 20, 1),
                 (65, 64, 3), (128, 7, 1), (129, 8, 9)):
        lens = [(n + int(rng.integers(0, 80)), n) for n in news]
        for part in (lens, lens[:2], lens[:1]):
            p, table, q_start, kv_len = make_batch(rng, part, 16, 2, hd, 8)
            q = rng.standard_normal((q_start[-1], 8, hd)).astype(np.float32)
            args = (q, p, q_start, kv_len, table, hd ** -0.5)
            check(attend(gpu, *args), *args)


@pytest.mark.parametrize("nh,nkv,page,block,order", [(8, 2, 8, 8, "head"), (10, 2, 64, 16, "token"),
                                                     (16, 1, 32, 32, "head")])
def test_attention_long_chunks_of_small_heads(gpu, nh, nkv, page, block, order):
    rng = np.random.default_rng(63 + nh)
    n = 2100 // (nh // nkv) + 5
    lens = [(n + 61, n), (40, 1), (90, 3), (0, 0), (200, 33)]
    p, table, q_start, kv_len = make_batch(rng, lens, page, nkv, 64, block, order, trash=np.nan)
    q = rng.standard_normal((q_start[-1] + 2, nh, 64)).astype(np.float32)
    args = (q, p, q_start, kv_len, table, 0.125)
    check(attend(gpu, *args), *args)
    seen = np.minimum(rng.integers(0, n + 90, q_start[-1] + 2), np.repeat(kv_len, np.diff(q_start)).max()).astype(np.int32)
    seen[5:40] = 0
    check(attend(gpu, *args, seen=seen), *args, seen)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_broken_queries(gpu, new):
    """An infinity or NaN in a row's query makes that head's output NaN, and no other."""
    rng = np.random.default_rng(65)
    p, table, q_start, kv_len = make_batch(rng, [(120, new), (50, 1)], 16, 2, 128, 16)
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    args = (p, q_start, kv_len, table, 128 ** -0.5)
    clean = attend(gpu, q, *args)
    q[0, 2, 5], q[new - 1, 6, 127] = np.inf, np.nan
    got = attend(gpu, q, *args)
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 2] = bad[new - 1, 6] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


def test_offsets_past_32_bits(gpu):
    """Pages 2^32 bytes apart: write and attention reach them."""
    rng = np.random.default_rng(14)
    hd, page, stride, T, nh = 64, 16, 1 << 32, 32, 4
    far = [gpu.Buf(stride + page * hd), dev(gpu, np.ones((2, 1, 2), np.float32)), gpu.Buf(stride + page * hd),
           dev(gpu, np.ones((2, 1, 2), np.float32))]
    p = PoolI8(2, page, 1, hd, 8)
    near = upload(gpu, p)
    qkv = rng.standard_normal((T, (nh + 2) * hd)).astype(np.float32)
    slots = pos = np.arange(T, dtype=np.int32)
    outs = []
    for bufs, strides in ((far, (stride, hd, hd)), (near, p.strides())):
        cache = gpu.PagedCacheI8(gpu.PagedCache(bufs[0], bufs[2], gpu.I8, 2, page, 1, hd, strides), bufs[1], bufs[3], 8)
        qb = gpu.Buf.empty((T, nh, hd))
        gpu.rope_qknorm_paged_i8(dev(gpu, qkv), T, nh, cache, dev(gpu, pos), dev(gpu, slots), 1e4, None, None, 0, None,
                                 None, 1e-5, qb)
        for new in (T, 1):
            arrays = [dev(gpu, a, np.int32) for a in ([0, new], [T], [[1, 0]])]
            batch = gpu.PagedBatch(1, T, 2, new, *arrays)
            out, ws = dev(gpu, np.zeros((T, nh, hd), np.float32)), Ws(gpu, nh, cache, batch)
            gpu.paged_attention_i8(qb, nh, cache, batch, 0.125, out, ws.b, ws.n)
            outs.append(out.numpy())
    assert np.abs(outs[0]).max() > 0.1
    np.testing.assert_array_equal(outs[0], outs[2])
    np.testing.assert_array_equal(outs[1], outs[3])


def test_attention_same_result_each_time(gpu):
    rng = np.random.default_rng(15)
    p, table, q_start, kv_len = make_batch(rng, [(900, 1), (500, 60), (40, 3)], 16, 2, 128, 16)
    q = rng.standard_normal((q_start[-1], 8, 128)).astype(np.float32)
    first = attend(gpu, q, p, q_start, kv_len, table, 0.1)
    for _ in range(3):
        np.testing.assert_array_equal(attend(gpu, q, p, q_start, kv_len, table, 0.1), first)


# ------------------------------------------------------------------ together

class Step:
    """A server's step in 8 bits: projection, write, attention, output projection onto the residual."""

    def __init__(self, gpu, seed, lens, page=16, block=16, nh=8, nkv=2, hd=64, H=256):
        rng = np.random.default_rng(seed)
        self.gpu, self.nh, self.hd, self.H = gpu, nh, hd, H
        self.p = random_pool(rng, sum(-(-kv // page) for kv, _ in lens) + 1, page, nkv, hd, block)
        self.p.ks[:] = self.p.vs[:] = np.float32(0.02)
        perm, at = rng.permutation(self.p.n_pages), 0
        width = max(-(-kv // page) for kv, _ in lens)
        self.table = np.full((len(lens), width), -1, np.int32)
        pos, slots = [], []
        for r, (kv, n) in enumerate(lens):
            need = -(-kv // page)
            self.table[r, :need] = perm[at:at + need]
            at += need
            for i in range(kv - n, kv):
                pos.append(i)
                slots.append(self.table[r, i // page] * page + i % page)
        self.pos, self.slots = np.array(pos, np.int32), np.array(slots, np.int32)
        self.q_start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
        self.kv = np.array([kv for kv, _ in lens], np.int32)
        T, self.nq = len(pos), (nh + 2 * nkv) * hd
        self.T = T
        self.x = rng.standard_normal((T, H)).astype(np.float32)
        self.wq, self.wqs = Q.quantize(rng.standard_normal((self.nq, H)).astype(np.float32))
        self.wo, self.wos = Q.quantize(rng.standard_normal((H, nh * hd)).astype(np.float32) * 0.1)
        self.bufs = upload(gpu, self.p)
        self.cache = cache_of(gpu, self.p, self.bufs)
        d = lambda a: dev(gpu, a)  # noqa: E731
        self.batch = gpu.PagedBatch(len(lens), T, width, int(np.diff(self.q_start).max()), d(self.q_start), d(self.kv),
                                    d(self.table), d(self.pos), d(self.slots))
        self.dx, self.dwq, self.dwqs, self.dwo, self.dwos = d(self.x), d(self.wq), d(self.wqs), d(self.wo), d(self.wos)
        self.qkv, self.q, self.att, self.out = (gpu.Buf.empty((T, n)) for n in (self.nq, nh * hd, nh * hd, H))
        self.n1, self.n2 = gpu.linear_i8_ws(T, H, self.nq), gpu.linear_i8_ws(T, nh * hd, H)
        self.ws1, self.ws2 = gpu.Buf(self.n1), gpu.Buf(self.n2)
        self.wsa = Ws(gpu, nh, self.cache, self.batch)

    def run(self, stream=None):
        g, b = self.gpu, self.batch
        g.linear_i8(self.dx, self.dwq, self.dwqs, None, self.T, self.H, self.nq, self.qkv, self.ws1, self.n1, stream)
        g.rope_qknorm_paged_i8(self.qkv, self.T, self.nh, self.cache, b.keep[3], b.keep[4], 1e4, None, None, 0, None,
                               None, 1e-5, self.q, stream)
        g.paged_attention_i8(self.q, self.nh, self.cache, b, self.hd ** -0.5, self.att, self.wsa.b, self.wsa.n, stream)
        g.linear_i8(self.att, self.dwo, self.dwos, self.dx, self.T, self.nh * self.hd, self.H, self.out, self.ws2,
                    self.n2, stream)

    def check(self):
        """Each call against its reference, from what the one before it gave."""
        xq, xs = Q.quantize(self.x)
        qkv = self.qkv.numpy()
        same_bits(qkv, Q.gemm(xq, xs, self.wq, self.wqs))
        q, k, v, qm, _ = append_ref(qkv, self.nh, self.p.nkv, self.hd, self.pos, 1e4, None, None, None, None, 1e-5)
        got_q = self.q.numpy().reshape(q.shape)
        assert (np.abs(got_q - q) <= APPEND_TOL * qm).all()
        self.p.write(k.astype(np.float32), self.slots, "k")
        self.p.write(v.astype(np.float32), self.slots, "v")
        same_pool(download(self.p, self.bufs), self.p)
        att = self.att.numpy()
        check(att.reshape(q.shape), got_q, self.p, self.q_start, self.kv, self.table, self.hd ** -0.5)
        aq, asc = Q.quantize(att)
        same_bits(self.out.numpy(), Q.gemm(aq, asc, self.wo, self.wos, self.x))


@pytest.mark.parametrize("lens", [[(100, 1), (37, 1), (5, 1)], [(90, 5), (64, 3), (16, 16)], [(200, 150), (30, 1)]])
def test_step(gpu, lens):
    s = Step(gpu, 21, lens)
    s.run()
    s.check()


def test_two_streams_at_once(gpu):
    steps = [Step(gpu, 30 + i, [(120, 40), (60, 1)]) for i in range(2)]
    streams = [gpu.Stream() for _ in steps]
    gpu.sync()
    for _ in range(3):  # a write again gives the same codes: the block begins anew, or its scale has grown already
        for s, st in zip(steps, streams):
            s.run(st.h)
    for s, st in zip(steps, streams):
        st.synchronize()
        s.check()


def test_captured_step(gpu):
    """A step in a graph, replayed between eager work: the same bits each time."""
    s, other = Step(gpu, 40, [(120, 40), (60, 1), (33, 2)]), Step(gpu, 41, [(50, 3)])
    st = gpu.Stream()
    s.run(st.h)
    st.synchronize()
    want = s.out.numpy()
    g = gpu.Graph(st, lambda: s.run(st.h))
    for i in range(4):
        other.run()
        gpu.sync()
        s.out.zero()
        gpu.sync()
        g.launch()
        st.synchronize()
        np.testing.assert_array_equal(s.out.numpy(), want)
    s.check()
    g.close()
