"""Paged serving on the GPU at the ends of its ranges, against plain numpy in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from paged_ref import BF16, EPS32, F16, F32, Pool
from test_paged_gpu import (PlanBufs, VerifyBufs, Ws, attend, cache_of, check_attention, dev, greedy_model, make_batch,
                            upload)

pytestmark = pytest.mark.gpu


def test_attention_long_request_in_tiles_of_one_token(gpu):
    """50000 rows of one request, 16 query heads per kv head, in the streams' tiles of 16 rows
    (max_new only chooses the kernel): a tile is one token, and the tiles' nominal lengths add up
    to 1.25e9.  Every row sees at most 40 keys, so that plain products can follow."""
    rng = np.random.default_rng(70)
    n, nh, hd, page = 50000, 16, 64, 64
    pool, table, q_start, kv_len = make_batch(rng, [(n, n)], page, 1, hd, F16)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    seen = rng.integers(0, 41, n).astype(np.int32)
    got = attend(gpu, q, pool, q_start, kv_len, table, hd ** -0.5, seen=seen, max_new=1)
    k, v = (np.stack([R.decode(pool.at(a, table[0, 0], i), F16)[0] for i in range(40)]) for a in (pool.k, pool.v))
    for t0 in range(0, n, 5000):
        x = q[t0:t0 + 5000].astype(np.float64)
        s = x @ k.T * hd ** -0.5
        gone = np.arange(40) >= seen[t0:t0 + 5000, None, None]
        w = np.exp(np.where(gone, -np.inf, s))
        w /= np.maximum(w.sum(-1, keepdims=True), 1e-300)
        bound = R.attention_bound((np.abs(x) @ np.abs(k).T).max(-1) * hd ** -0.5, w @ np.abs(v), hd, 40)
        assert (np.abs(got[t0:t0 + 5000] - w @ v) <= bound).all()


# max_new that sends a request of 40 rows and 4 query heads per kv head to the streams' tiles of 16
# rows, of 32, and to the tiles of 256
KERNELS = {"stream16": 1, "stream32": 8, "tiles": 1 << 20}


def at(pool, a, table, r, j):
    """Storage [nkv][hd] of a's (pool.k or pool.v) key j of request r."""
    return pool.at(a, table[r, j // pool.page], j % pool.page)


def scale_values(pool, f):
    """Values of a pool by a factor per [page][position]."""
    pool.v = R.encode(R.decode(pool.v, pool.wtype).astype(np.float32) * f[:, None, :, None].astype(np.float32), pool.wtype)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("wtype,scale", [(F32, 1.0), (F32, 1e-6), (F32, 1e-10), (F16, 1.0), (F16, 1e-3), (BF16, 1.0),
                                         (BF16, 1e-6), (BF16, 1e-10)])
def test_attention_zero_value_rows(gpu, wtype, scale, kernel):
    """Keys whose value is zero take their weight and leave the others' accuracy alone, whatever size
    the others' values have."""
    rng = np.random.default_rng(71)
    for zeros in ((150,), range(0, 300, 3), range(300)):
        pool, table, q_start, kv_len = make_batch(rng, [(300, 40)], 16, 2, 128, wtype)
        scale_values(pool, np.full((pool.n_pages, 16), scale))
        for j in zeros:
            at(pool, pool.v, table, 0, j)[:] = 0
        q = (rng.standard_normal((40, 8, 128)) * 0.5).astype(np.float32)
        args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
        check_attention(attend(gpu, *args, max_new=KERNELS[kernel]), *args)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("small,big,kv", [(0.01, 1e28, 300), (0.01, 1e28, 3000), (1e-15, 1e10, 300), (1e-17, 3e10, 3000),
                                          (0.01, 1e38, 300), (1e-6, 1e12, 3000)])
@pytest.mark.parametrize("wtype", [F32, BF16])
def test_attention_values_of_very_different_size(gpu, wtype, small, big, kv, kernel):
    """Equal scores: the weight of a small value counts in full beside a large one, in one piece and
    over many, and rows that do not see the large one keep the small ones' accuracy."""
    rng = np.random.default_rng(72)
    pool, table, q_start, kv_len = make_batch(rng, [(kv, 40)], 16, 2, 128, wtype)
    pool.k[:] = 0
    f = np.full((pool.n_pages, 16), small)
    for j in [kv - 30] if big > 1e30 else [kv - 30, 40, kv // 2]:
        f[table[0, j // 16], j % 16] = big
    scale_values(pool, f)
    q = rng.standard_normal((40, 8, 128)).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    check_attention(attend(gpu, *args, max_new=KERNELS[kernel]), *args)
    seen = rng.integers(0, kv + 1, 40).astype(np.int32)
    seen[:9] = (40, 41, 39, 7, kv // 2, kv // 2 + 1, kv - 30, kv - 29, kv)
    check_attention(attend(gpu, *args, seen=seen, max_new=KERNELS[kernel]), *args, seen)


def check_rows(got, want, bound, rows):
    """Rows x heads of a mask: finite, and within bound of want."""
    assert np.isfinite(got[rows]).all() and (np.abs(got - want)[rows] <= bound[rows]).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_infinities_make_rows_nan(gpu, wtype, sign, kernel):
    """One infinite element of a key or of q: NaN wherever a row sees it, whatever its product's sign,
    whichever kernel, on the key-by-key path too; other rows and heads notice nothing."""
    rng = np.random.default_rng(73)
    kv, n, j = 300, 40, 275              # row i sees keys 0 .. 260 + i
    for odd_value in (False, True):
        pool, table, q_start, kv_len = make_batch(rng, [(kv, n)], 16, 2, 128, wtype)
        q = rng.standard_normal((n, 8, 128)).astype(np.float32)
        q[:, :, 17] = np.where(rng.random((n, 8)) < 0.5, 1.0, -1.0)
        args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
        want, dot, pv = R.attention(*args)
        bound = R.attention_bound(dot, pv, 128, kv)
        hit = np.zeros((n, 8), bool)
        hit[j - 260:, :4] = True
        key, value = at(pool, pool.k, table, 0, j), at(pool, pool.v, table, 0, kv - 1)
        key[0, 17] = R.encode(np.float32([sign * np.inf]), wtype)[0]
        if odd_value:                    # of the last row's own key: the pieces with it go key by key
            value[0, :] = R.encode(np.float32([np.nan]), wtype)[0]
        got = attend(gpu, *args, max_new=KERNELS[kernel])
        assert np.isnan(got[hit]).all()
        check_rows(got, want, bound, ~hit)
        # q: every key has the other sign there, so that every score is -inf
        pool.k[..., 17] = R.encode(np.float32([-sign]), wtype)[0]
        q[:, :, 17] = 1.0
        want, dot, pv = R.attention(*args)
        bound = R.attention_bound(dot, pv, 128, kv)
        hit[:] = False
        q[7, 2, 17] = q[39, 5, 17] = sign * np.inf
        hit[7, 2] = hit[39, 5] = True
        got = attend(gpu, *args, max_new=KERNELS[kernel])
        assert np.isnan(got[hit]).all()
        if odd_value:
            hit[39, :4] = True           # they see the value that is NaN
        check_rows(got, want, bound, ~hit)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_large_queries(gpu, wtype, kernel):
    """Scores of 1e35: the best key takes all, where it leads by more than an f32 product's error."""
    rng = np.random.default_rng(74)
    pool, table, q_start, kv_len = make_batch(rng, [(300, 40)], 16, 2, 128, wtype)
    q = (rng.standard_normal((40, 8, 128)) * 1e35).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, 128 ** -0.5)
    got = attend(gpu, *args, max_new=KERNELS[kernel])
    assert np.isfinite(got).all()
    k = np.stack([R.decode(at(pool, pool.k, table, 0, j), wtype) for j in range(300)])
    v = np.stack([R.decode(at(pool, pool.v, table, 0, j), wtype) for j in range(300)])
    clear = 0
    for t in range(40):
        for h in range(8):
            s = k[:261 + t, h // 4] @ q[t, h].astype(np.float64)
            best = np.argsort(s)[-2:]
            if s[best[1]] - s[best[0]] > (128 + 8) * 2 * EPS32 * (np.abs(k[:, h // 4]) @ np.abs(q[t, h])).max() * 2:
                clear += 1
                # a weight of one, in pieces of 22 bits, and the division; small elements to 2^-38 of
                # their row's largest
                x = v[best[1], h // 4]
                assert (np.abs(got[t, h] - x) <= 8 * EPS32 * np.abs(x) + 2.0 ** -38 * np.abs(x).max()).all()
    assert clear > 250


def layer(gpu):
    att = gpu.Attn(512, 8, 2, 128, 32)
    att.synth(0, seed=5, std=0.05)
    return att


def test_layer_rows_of_nobody_keep_nothing_of_earlier_calls(gpu):
    """Rows behind the last sequence give zeros, and a row without a slot the same as in a new context;
    the other rows' bits do not depend on what ran before either."""
    rng = np.random.default_rng(75)
    nh, nkv, hd, page = 8, 2, 128, 16
    i32 = lambda a: dev(gpu, a, np.int32)  # noqa: E731
    x = rng.standard_normal((12, 512)).astype(np.float32)
    pool = Pool(4, page, nkv, hd, F16)

    def step(att, x, n, slots):
        kb, vb = upload(gpu, pool)
        cache = cache_of(gpu, pool, kb, vb)
        batch = gpu.PagedBatch(1, len(x), 2, n, i32([0, n]), i32([n]), i32([1, 3]), i32(range(len(x))), i32(slots))
        ws, out = Ws(gpu, nh, cache, batch), dev(gpu, np.full(x.shape, 7.0, np.float32))
        att.forward_paged(dev(gpu, x), cache, batch, out, ws.b, ws.n)
        return out.numpy()

    slots = page + np.arange(12)
    few = np.where(np.arange(12) < 8, slots, -1)
    few[5] = 4 * page + 1                                # outside the pool: no key, and no query
    for padding in (few, np.where(np.arange(12) == 5, -1, slots)):  # rows of nobody with slots too
        used, new = layer(gpu), layer(gpu)
        step(used, np.full((12, 512), np.nan, np.float32), 12, slots)
        got, want = step(used, x, 8, padding), step(new, x, 8, padding)
        assert np.isfinite(got).all() and (got[8:] == 0).all()
        np.testing.assert_array_equal(got, want)
        used.close()
        new.close()


def test_model_that_drops_tokens_is_refused(gpu):
    """Under token dropping a request's experts depend on the rows beside it, those of nobody among
    them: refused, with nothing written."""
    H, nh, nkv, hd, V, L, T = 256, 8, 2, 64, 500, 2, 32
    mc = gpu.Config(H, 128, 8, 2, L, T, gpu.F32, 1, 1, 1.0, 0, 0, 0, 0)
    mc.drop_tokens, mc.capacity_factor, mc.min_capacity = 1, 1.0, 1
    ac = gpu.AttnConfig(H, nh, nkv, hd, L, T, 0, 1e-5, 10000.0, 0)
    h = C.c_void_p()
    gpu.check(gpu.lib().hy_model_create(C.byref(gpu.ModelConfig(mc, ac, V)), C.byref(h)))
    m = gpu.Model.__new__(gpu.Model)
    m.h, m.H, m.V, m.L = h, H, V, L
    m.attn = gpu.Attn(H, nh, nkv, hd, T, handle=C.c_void_p(gpu.lib().hy_model_attn(h)))
    m.moe = gpu.Moe.__new__(gpu.Moe)
    m.moe.h, m.moe.owned = gpu.lib().hy_model_moe(h), False
    m.moe.H, m.moe.I, m.moe.E, m.moe.K, m.moe.wtype = H, 128, 8, 2, gpu.F32
    m.synth_globals(seed=3, std=0.5)
    for l in range(L):
        m.attn.synth(l, seed=7 + l, std=0.08)
        m.moe.synth(l, seed=9 + l, std=0.05)
    pool = Pool(4 * L, 16, nkv, hd, F32, fill=3.0)
    kb, vb = upload(gpu, pool)
    i32 = lambda *a: dev(gpu, np.array(a, np.int32))  # noqa: E731
    cache = gpu.PagedCache(kb, vb, F32, 4, 16, nkv, hd, layer_stride=4 * nkv * 16 * hd)
    batch = gpu.PagedBatch(1, 2, 4, 2, i32(0, 2), i32(2), i32(0, 1, 2, 3), i32(0, 1), i32(0, 1))
    ws, logits = Ws(gpu, nh, cache, batch), dev(gpu, np.full((2, V), 8.0, np.float32))
    with pytest.raises(gpu.HyError, match="drop"):
        m.forward_paged(i32(4, 5), cache, batch, logits, ws.b, ws.n)
    gpu.sync()
    np.testing.assert_array_equal(kb.numpy(), pool.k)
    assert (logits.numpy() == 8.0).all()
    m.close()


def test_layers_that_would_overlap_are_refused(gpu):
    """A context of several layers: pools that share elements are refused for every layer, pools side by
    side, interleaved by page, by position and by head are taken."""
    H, nh, nkv, hd, page, n_pages, L = 256, 8, 2, 64, 16, 4, 3
    att = gpu.Attn(H, nh, nkv, hd, 16, num_layers=L)
    for l in range(L):
        att.synth(l, seed=5 + l, std=0.05)
    one = n_pages * nkv * page * hd
    kb, vb = gpu.Buf(2 * L * (one + 64)), gpu.Buf(2 * L * (one + 64))
    i32 = lambda n: dev(gpu, np.zeros(n, np.int32))  # noqa: E731
    x, out = dev(gpu, np.zeros((8, H), np.float32)), gpu.Buf.empty((8, H))

    def call(layer, layer_stride, strides=(0, 0, 0)):
        c = gpu.PagedCache(kb, vb, F16, n_pages, page, nkv, hd, strides, layer_stride)
        b = gpu.PagedBatch(1, 8, 4, 8, i32(2), i32(1), i32(4), i32(8), i32(8))
        ws = Ws(gpu, nh, c, b)
        att.forward_paged(x, c, b, out, ws.b, ws.n, layer=layer)

    per = nkv * page * hd                                   # of a page
    good = [(one, (0, 0, 0)), (one + 64, (0, 0, 0)),        # one behind the other
            (per, (L * per, page * hd, hd)),                # a page's layers together
            (hd, (L * per, L * page * hd, L * hd)),         # a position's
            (page * hd, (L * per, L * page * hd, hd)),      # a head's
            (per, (L * per, hd, nkv * hd))]                 # pages of [position][head], their layers together
    for stride, strides in good:
        for layer in range(L):
            call(layer, stride, strides)
    bad = [(0, (0, 0, 0)), (8, (0, 0, 0)), (hd, (0, 0, 0)), (per, (0, 0, 0)), (one - 8, (0, 0, 0)),
           (per, ((L - 1) * per, page * hd, hd)),           # too few elements between pages
           (per - 8, (L * per, page * hd, hd)),
           (hd - 8, (L * per, L * page * hd, L * hd)),
           (hd, (L * per, L * page * hd, (L - 1) * hd))]
    for stride, strides in bad:
        for layer in range(L):
            with pytest.raises(gpu.HyError, match="layer_stride"):
                call(layer, stride, strides)
    gpu.sync()
    att.close()


@pytest.mark.parametrize("probs", [False, True])
def test_verify_row_starts_out_of_order(gpu, probs):
    """Starts that go back leave rows that no request's slices were written for: over a workspace of
    zeros their tokens are -1 or of the vocabulary, and nothing outside the logits is read."""
    rng = np.random.default_rng(76)
    V, n = 20000, 9
    logits = rng.standard_normal((n, V)).astype(np.float32)
    draft = np.full((n, V), 1 / V, np.float32) if probs else None
    for starts in ([0, 3, 1, 4], [5, 2, 9, 0], [0, 9, 9, 3], [7, 9, 0, 5]):
        b = VerifyBufs(gpu, logits, draft, np.arange(n), starts, None, np.full(n, 0.9), np.full(3, 0.5), n)
        b.ws = dev(gpu, np.zeros(b.n // 4 + 1, np.float32))
        b.run()
        accepted, tokens = b.result()
        assert ((accepted >= -1) & (accepted < n)).all() and ((tokens >= -1) & (tokens < V)).all()


def test_server_step_with_prompts_drafts_and_waiting_requests(gpu):
    """The loop that include/hy_paged.h describes, with everything in one step: prompts in pieces,
    last tokens with drafts, requests that find no pages and come again (where nobody finds any, the last
    one gives up its pages and starts again with what it has), rows of nobody.
    Verification takes all rows' logits as they are, two row starts per request.  The text equals
    greedy decoding by hy_model_forward."""
    m, nh, nkv, hd, V, L = greedy_model(gpu)
    rng = np.random.default_rng(77)
    prompts = [rng.integers(0, V, n).tolist() for n in (9, 23, 1, 14)]
    n, steps, piece, max_drafts = len(prompts), 12, 8, 4
    asked, want = [len(p) for p in prompts], []
    for p in prompts:
        seq = list(p)
        for _ in range(steps):
            lb = gpu.Buf.empty((len(seq), V))
            m.forward(dev(gpu, seq, np.int32), len(seq), lb)
            last = np.sort(lb.numpy()[-1])
            assert last[-1] - last[-2] > 1e-4 * abs(last[-1])  # no near tie decides
            seq.append(int(np.argmax(lb.numpy()[-1])))
        want.append(seq[len(p):])
    page, n_pages, max_pages = 8, 8, 8
    pool = Pool(n_pages * L, page, nkv, hd, F32, fill=np.nan)
    kb, vb = upload(gpu, pool)
    cache = gpu.PagedCache(kb, vb, F32, n_pages, page, nkv, hd, layer_stride=n_pages * nkv * page * hd)
    held, table = np.zeros(n, np.int32), np.zeros((n, max_pages), np.int32)
    free, n_free, cached = rng.permutation(n_pages).astype(np.int32), n_pages, np.zeros(n, np.int64)
    done, kinds, accepted_drafts = [[] for _ in prompts], set(), 0
    drafts = [[] for _ in prompts]
    for _ in range(80):
        if min(len(d) for d in done) >= steps:
            break
        rows, context = [], []
        for r, p in enumerate(prompts):                      # p: what runs without drafts
            if len(done[r]) >= steps:                        # ended: its pages go back
                rows.append([])
                context.append(0)
                cached[r] = 0
            elif cached[r] < len(p):                         # a piece of the prompt
                rows.append(p[cached[r]:cached[r] + piece])
                context.append(len(rows[-1]) - (cached[r] + len(rows[-1]) == len(p)))
            else:
                rows.append([done[r][-1]] + drafts[r])
                context.append(0)
        new = np.array([len(x) for x in rows])
        n_rows = int(new.sum()) + 2
        plan = PlanBufs(gpu, cached, new, held, table, free, n_free, n_rows, page, n_pages)
        plan.run(in_place=True)
        batch = gpu.PagedBatch(n, n_rows, max_pages, int(new.max()), plan.q_start, plan.kv_len, plan.table,
                               plan.positions, plan.slots)
        ids = np.array(sum(rows, []) + [V + 3, -1], np.int32)
        logits, ws = gpu.Buf.empty((n_rows, V)), Ws(gpu, nh, cache, batch)
        m.forward_paged(dev(gpu, ids), cache, batch, logits, ws.b, ws.n)
        start = np.concatenate([[0], np.cumsum(new)])
        starts = np.append(np.stack([start[:-1], start[:-1] + context], 1).ravel(), start[-1])
        ver = VerifyBufs(gpu, np.zeros((n_rows, V), np.float32), None, ids, starts, np.zeros(2 * n), np.zeros(n_rows),
                         np.zeros(2 * n), 1 + max_drafts)
        ver.logits = logits
        ver.run()
        accepted, tokens = (x[1::2] for x in ver.result())
        held, table, free, n_free = plan.held.numpy(), plan.table.numpy(), plan.free.numpy(), int(plan.n_free.numpy()[0])
        status = plan.status.numpy()
        kinds.add(tuple(sorted({"waits" if s else "prompt" if c else "drafts" if len(x) > 1 else "token"
                                for s, c, x in zip(status, context, rows) if len(x)})))
        if not any(len(x) and not s for s, x in zip(status, rows)):
            r = max(r for r in range(n) if rows[r] and held[r])
            prompts[r], cached[r], drafts[r] = prompts[r] + done[r][len(prompts[r]) - asked[r]:], 0, []
        for r in range(n):
            if status[r] or not rows[r]:
                continue
            cached[r] += context[r]
            if context[r] < len(rows[r]):
                cached[r] += 1 + accepted[r]
                done[r] += tokens[r, :accepted[r] + 1].tolist()
                accepted_drafts += int(accepted[r])
            else:
                assert accepted[r] == -1
            known = want[r][len(done[r]):len(done[r]) + int(rng.integers(0, max_drafts + 1))]
            drafts[r] = [t if rng.random() < 0.8 else (t + 1) % V for t in known]
    m.close()
    assert [d[:steps] for d in done] == want
    assert accepted_drafts > 8 and any({"waits", "drafts", "prompt"} <= set(k) for k in kinds), kinds


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_attention_small_weights_of_large_values(gpu, wtype, kernel):
    """Weights down to 2^-40 of the largest, of values up to 2^25 times the others'.  Beside an f32
    evaluation's error: over f16 a weight is off by up to 2^-31 of the largest one (f16 pieces of
    2^6 times it end at 2^-24, half a step 2^-25), in the tiles of the others a weight times 2^e,
    e the exponent of its value row's largest, by as much of the largest such product."""
    rng = np.random.default_rng(79)
    kv, n, hd = 300, 40, 128
    pool, table, q_start, kv_len = make_batch(rng, [(kv, n)], 16, 2, hd, wtype, k_std=0.01)
    q = (rng.standard_normal((n, 8, hd)) * 0.01).astype(np.float32)
    q[:, :, 0] = 8.0
    depth = rng.integers(0, 41, kv)
    depth[0] = 0
    for j in range(kv):
        at(pool, pool.k, table, 0, j)[:, 0] = R.encode(np.full(2, -depth[j] * np.log(2) * hd ** 0.5 / 8, np.float32), wtype)
        x = rng.standard_normal((2, hd)).astype(np.float32) * np.float32(2.0 ** -10 if depth[j] < 20 else 2.0 ** 13)
        at(pool, pool.v, table, 0, j)[:] = R.encode(x, wtype)
    args = (q, pool, q_start, kv_len, table, hd ** -0.5)
    want, dot, pv = R.attention(*args)
    bound = R.attention_bound(dot, pv, hd, kv)
    k = np.stack([R.decode(at(pool, pool.k, table, 0, j), wtype) for j in range(kv)])
    v = np.abs(np.stack([R.decode(at(pool, pool.v, table, 0, j), wtype) for j in range(kv)]))
    for t in range(n):
        for h in range(8):
            p = R.softmax64(k[:kv - n + t + 1, h // 4] @ q[t, h].astype(np.float64) * hd ** -0.5)
            seen = v[:len(p), h // 4]
            size = 2.0 ** np.floor(np.log2(seen.max(1)))
            bound[t, h] += 2.0 ** -31 * (p.max() * seen.sum(0) if wtype == F16
                                         else (p * size).max() * (seen / size[:, None]).sum(0))
    got = attend(gpu, *args, max_new=KERNELS[kernel])
    assert (np.abs(got - want) <= bound).all()


def test_captured_model_step(gpu):
    """hy_model_forward_paged of a padded batch in one graph, replayed with other contents, with eager
    calls of another context and synchronizations between: every replay equals the eager call."""
    rng = np.random.default_rng(78)
    nh, nkv, hd, page, V, L = 8, 2, 64, 8, 500, 2
    n_pages, max_pages, lens = 20, 5, [(17, 9), (30, 1), (6, 6)]

    class Step:
        def __init__(self):
            self.m = greedy_model(gpu)[0]
            self.pool = Pool(n_pages * L, page, nkv, hd, BF16)
            self.kb, self.vb = upload(gpu, self.pool)
            self.cache = gpu.PagedCache(self.kb, self.vb, BF16, n_pages, page, nkv, hd,
                                        layer_stride=n_pages * nkv * page * hd)
            self.n_rows = 18
            i32 = lambda a: dev(gpu, a, np.int32)  # noqa: E731
            table = np.arange(15).reshape(3, 5)
            pos = [kv - n + i for kv, n in lens for i in range(n)]
            req = [r for r, (_, n) in enumerate(lens) for _ in range(n)]
            slots = [table[r, p // page] * page + p % page for r, p in zip(req, pos)] + [-1, -1]
            self.batch = gpu.PagedBatch(3, self.n_rows, max_pages, 9, i32([0, 9, 10, 16]), i32([kv for kv, _ in lens]),
                                        i32(table), i32(pos + [0, 0]), i32(slots))
            self.ids, self.logits = i32(np.zeros(18)), dev(gpu, np.zeros((18, V), np.float32))
            self.ws = Ws(gpu, nh, self.cache, self.batch)

        def fill(self, ids):
            gpu.check(gpu.lib().hy_memcpy_h2d(self.ids.ptr, ids.ctypes.data, ids.nbytes))

        def run(self, st):
            self.m.forward_paged(self.ids, self.cache, self.batch, self.logits, self.ws.b, self.ws.n, st)

    st, a, b = gpu.Stream(), Step(), Step()
    a.run(st.h)                      # what a first call sets up is set up
    st.synchronize()
    g = gpu.Graph(st, lambda: a.run(st.h))
    try:
        for rep in range(4):
            ids = rng.integers(0, V, 18).astype(np.int32)
            a.fill(ids)
            b.fill(ids)
            b.run(st.h)
            st.synchronize()
            g.launch()
            st.synchronize()
            for p, q in ((a.kb, b.kb), (a.vb, b.vb), (a.logits, b.logits)):
                np.testing.assert_array_equal(p.numpy(), q.numpy())
            assert np.isfinite(a.logits.numpy()).all()
    finally:
        g.close()
        st.close()
        a.m.close()
        b.m.close()
