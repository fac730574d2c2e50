"""The attention layer and the backbone over a paged cache of 8 bits, with and without their products in 8
bits (include/hy_int8.h)."""
import numpy as np
import pytest

import int8_ref as Q
from int8_ref import PoolI8
from test_int8_gpu import Ws, cache_of, download, same_bits, same_pool, upload
from test_paged_gpu import PlanBufs, dev

pytestmark = pytest.mark.gpu


def plan_of(gpu, cached, news, held, table, free, n_free, page, n_pages, pad=0):
    p = PlanBufs(gpu, cached, news, held, table, free, n_free, int(sum(news)) + pad, page, n_pages)
    p.run(in_place=True)
    return p, gpu.PagedBatch(p.R, p.n_rows, p.max_pages, int(max(news)), p.q_start, p.kv_len, p.table, p.positions,
                             p.slots)


def layer_of(gpu, rng, H, nh, nkv, hd, max_tokens=128):
    att = gpu.Attn(H, nh, nkv, hd, max_tokens)
    w = [(rng.standard_normal(s) * 0.05).astype(np.float32) for s in (((nh + 2 * nkv) * hd, H), (H, nh * hd))]
    n = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    att.upload(*w, *n)
    return att, w, n


@pytest.mark.parametrize("H,nh,nkv,hd", [(512, 8, 2, 128), (256, 4, 1, 64)])
def test_layer_is_its_calls(gpu, H, nh, nkv, hd):
    """The layer with products in 8 bits: the same bits as its calls one after another, over several steps, rows
    of nobody among them."""
    rng = np.random.default_rng(50)
    att, (wqkv, wo), (qn, kn) = layer_of(gpu, rng, H, nh, nkv, hd)
    att.quantize_i8()
    (cq, sq), (co, so) = (tuple(dev(gpu, a) for a in Q.quantize(w)) for w in (wqkv, wo))
    page, n_pages, max_pages, pad = 16, 24, 8, 3
    pools = [PoolI8(n_pages, page, nkv, hd, 16) for _ in range(2)]
    bufs = [upload(gpu, p) for p in pools]
    caches = [cache_of(gpu, p, b) for p, b in zip(pools, bufs)]
    held, table = np.zeros(3, np.int32), np.zeros((3, max_pages), np.int32)
    free, n_free, cached = rng.permutation(n_pages).astype(np.int32), n_pages, np.zeros(3, np.int64)
    for news in ([40, 3, 1], [1, 30, 5], [33, 1, 1], [1, 1, 1]):
        p, batch = plan_of(gpu, cached, news, held, table, free, n_free, page, n_pages, pad)
        assert (p.status.numpy() == 0).all()
        T = p.n_rows
        x = dev(gpu, rng.standard_normal((T, H)).astype(np.float32))
        out, ws = dev(gpu, np.full((T, H), 9.0, np.float32)), Ws(gpu, nh, caches[0], batch)
        att.forward_paged_i8(x, caches[0], batch, out, ws.b, ws.n)
        qkv, q = gpu.Buf.empty((T, (nh + 2 * nkv) * hd)), dev(gpu, np.zeros((T, nh * hd), np.float32))
        merged, want = dev(gpu, np.zeros((T, nh * hd), np.float32)), gpu.Buf.empty((T, H))
        n1, n2 = gpu.linear_i8_ws(T, H, (nh + 2 * nkv) * hd), gpu.linear_i8_ws(T, nh * hd, H)
        lw = gpu.Buf(max(n1, n2))
        gpu.linear_i8(x, cq, sq, None, T, H, (nh + 2 * nkv) * hd, qkv, lw, n1)
        gpu.rope_qknorm_paged_i8(qkv, T, nh, caches[1], p.positions, p.slots, 10000.0, None, None, 0, dev(gpu, qn),
                                 dev(gpu, kn), 1e-5, q)
        gpu.paged_attention_i8(q, nh, caches[1], batch, 1.0 / np.sqrt(np.float32(hd)), merged, ws.b, ws.n)
        gpu.linear_i8(merged, co, so, None, T, nh * hd, H, want, lw, n2)
        got = out.numpy()
        same_bits(got, want.numpy())
        assert (got[T - pad:] == 0).all() and (got[:T - pad] != 0).any(axis=1).all()
        a, b = (download(pl, bf) for pl, bf in zip(pools, bufs))
        same_pool(a, b)
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        cached = cached + news
    att.close()


@pytest.mark.parametrize("quantized", [False, True])
def test_layer_in_chunks_is_near_one_prompt(gpu, quantized):
    """Against the f32 layer over the whole prompt.  A block's largest of 16 x 128 normal values is 3.5 to 4.5 of
    their size, a step 1/127 of it, its rounding 1 / sqrt(12) of a step: 1 % of a value, and 1 % of a score of q
    and k of rms 1 (its other terms' errors are independent), so 1 % of a weight; three growths of a block's
    scale at most double both.  Products in 8 bits round tokens and weights by 0.8 and 0.9 % in each of two:
    6 % in all if nothing cancelled."""
    rng = np.random.default_rng(51)
    H, nh, nkv, hd, T, page = 512, 8, 2, 128, 75, 16
    att, _, _ = layer_of(gpu, rng, H, nh, nkv, hd)
    x = rng.standard_normal((T, H)).astype(np.float32)
    want = att.run(x)
    if quantized:
        att.quantize_i8()
    pool = PoolI8(8, page, nkv, hd, 16)
    bufs = upload(gpu, pool)
    cache = cache_of(gpu, pool, bufs)
    held, table, free, n_free, at, got = np.zeros(1, np.int32), np.zeros((1, 5), np.int32), np.arange(8, dtype=np.int32), 8, 0, []
    for new in (40, 1, 1, 1, 30, 2):
        p, batch = plan_of(gpu, [at], [new], held, table, free, n_free, page, 8)
        out, ws = gpu.Buf.empty((new, H)), Ws(gpu, nh, cache, batch)
        att.forward_paged_i8(dev(gpu, x[at:at + new]), cache, batch, out, ws.b, ws.n)
        got.append(out.numpy())
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        at += new
    att.close()
    got = np.concatenate(got)
    assert np.linalg.norm(got - want) <= 0.06 * np.linalg.norm(want)


def test_loading_drops_the_codes(gpu):
    """New weights are used, not the old ones' codes; held in 8 bits again they give what a fresh layer gives."""
    rng = np.random.default_rng(52)
    H, nh, nkv, hd = 256, 4, 1, 64
    att, _, _ = layer_of(gpu, rng, H, nh, nkv, hd)
    att.quantize_i8()
    fresh, w, n = layer_of(gpu, rng, H, nh, nkv, hd)
    att.upload(*w, *n)
    outs = []
    x = dev(gpu, rng.standard_normal((5, H)).astype(np.float32))

    def run(a):
        p = PoolI8(2, 16, nkv, hd, 8)
        cache = cache_of(gpu, p, upload(gpu, p))
        i32 = lambda *v: dev(gpu, np.array(v, np.int32))  # noqa: E731
        batch = gpu.PagedBatch(1, 5, 1, 5, i32(0, 5), i32(5), i32(1), i32(0, 1, 2, 3, 4), i32(16, 17, 18, 19, 20))
        out, ws = gpu.Buf.empty((5, H)), Ws(gpu, nh, cache, batch)
        a.forward_paged_i8(x, cache, batch, out, ws.b, ws.n)
        return out.numpy()
    outs = [run(att), run(fresh)]
    same_bits(*outs)
    att.quantize_i8()
    att.quantize_i8()          # twice is once
    fresh.quantize_i8()
    again = [run(att), run(fresh)]
    same_bits(*again)
    assert (again[0] != outs[0]).any()
    att.close()
    fresh.close()


def model_of(gpu, L):
    H, I, E, K, nh, nkv, hd, V = 256, 128, 4, 4, 8, 2, 64, 500
    m = gpu.Model(H, I, E, K, gpu.F32, nh, nkv, hd, V, L, 64)
    m.synth_globals(seed=3, std=0.5)
    for l in range(L):
        m.attn.synth(l, seed=7 + l, std=0.08)
        m.moe.synth(l, seed=9 + l, std=0.05)
    return m, nh, nkv, hd, V


def model_cache(gpu, L, n_pages, nkv, hd, page=16, block=16, stride=None):
    k, v = (dev(gpu, np.zeros(L * n_pages * nkv * page * hd, np.int8)) for _ in range(2))
    n = n_pages * nkv * (page // block)
    ks, vs = (dev(gpu, np.zeros(L * n, np.float32)) for _ in range(2))
    pool = gpu.PagedCache(k, v, gpu.I8, n_pages, page, nkv, hd, layer_stride=n_pages * nkv * page * hd)
    return gpu.PagedCacheI8(pool, ks, vs, block, n if stride is None else stride), (k, v, ks, vs)


@pytest.mark.parametrize("quantized", [False, True])
def test_model_step_in_a_graph(gpu, quantized):
    """The backbone's step, eager and captured: the same bits; near the f32 backbone (every expert takes every
    token, so nothing turns on a rounding; the layers' 6 % each, halved by the residual, and the lm_head's 1 %)."""
    L, T = 2, 20
    m, nh, nkv, hd, V = model_of(gpu, L)
    rng = np.random.default_rng(53)
    ids = rng.integers(0, V, T).astype(np.int32)
    lb = gpu.Buf.empty((T, V))
    m.forward(dev(gpu, ids), T, lb)
    want = lb.numpy()
    if quantized:
        m.quantize_i8()
    st = gpu.Stream()
    i32 = lambda a: dev(gpu, np.array(a, np.int32))  # noqa: E731
    outs = []
    for _ in range(2):
        cache, keep = model_cache(gpu, L, 4, nkv, hd)
        batch = gpu.PagedBatch(1, T, 4, T, i32([0, T]), i32([T]), i32([2, 0, 1, 3]), i32(range(T)),
                               i32([(2 if t < 16 else 0) * 16 + t % 16 for t in range(T)]))
        out, ws, idb = dev(gpu, np.zeros((T, V), np.float32)), Ws(gpu, nh, cache, batch), dev(gpu, ids)
        outs.append((out, cache, batch, ws, idb, keep))
    out, cache, batch, ws, idb, _ = outs[0]
    m.forward_paged_i8(idb, cache, batch, out, ws.b, ws.n, st.h)
    st.synchronize()
    eager = out.numpy()
    assert np.linalg.norm(eager - want) <= 0.1 * np.linalg.norm(want)
    out, cache, batch, ws, idb, _ = outs[1]
    g = gpu.Graph(st, lambda: m.forward_paged_i8(idb, cache, batch, out, ws.b, ws.n, st.h))
    for _ in range(3):
        out.zero()
        gpu.sync()
        g.launch()
        st.synchronize()
        same_bits(out.numpy(), eager)
    g.close()
    st.close()
    m.close()


def test_refusals_of_layer_and_model(gpu):
    """Refused before anything is written: scales of layers that would overlap, other heads, layers without
    weights, nulls."""
    L = 2
    m, nh, nkv, hd, V = model_of(gpu, L)
    i32 = lambda *a: dev(gpu, np.array(a, np.int32))  # noqa: E731
    batch = gpu.PagedBatch(1, 2, 4, 2, i32(0, 2), i32(2), i32(0, 1, 2, 3), i32(0, 1), i32(0, 1))
    good, keep = model_cache(gpu, L, 4, nkv, hd)
    ws = Ws(gpu, nh, good, batch)
    logits = dev(gpu, np.full((2, V), 8.0, np.float32))
    ids, x = i32(4, 5), gpu.Buf.empty((2, 256))
    short, k2 = model_cache(gpu, L, 4, nkv, hd, stride=4 * nkv - 1)
    other, k3 = model_cache(gpu, L, 4, 1, hd)
    for cache in (short, other):
        with pytest.raises(gpu.HyError):
            m.forward_paged_i8(ids, cache, batch, logits, ws.b, ws.n)
        with pytest.raises(gpu.HyError):
            m.attn.forward_paged_i8(x, cache, batch, x, ws.b, ws.n)
    with pytest.raises(gpu.HyError):
        m.forward_paged_i8(ids, good, batch, logits, ws.b, ws.n - 1)
    lib, bad = gpu.lib(), -1
    assert lib.hy_model_forward_paged_i8(m.h, ids.ptr, None, batch, logits.ptr, ws.b.ptr, ws.n, None) == bad
    assert lib.hy_attn_forward_paged_i8(m.attn.h, 0, x.ptr, None, batch, None, None, 0, x.ptr, ws.b.ptr, ws.n, None) == bad
    assert lib.hy_attn_quantize_i8(m.attn.h, L) == bad
    gpu.sync()
    assert (logits.numpy() == 8.0).all() and not any(b.numpy().any() for b in keep + k2 + k3)
    empty = gpu.Attn(256, 8, 2, 64, 16)
    with pytest.raises(gpu.HyError):
        empty.quantize_i8()
    with pytest.raises(gpu.HyError):
        empty.forward_paged_i8(x, good, batch, x, ws.b, ws.n)
    empty.close()
    m.forward_paged_i8(ids, good, batch, logits, ws.b, ws.n)
    assert np.isfinite(logits.numpy()).all() and keep[0].numpy().any()
    m.close()
