"""Several layers over one paged cache of 8 bits: each has its own pool and its own scales, layer_stride and
layer_scale_stride apart, over the steps of a server (include/hy_int8.h)."""
import numpy as np
import pytest

from int8_ref import PoolI8
from test_int8_gpu import Ws, cache_of, same_bits, upload
from test_int8_layer_gpu import model_of, plan_of
from test_paged_gpu import dev

pytestmark = pytest.mark.gpu

MARK_CODE, MARK_SCALE = 77, 1234.5  # of what lies between the layers


class Layers:
    """L pools of one cache with room between the layers, codes and scales."""

    def __init__(self, gpu, L, n_pages, page, nkv, hd, block, gap=48, scale_gap=5):
        self.n, self.ns = n_pages * nkv * page * hd, n_pages * nkv * (page // block)
        self.L, self.step, self.scale_step = L, self.n + gap, self.ns + scale_gap
        self.codes = [dev(gpu, np.full(L * self.step, MARK_CODE, np.int8)) for _ in range(2)]
        self.scales = [dev(gpu, np.full(L * self.scale_step, MARK_SCALE, np.float32)) for _ in range(2)]
        pool = gpu.PagedCache(*self.codes, gpu.I8, n_pages, page, nkv, hd, layer_stride=self.step)
        self.cache = gpu.PagedCacheI8(pool, *self.scales, block, self.scale_step)

    def layer(self, l):
        """The layer's codes of K, V and scales of K, V, as they lie."""
        return [b.numpy()[l * w:l * w + n] for bs, w, n in ((self.codes, self.step, self.n),
                                                            (self.scales, self.scale_step, self.ns)) for b in bs]

    def check_gaps(self):
        for bs, w, n, mark in ((self.codes, self.step, self.n, MARK_CODE),
                               (self.scales, self.scale_step, self.ns, MARK_SCALE)):
            for b in bs:
                assert (b.numpy().reshape(self.L, w)[:, n:] == mark).all()


STEPS = [20, 1, 1, 5, 1, 9, 3]  # a prompt, single tokens, drafts that end inside a block


@pytest.mark.parametrize("quantized", [False, True])
def test_layers_of_a_context(gpu, quantized):
    """Each of three layers, in turn and over all steps: outputs, codes and scales are the same bits as those of a
    context of one layer with its own cache; nothing between the layers is written."""
    L, H, nh, nkv, hd, page, block, n_pages = 3, 256, 8, 2, 64, 16, 8, 5
    rng = np.random.default_rng(90)
    att, alone = gpu.Attn(H, nh, nkv, hd, 32, num_layers=L), [gpu.Attn(H, nh, nkv, hd, 32) for _ in range(L)]
    for l in range(L):
        w = [(rng.standard_normal(s) * 0.1).astype(np.float32) for s in (((nh + 2 * nkv) * hd, H), (H, nh * hd))]
        w += [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        for a, at in ((att, l), (alone[l], 0)):
            a.upload(*w, layer=at)
            if quantized:
                a.quantize_i8(at)
    many = Layers(gpu, L, n_pages, page, nkv, hd, block)
    pools = [PoolI8(n_pages, page, nkv, hd, block, fill=MARK_CODE, scale_fill=MARK_SCALE) for _ in range(L)]
    bufs = [upload(gpu, p) for p in pools]
    held, table, free, n_free, at = np.zeros(1, np.int32), np.zeros((1, 4), np.int32), rng.permutation(n_pages).astype(np.int32), n_pages, 0
    for new in STEPS:
        p, batch = plan_of(gpu, [at], [new], held, table, free, n_free, page, n_pages)
        assert (p.status.numpy() == 0).all()
        outs = []
        for l in rng.permutation(L):
            x = dev(gpu, (rng.standard_normal((new, H)) * 3 ** l).astype(np.float32))
            got, want, ws = gpu.Buf.empty((new, H)), gpu.Buf.empty((new, H)), Ws(gpu, nh, many.cache, batch)
            att.forward_paged_i8(x, many.cache, batch, got, ws.b, ws.n, layer=int(l))
            alone[l].forward_paged_i8(x, cache_of(gpu, pools[l], bufs[l]), batch, want, ws.b, ws.n)
            same_bits(got.numpy(), want.numpy())
            outs.append(got.numpy())
        assert not np.array_equal(outs[0], outs[1])
        for l in range(L):
            k, ks, v, vs = (b.numpy().ravel() for b in bufs[l])
            for a, b in zip(many.layer(l), (k, v, ks, vs)):
                np.testing.assert_array_equal(a, b)
        many.check_gaps()
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        at += new
    att.close()
    for a in alone:
        a.close()


@pytest.mark.parametrize("quantized", [False, True])
def test_model_over_steps(gpu, quantized):
    """The backbone of two layers step by step, near the f32 backbone over all tokens at once, each step's rows by
    themselves.  Every expert takes every token, so nothing turns on a rounding: the layers' 6 % each (half a step
    of codes, doubled by the growths of a block's scale, and products in 8 bits), halved by the residual, and
    the lm_head's 1 %."""
    L, page, block, n_pages = 2, 16, 16, 4
    m, nh, nkv, hd, V = model_of(gpu, L)
    rng = np.random.default_rng(91)
    T = sum(STEPS)
    ids = rng.integers(0, V, T).astype(np.int32)
    lb = gpu.Buf.empty((T, V))
    m.forward(dev(gpu, ids), T, lb)
    want = lb.numpy()
    if quantized:
        m.quantize_i8()
    many = Layers(gpu, L, n_pages, page, nkv, hd, block)
    held, table, free, n_free, at = np.zeros(1, np.int32), np.zeros((1, 3), np.int32), np.array([2, 0, 3, 1], np.int32), n_pages, 0
    for new in STEPS:
        p, batch = plan_of(gpu, [at], [new], held, table, free, n_free, page, n_pages)
        assert (p.status.numpy() == 0).all()
        out, ws = gpu.Buf.empty((new, V)), Ws(gpu, nh, many.cache, batch)
        m.forward_paged_i8(dev(gpu, ids[at:at + new]), many.cache, batch, out, ws.b, ws.n)
        got, ref = out.numpy(), want[at:at + new]
        assert np.linalg.norm(got - ref) <= 0.1 * np.linalg.norm(ref)
        held, table, free, n_free = p.held.numpy(), p.table.numpy(), p.free.numpy(), int(p.n_free.numpy()[0])
        at += new
        many.check_gaps()
        for l in range(L):  # the blocks that hold tokens, and no others
            for codes, scales in zip(many.layer(l)[:2], many.layer(l)[2:]):
                used = np.zeros(n_pages, bool)
                used[table[0, :-(-at // page)]] = True
                np.testing.assert_array_equal((scales.reshape(n_pages, -1) != MARK_SCALE).all(1), used)
                np.testing.assert_array_equal((codes.reshape(n_pages, -1) != MARK_CODE).any(1), used)
    assert not any(np.array_equal(a, b) for a, b in zip(many.layer(0), many.layer(1)))
    m.close()


def test_graph_and_new_weights(gpu):
    """A captured layer goes on with the codes there are when weights are loaded, and takes the new ones where they are
    quantized again; calls take the loaded weights at once."""
    H, nh, nkv, hd, T = 256, 8, 2, 64, 6
    rng = np.random.default_rng(92)
    att = gpu.Attn(H, nh, nkv, hd, 16)

    def load():
        att.upload(*[(rng.standard_normal(s) * 0.1).astype(np.float32) for s in (((nh + 2 * nkv) * hd, H), (H, nh * hd))],
                   np.ones(hd, np.float32), np.ones(hd, np.float32))
    i32 = lambda *v: dev(gpu, np.array(v, np.int32))  # noqa: E731
    pool = PoolI8(1, 16, nkv, hd, 16)
    cache = cache_of(gpu, pool, upload(gpu, pool))
    batch = gpu.PagedBatch(1, T, 1, T, i32(0, T), i32(T), i32(0), i32(*range(T)), i32(*range(T)))
    x, out, ws = dev(gpu, rng.standard_normal((T, H)).astype(np.float32)), gpu.Buf.empty((T, H)), Ws(gpu, nh, cache, batch)
    st = gpu.Stream()

    def call(run):
        out.zero()
        gpu.sync()
        run()
        st.synchronize()
        return out.numpy()
    eager = lambda: call(lambda: att.forward_paged_i8(x, cache, batch, out, ws.b, ws.n, stream=st.h))  # noqa: E731
    load()
    att.quantize_i8()
    old = eager()
    g = gpu.Graph(st, lambda: att.forward_paged_i8(x, cache, batch, out, ws.b, ws.n, stream=st.h))
    same_bits(call(g.launch), old)
    load()
    plain = eager()
    assert (plain != old).any()
    same_bits(call(g.launch), old)
    att.quantize_i8()
    new = eager()
    assert (new != old).any() and (new != plain).any()
    for _ in range(3):
        same_bits(call(g.launch), new)
        same_bits(eager(), new)
    g.close()
    st.close()
    att.close()
