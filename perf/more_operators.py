"""The operators of serving in 8 bits as measurable cases: the product of tokens and weights
in 8-bit integers with a scale per token and per channel, the rotary + QK-norm write into a
paged cache of 8-bit integers with a scale per block of tokens and head, and attention over
that cache -- in plain torch (own = False) or through the entry points of include/hy_int8.h
(own = True).

A case is a dict of plain values.  listed() gives the named ones, draw() further ones of
the same ranges, prepare() what a server holds before the call, run() one pass, exact() its
outputs in 64 bits, work() what a pass cannot do without.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.getcwd()
_I8 = 24
_EPS = 1e-5
_THETA = 10000.0
_TINY = 2.0 ** -126  # a scale below is 0
_VOCAB, _HIDDEN, _QKV = 133120, 4096, 6144  # HunyuanImage-3's
_BIG = {"nh": 32, "nkv": 8, "hd": 128}  # its attention heads


def _hy():
    if "hy3moe" not in sys.modules:
        pkg = os.path.join(_ROOT, "hunyuan-image-3-80b.cpp_amd")
        spec = importlib.util.spec_from_file_location("hy3moe", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["hy3moe"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["hy3moe"].hy_moe


class _Dev:
    """A torch tensor as the binding takes device buffers (it reads .ptr only)."""

    def __init__(self, t):
        self.t = t
        self.ptr = t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one chat's new token through the attention's input projection
        dict(name="linear_t1", kind="linear", T=1, K=_HIDDEN, N=_QKV, resid=False),
        # a step's tokens through the vocabulary's projection: the largest read of weights
        dict(name="linear_head_t16", kind="linear", T=16, K=_HIDDEN, N=_VOCAB, resid=False),
        # a step of chunks and single tokens, the attention's output onto the residual
        dict(name="linear_t300", kind="linear", T=300, K=_HIDDEN, N=_HIDDEN, resid=True),
        # an image's 64 x 64 tokens
        dict(name="linear_t4096", kind="linear", T=4096, K=_HIDDEN, N=_QKV, resid=False),
        # one request's drafted tokens behind 100 cached ones: a block that holds tokens already
        dict(name="append_t5", kind="append", T=5, ctx=100, page=16, block=16, table=False, pad=0, **_BIG),
        # an image's tokens behind a short prompt, 2D rotary tables
        dict(name="append_t4096", kind="append", T=4096, ctx=100, page=64, block=16, table=True, pad=0, **_BIG),
        # one chat, one new token
        dict(name="attn_one", kind="attn", R=1, ctx=1000, new=1, mode="decode", page=16, block=16, spans=False, pad=0,
             **_BIG),
        # a busy server's decode step over long ragged caches
        dict(name="attn_decode", kind="attn", R=64, ctx=8000, new=1, mode="decode", page=16, block=16, spans=False,
             pad=0, **_BIG),
        # the check of up to five drafted tokens per request
        dict(name="attn_draft", kind="attn", R=32, ctx=2900, new=6, mode="draft", page=64, block=32, spans=False,
             pad=5, **_BIG),
        # a chunk of a long prompt behind what is cached
        dict(name="attn_chunk", kind="attn", R=1, ctx=8192, new=2048, mode="chunk", page=64, block=64, spans=False,
             pad=0, **_BIG),
        # chunks and single tokens together, the chunks' image spans seen as a whole
        dict(name="attn_mixed", kind="attn", R=12, ctx=4500, new=700, mode="mixed", page=32, block=8, spans=True,
             pad=3, **_BIG),
        # prompts without a past, small heads
        dict(name="attn_prompt", kind="attn", R=5, ctx=0, new=1500, mode="chunk", page=16, block=16, spans=False,
             pad=0, nh=16, nkv=4, hd=64),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm, any residue."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / (1.5e15 if c["kind"] == "linear" else 4e14))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "append", "append", "attn", "attn", "attn", "attn"])
    if kind == "linear":
        # few tokens of a decode step, or chunks; a model's widths, or any
        T = rng.choice([_spread(rng, 1, 64), _spread(rng, 1, 8192)])
        return dict(kind="linear", T=T, K=rng.choice([_HIDDEN, _HIDDEN, 2048, 16 * _spread(rng, 16, 512)]),
                    N=rng.choice([_HIDDEN, _QKV, _VOCAB if T <= 256 else _QKV, _spread(rng, 256, 32003)]),
                    resid=rng.random() < 0.4)
    page = rng.choice([8, 16, 16, 32, 64, 128])
    block = rng.choice([b for b in (8, 16, 16, 32, 64, 128) if b <= page])
    heads = rng.choice([_BIG, _BIG, _BIG, dict(nh=16, nkv=4, hd=64), dict(nh=16, nkv=4, hd=128),
                        dict(nh=8, nkv=8, hd=128), dict(nh=16, nkv=2, hd=64), dict(nh=20, nkv=4, hd=128)])
    if kind == "append":
        return dict(kind="append", T=_spread(rng, 1, 8192), ctx=rng.choice([0, _spread(rng, 1, 5000)]), page=page,
                    block=block, table=rng.random() < 0.4, pad=rng.choice([0, 0, 3, 40]), **heads)
    mode = rng.choice(["decode", "decode", "draft", "chunk", "mixed"])
    if mode == "decode":
        R, new = _spread(rng, 1, 192), 1
        ctx = _spread(rng, 1, min(32000, 800000 // R))
    elif mode == "draft":
        R, new = _spread(rng, 1, 96), rng.randint(2, 16)
        ctx = _spread(rng, 1, min(16000, 400000 // R))
    else:
        R = _spread(rng, 1, 16)
        new, ctx = _spread(rng, 9, max(9, 4096 // R)), rng.choice([0, _spread(rng, 1, max(1, 32000 // R))])
    return dict(kind="attn", R=R, ctx=ctx, new=new, mode=mode, page=page, block=block,
                spans=mode in ("chunk", "mixed") and rng.random() < 0.4, pad=rng.choice([0, 0, 3, 17]), **heads)


def _lens(c):
    """Cached and new lengths of a case's requests: ragged, the same for every seed."""
    g = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    ctx, new = [], []
    for r in range(c["R"]):
        n, lo, hi = c["new"], c["ctx"] // 4, c["ctx"]
        if r:
            n = g.randint(1, n) if c["mode"] != "mixed" or r % 2 else 1
        ctx.append(hi if r == 0 else g.randint(lo, hi))
        new.append(n)
    return ctx, new


# ------------------------------------------------------------------ inputs

def _gen(seed, *path):
    g = torch.Generator(device="cuda")
    k = seed & 0xFFFFFFFF
    for p in path:
        k = (k * 1000003 + p + 1) & 0x7FFFFFFFFFFFFFFF
    g.manual_seed(k)
    return g


def _randn(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


class _State:
    pass


def _scale(big):
    """Scales of groups whose largest magnitudes are given, and their reciprocals (0 for 0): each
    rounded to 32 bits once (a quotient in 64 bits rounds to the 32-bit quotient)."""
    d = (big.double() / 127.0).float()
    d = torch.where(d < _TINY, torch.zeros_like(d), d)
    return d, _inverse(d)


def _inverse(d):
    return torch.where(d > 0, (1.0 / d.double()).float(), torch.zeros_like(d))


def _quantize(x):
    """8-bit codes of the rows of x (f32) and their scales."""
    d, inv = _scale(x.abs().amax(-1))
    return torch.round(x * inv[..., None]).to(torch.int8), d


def _tables(c, seed, lens):
    """A random assignment of pages to requests: table [R][max_pages], pages in all."""
    need = [-(-n // c["page"]) for n in lens]
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    width = max(1, max(need))
    table = torch.zeros((len(lens), width), device="cuda", dtype=torch.int32)
    at = torch.arange(width, device="cuda")[None, :]
    n = _ints(need).long()[:, None]
    first = torch.cumsum(n, 0) - n
    table[at < n] = perm[(first + at)[at < n]]
    return table, n_pages


def _pool(c, seed, n_pages):
    """Codes [page][kv head][position][head_dim] and scales [page][kv head][block] of keys (rms 1,
    behind a QK-norm) and values (of differing size)."""
    P, B, g, hd = n_pages, c["page"] // c["block"], c["nkv"], c["hd"]
    out = []
    for what in (3, 4):
        x = _randn((P, g, B, c["block"], hd), _gen(seed, what))
        if what == 4:
            x = x * torch.exp(_randn((P, g, B, c["block"], 1), _gen(seed, 5), 0.5))
        q, d = _quantize(x.view(P, g, B, -1))
        out += [q.view(P, g, c["page"], hd), d.contiguous()]
    return out


def _prepare_linear(c, seed):
    s = _State()
    s.x = _randn((c["T"], c["K"]), _gen(seed, 2))
    s.x *= torch.exp(_randn((1, c["K"]), _gen(seed, 3), 0.7))  # some channels of a model's activations are large
    w = torch.empty((c["N"], c["K"]), device="cuda", dtype=torch.int8)
    d = torch.empty(c["N"], device="cuda")
    g = _gen(seed, 4)
    for i in range(0, c["N"], 16384):
        n = min(16384, c["N"] - i)
        w[i: i + n], d[i: i + n] = _quantize(_randn((n, c["K"]), g, 0.02))
    s.w, s.w_scale = w, d
    s.resid = _randn((c["T"], c["N"]), _gen(seed, 5)) if c["resid"] else None
    s.out = torch.zeros((c["T"], c["N"]), device="cuda")
    s.ws = None
    return s


def _freqs(hd):
    return _THETA ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)


def _prepare_append(c, seed):
    s = _State()
    T, hd, page, ctx = c["T"], c["hd"], c["page"], c["ctx"]
    s.n_rows = T + c["pad"]
    # the pages from the one that the first new token falls into on
    first = ctx // page * page
    table, s.n_pages = _tables(c, seed, [ctx + T - first])
    pos = torch.arange(ctx, ctx + T, device="cuda")
    slot = table[0, (pos - first) // page].long() * page + pos % page
    s.positions, s.slots = torch.zeros(s.n_rows, device="cuda", dtype=torch.int32), _ints([-1] * s.n_rows)
    s.positions[:T], s.slots[:T] = pos.int(), slot.int()
    s.qkv = _randn((s.n_rows, (c["nh"] + 2 * c["nkv"]) * hd), _gen(seed, 2))
    s.qn, s.kn = 1.0 + _randn((hd,), _gen(seed, 3), 0.1), 1.0 + _randn((hd,), _gen(seed, 4), 0.1)
    s.cos = s.sin = None
    s.n_pos = ctx + T if c["table"] else 0
    if c["table"]:
        ang = torch.arange(s.n_pos, device="cuda", dtype=torch.float64)[:, None] * _freqs(hd)
        s.cos = torch.cos(ang).float().repeat_interleave(2, dim=1).contiguous()
        s.sin = torch.sin(ang).float().repeat_interleave(2, dim=1).contiguous()
    s.k, s.ks, s.v, s.vs = _pool(c, seed, s.n_pages)
    s.q = torch.zeros((s.n_rows, c["nh"], hd), device="cuda")
    return s


def _prepare_attn(c, seed):
    s = _State()
    ctx, new = _lens(c)
    total = [a + b for a, b in zip(ctx, new)]
    s.n_rows = sum(new) + c["pad"]
    s.table, s.n_pages = _tables(c, seed, total)
    s.max_pages, s.max_new = s.table.shape[1], max(new)
    s.q_start = _ints([sum(new[:i]) for i in range(len(new) + 1)])
    s.kv_len = _ints(total)
    s.seen = None
    if c["spans"]:
        # text and images in turns: the tokens of an image see the whole of it
        seen = []
        for a, n in zip(ctx, new):
            g = random.Random(a * 7919 + n)
            i = 0
            while i < n:
                span = min(n - i, g.randint(1, 256))
                image = g.random() < 0.5
                seen += [a + i + span if image else a + i + j + 1 for j in range(span)]
                i += span
        s.seen = _ints(seen + [0] * c["pad"])
    # queries and keys have passed the QK-norm (rms about 1); a factor 2 for peaked scores
    s.q = _randn((s.n_rows, c["nh"], c["hd"]), _gen(seed, 2), 2.0)
    s.k, s.ks, s.v, s.vs = _pool(c, seed, s.n_pages)
    s.scale = 1.0 / math.sqrt(c["hd"])
    s.out = torch.zeros((s.n_rows, c["nh"], c["hd"]), device="cuda")
    s.ws = None
    return s


def prepare(case, seed):
    s = {"linear": _prepare_linear, "append": _prepare_append, "attn": _prepare_attn}[case["kind"]](case, seed)
    s.case = case
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ plain forms

def _plain_linear(s, c):
    xq, d = _quantize(s.x)
    y = torch.matmul(xq.float(), s.w.t().float())
    y = y * d[:, None] * s.w_scale
    return y if s.resid is None else y + s.resid


def _blocks(codes, c):
    """[page][kv head][position][hd] as [block][kv head][position in it][hd]."""
    P, g, page, hd = codes.shape
    return codes.view(P, g, page // c["block"], c["block"], hd).transpose(1, 2).reshape(-1, g, c["block"], hd)


def _values(codes, scales):
    """What a pool holds."""
    P, g, page, hd = codes.shape
    return (codes.view(P, g, scales.shape[2], -1, hd) * scales[..., None, None]).view(P, g, page, hd)


def _write(codes, scales, y, slot, c):
    """Rows y [T][kv head][hd] at their slots: a block whose first position is among them begins anew, others
    keep what they hold at a scale that no row passes."""
    P, g, page, hd = codes.shape
    blk, at = slot // c["block"], slot % c["block"]
    old = scales.transpose(1, 2).reshape(-1, g)
    n = old.shape[0]
    big = torch.zeros((n, g), device="cuda").scatter_reduce(0, blk[:, None].expand(-1, g), y.abs().amax(-1), "amax")
    touched, fresh = torch.zeros(n, device="cuda", dtype=torch.bool), torch.zeros(n, device="cuda", dtype=torch.bool)
    touched[blk] = True
    fresh[blk[at == 0]] = True
    kept = torch.where(fresh[:, None], 0.0, old)
    d = torch.where(touched[:, None], torch.maximum(kept, _scale(big)[0]), old)
    inv = _inverse(d)
    ratio = torch.where(d > 0, (kept.double() / d.double()).float(), torch.zeros_like(d))
    fac = torch.where(touched[:, None], ratio, 1.0)
    q = torch.round(_blocks(codes, c) * fac[:, :, None, None])
    q[blk, :, at] = torch.round(y * inv[blk][:, :, None])
    codes.copy_(q.view(P, -1, g, c["block"], hd).transpose(1, 2).reshape(P, g, page, hd))
    scales.copy_(d.view(P, -1, g).transpose(1, 2))


def _plain_append(s, c):
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    live = s.slots >= 0
    x = s.qkv[live].view(-1, nh + 2 * nkv, hd)
    pos, slot = s.positions[live].long(), s.slots[live].long()
    if s.cos is not None:
        cs, sn = s.cos[pos][:, None, ::2].double(), s.sin[pos][:, None, ::2].double()
    else:
        ang = pos.double()[:, None] * _freqs(hd)
        cs, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    # in 64 bits: a key next to the border between two codes goes to the right one
    a, b = x[:, : nh + nkv, ::2].double(), x[:, : nh + nkv, 1::2].double()
    rot = torch.stack([a * cs - b * sn, a * sn + b * cs], dim=-1).flatten(2)
    rot = rot / torch.sqrt((rot * rot).mean(-1, keepdim=True) + _EPS)
    s.q[live] = (rot[:, :nh] * s.qn).float()
    _write(s.k, s.ks, (rot[:, nh:] * s.kn).float(), slot, c)
    _write(s.v, s.vs, x[:, nh + nkv:], slot, c)
    return [s.q, _values(s.k, s.ks), _values(s.v, s.vs), s.ks, s.vs]


def _padded(s, c):
    """Token rows [R][max_new] and their mask, keys seen [R][max_new], slots [R][max_kv]."""
    start = s.q_start.long()
    n = start[1:] - start[:-1]
    i = torch.arange(s.max_new, device="cuda")[None, :]
    there = i < n[:, None]
    rows = torch.where(there, start[:-1, None] + i, 0)
    kv = s.kv_len.long()[:, None]
    seen = kv - n[:, None] + i + 1 if s.seen is None else torch.minimum(s.seen[rows].long(), kv)
    j = torch.arange(s.max_pages * c["page"], device="cuda")[None, :]
    return rows, there, seen, s.table[:, j[0] // c["page"]].long(), j


def _plain_attn(s, c):
    nh, nkv, hd, P = c["nh"], c["nkv"], c["hd"], c["page"]
    rows, there, seen, page, j = _padded(s, c)
    R, N = rows.shape
    at = j % P
    in_len = (j < s.kv_len[:, None])[:, :, None, None]
    k = s.k[page, :, at] * s.ks[page, :, at // c["block"]][..., None]
    k = torch.where(in_len, k, 0.0).permute(0, 2, 3, 1).contiguous()  # [R][nkv][hd][keys]
    v = s.v[page, :, at] * s.vs[page, :, at // c["block"]][..., None]
    v = torch.where(in_len, v, 0.0).permute(0, 2, 1, 3).contiguous()  # [R][nkv][keys][hd]
    q = s.q[rows].view(R, N, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4).reshape(R, nkv, -1, hd) * s.scale
    sc = torch.matmul(q, k).view(R, nkv, N, nh // nkv, -1)
    sc = sc.masked_fill((j[:, None, :] >= seen[:, :, None])[:, None, :, None, :], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(sc - m)
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.matmul(e.view(R, nkv, -1, e.shape[-1]), v).view(R, nkv, N, nh // nkv, hd)
    s.out[rows[there]] = o.permute(0, 2, 1, 3, 4).reshape(R, N, nh, hd)[there]
    return s.out


# ------------------------------------------------------------------ the framework's calls

def _own_linear(s, c):
    hy = _hy()
    if s.ws is None:
        s.ws = torch.empty(hy.linear_i8_ws(c["T"], c["K"], c["N"]), dtype=torch.uint8, device="cuda")
    hy.linear_i8(_Dev(s.x), _Dev(s.w), _Dev(s.w_scale), None if s.resid is None else _Dev(s.resid), c["T"], c["K"],
                 c["N"], _Dev(s.out), _Dev(s.ws), s.ws.numel(), _stream())
    return s.out


def _cache(s, c):
    hy = _hy()
    return hy.PagedCacheI8(hy.PagedCache(_Dev(s.k), _Dev(s.v), _I8, s.n_pages, c["page"], c["nkv"], c["hd"]),
                           _Dev(s.ks), _Dev(s.vs), c["block"])


def _own_append(s, c):
    _hy().rope_qknorm_paged_i8(_Dev(s.qkv), s.n_rows, c["nh"], _cache(s, c), _Dev(s.positions), _Dev(s.slots), _THETA,
                               None if s.cos is None else _Dev(s.cos), None if s.sin is None else _Dev(s.sin), s.n_pos,
                               _Dev(s.qn), _Dev(s.kn), _EPS, _Dev(s.q), _stream())
    return [s.q, _values(s.k, s.ks), _values(s.v, s.vs), s.ks, s.vs]


def _own_attn(s, c):
    hy = _hy()
    cache = _cache(s, c)
    batch = hy.PagedBatch(c["R"], s.n_rows, s.max_pages, s.max_new, _Dev(s.q_start), _Dev(s.kv_len), _Dev(s.table),
                          seen=None if s.seen is None else _Dev(s.seen))
    if s.ws is None:
        s.ws = torch.empty(hy.paged_attention_i8_ws(c["nh"], cache, batch), dtype=torch.uint8, device="cuda")
    hy.paged_attention_i8(_Dev(s.q), c["nh"], cache, batch, s.scale, _Dev(s.out), _Dev(s.ws), s.ws.numel(), _stream())
    return s.out


def run(s):
    c = s.case
    kind = c["kind"]
    if own:
        if kind == "linear":
            return _own_linear(s, c)
        if kind == "append":
            return _own_append(s, c)
        return _own_attn(s, c)
    if kind == "linear":
        return _plain_linear(s, c)
    if kind == "append":
        return _plain_append(s, c)
    return _plain_attn(s, c)


# ------------------------------------------------------------------ 64 bits

def _f32(x):
    """Rounded to 32 bits, in 64."""
    return x.float().double()


def _exact_scale(big):
    """d = a / 127 and 1 / d, each rounded to 32 bits; none below 2^-126."""
    d = _f32(big / 127.0)
    d = d * (d >= _TINY)
    return d, torch.nan_to_num(_f32(d.reciprocal()), posinf=0.0)


def _exact_linear(s, c):
    if 2.0 * c["T"] * c["K"] * c["N"] > 4e12:
        return None
    x = s.x.double()
    d, inv = _exact_scale(x.abs().max(dim=1).values)
    q = _f32(x * inv[:, None]).round()  # the product rounded to 32 bits, then to a whole number
    out = s.out.double()
    for i in range(0, c["N"], 8192):
        w = s.w[i: i + 8192].double()
        out[:, i: i + 8192] = torch.mm(q, w.t().contiguous()) * d[:, None] * s.w_scale[i: i + 8192].double()
    return out if s.resid is None else out + s.resid.double()


def _exact_write(codes, scales, y, slot, c):
    """Block by block on the host's order of blocks; values, scales."""
    P, g, page, hd = codes.shape
    B = c["block"]
    held = (codes.double().view(P, g, page // B, B, hd)).clone()
    d_all = scales.double()
    order = torch.div(slot, B, rounding_mode="floor").tolist()
    lo = 0
    while lo < len(order):  # rows of one block lie side by side
        hi = lo
        while hi < len(order) and order[hi] == order[lo]:
            hi += 1
        p, b = divmod(order[lo], page // B)
        off = int(slot[lo]) % B
        rows = y[lo:hi]
        old = d_all[p, :, b] * (0.0 if off == 0 else 1.0)
        d = torch.maximum(old, _exact_scale(rows.abs().amax(dim=(0, 2)))[0])
        inv = torch.nan_to_num(_f32(d.reciprocal()), posinf=0.0)
        keep = torch.nan_to_num(_f32(old / d))
        cell = _f32(held[p, :, b] * keep[:, None, None]).round()
        cell[:, off: off + hi - lo] = _f32(rows.transpose(0, 1) * inv[:, None, None]).round()
        held[p, :, b], d_all[p, :, b] = cell, d
        lo = hi
    return (held * d_all[..., None, None]).view(P, g, page, hd), d_all


def _exact_append(s, c):
    nh, nkv, hd, T = c["nh"], c["nkv"], c["hd"], c["T"]
    x = s.qkv[:T].double().view(T, nh + 2 * nkv, hd // 2, 2)
    pos, slot = s.positions[:T].long(), s.slots[:T].long()
    if s.cos is not None:
        z = torch.complex(s.cos[pos, ::2].double(), s.sin[pos, ::2].double())
    else:
        z = torch.polar(torch.ones((T, hd // 2), device="cuda", dtype=torch.float64), pos.double()[:, None] * _freqs(hd))
    y = torch.view_as_real(torch.view_as_complex(x[:, : nh + nkv].contiguous()) * z[:, None]).flatten(2)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS)
    q = s.q.double()
    q[:T] = y[:, :nh] * s.qn.double()
    k, ks = _exact_write(s.k, s.ks, _f32(y[:, nh:] * s.kn.double()), slot, c)
    v, vs = _exact_write(s.v, s.vs, x[:, nh + nkv:].flatten(2), slot, c)
    return [q, k, v, ks, vs]


def _exact_attn(s, c):
    nh, nkv, P, B = c["nh"], c["nkv"], c["page"], c["block"]
    out = s.out.double()
    start, kv = s.q_start.tolist(), s.kv_len.tolist()
    for r in range(c["R"]):
        n, L = start[r + 1] - start[r], kv[r]
        j = torch.arange(L, device="cuda")
        page = s.table[r].long()[j // P]
        k = s.k[page, :, j % P].double() * s.ks[page, :, j % P // B].double()[..., None]
        v = s.v[page, :, j % P].double() * s.vs[page, :, j % P // B].double()[..., None]
        seen = torch.arange(L - n + 1, L + 1, device="cuda") if s.seen is None else s.seen[start[r]: start[r + 1]]
        for h in range(nh):
            sc = s.q[start[r]: start[r + 1], h].double() @ k[:, h // (nh // nkv)].t().contiguous() * s.scale
            p = torch.softmax(torch.where(j[None, :] < seen[:, None], sc, -math.inf), dim=1)
            out[start[r]: start[r + 1], h] = p @ v[:, h // (nh // nkv)].contiguous()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attn": _exact_attn}[case["kind"]](s, case)


# ------------------------------------------------------------------ floors

def work(case):
    c, kind = case, case["kind"]
    if kind == "linear":
        T, K, N = c["T"], c["K"], c["N"]
        return {"bytes": float(4 * T * K + N * K + 4 * N + 4 * T * N * (2 if c["resid"] else 1)),
                "flops": 2.0 * T * K * N}
    hd = c["hd"]
    if kind == "append":
        T = c["T"]
        blocks = T // c["block"] + 1
        return {"bytes": float(T * hd * (4 * (c["nh"] + 2 * c["nkv"]) + 4 * c["nh"] + 2 * c["nkv"])
                               + 8 * blocks * c["nkv"] + (8 * T * hd if c["table"] else 0)),
                "flops": 12.0 * T * hd * (c["nh"] + c["nkv"])}
    ctx, new = _lens(c)
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(ctx, new))
    keys = sum(a + n for a, n in zip(ctx, new))
    return {"bytes": float(8 * sum(new) * c["nh"] * hd + 2 * keys * c["nkv"] * hd
                           + 8 * keys * c["nkv"] / c["block"]),
            "flops": 4.0 * pairs * c["nh"] * hd}
