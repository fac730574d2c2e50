"""The operators of paged serving as measurable cases: block tables and slot maps, the
rotary + QK-norm write into a paged cache, attention of new tokens over it, and the
verification of drafted tokens -- in plain torch (own = False) or through the entry points
of include/hy_paged.h (own = True).

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
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPES = {"f32": 0, "f16": 1, "bf16": 30}
_EPS = 1e-5
_THETA = 10000.0
_VOCAB = 133120  # HunyuanImage-3's
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
        # eight chats, one new token each: the smallest step's tables
        dict(name="plan_r8", kind="plan", R=8, ctx=2000, new=1, page=16, pad=0),
        # a full server: a thousand requests, some starting, some ending, some prompts
        dict(name="plan_r1024", kind="plan", R=1024, ctx=8000, new=48, page=16, pad=100),
        # one request's drafted tokens into a 16-bit cache
        dict(name="append_f16_t5", kind="append", dt="f16", T=5, page=16, table=False, pad=0, **_BIG),
        # an image's 64 x 64 tokens, 2D rotary tables, unrounded cache
        dict(name="append_f32_t4096", kind="append", dt="f32", T=4096, page=64, table=True, pad=0, **_BIG),
        # one chat, one new token
        dict(name="attn_one_f32", kind="attn", dt="f32", R=1, ctx=1000, new=1, mode="decode", page=16, spans=False,
             pad=0, **_BIG),
        # a busy server's decode step over long ragged caches
        dict(name="attn_decode_bf16", kind="attn", dt="bf16", R=64, ctx=8000, new=1, mode="decode", page=16,
             spans=False, pad=0, **_BIG),
        # the check of up to five drafted tokens per request
        dict(name="attn_draft_f16", kind="attn", dt="f16", R=32, ctx=2900, new=6, mode="draft", page=16, spans=False,
             pad=5, **_BIG),
        # a chunk of a long prompt behind what is cached, unrounded cache: the largest call
        dict(name="attn_chunk_f32", kind="attn", dt="f32", R=1, ctx=8192, new=2048, mode="chunk", page=64, spans=False,
             pad=0, **_BIG),
        # chunks and single tokens together, the chunks' image spans seen as a whole
        dict(name="attn_mixed_bf16", kind="attn", dt="bf16", R=12, ctx=4500, new=700, mode="mixed", page=32, spans=True,
             pad=3, **_BIG),
        # prompts without a past, small heads
        dict(name="attn_prompt_f16", kind="attn", dt="f16", R=5, ctx=0, new=1500, mode="chunk", page=16, spans=False,
             pad=0, nh=16, nkv=4, hd=64),
        # four requests, four drafts each, a drafter that gives no probabilities
        dict(name="verify_r4", kind="verify", R=4, new=5, V=_VOCAB, probs=False, pad=0),
        # a busy server: up to five drafts each, sampled drafts, some requests greedy
        dict(name="verify_r64", kind="verify", R=64, new=6, V=_VOCAB, probs=True, pad=2),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm, any residue."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 5e12, w["flops"] / 4e14)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _draw(rng):
    kind = rng.choice(["plan", "append", "attn", "attn", "attn", "attn", "verify"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind == "plan":
        return dict(kind="plan", R=_spread(rng, 1, 2048), ctx=_spread(rng, 1, 16000),
                    new=rng.choice([1, 1, 8, _spread(rng, 1, 64)]), page=page, pad=rng.choice([0, 0, 7, 100]))
    heads = rng.choice([_BIG, _BIG, _BIG, dict(nh=16, nkv=4, hd=64), dict(nh=16, nkv=4, hd=128),
                        dict(nh=8, nkv=8, hd=128), dict(nh=16, nkv=2, hd=64), dict(nh=20, nkv=4, hd=128)])
    dt = rng.choice(["f32", "f16", "bf16"])
    if kind == "append":
        return dict(kind="append", dt=dt, T=_spread(rng, 1, 8192), page=page, table=rng.random() < 0.4,
                    pad=rng.choice([0, 0, 3, 40]), **heads)
    if kind == "verify":
        return dict(kind="verify", R=_spread(rng, 1, 64), new=rng.randint(1, 8),
                    V=rng.choice([_VOCAB, _VOCAB, 32000, 32003, 8000]), probs=rng.random() < 0.6,
                    pad=rng.choice([0, 0, 3]))
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
    return dict(kind="attn", dt=dt, R=R, ctx=ctx, new=new, mode=mode, page=page,
                spans=mode in ("chunk", "mixed") and rng.random() < 0.4, pad=rng.choice([0, 0, 3, 17]), **heads)


def _lens(c):
    """Cached and new lengths of a case's requests: ragged, the same for every seed."""
    g = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    ctx, new = [], []
    for r in range(c["R"]):
        n, lo, hi = c["new"], c["ctx"] // 4, c["ctx"]
        if r and c["kind"] != "plan":
            n = g.randint(1, n) if c.get("mode") != "mixed" or r % 2 else 1
        ctx.append(hi if r == 0 else g.randint(lo, hi))
        new.append(n)
    if c["kind"] == "plan":
        for r in range(c["R"]):
            what = g.random()
            if what < 0.05:
                ctx[r], new[r] = 0, 0  # ended: gives its pages back
            elif what < 0.10:
                ctx[r] = 0  # starts
            elif what < 0.9 and c["R"] > 8:
                new[r] = 1
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


def _prepare_plan(c, seed):
    s = _State()
    ctx, new = _lens(c)
    g = random.Random(c["R"] * 7919 + c["ctx"])
    # held: what the last step left; a few requests hold more (drafts not taken)
    held = [-(-x // c["page"]) + (g.randint(0, 2) if g.random() < 0.3 else 0) for x in ctx]
    held = [h + g.randint(1, 40) if x == 0 and n == 0 else h for h, x, n in zip(held, ctx, new)]
    s.n_rows = sum(new) + c["pad"]
    s.max_pages = max(max(held), max(-(-(x + n) // c["page"]) for x, n in zip(ctx, new)))
    s.n_pages = sum(held) + c["R"] // 2 + 5
    perm = torch.randperm(s.n_pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    s.cached, s.new, s.held = _ints(ctx), _ints(new), _ints(held)
    s.table = torch.full((c["R"], s.max_pages), -1, device="cuda", dtype=torch.int32)
    at = torch.arange(s.max_pages, device="cuda")[None, :]
    h = s.held.long()[:, None]
    first = torch.cumsum(h, 0) - h
    s.table[at < h] = perm[(first + at)[at < h]]
    s.free = torch.zeros(s.n_pages, device="cuda", dtype=torch.int32)
    n = s.n_pages - sum(held)
    s.free[:n] = perm[sum(held):]
    s.n_free = _ints([n])
    R = c["R"]
    s.held_out, s.n_free_out = torch.empty_like(s.held), torch.empty_like(s.n_free)
    s.q_start, s.kv_len, s.status = _ints([0] * (R + 1)), _ints([0] * R), _ints([0] * R)
    s.positions, s.slots = _ints([0] * s.n_rows), _ints([0] * s.n_rows)
    return s


def _prepare_append(c, seed):
    s = _State()
    T, hd, page = c["T"], c["hd"], c["page"]
    # T tokens of one request behind 100 cached ones
    ctx = 100
    s.n_rows = T + c["pad"]
    table, s.n_pages = _tables(c, seed, [ctx + T])
    pos = torch.arange(ctx, ctx + T, device="cuda")
    slot = table[0, pos // page].long() * page + pos % page
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
    s.k = torch.zeros((s.n_pages, c["nkv"], page, hd), device="cuda", dtype=_DT[c["dt"]])
    s.v = torch.zeros_like(s.k)
    s.q = torch.zeros((s.n_rows, c["nh"], hd), device="cuda")
    return s


def _freqs(hd):
    return _THETA ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)


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
    shape = (s.n_pages, c["nkv"], c["page"], c["hd"])
    s.k = _randn(shape, _gen(seed, 3)).to(_DT[c["dt"]])
    s.v = _randn(shape, _gen(seed, 4)).to(_DT[c["dt"]])
    s.scale = 1.0 / math.sqrt(c["hd"])
    s.out = torch.zeros((s.n_rows, c["nh"], c["hd"]), device="cuda")
    s.ws = None
    return s


def _prepare_verify(c, seed):
    s = _State()
    _, new = _lens(dict(c, ctx=0))
    R, V = c["R"], c["V"]
    s.n_rows, s.max_new = sum(new) + c["pad"], max(new)
    s.q_start = _ints([sum(new[:i]) for i in range(R + 1)])
    # a head of likely tokens over a tail, another head on each row
    g = _gen(seed, 2)
    s.logits = _randn((s.n_rows, V), g, 2.0)
    head = torch.randint(0, V, (s.n_rows, 8), generator=g, device="cuda")
    s.logits.scatter_add_(1, head, _randn((s.n_rows, 8), g, 2.0) + 10.0)
    s.temp = 0.6 + 0.5 * torch.rand(R, generator=g, device="cuda")
    s.temp[3::4] = 0.0  # greedy
    # the drafter: the target's logits, a little off
    d = torch.softmax(s.logits * 0.9 + _randn((s.n_rows, V), g, 0.5), dim=1)
    ids = torch.multinomial(d, 1, generator=g)[:, 0] if c["probs"] else d.argmax(1)
    s.ids = torch.roll(ids, 1).int()
    s.draft = d if c["probs"] else None
    s.u_accept = torch.rand(s.n_rows, generator=g, device="cuda")
    s.u_sample = torch.rand(R, generator=g, device="cuda")
    s.accepted = _ints([0] * R)
    s.tokens = torch.zeros((R, s.max_new), device="cuda", dtype=torch.int32)
    s.ws = None
    return s


def prepare(case, seed):
    s = {"plan": _prepare_plan, "append": _prepare_append, "attn": _prepare_attn,
         "verify": _prepare_verify}[case["kind"]](case, seed)
    s.case = case
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ plain forms

def _plain_plan(s, c):
    P, R = c["page"], c["R"]
    cached, new, held = s.cached.long(), s.new.long(), s.held.long()
    rows = torch.where((new >= 0) & (new <= s.n_rows), new, 0)
    incl = torch.cumsum(rows, 0)
    start = incl - rows
    q_start = torch.cat([torch.zeros_like(incl[:1]), incl]).clamp(max=s.n_rows)
    length = cached + new
    want = (length + P - 1) // P
    bad = (cached < 0) | (new < 0) | (start + new > s.n_rows) | (held < 0) | (held > s.max_pages)
    longer = ~bad & (want > s.max_pages)
    ok = ~bad & ~longer
    excess = torch.where(ok, (held - want).clamp(min=0), 0)
    need = torch.where(ok, (want - held).clamp(min=0), 0)
    n_free = s.n_free.long().clamp(0, s.n_pages)
    at = torch.arange(s.max_pages, device="cuda")[None, :]
    # pages given back go on the stack, in order; behind its end is a place for what does not exist
    give = ok[:, None] & (at >= want[:, None]) & (at < held[:, None])
    to = n_free + (torch.cumsum(excess, 0) - excess)[:, None] + at - want[:, None]
    stack = torch.cat([s.free, s.free[:1]])
    stack[torch.where(give & (to < s.n_pages), to, s.n_pages)] = s.table
    n1 = (n_free + excess.sum()).clamp(max=s.n_pages)
    upto = torch.cumsum(need, 0)
    served = ok & ((need == 0) | (upto <= n1))
    take = served[:, None] & (at >= held[:, None]) & (at < want[:, None])
    frm = n1 - 1 - (upto - need)[:, None] - at + held[:, None]
    s.table.copy_(torch.where(take, stack[torch.where(take, frm, 0)], s.table))
    s.free.copy_(stack[: s.n_pages])
    held_out = torch.where(served, want, held)
    n_out = n1 - torch.where(served, need, 0).sum()
    status = torch.where(bad, 3, torch.where(longer, 2, torch.where(served, 0, 1)))
    t = torch.arange(s.n_rows, device="cuda")
    r = torch.searchsorted(incl, t, right=True).clamp(max=R - 1)
    live = (t < incl[-1]) & served[r]
    pos = torch.where(live, cached[r] + t - start[r], 0)
    page = s.table[r, pos // P].long()
    slot = torch.where(live & (page >= 0) & (page < s.n_pages), page * P + pos % P, -1)
    return [s.table, held_out.int(), s.free, n_out.int(), q_start.int(), torch.where(served, length, 0).int(),
            pos.int(), slot.int(), status.int()]


def _plain_append(s, c):
    nh, nkv, hd, P = c["nh"], c["nkv"], c["hd"], c["page"]
    live = s.slots >= 0
    x = s.qkv[live].view(-1, nh + 2 * nkv, hd)
    pos, slot = s.positions[live].long(), s.slots[live].long()
    if s.cos is not None:
        cs, sn = s.cos[pos][:, None, ::2], s.sin[pos][:, None, ::2]
    else:
        ang = pos.double()[:, None] * _freqs(hd)
        cs, sn = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    a, b = x[:, : nh + nkv, ::2], x[:, : nh + nkv, 1::2]
    rot = torch.stack([a * cs - b * sn, a * sn + b * cs], dim=-1).flatten(2)
    rot = rot / torch.sqrt((rot * rot).mean(-1, keepdim=True) + _EPS)
    s.q[live] = rot[:, :nh] * s.qn
    s.k[slot // P, :, slot % P] = (rot[:, nh:] * s.kn).to(s.k.dtype)
    s.v[slot // P, :, slot % P] = x[:, nh + nkv:].to(s.v.dtype)
    return [s.q, s.k, s.v]


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
    in_len = (j < s.kv_len[:, None])[:, :, None, None]
    k = torch.where(in_len, s.k[page, :, j % P].float(), 0.0).permute(0, 2, 3, 1).contiguous()  # [R][nkv][hd][keys]
    v = torch.where(in_len, s.v[page, :, j % P].float(), 0.0).permute(0, 2, 1, 3).contiguous()  # [R][nkv][keys][hd]
    q = s.q[rows].view(R, N, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4).reshape(R, nkv, -1, hd) * s.scale
    sc = torch.matmul(q, k).view(R, nkv, N, nh // nkv, -1)
    sc = sc.masked_fill((j[:, None, :] >= seen[:, :, None])[:, None, :, None, :], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(sc - m)
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.matmul(e.view(R, nkv, -1, e.shape[-1]), v).view(R, nkv, N, nh // nkv, hd)
    s.out[rows[there]] = o.permute(0, 2, 1, 3, 4).reshape(R, N, nh, hd)[there]
    return s.out


def _plain_verify(s, c):
    V, N = c["V"], s.max_new
    start = s.q_start.long()
    n = start[1:] - start[:-1]
    total = s.n_rows - c["pad"]
    t = torch.arange(total, device="cuda")
    r = torch.searchsorted(start, t, right=True) - 1
    l = s.logits[:total].double()
    m = l.amax(1, keepdim=True)
    ids = torch.arange(V, device="cuda")
    best = torch.where(l == m, ids, V).amin(1)
    greedy = s.temp[r] <= 0
    w = torch.exp((l - m) / torch.where(greedy, 1.0, s.temp[r].double())[:, None])
    p = w / w.sum(1, keepdim=True)
    x = s.ids[(t + 1).clamp(max=s.n_rows - 1)].long()
    q_x = s.draft[t, x].double() if s.draft is not None else torch.ones_like(p[:, 0])
    take = torch.where(greedy, x == best, s.u_accept[:total].double() * q_x < p[t, x])
    i = torch.arange(N, device="cuda")[None, :]
    row = (start[:-1, None] + i).clamp(max=total - 1)
    is_draft = i < (n - 1)[:, None]
    accepted = torch.cumprod((take[row] & is_draft).int(), 1).sum(1)
    last = start[:-1] + accepted
    refused = accepted < n - 1
    q = s.draft[last].double() if s.draft is not None else (ids[None, :] == x[last][:, None]).double()
    rest = torch.where(refused[:, None] & (p[last] > q), p[last] - q, torch.where(refused[:, None], 0.0, p[last]))
    if s.draft is None:  # the drafter's token was certain
        rest = torch.where(refused[:, None] & (q > 0), 0.0, p[last])
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p[last])
    cdf = torch.cumsum(rest, 1)
    over = cdf > s.u_sample.double()[:, None] * cdf[:, -1:]
    tok = torch.where(over, ids, V).amin(1)
    tok = torch.where(tok < V, tok, torch.where(rest > 0, ids, -1).amax(1))
    tok = torch.where(greedy[last], best[last], tok)
    drafts = x[row]
    tokens = torch.where(i < accepted[:, None], drafts, torch.where(i == accepted[:, None], tok[:, None], -1))
    return [accepted.int(), tokens.int()]


# ------------------------------------------------------------------ the framework's calls

def _own_plan(s, c):
    _hy().paged_plan(_Dev(s.cached), _Dev(s.new), c["R"], s.n_rows, c["page"], s.max_pages, s.n_pages, _Dev(s.table),
                     _Dev(s.held), _Dev(s.held_out), _Dev(s.free), _Dev(s.n_free), _Dev(s.n_free_out),
                     _Dev(s.q_start), _Dev(s.kv_len), _Dev(s.positions), _Dev(s.slots), _Dev(s.status), _stream())
    return [s.table, s.held_out, s.free, s.n_free_out[0], s.q_start, s.kv_len, s.positions, s.slots, s.status]


def _cache(s, c):
    return _hy().PagedCache(_Dev(s.k), _Dev(s.v), _TYPES[c["dt"]], s.n_pages, c["page"], c["nkv"], c["hd"])


def _own_append(s, c):
    _hy().rope_qknorm_paged(_Dev(s.qkv), s.n_rows, c["nh"], _cache(s, c), _Dev(s.positions), _Dev(s.slots), _THETA,
                            None if s.cos is None else _Dev(s.cos), None if s.sin is None else _Dev(s.sin), s.n_pos,
                            _Dev(s.qn), _Dev(s.kn), _EPS, _Dev(s.q), _stream())
    return [s.q, s.k, s.v]


def _own_attn(s, c):
    hy = _hy()
    cache = _cache(s, c)
    batch = hy.PagedBatch(c["R"], s.n_rows, s.max_pages, s.max_new, _Dev(s.q_start), _Dev(s.kv_len), _Dev(s.table),
                          seen=None if s.seen is None else _Dev(s.seen))
    if s.ws is None:
        s.ws = torch.empty(hy.paged_attention_ws(c["nh"], cache, batch), dtype=torch.uint8, device="cuda")
    hy.paged_attention(_Dev(s.q), c["nh"], cache, batch, s.scale, _Dev(s.out), _Dev(s.ws), s.ws.numel(), _stream())
    return s.out


def _own_verify(s, c):
    hy = _hy()
    if s.ws is None:
        s.ws = torch.empty(hy.verify_drafts_ws(c["R"], s.n_rows, c["V"]), dtype=torch.uint8, device="cuda")
    hy.verify_drafts(_Dev(s.logits), None if s.draft is None else _Dev(s.draft), _Dev(s.ids), _Dev(s.q_start), c["R"],
                     s.n_rows, s.max_new, c["V"], _Dev(s.temp), _Dev(s.u_accept), _Dev(s.u_sample), _Dev(s.accepted),
                     _Dev(s.tokens), _Dev(s.ws), s.ws.numel(), _stream())
    return [s.accepted, s.tokens]


def run(s):
    c = s.case
    kind = c["kind"]
    if own:
        if kind == "plan":
            return _own_plan(s, c)
        if kind == "append":
            return _own_append(s, c)
        if kind == "attn":
            return _own_attn(s, c)
        return _own_verify(s, c)
    if kind == "plan":
        r = _plain_plan(s, c)
        return r[:3] + [r[3][0]] + r[4:]
    if kind == "append":
        return _plain_append(s, c)
    if kind == "attn":
        return _plain_attn(s, c)
    return _plain_verify(s, c)


# ------------------------------------------------------------------ 64 bits

def _exact_plan(s, c):
    """Request by request on the host."""
    P = c["page"]
    table, free = s.table.cpu().tolist(), s.free.cpu().tolist()
    cached, new, held = s.cached.tolist(), s.new.tolist(), s.held.tolist()
    n = s.n_free.tolist()[0]
    q_start = [0]
    for x in new:
        q_start.append(q_start[-1] + x)
    want = [-(-(a + b) // P) for a, b in zip(cached, new)]
    for r in range(c["R"]):
        for k in range(want[r], held[r]):
            free[n] = table[r][k]
            n += 1
    status, out_of = [0] * c["R"], False
    for r in range(c["R"]):
        need = max(0, want[r] - held[r])
        out_of = out_of or need > n
        if need and out_of:
            status[r] = 1
            continue
        for k in range(need):
            n -= 1
            table[r][held[r] + k] = free[n]
        held[r] = want[r]
    pos, slot = [0] * s.n_rows, [-1] * s.n_rows
    for r in range(c["R"]):
        for i in range(new[r] if status[r] == 0 else 0):
            at = cached[r] + i
            pos[q_start[r] + i], slot[q_start[r] + i] = at, table[r][at // P] * P + at % P
    kv = [a + b if st == 0 else 0 for a, b, st in zip(cached, new, status)]
    return [_ints(table), _ints(held), _ints(free), _ints(n), _ints(q_start), _ints(kv), _ints(pos), _ints(slot),
            _ints(status)]


def _exact_append(s, c):
    nh, nkv, hd, P, T = c["nh"], c["nkv"], c["hd"], c["page"], c["T"]
    x = s.qkv[:T].double().view(T, nh + 2 * nkv, hd // 2, 2)
    pos, slot = s.positions[:T].long(), s.slots[:T].long()
    if s.cos is not None:
        z = torch.complex(s.cos[pos, ::2].double(), s.sin[pos, ::2].double())
    else:
        z = torch.polar(torch.ones((T, hd // 2), device="cuda", dtype=torch.float64), pos.double()[:, None] * _freqs(hd))
    y = torch.view_as_real(torch.view_as_complex(x[:, : nh + nkv].contiguous()) * z[:, None]).flatten(2)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS)
    q, k, v = s.q.double(), s.k.double(), s.v.double()
    q[:T] = y[:, :nh] * s.qn.double()
    k[slot // P, :, slot % P] = y[:, nh:] * s.kn.double()
    v[slot // P, :, slot % P] = x[:, nh + nkv:].flatten(2)
    return [q, k, v]


def _exact_attn(s, c):
    nh, nkv, hd, P = c["nh"], c["nkv"], c["hd"], c["page"]
    out = s.out.double()
    start, kv = s.q_start.tolist(), s.kv_len.tolist()
    for r in range(c["R"]):
        n, L = start[r + 1] - start[r], kv[r]
        j = torch.arange(L, device="cuda")
        page = s.table[r].long()[j // P]
        k, v = s.k[page, :, j % P].double(), s.v[page, :, j % P].double()
        seen = torch.arange(L - n + 1, L + 1, device="cuda") if s.seen is None else s.seen[start[r]: start[r + 1]]
        for h in range(nh):
            sc = s.q[start[r]: start[r + 1], h].double() @ k[:, h // (nh // nkv)].t().contiguous() * s.scale
            p = torch.softmax(torch.where(j[None, :] < seen[:, None], sc, -math.inf), dim=1)
            out[start[r]: start[r + 1], h] = p @ v[:, h // (nh // nkv)].contiguous()
    return out


def _exact_verify(s, c):
    """Token by token, as the definition reads."""
    accepted, tokens = [], []
    start = s.q_start.tolist()
    u, us, temp, ids = s.u_accept.tolist(), s.u_sample.tolist(), s.temp.double().tolist(), s.ids.tolist()
    for r in range(c["R"]):
        got = []
        for row in range(start[r], start[r + 1]):
            l = s.logits[row].double()
            x = ids[row + 1] if row + 1 < start[r + 1] else None
            if temp[r] <= 0:
                tok = int((l == l.max()).nonzero()[0])
                got.append(tok)
                if tok != x:
                    break
                continue
            p = torch.softmax(l / temp[r], dim=0)
            if x is None:
                rest = p
            else:
                q = torch.zeros_like(p).index_fill_(0, torch.tensor([x], device="cuda"), 1.0) if s.draft is None \
                    else s.draft[row].double()
                if u[row] * float(q[x]) < float(p[x]):
                    got.append(x)
                    continue
                rest = (p - q).clamp(min=0)
            cdf = rest.cumsum(0)
            got.append(int((cdf > us[r] * cdf[-1]).nonzero()[0]))
            break
        accepted.append(len(got) - 1)
        tokens.append(got + [-1] * (s.max_new - len(got)))
    return [_ints(accepted), _ints(tokens)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attn": _exact_attn,
            "verify": _exact_verify}[case["kind"]](s, case)


# ------------------------------------------------------------------ floors

def work(case):
    c, kind = case, case["kind"]
    if kind == "plan":
        _, new = _lens(c)
        moved = sum(new) // c["page"] + c["R"] // 8
        return {"bytes": 4.0 * (7 * c["R"] + 3 * moved + 2 * (sum(new) + c["pad"])), "flops": 0.0}
    if kind == "append":
        el = {"f32": 4, "f16": 2, "bf16": 2}[c["dt"]]
        T, hd = c["T"], c["hd"]
        return {"bytes": float(T * hd * (4 * (c["nh"] + 2 * c["nkv"]) + 4 * c["nh"] + 2 * el * c["nkv"])
                               + (8 * T * hd if c["table"] else 0)),
                "flops": 12.0 * T * hd * (c["nh"] + c["nkv"])}
    if kind == "attn":
        el = {"f32": 4, "f16": 2, "bf16": 2}[c["dt"]]
        ctx, new = _lens(c)
        pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(ctx, new))
        return {"bytes": float(8 * sum(new) * c["nh"] * c["hd"]
                               + 2 * el * sum(a + n for a, n in zip(ctx, new)) * c["nkv"] * c["hd"]),
                "flops": 4.0 * pairs * c["nh"] * c["hd"]}
    _, new = _lens(dict(c, ctx=0))
    return {"bytes": 4.0 * c["V"] * (sum(new) + (c["R"] if c["probs"] else 0)), "flops": 4.0 * c["V"] * sum(new)}
