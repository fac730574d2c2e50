"""Paged serving without a device: exported names, struct layouts, and the refusals, which
come before anything is launched."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED = 0, -1, -2
P = 4096  # a pointer that is never followed


class At:
    ptr = P


def test_library_exports_paged_header(hy):
    syms = hy.header_symbols(hy.PAGED_HEADER)
    assert {"hy_paged_plan", "hy_rope_qknorm_paged", "hy_paged_attention", "hy_verify_drafts",
            "hy_attn_forward_paged", "hy_model_forward_paged"} <= set(syms)
    assert not [s for s in syms if not hasattr(hy.lib(), s)]


def test_signatures_match_header(hy):
    text = re.sub(r"/\*.*?\*/", "", open(hy.PAGED_HEADER).read(), flags=re.S)
    for name in hy.header_symbols(hy.PAGED_HEADER):
        params = re.search(name + r"\s*\(([^)]*)\)", text).group(1).split(",")
        assert len(hy._SIGS[name][1]) == len(params), name


def test_struct_layouts_match_header(hy, tmp_path):
    structs = {"hy_paged_cache": hy.PagedCache, "hy_paged_batch": hy.PagedBatch}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "hy_paged.h"', 'int main(void) {']
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            cname, f, v = line.split()
            py = structs[cname]
            assert int(v) == (C.sizeof(py) if f == "size" else getattr(py, f).offset), line


def _cache(hy, **kw):
    c = hy.PagedCache(At, At, hy.F16, 10, 16, 8, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _batch(hy, **kw):
    b = hy.PagedBatch(2, 7, 5, 4, At, At, At, At, At)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_CACHE = [
    (dict(k_dev=None), INVALID), (dict(v_dev=None), INVALID), (dict(type=2), UNSUPPORTED), (dict(type=8), UNSUPPORTED),
    (dict(page_size=4), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED), (dict(page_size=8192), UNSUPPORTED),
    (dict(page_size=0), UNSUPPORTED), (dict(n_pages=0), INVALID), (dict(n_pages=1 << 27), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(n_kv_heads=0), INVALID), (dict(n_kv_heads=5), INVALID),
    (dict(k_dev=P + 8), INVALID), (dict(v_dev=P + 2), INVALID),
    (dict(page_stride=1 << 14), INVALID),                                               # some strides 0
    (dict(page_stride=1 << 14, head_stride=2048, token_stride=132), INVALID),           # not 16 bytes
    (dict(page_stride=1 << 14, head_stride=2048, token_stride=64), INVALID),            # below head_dim
    (dict(page_stride=1 << 41, head_stride=2048, token_stride=128), INVALID),
    (dict(page_stride=1 << 14, head_stride=2048, token_stride=(1 << 24) + 128), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", BAD_CACHE)
def test_cache_refused(hy, kw, code):
    L = hy.lib()
    c, b = _cache(hy, **kw), _batch(hy)
    assert L.hy_paged_attention(P, 32, c, b, 1.0, P, P, 1 << 40, None) == code
    assert L.hy_last_error().decode()
    assert L.hy_paged_attention_ws(32, c, b) == 0
    assert L.hy_rope_qknorm_paged(P, 7, 32, c, P, P, 1e4, None, None, 0, P, P, 1e-5, P, None) == code


@pytest.mark.parametrize("kw", [
    dict(n_req=0), dict(n_req=4097), dict(n_rows=0), dict(n_rows=(1 << 20) + 1), dict(max_pages=0),
    dict(max_pages=(1 << 26) + 1), dict(q_start_dev=None), dict(kv_len_dev=None), dict(table_dev=None)])
def test_batch_refused(hy, kw):
    L = hy.lib()
    c, b = _cache(hy), _batch(hy, **kw)
    assert L.hy_paged_attention(P, 32, c, b, 1.0, P, P, 1 << 40, None) == INVALID
    assert L.hy_last_error().decode()
    assert L.hy_paged_attention_ws(32, c, b) == 0
    with pytest.raises(hy.HyError):
        hy.paged_attention_ws(32, c, b)


def test_attention_refused(hy):
    L = hy.lib()
    c, b = _cache(hy), _batch(hy)
    need = L.hy_paged_attention_ws(32, c, b)
    assert need > 0
    good = dict(q=P, nh=32, scale=0.1, out=P, ws=P, n=need)
    for kw in (dict(q=None), dict(out=None), dict(ws=None), dict(n=need - 1), dict(ws=P + 4), dict(q=P + 4),
               dict(out=P + 8), dict(scale=float("nan")), dict(scale=float("inf")), dict(nh=12), dict(nh=0),
               dict(nh=2048)):
        a = {**good, **kw}
        assert L.hy_paged_attention(a["q"], a["nh"], c, b, a["scale"], a["out"], a["ws"], a["n"], None) == INVALID, kw
    assert L.hy_paged_attention(P, 32, None, b, 0.1, P, P, need, None) == INVALID
    assert L.hy_paged_attention(P, 32, c, None, 0.1, P, P, need, None) == INVALID


def test_append_refused(hy):
    L = hy.lib()
    good = dict(qkv=P, n=7, pos=P, slots=P, theta=1e4, cos=None, sin=None, n_pos=0, eps=1e-5, q=P, qn=P)
    for kw in (dict(qkv=None), dict(pos=None), dict(slots=None), dict(q=None), dict(n=0), dict(n=(1 << 20) + 1),
               dict(theta=-1.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(cos=P, n_pos=4),
               dict(sin=P, n_pos=4), dict(cos=P, sin=P, n_pos=0), dict(eps=-1.0), dict(eps=float("nan")),
               dict(qkv=P + 4), dict(q=P + 8), dict(qn=P + 4), dict(cos=P + 4, sin=P, n_pos=4)):
        a = {**good, **kw}
        rc = L.hy_rope_qknorm_paged(a["qkv"], a["n"], 32, _cache(hy), a["pos"], a["slots"], a["theta"], a["cos"],
                                    a["sin"], a["n_pos"], a["qn"], P, a["eps"], a["q"], None)
        assert rc == INVALID, kw


def test_plan_refused(hy):
    L = hy.lib()
    sizes = dict(n_req=3, n_rows=9, page=16, max_pages=4, n_pages=12)
    for kw, code in ((dict(n_req=0), INVALID), (dict(n_req=4097), INVALID), (dict(n_rows=0), INVALID),
                     (dict(n_rows=(1 << 20) + 1), INVALID), (dict(page=12), UNSUPPORTED), (dict(page=4), UNSUPPORTED),
                     (dict(max_pages=0), INVALID), (dict(max_pages=1 << 27), INVALID), (dict(n_pages=0), INVALID),
                     (dict(n_pages=1 << 27), INVALID)):
        a = {**sizes, **kw}
        assert L.hy_paged_plan(P, P, *a.values(), *[P] * 11, None) == code, kw
    for i in range(13):
        ptrs = [P] * 13
        ptrs[i] = None
        assert L.hy_paged_plan(*ptrs[:2], *sizes.values(), *ptrs[2:], None) == INVALID, i


def test_verify_refused(hy):
    L = hy.lib()
    need = L.hy_verify_drafts_ws(2, 9, 1000)
    assert need > 0
    good = dict(logits=P, draft=P, ids=P, qs=P, n_req=2, n_rows=9, max_new=5, vocab=1000, temp=P, ua=P, us=P, acc=P,
                tok=P, ws=P, n=need)
    for kw in (dict(logits=None), dict(ids=None), dict(qs=None), dict(ua=None), dict(us=None), dict(acc=None),
               dict(tok=None), dict(ws=None), dict(n=need - 1), dict(ws=P + 4), dict(n_req=0), dict(n_req=4097),
               dict(n_rows=0), dict(n_rows=(1 << 20) + 1), dict(max_new=0), dict(max_new=(1 << 20) + 1),
               dict(vocab=0), dict(vocab=(1 << 22) + 1)):
        a = {**good, **kw}
        assert L.hy_verify_drafts(*a.values(), None) == INVALID, kw
        assert L.hy_last_error().decode()
    for bad in ((0, 9, 1000), (2, 0, 1000), (2, 9, 0), (2, 9, (1 << 22) + 1)):
        assert L.hy_verify_drafts_ws(*bad) == 0
        with pytest.raises(hy.HyError):
            hy.verify_drafts_ws(*bad)


def test_context_calls_refuse_null(hy):
    L = hy.lib()
    assert L.hy_attn_forward_paged(None, 0, P, _cache(hy), _batch(hy), None, None, 0, P, P, 1 << 40, None) == INVALID
    assert L.hy_model_forward_paged(None, P, _cache(hy), _batch(hy), P, P, 1 << 40, None) == INVALID


def test_verify_refuses_what_no_launch_covers(hy):
    L = hy.lib()
    n_rows, vocab = 1 << 20, (1 << 16) + 1     # past 2^36 logits
    assert L.hy_verify_drafts_ws(4, n_rows, vocab) == 0
    assert L.hy_verify_drafts(P, None, P, P, 4, n_rows, 5, vocab, None, P, P, P, P, P, 1 << 62, None) == UNSUPPORTED
    assert L.hy_last_error().decode()
    assert L.hy_verify_drafts_ws(4, n_rows, vocab - 1) > 0


def test_workspace_is_bounded(hy):
    """What the header promises, over every choice of kernels."""
    L = hy.lib()
    for t in (0, 1, 30):
        for hd in (64, 128):
            for nkv, nh in ((1, 1), (1, 64), (8, 32), (8, 1024)):
                for n_req in (1, 2, 3, 4096):
                    for max_new in (0, 1, 4, 8, 16, 33, 700, 1 << 20):
                        n = L.hy_paged_attention_ws(nh, _cache(hy, type=t, head_dim=hd, n_kv_heads=nkv),
                                                    _batch(hy, n_req=n_req, n_rows=1 << 20, max_new=max_new))
                        assert 0 < n <= 103_000_000
