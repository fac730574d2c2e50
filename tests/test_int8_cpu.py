"""Serving in 8 bits without a device: exported names, signatures, struct layouts, and the refusals,
which come before anything is launched."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import int8_ref as Q

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -2
P = 4096  # a pointer that is never followed


class At:
    ptr = P


def test_library_exports_header(hy):
    syms = hy.header_symbols(hy.INT8_HEADER)
    assert {"hy_quantize_rows_i8", "hy_gemm_i8", "hy_linear_i8", "hy_rope_qknorm_paged_i8",
            "hy_paged_attention_i8"} <= set(syms)
    assert not [s for s in syms if not hasattr(hy.lib(), s)]
    text = re.sub(r"/\*.*?\*/", "", open(hy.INT8_HEADER).read(), flags=re.S)
    for name in syms:
        params = re.search(name + r"\s*\(([^)]*)\)", text).group(1).split(",")
        assert len(hy._SIGS[name][1]) == len(params), name


def test_struct_layout_matches_header(hy, tmp_path):
    py = hy.PagedCacheI8
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "hy_int8.h"', 'int main(void) {',
             'printf("size %zu\\n", sizeof(hy_paged_cache_i8));']
    lines += [f'printf("{f} %zu\\n", offsetof(hy_paged_cache_i8, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            f, v = line.split()
            assert int(v) == (C.sizeof(py) if f == "size" else getattr(py, f).offset), line


def _cache(hy, block=16, ks=P, vs=P, **kw):
    c = hy.PagedCache(At, At, hy.I8, 10, 16, 8, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    c8 = hy.PagedCacheI8(c, At, At, block)
    c8.k_scale_dev, c8.v_scale_dev = ks, vs
    return c8


def _batch(hy, **kw):
    b = hy.PagedBatch(2, 7, 5, 4, At, At, At, At, At)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("kw,code", [
    (dict(k_dev=None), INVALID), (dict(v_dev=None), INVALID), (dict(ks=None), INVALID), (dict(vs=None), INVALID),
    (dict(ks=P + 2), INVALID), (dict(vs=P + 1), INVALID), (dict(type=0), UNSUPPORTED), (dict(type=1), UNSUPPORTED),
    (dict(type=8), UNSUPPORTED), (dict(block=0), UNSUPPORTED), (dict(block=4), UNSUPPORTED),
    (dict(block=12), UNSUPPORTED), (dict(block=32), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(page_size=8192), UNSUPPORTED), (dict(n_pages=0), INVALID), (dict(n_pages=1 << 27), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(n_kv_heads=5), INVALID), (dict(k_dev=P + 8), INVALID),
    (dict(page_stride=1 << 14), INVALID), (dict(page_stride=1 << 14, head_stride=2048, token_stride=136), INVALID),
    (dict(page_stride=1 << 14, head_stride=2048, token_stride=64), INVALID)])
def test_cache_refused(hy, kw, code):
    L = hy.lib()
    c, b = _cache(hy, **kw), _batch(hy)
    assert L.hy_paged_attention_i8(P, 32, c, b, 1.0, P, P, 1 << 40, None) == code
    assert L.hy_last_error().decode()
    assert L.hy_paged_attention_i8_ws(32, c, b) == 0
    assert L.hy_rope_qknorm_paged_i8(P, 7, 32, c, P, P, 1e4, None, None, 0, P, P, 1e-5, P, None) == code
    with pytest.raises(hy.HyError):
        hy.paged_attention_i8_ws(32, c, b)


def test_other_calls_refuse_the_type(hy):
    """The calls of hy_paged.h know nothing of scales."""
    L, c = hy.lib(), hy.PagedCache(At, At, hy.I8, 10, 16, 8, 128)
    assert L.hy_paged_attention(P, 32, c, _batch(hy), 1.0, P, P, 1 << 40, None) == UNSUPPORTED
    assert L.hy_rope_qknorm_paged(P, 7, 32, c, P, P, 1e4, None, None, 0, P, P, 1e-5, P, None) == UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(n_req=0), dict(n_req=4097), dict(n_rows=0), dict(n_rows=(1 << 20) + 1), dict(max_pages=0),
    dict(max_pages=(1 << 26) + 1), dict(q_start_dev=None), dict(kv_len_dev=None), dict(table_dev=None)])
def test_batch_refused(hy, kw):
    L = hy.lib()
    c, b = _cache(hy), _batch(hy, **kw)
    assert L.hy_paged_attention_i8(P, 32, c, b, 1.0, P, P, 1 << 40, None) == INVALID
    assert L.hy_paged_attention_i8_ws(32, c, b) == 0


def test_attention_refused(hy):
    L = hy.lib()
    c, b = _cache(hy), _batch(hy)
    need = L.hy_paged_attention_i8_ws(32, c, b)
    assert need > 0
    good = dict(q=P, nh=32, scale=0.1, out=P, ws=P, n=need)
    for kw in (dict(q=None), dict(out=None), dict(ws=None), dict(n=need - 1), dict(ws=P + 4), dict(q=P + 4),
               dict(out=P + 8), dict(scale=float("nan")), dict(scale=float("inf")), dict(nh=12), dict(nh=0),
               dict(nh=2048)):
        a = {**good, **kw}
        assert L.hy_paged_attention_i8(a["q"], a["nh"], c, b, a["scale"], a["out"], a["ws"], a["n"], None) == INVALID, kw
    assert L.hy_paged_attention_i8(P, 32, None, b, 0.1, P, P, need, None) == INVALID
    assert L.hy_paged_attention_i8(P, 32, c, None, 0.1, P, P, need, None) == INVALID


def test_append_refused(hy):
    L = hy.lib()
    good = dict(qkv=P, n=7, pos=P, slots=P, theta=1e4, cos=None, sin=None, n_pos=0, eps=1e-5, q=P, qn=P)
    for kw in (dict(qkv=None), dict(pos=None), dict(slots=None), dict(q=None), dict(n=0), dict(n=(1 << 20) + 1),
               dict(theta=-1.0), dict(theta=float("nan")), dict(cos=P, n_pos=4), dict(sin=P, n_pos=4),
               dict(cos=P, sin=P, n_pos=0), dict(eps=-1.0), dict(eps=float("nan")), dict(qkv=P + 4), dict(q=P + 8),
               dict(qn=P + 4), dict(cos=P + 4, sin=P, n_pos=4)):
        a = {**good, **kw}
        rc = L.hy_rope_qknorm_paged_i8(a["qkv"], a["n"], 32, _cache(hy), a["pos"], a["slots"], a["theta"], a["cos"],
                                       a["sin"], a["n_pos"], a["qn"], P, a["eps"], a["q"], None)
        assert rc == INVALID, kw
    assert L.hy_rope_qknorm_paged_i8(P, 7, 32, None, P, P, 1e4, None, None, 0, P, P, 1e-5, P, None) == INVALID


def test_products_refused(hy):
    L = hy.lib()
    for bad in ((0, 64, 8), ((1 << 20) + 1, 64, 8), (4, 0, 8), (4, 72, 8), (4, 1 << 17, 8), (4, 64, 0),
                (4, 64, (1 << 22) + 1)):
        assert L.hy_gemm_i8_ws(*bad) == 0 and L.hy_linear_i8_ws(*bad) == 0
        assert L.hy_gemm_i8(P, P, P, P, None, *bad, P, P, 1 << 62, None) == INVALID
        assert L.hy_linear_i8(P, P, P, None, *bad, P, P, 1 << 62, None) == INVALID
        with pytest.raises(hy.HyError):
            hy.gemm_i8_ws(*bad)
        with pytest.raises(hy.HyError):
            hy.linear_i8_ws(*bad)
    need = L.hy_gemm_i8_ws(4, 64, 8)
    assert need >= 16
    good = dict(x=P, xs=P, w=P, ws=P, r=None, T=4, K=64, N=8, out=P, wsp=P, n=need)
    for kw in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(wsp=None),
               dict(n=need - 1), dict(wsp=P + 4), dict(x=P + 8), dict(w=P + 1), dict(out=P + 2), dict(r=P + 3),
               dict(xs=P + 1), dict(ws=P + 2)):
        assert L.hy_gemm_i8(*{**good, **kw}.values(), None) == INVALID, kw
        assert L.hy_last_error().decode()
    need = L.hy_linear_i8_ws(4, 64, 8)
    assert need >= 4 * 64 + 16
    good = dict(x=P, w=P, ws=P, r=None, T=4, K=64, N=8, out=P, wsp=P, n=need)
    for kw in (dict(x=None), dict(w=None), dict(ws=None), dict(out=None), dict(wsp=None), dict(n=need - 1),
               dict(wsp=P + 8), dict(x=P + 8), dict(w=P + 1), dict(out=P + 2), dict(r=P + 3), dict(ws=P + 2)):
        assert L.hy_linear_i8(*{**good, **kw}.values(), None) == INVALID, kw
    for kw in (dict(x=None), dict(c=None), dict(s=None), dict(r=0), dict(r=(1 << 24) + 1), dict(n=0), dict(n=24),
               dict(n=1 << 17), dict(x=P + 4), dict(c=P + 4), dict(s=P + 1)):
        a = {**dict(x=P, r=3, n=64, c=P, s=P), **kw}
        assert L.hy_quantize_rows_i8(*a.values(), None) == INVALID, kw


def test_context_calls_refuse_null(hy):
    L = hy.lib()
    assert L.hy_attn_forward_paged_i8(None, 0, P, _cache(hy), _batch(hy), None, None, 0, P, P, 1 << 40, None) == INVALID
    assert L.hy_model_forward_paged_i8(None, P, _cache(hy), _batch(hy), P, P, 1 << 40, None) == INVALID
    assert L.hy_attn_quantize_i8(None, 0) == INVALID and L.hy_model_quantize_i8(None) == INVALID


def test_workspace_is_bounded(hy):
    L = hy.lib()
    for hd in (64, 128):
        for nkv, nh in ((1, 1), (1, 64), (8, 32), (8, 1024)):
            for n_req in (1, 2, 3, 4096):
                for max_new in (0, 1, 4, 8, 16, 33, 700, 1 << 20):
                    n = L.hy_paged_attention_i8_ws(nh, _cache(hy, head_dim=hd, n_kv_heads=nkv),
                                                   _batch(hy, n_req=n_req, n_rows=1 << 20, max_new=max_new))
                    assert 0 < n <= 103_000_000


def test_reference_pool_growth():
    """The references' own steps: a block that grows keeps its values to half a step per growth."""
    rng = np.random.default_rng(1)
    p = Q.PoolI8(2, 16, 1, 64, 16, fill=55, scale_fill=99.0)
    y = rng.standard_normal((16, 1, 64)).astype(np.float32) * np.linspace(0.5, 4, 16)[:, None, None].astype(np.float32)
    for i in range(16):
        p.write(y[i:i + 1], [16 + i], "k")
    got = p.values().k[1, 0]
    assert np.abs(got - y[:, 0]).max() <= p.ks[1, 0, 0] * (0.5 + 15 * 0.5) * 1.001
    assert (p.k[0] == 55).all() and (p.v == 55).all() and p.ks[1, 0, 0] == np.float32(np.abs(y).max() / np.float32(127))
    p.write(y[:3], [16, 17, 18], "k")  # begins anew
    assert (p.k[1, 0, 3:] == 0).all() and p.ks[1, 0, 0] == np.float32(np.abs(y[:3]).max() / np.float32(127))
