"""Paged serving at the ends of its ranges, without a device: the arithmetic that finds a worker's
items."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = """
#include "hy_paged_part.hpp"
extern "C" int upto32(int n, int tau, int full, long long base, int k) {
    const hy::PartReq q{0, n, 0, 0, full, base, 0};
    return q.upto<int>(tau, k);
}
extern "C" long long upto64(int n, int tau, int full, long long base, long long k) {
    const hy::PartReq q{0, n, 0, 0, full, base, 0};
    return q.upto<int64_t>(tau, (int64_t)k);
}
"""


@pytest.fixture(scope="module")
def part(tmp_path_factory):
    """The host's side of csrc/hy_paged_part.hpp."""
    d = tmp_path_factory.mktemp("part")
    (d / "shim.hip").write_text(SHIM)
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-host-only", "-std=c++17", "-O1", "-fwrapv", "-shared", "-fPIC",
                    f"-I{ROOT}/include", f"-I{ROOT}/hunyuan-image-3-80b.cpp_amd/csrc", str(d / "shim.hip"), "-o",
                    str(d / "shim.so")], check=True)
    lib = C.CDLL(str(d / "shim.so"))
    lib.upto32.argtypes = [C.c_int, C.c_int, C.c_int, C.c_longlong, C.c_int]
    lib.upto64.argtypes = [C.c_int, C.c_int, C.c_int, C.c_longlong, C.c_longlong]
    lib.upto64.restype = C.c_longlong
    return lib


@pytest.mark.parametrize("tau", [1, 2, 4, 16, 256])
@pytest.mark.parametrize("base", [16, 256, 5000])
def test_nominal_lengths_in_32_bits(part, tau, base):
    """Wherever a request's nominal length fits 32 bits, so do its tiles' starts: the largest
    request of each kind, and some below it.  Tiles of one token are the ones whose f (f + 1)
    passes 2^31 while half of it does not."""
    def length(n, k):
        return k * base + tau * (min(k, n // tau) * (min(k, n // tau) + 1) // 2) + max(k - n // tau, 0) * n

    for limit in (2 ** 31 - 1, 2 ** 30, 10 ** 6):
        lo, hi = 1, 1 << 20
        while lo + 1 < hi:  # the largest n whose tiles end below limit
            mid = (lo + hi) // 2
            lo, hi = (mid, hi) if length(mid, -(-mid // tau)) <= limit else (lo, mid)
        n = lo
        tiles = -(-n // tau)
        for k in {0, 1, 2, tiles // 3, tiles // 2, 46340, 46341, tiles - 1, tiles}:
            if 0 <= k <= tiles:
                want = length(n, k)
                assert part.upto32(n, tau, n // tau, base, k) == want, (n, k)
                assert part.upto64(n, tau, n // tau, base, k) == want, (n, k)
