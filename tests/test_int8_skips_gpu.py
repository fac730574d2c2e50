"""The quantizing write of an 8-bit cache, rows whose position lies outside the rotary tables: they have a slot,
behind or before those of live rows, and are skipped all the same (include/hy_int8.h)."""
import numpy as np
import pytest

from test_int8_gpu import append, download, random_pool, same_pool, upload
from test_paged_gpu import APPEND_TOL, append_ref

pytestmark = pytest.mark.gpu

N_POS = 40  # of the tables


def outside(i):
    """A position that the tables do not have."""
    return (N_POS, -1, 2 ** 31 - 1, -2 ** 31, N_POS + 1)[i % 5]


def check(gpu, nh, nkv, hd, page, block, slots, bad):
    """Rows at consecutive or other slots, those in bad outside the tables: queries, codes and scales as if they
    were not there."""
    rng = np.random.default_rng(len(slots) + block)
    slots = np.asarray(slots, np.int32)
    T = len(slots)
    p = random_pool(rng, int(slots.max()) // page + 2, page, nkv, hd, block)
    pos = rng.integers(0, N_POS, T).astype(np.int32)
    for i, t in enumerate(bad):
        pos[t] = outside(i)
    live = np.setdiff1d(np.arange(T), bad)
    ang = rng.random((N_POS, hd // 2)) * 6
    cos, sin = (np.repeat(f(ang), 2, axis=1).astype(np.float32) for f in (np.cos, np.sin))
    # live rows' values small beside the held ones in every third block, so that a scale is kept there
    qkv = rng.standard_normal((T, (nh + 2 * nkv) * hd)).astype(np.float32)
    qkv[slots // block % 3 == 0] *= np.float32(1e-3)
    qkv[bad] *= np.float32(100)  # shows in a scale that it got into
    bufs = upload(gpu, p)
    got = append(gpu, p, bufs, qkv, pos, slots, nh, 0.0, cos, sin)
    eps = float(np.float32(1e-5))  # as the call gets it: beside values of 1e-3 its last bits show in a code
    q, k, v, qm, _ = append_ref(qkv[live], nh, nkv, hd, pos[live], 0, cos, sin, None, None, eps)
    assert (np.abs(got[live] - q) <= APPEND_TOL * qm).all()
    assert (got[bad] == 5.0).all()
    p.write(k.astype(np.float32), slots[live], "k")
    p.write(v.astype(np.float32), slots[live], "v")
    same_pool(download(p, bufs), p)


@pytest.mark.parametrize("hd", [64, 128])
def test_first_and_last_rows_of_blocks(gpu, hd):
    """A block without its first row goes on at the scale it has; a run ends before a row that is skipped."""
    slots = np.r_[32:48, 64:80, 96:105, 7:16, 48:64]
    at = {int(s): i for i, s in enumerate(slots)}
    bad = [at[s] for s in (32, 64, 65, 66, 104, 15, 63, 62)]
    check(gpu, 4, 2, hd, 32, 16, slots, bad)
    check(gpu, 4, 2, hd, 32, 8, slots, [at[s] for s in (32, 40, 41, 71, 70, 96, 104, 15, 56, 57, 58)])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [300, 512, 513, 700])
def test_first_rows_at_groups_ends(gpu, hd, T):
    """Rows 15, 31, .. begin their blocks: past 512 rows a work group goes through 16, and what stands before its
    first one decides whether that goes on."""
    bad = [t for t in range(15, T, 16) if t // 16 % 2 == 0 or t // 16 % 5 == 1]
    check(gpu, 2, 1, hd, 64, 16, np.arange(1, T + 1), bad)
    check(gpu, 2, 1, hd, 64, 16, np.arange(1, T + 1), [t - 1 for t in bad])  # the last rows of the blocks before


@pytest.mark.parametrize("live", [63, 64, 65, 127, 128, 150, 200])
def test_ends_of_long_runs(gpu, live):
    """Runs of more rows than a wave looks at end where a position is outside, too."""
    check(gpu, 3, 1, 64, 256, 256, np.arange(256 + 20, 512 + 70), np.r_[live:236, 236:236 + live % 7])
