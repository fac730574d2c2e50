"""Attention over 8-bit caches whose values are large or small (include/hy_int8.h): f32 accuracy whatever
the scales' size.

All value scales times a power of two, and what comes out is to be the same power of two times what it was, bit for
bit: keys whose codes are 0 at the head of every block and negative behind it, under queries that are not negative,
make 0 every row's largest score wherever it begins, so that the running maximum is a whole number, the products'
exponents differ by whole numbers alone, and no rounding falls differently.  A weight's exponent that was rounded
at the size of its value's logarithm (2^-19 where that is 50: 1.3e-6 of the weight) falls differently at once."""
import numpy as np
import pytest

import test_int8_gpu as I8

pytestmark = pytest.mark.gpu


def level_batch(rng, lens, hd, block=8):
    """As I8.make_batch, the first key of each block zeros, the others negative, V's scales across nine powers
    of two; queries of 4 heads that are not negative."""
    p, table, q_start, kv_len = I8.make_batch(rng, lens, 16, 1, hd, block)
    p.k = -np.abs(p.k)
    p.k[:, :, ::block] = 0
    p.vs = np.exp2(rng.uniform(-4.5, 4.5, p.vs.shape)).astype(np.float32)
    p.ks = (0.05 * rng.random(p.ks.shape) / 60).astype(np.float32)  # scores down to -1 or so
    q = np.abs(rng.standard_normal((q_start[-1], 4, hd))).astype(np.float32)
    return p, q, table, q_start, kv_len


def check_powers(gpu, lens, hd, bad_page=False):
    rng = np.random.default_rng(hd + sum(n for _, n in lens))
    p, q, table, q_start, kv_len = level_batch(rng, lens, hd)
    if bad_page:
        table[0, 1] = -1
    run = lambda: I8.attend(gpu, q, p, q_start, kv_len, table, hd ** -0.5)  # noqa: E731
    want = run()
    assert np.isfinite(want).all() and want.any()
    I8.check(want, q, p, q_start, kv_len, table, hd ** -0.5)
    vs = p.vs
    for e in (-54, -37, 13, 29):
        p.vs = np.ldexp(vs, e).astype(np.float32)
        got = np.ldexp(run().astype(np.float64), -e)
        np.testing.assert_array_equal(got, want.astype(np.float64), err_msg=str(e))


# tiles of 256 rows: whole blocks of keys and the last ones of each row, in one piece and in many
@pytest.mark.parametrize("bad_page", [False, True])
@pytest.mark.parametrize("hd,lens", [(128, [(90, 90)]), (128, [(3000, 70)]), (128, [(400, 300), (70, 70)]),
                                     (64, [(200, 200)]), (64, [(2500, 250)])])
def test_powers_of_two_tiles(gpu, hd, lens, bad_page):
    check_powers(gpu, lens, hd, bad_page)


# streams of 16 and of 32 rows: turns that every row sees whole, and the last ones
@pytest.mark.parametrize("bad_page", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[(50, 1)], [(700, 1), (20, 1), (130, 1)], [(300, 3), (17, 2)], [(6000, 4)], [(400, 7), (33, 5)],
                                  [(2000, 8)]])
def test_powers_of_two_streams(gpu, hd, lens, bad_page):
    check_powers(gpu, lens, hd, bad_page)


@pytest.mark.parametrize("hd,lens", [(128, [(90, 90)]), (64, [(200, 200)])])
def test_larger_scales_in_tiles(gpu, hd, lens):
    """Past 2^34 value scales are not defined where small ones stand beside them; tiles take large ones alike, up
    to f32's range for the sums."""
    rng = np.random.default_rng(5)
    p, q, table, q_start, kv_len = level_batch(rng, lens, hd)
    vs = p.vs
    for e in (40, 70, 100):
        p.vs = np.ldexp(vs, e).astype(np.float32)
        args = (q, p, q_start, kv_len, table, hd ** -0.5)
        I8.check(I8.attend(gpu, *args), *args)
