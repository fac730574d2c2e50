"""Every piece of a weight reaches the matrix cores: near-equal weights that f16 does not hold, over values
of one size, where a lost remainder (2^-12 of its weight) shows in the norm.

Scores up to 1/2 in size: check_attention's normwise bound is then 2^-23 (2 (sqrt(hd) + 4) + 8), 4.6e-6 for
head_dim 128; remainders lost for one key in 16 and one dim in 8 leave 1.3e-5."""
import numpy as np
import pytest

import int8_ref as Q
import test_int8_gpu as I8
import test_paged_gpu as P
from paged_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu



@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 6, 90, 700])
@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_near_equal_weights(gpu, wtype, new, hd):
    rng = np.random.default_rng(70 + new)
    pool, table, q_start, kv_len = P.make_batch(rng, [(800, new)] * (3 if new > 1 else 1), 16, 1, hd, wtype)
    q = (rng.standard_normal((q_start[-1], 4, hd)) * 0.03).astype(np.float32)
    args = (q, pool, q_start, kv_len, table, hd ** -0.5)
    P.check_attention(P.attend(gpu, *args), *args)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 6, 90, 700])
def test_near_equal_weights_i8(gpu, new, hd):
    rng = np.random.default_rng(80 + new)
    p, table, q_start, kv_len = I8.make_batch(rng, [(800, new)] * (3 if new > 1 else 1), 16, 1, hd, 16, v_spread=0.2)
    q = (rng.standard_normal((q_start[-1], 4, hd)) * 0.03).astype(np.float32)
    args = (q, p, q_start, kv_len, table, hd ** -0.5)
    Q.check_attention(I8.attend(gpu, *args), *args)
