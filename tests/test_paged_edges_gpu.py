"""Paged serving on the GPU at the ends of its ranges, against plain numpy in 64 bits."""
import numpy as np
import pytest

import paged_ref as R
from paged_ref import F16
from test_paged_gpu import attend, make_batch

pytestmark = pytest.mark.gpu


def test_attention_long_request_in_tiles_of_one_token(gpu):
    """50000 rows of one request, 16 query heads per kv head, in the streams' tiles of 16 rows
    (max_new only chooses the kernel): a tile is one token, and the tiles' nominal lengths add up
    to 1.25e9.  Every row sees at most 40 keys, so that plain products can follow."""
    rng = np.random.default_rng(70)
    n, nh, hd, page = 50000, 16, 64, 64
    pool, table, q_start, kv_len = make_batch(rng, [(n, n)], page, 1, hd, F16)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    seen = rng.integers(0, 41, n).astype(np.int32)
    got = attend(gpu, q, pool, q_start, kv_len, table, hd ** -0.5, seen=seen, max_new=1)
    k, v = (np.stack([R.decode(pool.at(a, table[0, 0], i), F16)[0] for i in range(40)]) for a in (pool.k, pool.v))
    for t0 in range(0, n, 5000):
        x = q[t0:t0 + 5000].astype(np.float64)
        s = x @ k.T * hd ** -0.5
        gone = np.arange(40) >= seen[t0:t0 + 5000, None, None]
        w = np.exp(np.where(gone, -np.inf, s))
        w /= np.maximum(w.sum(-1, keepdims=True), 1e-300)
        bound = R.attention_bound((np.abs(x) @ np.abs(k).T).max(-1) * hd ** -0.5, w @ np.abs(v), hd, 40)
        assert (np.abs(got[t0:t0 + 5000] - w @ v) <= bound).all()
