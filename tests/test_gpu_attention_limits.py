"""GPU: attention and norms at the ends of their ranges: lists across the tables
of a tile, values near the type's largest, scores of any size, NaN in one piece."""
import numpy as np
import pytest

import attention_ref as R
import test_gpu_block_attention as B

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Sparse lists that go on behind the first 1,024 blocks
# ---------------------------------------------------------------------------
def alike(rng, n, kv, block, lk, top, other):
    """Lists of neighbouring rows: one of `top` blocks for all, `other` entries of each row's its own."""
    nb = -(-lk // block)
    base = rng.permutation(nb)[:top]
    out = np.tile(base, (n, kv, 1))
    for i in range(n):
        for h in range(kv):
            out[i, h, rng.permutation(top)[:other]] = rng.integers(0, nb, other)
    return np.sort(out, -1).astype(np.int32)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,lk,heads,kv,d,block,chosen", [
    (64, 42000, 1, 1, 128, 32, [900, 1000, 1100, 1200]),
    (64, 42000, 1, 1, 96, 32, [0, 100, 1030]),
    (50, 42000, 2, 2, 128, 32, [0, 1000, 1024, 1025]),
    (64, 42000, 1, 1, 64, 32, [900, 1000, 1100, 1200]),
    (3, 100000, 32, 1, 128, 32, [5, 70, 1023, 1024, 2047, 2048, 2100, 3000]),   # a list across four tables
    (1, 70000, 64, 1, 96, 32, [3, 64, 640, 1500, 1501, 2100]),                  # one new row
    (60, 135000, 1, 1, 128, 128, [0, 63, 64, 1040]),
])
def test_blocks_of_all_rows_across_tables(s3dx, dtype, n, lk, heads, kv, d, block, chosen):
    rng = np.random.default_rng(lk + d)
    q, k, v = B.rows(rng, n, heads, d), B.rows(rng, lk, kv, d), B.rows(rng, lk, kv, d)
    sel = np.tile(np.array(chosen, np.int32), (n, kv, 1))
    got, lse, want = B.run_attend(s3dx, q, k, v, dtype, [n], [lk], block, sel)
    B.check(s3dx, dtype, got, lse, want)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("n,lk,heads,kv,d,block,top,causal", [
    (16, 80000, 8, 2, 128, 64, 32, True),    # in several pieces
    (100, 100000, 1, 1, 128, 64, 32, False),
    (64, 50000, 1, 1, 96, 32, 12, True),
    (64, 50000, 1, 1, 128, 32, 3, False),
    (64, 50000, 1, 1, 32, 32, 12, True),
])
def test_neighbours_lists_across_tables(s3dx, seed, n, lk, heads, kv, d, block, top, causal):
    rng = np.random.default_rng(1000 + seed)
    q, k, v = B.rows(rng, n, heads, d), B.rows(rng, lk, kv, d), B.rows(rng, lk, kv, d)
    sel = alike(rng, n, kv, block, lk, top, seed % 3)
    got, lse, want = B.run_attend(s3dx, q, k, v, s3dx.BF16, [n], [lk], block, sel, causal)
    B.check(s3dx, s3dx.BF16, got, lse, want)
