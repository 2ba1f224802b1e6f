"""GPU: attention and norms at the ends of their ranges: lists across the tables
of a tile, values near the type's largest, scores of any size, NaN in one piece,
caches with room behind their keys."""
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


# ---------------------------------------------------------------------------
# What weights are relative to
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d,lk", [(64, 5000), (128, 5000), (32, 5000)])
def test_a_row_keeps_its_weights_while_its_neighbours_maxima_rise(s3dx, dtype, d, lk):
    # Even rows: one score for all keys, hence the mean of the values.  Odd rows: scores that rise by more than 8 binary
    # orders at every step, so that the tile's bases move all the time.  All raw products are exact.  399 sequences
    # without rows keep the tile in one piece.
    n, scale = 32, 0.71
    q, k = np.zeros((n, 1, d), np.float32), np.zeros((lk, 1, d), np.float32)
    q[::2, 0, 0] = 2.0 ** 11 * np.arange(65, 81)
    q[1::2, 0, 1] = 1.0
    k[:, 0, 0], k[:, 0, 1] = 1.0, 16.0 * (np.arange(lk) // 32)
    v = np.where(np.arange(lk) < lk // 2, 1.0, -1.0).astype(np.float32)[:, None, None] * np.ones((1, 1, d), np.float32)
    dq, dk, dv = (R.dev(s3dx, R.stored(s3dx, a, dtype)[0]) for a in (q, k, v))
    o, lse = s3dx.DeviceArray((n, 1, d), R.store_type(s3dx, dtype)), s3dx.DeviceArray((n, 1), np.float32)
    qs, ks = B.starts(s3dx, [n] + [0] * 399), B.starts(s3dx, [lk] + [0] * 399)
    size = s3dx.block_attention_workspace_size(n, 1, 1, d, 400, 64, 0, lk)
    s3dx.block_attention(dq, dk, dv, dtype, n, lk, 1, 1, d, qs, ks, 400, 64, lk, o, lse, scale=scale,
                         workspace=s3dx.DeviceArray(max(1, size), np.uint8))
    got, l = R.values(s3dx, o, dtype)[::2], lse.download()[::2, 0].astype(np.float64)
    print("  off by", np.abs(got).max(), flush=True)
    # equal weights (rounded alike), a sum of lk terms above and below
    assert np.all(np.abs(got) <= 2 * (lk + 8) * R.U32)
    want = q[::2, 0, 0].astype(np.float64) * np.float64(np.float32(scale)) + np.log(lk)
    assert np.all(np.abs(l - want) <= 8 * R.U32 * want)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("lk", [1, 2, 5, 100, 700, 4000])
@pytest.mark.parametrize("n,d,listed", [(40, 64, False), (70, 128, False), (3, 96, False), (40, 64, True), (70, 128, True)])
def test_scores_from_a_million_to_1e30(s3dx, dtype, lk, n, d, listed):
    # equal scores, of either sign: the mean of the values, whatever their size
    rng = np.random.default_rng(lk + n)
    q, k, v = np.zeros((n, 1, d), np.float32), np.zeros((lk, 1, d), np.float32), B.rows(rng, lk, 1, d)
    q[:, 0, 0] = 10.0 ** rng.uniform(6, 12, n) * rng.choice([-1, 1], n)
    q[::7, 0, 0] *= 1e18
    k[:, 0, 0] = 1.0
    sel = np.tile(np.arange(-(-lk // 32), dtype=np.int32), (n, 1, 1)) if listed else None
    got, lse, _ = B.run_attend(s3dx, q, k, v, dtype, [n], [lk], 32, sel, scale=1.0)
    v64, q64 = R.stored(s3dx, v, dtype)[1][:, 0], R.stored(s3dx, q, dtype)[1][:, 0, 0]
    mean, size = v64.mean(0), np.abs(v64).mean(0)
    # weights are equal (bfloat16: rounded alike, their sum is not rounded so: 2^-8), sums of lk terms
    off = np.abs(got[:, 0] - mean) - R.half_step(s3dx, dtype) * np.abs(mean) * 1.01
    assert np.all(off <= (2 * (lk + 8) * R.U32 + (1.01 * R.UBF if dtype else 0)) * size), (np.abs(got[:, 0] - mean).max())
    assert np.all(np.abs(lse[:, 0] - (q64 + np.log(lk))) <= 8 * R.U32 * np.abs(q64) + 1e-6)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,lk,d", [(40, 300, 64), (70, 1300, 128), (3, 4000, 64)])
def test_one_score_far_above_the_others(s3dx, dtype, n, lk, d):
    # the key takes all; below: far scores among ordinary ones count for nothing
    rng = np.random.default_rng(n)
    for far in (1e9, 3e10, 1e12, 1e30):
        q, k, v = np.zeros((n, 1, d), np.float32), 0.1 * B.rows(rng, lk, 1, d), B.rows(rng, lk, 1, d)
        q[:, 0, 0], k[:, 0, 0] = 1.0, 0.0
        k[lk // 3, 0, 0] = far
        got, _, _ = B.run_attend(s3dx, q, k, v, dtype, [n], [lk], 32, scale=1.0)
        assert np.array_equal(got[:, 0], np.tile(R.stored(s3dx, v, dtype)[1][lk // 3, 0], (n, 1)))
        k[:, 0, 0] = np.where(np.arange(lk) % 5 == 0, np.float32(-far), 0.0)
        got, lse, _ = B.run_attend(s3dx, q, k, v, dtype, [n], [lk], 32, scale=1.0)
        v64 = R.stored(s3dx, v, dtype)[1][np.arange(lk) % 5 != 0, 0]
        off = np.abs(got[:, 0] - v64.mean(0)) - R.half_step(s3dx, dtype) * np.abs(v64.mean(0))
        assert np.all(off <= (2 * (lk + 8) * R.U32 + (1.01 * R.UBF if dtype else 0)) * np.abs(v64).mean(0))
        assert np.all(np.abs(lse[:, 0] - np.log(len(v64))) <= (lk + 8) * R.U32)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("power", [115, 121, 127])
@pytest.mark.parametrize("n,lk,d,top,causal", [(40, 100, 64, 0, False), (70, 700, 64, 0, False), (65, 1300, 128, 0, False),
                                               (3, 4000, 64, 0, False), (90, 600, 96, 0, False), (70, 700, 32, 0, True),
                                               (70, 700, 64, 9, False), (65, 1300, 128, 17, True), (3, 4000, 64, 30, False)])
def test_values_near_the_types_largest(s3dx, dtype, power, n, lk, d, top, causal):
    # Scores that rise by 7.9 binary orders from the first key to the last: weights are relative to the first ones' for long.
    rng = np.random.default_rng(n + lk)
    q, k, v = np.zeros((n, 2, d), np.float32), np.zeros((lk, 2, d), np.float32), B.rows(rng, lk, 2, d)
    q[:, :, 0] = 1.0
    k[:, :, 0] = (7.9 * np.log(2) / lk * np.arange(lk))[:, None]
    v = np.clip(np.exp(0.2 * v), 0.5, 1.9).astype(np.float32) * np.float32(2.0 ** power)
    v[:, :, ::2] *= -1
    sel = B.choose(rng, [n], [lk], 2, 32, top) if top else None
    got, lse, want = B.run_attend(s3dx, q, k, v, dtype, [n], [lk], 32, sel, causal, scale=1.0)
    assert np.isfinite(want[0]).all() and np.isfinite(got).all()
    B.check(s3dx, dtype, got, lse, want)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("lk,d,stretch,period", [(2048, 64, 256, 1024), (2048, 64, 128, 512), (2048, 128, 128, 512), (5000, 32, 256, 2048),
                                                 (5000, 64, 256, 2048), (5000, 128, 128, 1024), (300, 64, 32, 128)])
def test_nan_keys_that_are_all_of_a_piece(s3dx, dtype, lk, d, stretch, period):
    rng = np.random.default_rng(lk)
    q, k, v = B.rows(rng, 1, 1, d), B.rows(rng, lk, 1, d), B.rows(rng, lk, 1, d)
    k[np.arange(lk) % period < stretch] = np.nan
    got, lse, _ = B.run_attend(s3dx, q, k, v, dtype, [1], [lk], 64)
    assert np.isnan(got).all() and np.isnan(lse).all()


# ---------------------------------------------------------------------------
# FP32: how close to 64 bits over many elements
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,lk,heads,kv,d,top", [(100, 400, 2, 2, 64, 0), (200, 600, 2, 1, 32, 0), (100, 900, 2, 2, 64, 9), (3, 4000, 16, 4, 64, 30),
                                                 (60, 500, 2, 2, 128, 0), (60, 500, 2, 2, 96, 5)])
def test_float32_keeps_its_bits(s3dx, n, lk, heads, kv, d, top):
    # Three terms a value leave at most 2^-21 of a product, 2^-24.5 in the mean: a score of d products of about
    # 1.5 / sqrt(d) each is short by sqrt(d) 2^-21 at the very most, the values' products by 2^-21: 4e-6 in all, and less than
    # 1e-6 with the mean.  Two terms (2^-14 of a product and more) give 3e-5.
    rng = np.random.default_rng(n + d)
    q, k, v = B.rows(rng, n, heads, d), B.rows(rng, lk, kv, d), B.rows(rng, lk, kv, d)
    sel = B.choose(rng, [n], [lk], kv, 32, top) if top else None
    got, lse, want = B.run_attend(s3dx, q, k, v, s3dx.F32, [n], [lk], 32, sel)
    rel = np.linalg.norm(got - want[0]) / np.linalg.norm(want[0])
    print(f"  rel-L2 {rel:.2e} over {got.size}", flush=True)
    assert got.size > 2000 and rel <= 4e-6


# ---------------------------------------------------------------------------
# Norms of large rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d,pairs,adjacent,pad", [(64, 30, True, 0), (64, 24, False, 0), (64, 30, False, 0), (20, 10, True, 0), (64, 30, True, 1),
                                                  (128, 0, True, 0), (33, 0, True, 0)])
def test_norms_of_rows_of_any_size(s3dx, dtype, d, pairs, adjacent, pad):
    # x / sqrt(mean(x^2) + eps) is of order one however large x is, also where x^2 passes float32's range
    rng = np.random.default_rng(d + pairs)
    n, h = 41, 3
    x = rng.standard_normal((n, h * d + pad)).astype(np.float32) * np.exp2(np.linspace(-40, 125, n)).astype(np.float32)[:, None]
    x = np.clip(x, -3e38, 3e38)
    xs, xv = R.stored(s3dx, x, dtype)
    gain = (1 + 0.2 * rng.standard_normal((h, d))).astype(np.float32)
    pos = rng.integers(0, 64, (n, 1)).astype(np.int32)
    rot = s3dx.Rotary.per_axis(d, [pairs], 1000.0, s3dx.ROTARY_ADJACENT if adjacent else s3dx.ROTARY_HALVES) if pairs else None
    y = s3dx.DeviceArray((n, h, d), np.float32)
    s3dx.qk_norm_rotary(R.dev(s3dx, xs), None, dtype, n, h, 0, d, 1e-6, y, rotary=rot, positions=R.dev(s3dx, pos) if pairs else None,
                        position_stride=1, q_gain=R.dev(s3dx, gain), q_stride=h * d + pad, out_dtype=s3dx.F32)
    want = R.rms(xv[:, : h * d].reshape(n, h, d), gain, 1e-6)
    size = np.abs(want)
    if pairs:
        want, size = R.turn(want, pos, [0] * pairs, [1000.0 ** (-j / pairs) for j in range(pairs)], adjacent)
    off = np.abs(y.download() - want)
    # the sum of squares, its root, gain and scale, the turn (8 u), the output's rounding
    bound = ((d + 2) / 2 + 8 + 8 + 1) * R.U32 * (size + np.abs(want))
    assert np.all(off <= bound + 1e-37), np.argwhere(off > bound + 1e-37)[:4]


# ---------------------------------------------------------------------------
# Caches with room behind their keys
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("lens,room,heads,kv,d,block,top", [([150, 1, 190], 200, 8, 2, 128, 64, 2), ([3000, 2047, 64, 0], 3010, 4, 4, 64, 32, 20)])
def test_single_rows_over_caches_that_grow(s3dx, dtype, lens, room, heads, kv, d, block, top):
    # The room of a cache is a sequence without queries.  What it holds (NaN here) reaches nothing.
    rng = np.random.default_rng(room)
    b, lens = len(lens), list(lens)
    k, v = np.full((b * room, kv, d), np.nan, np.float32), np.full((b * room, kv, d), np.nan, np.float32)
    for s, n in enumerate(lens):
        k[s * room: s * room + n], v[s * room: s * room + n] = B.rows(rng, n, kv, d), B.rows(rng, n, kv, d)
    rows = s3dx.block_index_rows(b * room, 2 * b, block)
    codes, scale = s3dx.DeviceArray((kv, rows, d), np.int8), s3dx.DeviceArray((kv, rows), np.float32)
    qs = B.starts(s3dx, [1, 0] * b)
    for step in range(3):
        for s in range(b):   # a new key each
            k[s * room + lens[s]], v[s * room + lens[s]] = B.rows(rng, 1, kv, d)[0], B.rows(rng, 1, kv, d)[0]
            lens[s] += 1
        q = B.rows(rng, b, heads, d)
        (dq, q64), (dk, k64), (dv, v64) = ((R.dev(s3dx, st), val) for st, val in (R.stored(s3dx, a, dtype) for a in (q, k, v)))
        ks = B.starts(s3dx, [n for s in range(b) for n in (lens[s], room - lens[s])])
        s3dx.block_index(dk, dtype, b * room, kv, d, ks, 2 * b, block, codes, scale)
        sel = R.filled(s3dx, (b, kv, top), np.int32, 0x5A)
        s3dx.block_select(dq, dtype, b, b * room, heads, kv, d, qs, ks, 2 * b, block, top, max(lens), codes, scale, sel, causal=True, near=True)
        real = np.concatenate([np.arange(s * room, s * room + n) for s, n in enumerate(lens)])
        packed_k, packed_v = k64[real], v64[real]
        c, power, _ = R.index_of(packed_k, lens, block)
        want = R.select(q64, c, power, [1] * b, lens, block, top, True, True)
        assert np.array_equal(sel.download(), want)
        for chosen in (want, None):
            n = 0 if chosen is None else top
            o, lse = s3dx.DeviceArray((b, heads, d), R.store_type(s3dx, dtype)), s3dx.DeviceArray((b, heads), np.float32)
            ws = s3dx.DeviceArray(max(1, s3dx.block_attention_workspace_size(b, heads, kv, d, 2 * b, block, n, max(lens))), np.uint8)
            s3dx.block_attention(dq, dk, dv, dtype, b, b * room, heads, kv, d, qs, ks, 2 * b, block, max(lens), o, lse,
                                 None if chosen is None else sel, n, causal=True, workspace=ws)
            B.check(s3dx, dtype, R.values(s3dx, o, dtype), lse.download().astype(np.float64),
                    R.attend(q64, packed_k, packed_v, [1] * b, lens, block, chosen, d ** -0.5, True, dtype == s3dx.BF16))
