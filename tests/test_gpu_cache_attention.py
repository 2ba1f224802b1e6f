"""GPU: attention over the cache in 8 bits against a plain 64-bit implementation:
lengths from none to long, tiles of all heights, windows and first keys, steps and
scores of any size, queries that are not finite."""
import numpy as np
import pytest

import attention_ref as R
import cache_ref as K

pytestmark = pytest.mark.gpu


def run(s3dx, q, held, table, dtype, new, lens, causal=True, window=0, sinks=0, scale=None, pad=0, behind=0, max_k=None, stream=None,
        buffer=None):
    """The call's o and lse with the reference and its bounds; `behind`: rows behind the last sequence."""
    n, heads, d = q.shape
    bits, q64 = R.stored(s3dx, q, dtype)
    wide = np.full((n + behind, heads * d + pad), 0x7FC0 if dtype == s3dx.BF16 else np.nan, bits.dtype)
    wide[:n, : heads * d] = bits.reshape(n, -1)
    db = R.dev(s3dx, held.buffer()) if buffer is None else buffer
    cache = s3dx.KvCache(db, held.pages, held.kv, d, held.block)
    o = R.filled(s3dx, (n + behind, heads * d + pad), R.store_type(s3dx, dtype), 0x5A)
    lse = R.filled(s3dx, (n + behind, heads), np.float32, 0x5A)
    longest = max(lens) if max_k is None else max_k
    ws = R.filled(s3dx, max(1, cache.attention_workspace_size(n + behind, heads, len(new), max(0, longest), window, sinks)), np.uint8, 0xFF)
    dq, ds, dt, dl = R.dev(s3dx, wide), R.dev(s3dx, K.starts(new)), R.dev(s3dx, table), R.dev(s3dx, np.asarray(lens, np.int32))
    cache.attention(dq, dtype, n + behind, heads, ds, dt, table.shape[1], dl, len(new), max(0, longest), o, lse, heads * d + pad, heads * d + pad,
                    scale, causal, window, sinks, ws, stream=stream)
    s3dx.synchronize(stream)
    got, l, raw = R.values(s3dx, o, dtype), lse.download(), o.download()
    assert np.all(raw[n:].view(np.uint8) == 0x5A) and np.all(l[n:].view(np.uint8) == 0x5A)
    assert np.all(np.ascontiguousarray(raw[:, heads * d:]).view(np.uint8) == 0x5A)
    want = K.attend(q64, held, table, new, lens, float(np.float32(d ** -0.5 if scale is None else scale)), causal, window, sinks,
                    dtype == s3dx.BF16)
    return got[:n, : heads * d].reshape(n, heads, d), l[:n].astype(np.float64), want


CASES = [
    # new, lens, heads, kv, d, block, causal, window, sinks
    ([1], [1], 1, 1, 64, 64, True, 0, 0),
    ([1], [300], 12, 12, 64, 64, True, 0, 0),
    ([1], [63], 8, 2, 128, 64, False, 0, 0),
    ([1, 1, 1], [1, 64, 65], 4, 1, 32, 128, True, 0, 0),
    ([1] * 5, [1000, 3, 128, 4097, 64], 32, 8, 128, 64, True, 0, 0),
    ([1], [9000], 5, 1, 96, 128, True, 0, 0),
    ([1, 1], [5000, 4999], 2, 2, 64, 64, True, 700, 4),
    ([1], [5000], 8, 1, 128, 64, True, 64, 0),
    ([1], [5000], 8, 1, 128, 64, True, 1, 1),
    ([1], [900], 8, 2, 64, 64, True, 5000, 4),              # a window longer than the sequence
    ([1], [700], 4, 4, 64, 128, True, 100, 5000),           # first keys beyond the sequence
    ([100], [100], 3, 3, 64, 64, True, 0, 0),
    ([257], [257], 2, 2, 64, 64, True, 0, 0),
    ([90], [130], 2, 2, 32, 64, False, 0, 0),
    ([65], [200], 4, 4, 96, 128, True, 0, 0),
    ([200], [330], 4, 2, 128, 64, True, 0, 0),
    ([40], [256], 40, 1, 64, 64, True, 0, 0),               # a group wider than a tile
    ([129], [500], 5, 1, 64, 64, False, 0, 0),              # rows of a tile are not whole groups
    ([300], [600], 4, 2, 128, 64, True, 100, 7),            # a window that moves through tiles and blocks
    ([300], [300], 2, 1, 64, 128, True, 65, 70),            # first keys over more than one step
    ([150], [700], 6, 2, 96, 64, True, 200, 64),
    ([500], [500], 2, 2, 32, 64, True, 1, 0),               # each row sees itself alone
    ([33, 0, 1, 64, 7], [40, 20, 1, 64, 300], 8, 2, 64, 64, True, 0, 0),
    ([17, 3, 0, 40], [5, 0, 50, 90], 3, 1, 64, 64, True, 0, 0),      # more queries than keys, none of either
    ([17, 3, 0, 40], [5, 0, 50, 90], 3, 1, 128, 64, False, 0, 0),
    ([17, 3, 0, 40], [5, 0, 50, 90], 3, 1, 96, 128, True, 10, 2),
    ([2], [4000], 4, 4, 64, 128, False, 0, 0),
    ([20], [3000], 8, 2, 128, 64, True, 0, 0),              # several waves and workgroups a tile
    ([16], [3000], 2, 1, 64, 64, True, 0, 0),
    ([700], [900], 16, 4, 64, 64, True, 0, 0),              # more tiles than waves a tile
    ([400], [500], 32, 8, 128, 128, True, 0, 0),
    ([1] * 300, [70 + 3 * s for s in range(300)], 4, 1, 32, 64, True, 0, 0),
]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%s of %s %s" % (str(c[0])[:12], str(c[1])[:14], c[2:]))
def test_attention(s3dx, dtype, case):
    new, lens, heads, kv, d, block, causal, window, sinks = case
    rng = np.random.default_rng(sum(lens) + heads)
    held, table = K.filled(rng, kv, d, block, lens)
    q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
    got, lse, want = run(s3dx, q, held, table, dtype, new, lens, causal, window, sinks, pad=8, behind=3)
    K.check(s3dx, dtype, got, lse, want)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,lens,heads,kv,d", [
    ([300, 0, 700, 129], [300, 5, 900, 4000], 10, 10, 32),           # two heads beyond eight
    ([300, 0, 700, 129], [300, 5, 900, 4000], 3, 1, 128),
    ([0, 500, 1, 0, 260], [9, 700, 2, 0, 300], 12, 6, 64),
    ([200, 390], [1000, 390], 38, 19, 32),
    ([100] * 70, [100 + 2 * s for s in range(70)], 3, 3, 32),        # tiles by a bound
    ([100] * 70, [100 + 2 * s for s in range(70)], 12, 12, 32),      # ... more than run at once
    ([130] * 33, [150 + s for s in range(33)], 13, 13, 64),
    ([0] * 20 + [90] * 44, [64] * 64, 9, 9, 96),                     # 64 sequences, more queries than keys
])
def test_every_tile_is_computed(s3dx, new, lens, heads, kv, d, causal):
    rng = np.random.default_rng(sum(lens))
    held, table = K.filled(rng, kv, d, 64, lens)
    q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
    got, lse, want = run(s3dx, q, held, table, s3dx.BF16, new, lens, causal, behind=2)
    K.check(s3dx, s3dx.BF16, got, lse, want)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,heads,kv,d", [([1, 1], [2000, 300], 8, 2, 64), ([90], [260], 4, 2, 128), ([200], [200], 4, 4, 32)])
def test_work_is_cut_by_max_k_and_results_are_not(s3dx, dtype, new, lens, heads, kv, d):
    rng = np.random.default_rng(7)
    held, table = K.filled(rng, kv, d, 64, lens)
    q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
    for max_k in (0, 1, 64, 5000, 2 ** 20):
        got, lse, want = run(s3dx, q, held, table, dtype, new, lens, max_k=max_k)
        K.check(s3dx, dtype, got, lse, want, str(max_k))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,heads,kv,d,window,sinks", [
    ([1] * 8, [5, 0, 3000, 64, 700, 129, 1, 2000], 16, 8, 64, 0, 0),
    ([1] * 8, [9000] + [100] * 7, 32, 8, 128, 0, 0),                          # one that would take all
    ([2, 0, 3, 1, 0, 4, 1, 1], [700, 50, 2, 1500, 0, 900, 64, 333], 16, 8, 96, 0, 0),
    ([40] + [1] * 20, [2000] + [90 * s for s in range(20)], 12, 3, 32, 0, 0),   # several tiles of one
    ([1] * 64, [1 + 37 * (s * s % 61) for s in range(64)], 4, 1, 64, 0, 0),
    ([1] * 8, [5000, 40, 3000, 700, 64, 129, 1, 2000], 16, 8, 64, 600, 70),     # (a short window: pieces of one size)
    ([1] * 8, [14000, 12500, 300, 40, 700, 64, 129, 2000], 8, 8, 128, 11000, 70),
])
def test_workgroups_are_shared_out_by_lengths(s3dx, dtype, new, lens, heads, kv, d, window, sinks):
    # a max_k that speaks of long sequences; then with values' steps that make one sequence's rows go key by key
    rng = np.random.default_rng(sum(lens))
    held, table = K.filled(rng, kv, d, 64, lens)
    q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
    got, lse, want = run(s3dx, q, held, table, dtype, new, lens, True, window, sinks, max_k=2 ** 20, behind=2)
    K.check(s3dx, dtype, got, lse, want)
    longest = int(np.argmax(lens))
    blocks = -(-lens[longest] // 64)
    held.steps[table[longest, :blocks], :, 1] = np.ldexp(1.0, rng.choice([-60, -30, 0], (blocks, 1)))
    got, lse, want = run(s3dx, q, held, table, dtype, new, lens, True, window, sinks, max_k=2 ** 20, behind=2)
    K.check(s3dx, dtype, got, lse, want, "far")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,d", [([1], [1500], 64), ([40], [700], 128), ([100], [300], 96)])
def test_pages_that_are_none_count_for_nothing(s3dx, dtype, new, lens, d):
    rng = np.random.default_rng(9)
    held, table = K.filled(rng, 2, d, 64, lens)
    table[0, 1], table[0, 2], table[0, 4] = -1, held.pages, 2 ** 31 - 1
    # what no row sees holds anything: pages of nobody, places behind the last row
    buffer = held.buffer()
    raw = buffer[: -8 * held.pages * held.kv].reshape(held.pages, -1)
    steps = buffer[-8 * held.pages * held.kv:].view(np.float32).reshape(held.pages, -1)
    nobody = np.setdiff1d(np.arange(held.pages), table)
    raw[nobody], steps[nobody] = 255, np.nan
    q = rng.standard_normal((sum(new), 4, d)).astype(np.float32)
    got, lse, want = run(s3dx, q, held, table, dtype, new, lens, buffer=R.dev(s3dx, buffer))
    K.check(s3dx, dtype, got, lse, want)
    # ... all of them: nothing is seen
    got, lse, _ = run(s3dx, q, held, np.full_like(table, -1), dtype, new, lens)
    assert not got.any() and np.all(lse == -np.inf)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,heads,d", [([1], [3000], 4, 64), ([1], [200], 4, 128), ([70], [400], 2, 64)])
def test_steps_of_any_size(s3dx, dtype, new, lens, heads, d):
    # blocks' values (and keys) apart by up to 2^200, and blocks of zeros; large values where weights are small and elsewhere
    rng = np.random.default_rng(d)
    held, table = K.filled(rng, 1, d, 64, lens, spread=0.0)
    blocks = -(-lens[0] // 64)
    for name, powers in (("values", rng.integers(-8, 9, blocks)), ("far", rng.choice([-60, -30, 0], blocks)),
                         ("ends", rng.choice([-100, 119], blocks)), ("falling", -3 * np.arange(blocks)), ("rising", 2 * np.arange(blocks))):
        held.steps[table[0, :blocks], 0, 1] = np.ldexp(1.0, np.clip(powers, -106, 119))
        held.steps[table[0, 0], 0, 1] = 0.0 if name == "values" else held.steps[table[0, 0], 0, 1]
        held.codes[1, table[0, 0]] = 0 if name == "values" else held.codes[1, table[0, 0]]
        q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
        got, lse, want = run(s3dx, q, held, table, dtype, new, lens)
        K.check(s3dx, dtype, got, lse, want, name)
    held.steps[table[0, :blocks], 0, 1] = 0.01
    held.steps[table[0, :blocks], 0, 0] = np.ldexp(1.0, rng.choice([-106, -20, -7, -6], blocks))
    held.steps[table[0, blocks // 2], 0, 0] = 0.0
    held.codes[0, table[0, blocks // 2]] = 0
    held.steps[table[0, :blocks], 0, 1] = 2.0 ** -6
    got, lse, want = run(s3dx, q, held, table, dtype, new, lens)
    K.check(s3dx, dtype, got, lse, want, "keys")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("lk", [1, 5, 64, 700, 4000])
@pytest.mark.parametrize("n,d", [(1, 64), (40, 64), (70, 128)])
def test_equal_scores_of_any_size(s3dx, dtype, lk, n, d):
    # equal scores, of either sign, from a million to 1e30: the mean of the values
    rng = np.random.default_rng(lk + n)
    held, table = K.filled(rng, 1, d, 64, [lk])
    held.codes[0] = 0
    held.codes[0, :, :, :, 0] = 64
    held.steps[:, :, 0] = 2.0 ** -6
    q = np.zeros((n, 1, d), np.float32)
    q[:, 0, 0] = 10.0 ** rng.uniform(6, 12, n) * rng.choice([-1, 1], n)
    q[::7, 0, 0] *= 1e18
    got, lse, _ = run(s3dx, q, held, table, dtype, [n], [lk], False, scale=1.0)
    v, q64 = held.values(0, lk, table)[1][:, 0], R.stored(s3dx, q, dtype)[1][:, 0, 0]
    mean, size = v.mean(0), np.abs(v).mean(0)
    # weights are equal and a power of two but for the base's rounding (2^-0.5 .. 2^0.5 where it is in one part): rounded alike,
    # and their sum is not (2^-11); sums of lk terms
    off = np.abs(got[:, 0] - mean) - R.half_step(s3dx, dtype) * np.abs(mean) * 1.01
    assert np.all(off <= (2 * (lk + 10) * R.U32 + (1.01 * 2.0 ** -11 if dtype else 2.0 ** -21)) * size)
    assert np.all(np.abs(lse[:, 0] - (q64 + np.log(lk))) <= 8 * R.U32 * np.abs(q64) + 1e-6)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,lk,d", [(1, 4000, 64), (40, 300, 64), (70, 1300, 128)])
def test_one_score_far_from_the_others(s3dx, dtype, n, lk, d):
    rng = np.random.default_rng(n)
    for far in (1e3, 1e6, 1e9, 1e12, 1e30, -1e6, -1e30):
        held, table = K.filled(rng, 1, d, 64, [lk])
        held.codes[0] = 0
        at = lk // 3
        page, slot = table[0, at // 64], at % 64
        held.codes[0, page, 0, slot, 0] = 64 if far > 0 else -64
        held.steps[page, 0, 0] = 2.0 ** np.floor(np.log2(abs(far) / 64))
        q = np.zeros((n, 1, d), np.float32)
        q[:, 0, 0] = 1.0
        got, lse, want = run(s3dx, q, held, table, dtype, [n], [lk], False, scale=1.0)
        K.check(s3dx, dtype, got, lse, want, str(far))


@pytest.mark.parametrize("dtype", [0, 1])
def test_maxima_that_rise(s3dx, dtype):
    # one row's scores rise by 2^4 at every key, its neighbours' fall or stay: bases move all the time, each by its own
    rng = np.random.default_rng(2)
    for lk, d, n in ((300, 64, 40), (2000, 128, 3), (1000, 32, 20)):
        held, table = K.filled(rng, 1, d, 64, [lk])
        held.codes[0] = 0
        for j in range(lk):
            held.codes[0, table[0, j // 64], 0, j % 64, 0] = (j % 64) + 1
        for b in range(-(-lk // 64)):
            held.steps[table[0, b], 0, 0] = 2.0 ** (b % 7)
        q = np.zeros((n, 1, d), np.float32)
        q[:, 0, 0] = rng.choice([0.0, 0.01, 1.0, -1.0, 16.0], n)
        q[:, 0, 1] = 1.0
        got, lse, want = run(s3dx, q, held, table, dtype, [n], [lk], False, scale=0.71)
        K.check(s3dx, dtype, got, lse, want, str(lk))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,d", [([40], [200], 64), ([1, 1, 1], [3000, 50, 700], 128), ([50], [20], 32)])
def test_queries_that_are_not_finite(s3dx, dtype, new, lens, d):
    # their rows are NaN (or see nothing and are zeros), and no other
    rng = np.random.default_rng(5)
    held, table = K.filled(rng, 2, d, 64, lens)
    q = rng.standard_normal((sum(new), 4, d)).astype(np.float32)
    clean = run(s3dx, q, held, table, dtype, new, lens)
    K.check(s3dx, dtype, *clean)
    bad = np.zeros((sum(new), 4), bool)
    for i, (r, h, x) in enumerate([(0, 1, np.nan), (sum(new) - 1, 0, np.inf), (sum(new) // 2, 3, -np.inf)]):
        q[r, h, i * 7] = x
        bad[r, h] = True
    with np.errstate(invalid="ignore"):
        got, lse, _ = run(s3dx, q, held, table, dtype, new, lens)
    assert np.array_equal(got[~bad], clean[0][~bad]) and np.array_equal(lse[~bad], clean[1][~bad])
    sees = clean[1][bad] != -np.inf
    assert np.all(np.isnan(got[bad][sees])) and np.all(np.isnan(lse[bad][sees]))
    assert np.all(got[bad][~sees] == 0) and np.all(lse[bad][~sees] == -np.inf)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("power", [-120, -60, 60, 100])
def test_queries_of_any_size(s3dx, dtype, power):
    # scores stay ordinary: softmax_scale makes up for them as far as it may, the keys' steps for the rest
    rng = np.random.default_rng(power + 200)
    held, table = K.filled(rng, 2, 64, 64, [500, 90], spread=0.0)
    held.steps[:, :, 0] = np.ldexp(held.steps[:, :, 0], -power if power > 0 else min(-power, 110))
    q = (np.ldexp(rng.standard_normal((30, 4, 64)), power)).astype(np.float32)
    got, lse, want = run(s3dx, q, held, table, dtype, [10, 20], [500, 90])
    K.check(s3dx, dtype, got, lse, want)


def test_other_streams_graphs_and_shared_pages(s3dx):
    # single rows over sequences that share their first pages, captured once and replayed as they grow; each replay against the
    # eager call and the definition
    rng = np.random.default_rng(21)
    kv, d, heads, width, seqs = 2, 128, 8, 20, 4
    lens = np.array([700, 520, 641, 1000])
    held = K.Held(seqs * width, kv, d, 64)
    table = rng.permutation(seqs * width).reshape(seqs, width).astype(np.int32)
    held.write(*(K.rows(rng, int(lens.sum()), kv, d).astype(np.float64) for _ in range(2)), lens, lens, table)
    table[1:, :5] = table[0, :5]
    buffer = R.dev(s3dx, held.buffer())
    cache = s3dx.KvCache(buffer, held.pages, kv, d, 64)
    stream, other = s3dx.Stream(), s3dx.Stream()
    dk, dv = (s3dx.DeviceArray((seqs, kv, d), np.uint16) for _ in range(2))
    dq, o, o2 = (s3dx.DeviceArray((seqs, heads, d), np.uint16) for _ in range(3))
    lse, lse2 = (s3dx.DeviceArray((seqs, heads), np.float32) for _ in range(2))
    size = cache.attention_workspace_size(seqs, heads, seqs, 1280)
    assert size > 0
    ws, ws2 = (R.filled(s3dx, size, np.uint8, 0xFF) for _ in range(2))
    ds, dt, dl = R.dev(s3dx, K.starts([1] * seqs)), R.dev(s3dx, table), R.dev(s3dx, lens.astype(np.int32))

    def body():
        cache.write(dk, dv, s3dx.BF16, seqs, ds, dt, width, dl, seqs, stream=stream)
        cache.attention(dq, s3dx.BF16, seqs, heads, ds, dt, width, dl, seqs, 1280, o, lse, causal=True, window=900, sinks=3,
                        workspace=ws, stream=stream)

    # sizes for a window differ: the larger workspace serves both
    graph = R.Graph(s3dx, stream, body)
    for step in range(12):
        lens = lens + 1
        (kb, k64), (vb, v64) = (R.stored(s3dx, K.rows(rng, seqs, kv, d), s3dx.BF16) for _ in range(2))
        qb, q64 = R.stored(s3dx, rng.standard_normal((seqs, heads, d)).astype(np.float32), s3dx.BF16)
        for dev, host in ((dk, kb), (dv, vb), (dq, qb), (dl, lens.astype(np.int32))):
            dev.upload(host, stream)
        graph.launch()
        stream.synchronize()
        cache.attention(dq, s3dx.BF16, seqs, heads, ds, dt, width, dl, seqs, 1280, o2, lse2, causal=True, window=900, sinks=3,
                        workspace=ws2, stream=other)
        other.synchronize()
        held.write(k64, v64, [1] * seqs, lens, table)
        want = K.attend(q64, held, table, [1] * seqs, lens, float(np.float32(d ** -0.5)), True, 900, 3, True)
        K.check(s3dx, s3dx.BF16, R.values(s3dx, o, s3dx.BF16), lse.download().astype(np.float64), want, "step %d" % step)
        assert np.array_equal(o.download(), o2.download()) and np.array_equal(lse.download(), lse2.download())
    graph.close()


@pytest.mark.parametrize("new,lens,d", [([1, 1], [3000, 70], 64), ([20], [500], 96), ([150, 3], [200, 900], 128), ([2] * 66, [90] * 66, 32)])
def test_sequences_that_begin_behind_the_first_row(s3dx, new, lens, d):
    # rows before the first sequence, as those behind the last, stay as they were
    rng = np.random.default_rng(d)
    held, table = K.filled(rng, 2, d, 64, lens)
    n, before, behind, heads = sum(new), 5, 4, 4
    q = rng.standard_normal((n, heads, d)).astype(np.float32)
    bits, q64 = R.stored(s3dx, q, s3dx.BF16)
    wide = np.full((before + n + behind, heads * d), 0x7FC0, bits.dtype)
    wide[before:before + n] = bits.reshape(n, -1)
    cache = s3dx.KvCache(R.dev(s3dx, held.buffer()), held.pages, 2, d, 64)
    o, lse = R.filled(s3dx, wide.shape, np.uint16, 0x5A), R.filled(s3dx, (len(wide), heads), np.float32, 0x5A)
    ws = R.filled(s3dx, max(1, cache.attention_workspace_size(len(wide), heads, len(new), max(lens))), np.uint8, 0xFF)
    cache.attention(R.dev(s3dx, wide), s3dx.BF16, len(wide), heads, R.dev(s3dx, K.starts(new) + before), R.dev(s3dx, table), table.shape[1],
                    R.dev(s3dx, np.asarray(lens, np.int32)), len(new), max(lens), o, lse, causal=True, workspace=ws)
    s3dx.synchronize()
    got, l, raw = R.values(s3dx, o, s3dx.BF16), lse.download(), o.download()
    for rest in (slice(0, before), slice(before + n, None)):
        assert np.all(raw[rest] == 0x5A5A) and np.all(l[rest].view(np.uint32) == 0x5A5A5A5A)
    want = K.attend(q64, held, table, new, lens, float(np.float32(d ** -0.5)), True, 0, 0, True)
    K.check(s3dx, s3dx.BF16, got[before:before + n].reshape(n, heads, d), l[before:before + n].astype(np.float64), want)


def test_the_same_call_gives_the_same_bits(s3dx):
    rng = np.random.default_rng(4)
    for new, lens, heads, kv, d in (([1, 1], [3000, 777], 8, 2, 128), ([60], [900], 4, 2, 64)):
        held, table = K.filled(rng, kv, d, 64, lens)
        q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
        a, b = (run(s3dx, q, held, table, s3dx.BF16, new, lens) for _ in range(2))
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("new,lens,d", [([1], [300], 64), ([1, 1], [3000, 64], 128), ([40], [200], 96), ([200], [500], 64)])
def test_infinite_queries_whose_products_are_all_negative(s3dx, dtype, far, new, lens, d):
    # their scores are all -inf, and the rows NaN all the same; far: rows that go key by key
    rng = np.random.default_rng(11)
    held, table = K.filled(rng, 2, d, 64, lens)
    held.codes[0, ..., 3] = -1 - np.abs(held.codes[0, ..., 3]) % 127
    if far:
        held.steps[..., 1] = np.ldexp(1.0, rng.choice([-60, 0], held.steps[..., 1].shape))
        held.steps[table[0, 0], :, 1], held.steps[table[0, 1], :, 1] = 2.0 ** -60, 1.0
    q = rng.standard_normal((sum(new), 4, d)).astype(np.float32)
    clean = run(s3dx, q, held, table, dtype, new, lens)
    K.check(s3dx, dtype, *clean)
    bad = np.zeros((sum(new), 4), bool)
    for r, h, x in ((0, 1, 1.0), (sum(new) - 1, 2, 1.0), (sum(new) // 2, 3, 1.0)):
        q[r, h, 3] = x * np.inf
        bad[r, h] = True
    with np.errstate(invalid="ignore"):
        got, lse, _ = run(s3dx, q, held, table, dtype, new, lens)
    assert np.array_equal(got[~bad], clean[0][~bad]) and np.array_equal(lse[~bad], clean[1][~bad])
    assert np.all(np.isnan(got[bad])) and np.all(np.isnan(lse[bad]))
    # pages that are none: nothing is seen, and the rows are zeros
    with np.errstate(invalid="ignore"):
        got, lse, _ = run(s3dx, q, held, np.full_like(table, -1), dtype, new, lens)
    assert not got.any() and np.all(lse == -np.inf)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("new,lens,d", [([1], [300], 64), ([1, 1], [3000, 64], 128), ([40], [200], 96), ([200], [500], 64)])
def test_scores_beyond_float32(s3dx, dtype, far, new, lens, d):
    # products of -1 and -2 in units of 2^200: below float32's range they weigh nothing, above it they make a row NaN; far: rows that go
    # key by key
    rng = np.random.default_rng(13)
    held, table = K.filled(rng, 2, d, 64, lens)
    held.codes[0], held.steps[..., 0] = 0, 2.0 ** 100
    held.codes[0, ..., 1] = -rng.integers(1, 3, held.codes.shape[1:4])
    held.codes[0, ..., 2] = 0
    if far:
        held.steps[..., 1] = np.ldexp(1.0, rng.choice([-60, 0], held.steps[..., 1].shape))
        held.steps[table[0, 0], :, 1], held.steps[table[0, 1], :, 1] = 2.0 ** -60, 1.0
    q = np.zeros((sum(new), 4, d), np.float32)
    q[..., 0], q[..., 1] = 2.0 ** 120, 2.0 ** 100
    with np.errstate(all="ignore"):
        got, lse, _ = run(s3dx, q, held, table, dtype, new, lens)
        assert not got.any() and np.all(lse == -np.inf)
        q[0, 1, 1] = -(2.0 ** 100)
        got, lse, _ = run(s3dx, q, held, table, dtype, new, lens)
        assert np.all(np.isnan(got[0, 1])) and np.isnan(lse[0, 1])
        got[0, 1], lse[0, 1] = 0.0, -np.inf
        assert not got.any() and np.all(lse == -np.inf)
        # beside keys whose scores float32 holds they count for nothing: the mean of those keys' values
        here = table[0, 0]
        held.codes[0, here], held.steps[here, :, 0] = 0, 2.0 ** -6
        got, lse, _ = run(s3dx, q, held, table, dtype, new, lens, causal=False)
    mean = (held.codes[1, here, :, : min(64, lens[0])] * held.steps[here, :, 1, None, None]).mean(1)
    size = (np.abs(held.codes[1, here, :, : min(64, lens[0])]) * held.steps[here, :, 1, None, None]).mean(1)
    for r in range(new[0]):
        for h in range(4):
            if (r, h) == (0, 1):
                continue
            # weights are equal powers of two; sums of 64 terms; a logarithm of up to 16 to its last bit, times ln 2, and a sum
            assert np.all(np.abs(got[r, h] - mean[h // 2]) <= R.half_step(s3dx, dtype) * np.abs(mean[h // 2]) * 1.01 + 80 * R.U32 * size[h // 2])
            assert abs(lse[r, h] - np.log(64)) <= 2.0 ** -20 + 2.0 ** -21 + 4 * R.U32
