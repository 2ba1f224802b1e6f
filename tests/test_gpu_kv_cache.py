"""GPU: rows written to the cache in 8 bits and read back, code by code against the
definition in 64 bits."""
import numpy as np
import pytest

import attention_ref as R
import cache_ref as K

pytestmark = pytest.mark.gpu


class Side:
    """A cache on the device beside its reference; every byte begins as `fill`."""

    def __init__(self, s3dx, pages, kv, d, block, fill=0x5A):
        self.s3dx, self.held = s3dx, K.Held(pages, kv, d, block)
        size = s3dx.KvCache.size(pages, kv, d, block)
        self.buffer = R.filled(s3dx, (size,), np.uint8, fill)
        self.held.codes, self.held.steps = self.held.take(self.buffer.download())
        self.cache = s3dx.KvCache(self.buffer, pages, kv, d, block)
        self.touched = np.zeros((2, pages, kv, block, d), bool)  # places behind a last row may hold anything

    def write(self, k, v, dtype, new, lens, table, pad=0, behind=0, stream=None):
        s3dx, (n, kv, d) = self.s3dx, k.shape
        dev, exact = [], []
        for x in (k, v):
            bits, x64 = R.stored(s3dx, x, dtype)
            wide = np.full((n + behind, kv * d + pad), 0x7F7F if dtype == s3dx.BF16 else np.nan, bits.dtype)
            wide[:n, : kv * d] = bits.reshape(n, -1)
            dev.append(R.dev(s3dx, wide))
            exact.append(x64)
        ds, dt, dl = R.dev(s3dx, K.starts(new)), R.dev(s3dx, table), R.dev(s3dx, np.asarray(lens, np.int32))
        self.cache.write(dev[0], dev[1], dtype, n + behind, ds, dt, table.shape[1], dl, len(new), kv * d + pad, kv * d + pad, stream=stream)
        s3dx.synchronize(stream)
        self.held.write(*exact, new, lens, table)
        for s, m in enumerate(lens):
            for j in range(min(-(-max(0, m) // self.held.block), table.shape[1])):
                if 0 <= table[s, j] < self.held.pages and new[s]:
                    self.touched[:, table[s, j], :, max(0, m - j * self.held.block):] = True

    def check(self):
        codes, steps = self.held.take(self.buffer.download())
        assert np.array_equal(steps, self.held.steps, equal_nan=True)
        bad = (codes != self.held.codes) & ~self.touched
        assert not bad.any(), np.argwhere(bad)[:5]


CASES = [
    # new rows and lengths of the sequences, kv, d, block
    ([1], [1], 1, 32, 64), ([64], [64], 2, 64, 64), ([65], [65], 1, 128, 64), ([130], [200], 3, 96, 64), ([129], [129], 2, 32, 128),
    ([1], [65], 8, 128, 64), ([1, 1, 1], [1, 64, 200], 2, 64, 128), ([5], [70], 1, 96, 128),
    ([0, 17, 1, 200, 0], [10, 17, 33, 231, 0], 2, 128, 64),     # ragged, with and without rows before
    ([63, 2, 64], [127, 65, 128], 5, 64, 64),                    # into the middle and up to the end of blocks
    ([300], [1000], 16, 64, 64), ([3], [2], 1, 64, 64),          # more rows than the length says: the first has no place
    ([1] * 70, list(range(1, 141, 2)), 1, 32, 64),               # more sequences than lanes
]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("new,lens,kv,d,block", CASES)
def test_write_and_read(s3dx, dtype, new, lens, kv, d, block):
    rng = np.random.default_rng(sum(lens) + d)
    width = max(1, -(-max(lens) // block))
    side = Side(s3dx, width * len(lens) + 2, kv, d, block)
    table = rng.permutation(side.held.pages)[: width * len(lens)].reshape(len(lens), width).astype(np.int32)
    before = [max(0, m - n) for n, m in zip(new, lens)]
    if sum(before):
        side.write(K.rows(rng, sum(before), kv, d), K.rows(rng, sum(before), kv, d), dtype, before, before, table)
    # larger ones behind them: blocks' steps grow
    side.write(2.5 * K.rows(rng, sum(new), kv, d), 3.0 * K.rows(rng, sum(new), kv, d), dtype, new, lens, table, pad=8, behind=2)
    side.check()
    # all of it back, with rows behind the last sequence left as they were
    back = [max(0, m) for m in lens]
    n = sum(back) + 2
    out = [R.filled(s3dx, (n, kv * d + 8), R.store_type(s3dx, dtype), 0x5A) for _ in range(2)]
    side.cache.read(out[0], out[1], dtype, n, R.dev(s3dx, K.starts(back)), R.dev(s3dx, table), width, R.dev(s3dx, np.asarray(lens, np.int32)),
                    len(lens), kv * d + 8, kv * d + 8)
    want = [side.held.values(s, m, table) for s, m in enumerate(lens)]
    for w in (0, 1):
        got = R.values(s3dx, out[w], dtype)
        assert np.array_equal(got[: n - 2, : kv * d].reshape(-1, kv, d), np.concatenate([x[w] for x in want]))
        raw = out[w].download()
        assert np.all(raw[n - 2:].view(np.uint8) == 0x5A) and np.all(np.ascontiguousarray(raw[:, kv * d:]).view(np.uint8) == 0x5A)


@pytest.mark.parametrize("seqs", [64, 65])
@pytest.mark.parametrize("first", [0, 7])
def test_sequences_by_count_and_by_bound(s3dx, seqs, first):
    # as many sequences as lanes and one more, some empty, rows before the first one; what none of them has is neither written nor read
    rng = np.random.default_rng(seqs + first)
    kv, d = 2, 32
    new = [int(n) for n in rng.choice([0, 1, 5, 63, 64, 65, 130], seqs)]
    lens = [n + int(m) for n, m in zip(new, rng.choice([0, 1, 63, 64, 100], seqs))]
    width = -(-max(lens) // 64)
    side = Side(s3dx, width * seqs + 1, kv, d, 64)
    table = rng.permutation(side.held.pages)[: width * seqs].reshape(seqs, width).astype(np.int32)
    before = [m - n for n, m in zip(new, lens)]
    side.write(K.rows(rng, sum(before), kv, d), K.rows(rng, sum(before), kv, d), s3dx.BF16, before, before, table)
    total = first + sum(new) + 3
    k, v = (K.rows(rng, total, kv, d) for _ in range(2))
    (kb, k64), (vb, v64) = (R.stored(s3dx, x, s3dx.BF16) for x in (k, v))
    ds, dt, dl = R.dev(s3dx, K.starts(new) + first), R.dev(s3dx, table), R.dev(s3dx, np.asarray(lens, np.int32))
    side.cache.write(R.dev(s3dx, kb), R.dev(s3dx, vb), s3dx.BF16, total, ds, dt, width, dl, seqs)
    out = [R.filled(s3dx, (total, kv * d), np.uint16, 0x5A) for _ in range(2)]
    side.cache.read(out[0], out[1], s3dx.BF16, total, ds, dt, width, dl, seqs)
    s3dx.synchronize()
    here = slice(first, first + sum(new))
    side.held.write(k64[here], v64[here], new, lens, table)
    for s, m in enumerate(lens):
        for j in range(-(-m // 64)):
            side.touched[:, table[s, j], :, max(0, m - j * 64):] = True
    side.check()
    for w in (0, 1):
        got, raw = R.values(s3dx, out[w], s3dx.BF16), out[w].download()
        want = np.concatenate([side.held.values(s, m, table)[w][m - n:] for s, (n, m) in enumerate(zip(new, lens))])
        assert np.array_equal(got[here].reshape(want.shape), want)
        assert np.all(raw[:first] == 0x5A5A) and np.all(raw[first + sum(new):] == 0x5A5A)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("block", [64, 128])
def test_row_by_row(s3dx, dtype, block):
    # a sequence that grows by one to five rows at a time, its values by a hundredfold: codes are counted again as it goes
    rng = np.random.default_rng(block)
    side = Side(s3dx, 4, 2, 64, block)
    table, m = np.array([[3, 1]], np.int32), 0
    while m < block + 20:
        n = int(rng.integers(1, 6))
        m += n
        grow = 100.0 ** (m / block) * np.array([[[1.0], [0.01]]])
        side.write((grow * K.rows(rng, n, 2, 64)).astype(np.float32), (K.rows(rng, n, 2, 64) / grow).astype(np.float32), dtype, [n], [m], table)
        side.check()


def test_extremes(s3dx):
    # per head: zeros; below 2^-100; the type's largest; beside infinities and NaN; nothing finite; a power of two; a tie
    rng = np.random.default_rng(8)
    k = K.rows(rng, 70, 8, 32)
    k[:, 0] = 0.0
    k[:, 1] *= np.float32(2.0 ** -105)
    k[:, 2] *= np.float32(3e38) / np.abs(k[:, 2]).max()
    k[3, 3, 5], k[4, 3, 6], k[5, 3, 7], k[66, 3, 0] = np.inf, -np.inf, np.nan, -np.nan
    k[:, 4] = np.nan
    k[:, 5] = np.where(np.arange(70) % 2, 2.0 ** 100, -(2.0 ** -100))[:, None]
    k[:, 6] = np.float32(2.0 ** -100) * np.where(rng.random((70, 32)) < 0.5, 1.0, -1.0)
    k[:, 7] = (rng.integers(-255, 256, (70, 32)) * 0.5).astype(np.float32)
    k[0, 7, 0] = 64.0
    for dtype in (s3dx.F32, s3dx.BF16):
        for block in (64, 128):
            side = Side(s3dx, 3, 8, 32, block)
            table = np.array([[2, 0]], np.int32)
            side.write(k[:40], -k[:40], dtype, [40], [40], table)
            side.write(k[40:], -k[40:], dtype, [30], [70], table)
            side.check()
            out = [s3dx.DeviceArray((70, 8, 32), R.store_type(s3dx, dtype)) for _ in range(2)]
            side.cache.read(out[0], out[1], dtype, 70, R.dev(s3dx, K.starts([70])), R.dev(s3dx, table), 2, R.dev(s3dx, np.array([70], np.int32)), 1)
            for w in (0, 1):
                assert np.array_equal(R.values(s3dx, out[w], dtype), side.held.values(0, 70, table)[w])


def test_pages_that_are_none(s3dx):
    # outside the cache, outside the table, before place 0: not written, and zeros when read
    rng = np.random.default_rng(3)
    side = Side(s3dx, 5, 2, 64, 64)
    table = np.array([[0, -1, 4], [5, 1, 2 ** 31 - 1], [2, 3, -(2 ** 31)]], np.int32)
    new, lens = [192, 300, 140], [192, 150, 999]   # the last one's length is more than its table holds
    side.write(K.rows(rng, 632, 2, 64), K.rows(rng, 632, 2, 64), s3dx.F32, new, lens, table)
    side.check()
    out = [R.filled(s3dx, (632, 2, 64), np.float32, 0xFF) for _ in range(2)]
    args = (R.dev(s3dx, K.starts(new)), R.dev(s3dx, table), 3, R.dev(s3dx, np.array(lens, np.int32)), 3)
    side.cache.read(out[0], out[1], s3dx.F32, 632, *args)
    for w in (0, 1):
        got, at = out[w].download(), 0
        for s, (n, m) in enumerate(zip(new, [192, 150, 192])):
            want = np.zeros((n, 2, 64))
            want[max(0, n - m):] = side.held.values(s, m, table)[w][max(0, m - n):]
            assert np.array_equal(got[at: at + n], want), (w, s)
            at += n
    before = side.buffer.download()
    for lengths in ([-5, 0, -(2 ** 31)],):  # no rows at all
        dl = R.dev(s3dx, np.array(lengths, np.int32))
        dk = R.dev(s3dx, K.rows(rng, 632, 2, 64))
        side.cache.write(dk, dk, s3dx.F32, 632, args[0], args[1], 3, dl, 3)
        side.cache.read(out[0], out[1], s3dx.F32, 632, args[0], args[1], 3, dl, 3)
        assert np.array_equal(before, side.buffer.download()) and not out[0].download().any() and not out[1].download().any()


def test_two_streams_and_a_graph(s3dx):
    # one call captured, then replayed with other rows and lengths in its buffers, beside another cache's eager work
    rng = np.random.default_rng(12)
    kv, d, width = 4, 128, 4
    sides = [Side(s3dx, 9, kv, d, 64) for _ in range(2)]
    table = rng.permutation(9)[:8].reshape(2, width).astype(np.int32)
    stream, other = s3dx.Stream(), s3dx.Stream()
    dk, dv = (s3dx.DeviceArray((6, kv, d), np.uint16) for _ in range(2))
    out = [s3dx.DeviceArray((6, kv, d), np.uint16) for _ in range(2)]
    ds, dt, dl = R.dev(s3dx, K.starts([2, 4])), R.dev(s3dx, table), R.dev(s3dx, np.zeros(2, np.int32))

    def body(st=stream):
        sides[0].cache.write(dk, dv, s3dx.BF16, 6, ds, dt, width, dl, 2, stream=st)
        sides[0].cache.read(out[0], out[1], s3dx.BF16, 6, ds, dt, width, dl, 2, stream=st)

    graph = R.Graph(s3dx, stream, body)
    lens = np.zeros(2, np.int64)
    for step in range(40):
        lens += [2, 4]
        (kb, k64), (vb, v64) = (R.stored(s3dx, K.rows(rng, 6, kv, d) * (1 + step / 4), s3dx.BF16) for _ in range(2))
        dk.upload(kb, stream)
        dv.upload(vb, stream)
        dl.upload(lens.astype(np.int32), stream)
        graph.launch()
        if step % 10 == 0:
            sides[1].write(K.rows(rng, 30, kv, d), K.rows(rng, 30, kv, d), s3dx.F32, [10, 20], [10, 20], table, stream=other)
        stream.synchronize()
        sides[0].held.write(k64, v64, [2, 4], lens, table)
        for w in (0, 1):
            want = np.concatenate([sides[0].held.values(s, m, table)[w][m - n:] for s, (n, m) in enumerate(zip([2, 4], lens))])
            assert np.array_equal(R.values(s3dx, out[w], s3dx.BF16), want), step
    graph.close()
    for s, m in enumerate(lens):
        sides[0].touched[:, table[s, -(-m // 64) - 1], :, m % 64 or 64:] = True
        sides[0].touched[:, table[s, -(-m // 64):]] = True
    sides[0].check()
    sides[1].check()


def test_a_cache_beyond_32_bits(s3dx):
    # 2.2 GB of codes: pages whose offset passes 2^31
    kv, d, block, pages = 16, 128, 128, 4200
    rng = np.random.default_rng(6)
    buffer = s3dx.DeviceArray((s3dx.KvCache.size(pages, kv, d, block),), np.uint8)
    cache = s3dx.KvCache(buffer, pages, kv, d, block)
    table = np.array([[4199, 0, 4198, 2100]], np.int32)
    held = K.Held(4, kv, d, block)  # the same rows on four pages
    (kb, k64), (vb, v64) = (R.stored(s3dx, K.rows(rng, 500, kv, d), s3dx.BF16) for _ in range(2))
    held.write(k64, v64, [500], [500], np.array([[0, 1, 2, 3]], np.int32))
    ds, dt, dl = R.dev(s3dx, K.starts([500])), R.dev(s3dx, table), R.dev(s3dx, np.array([500], np.int32))
    cache.write(R.dev(s3dx, kb), R.dev(s3dx, vb), s3dx.BF16, 500, ds, dt, 4, dl, 1)
    out = [s3dx.DeviceArray((500, kv, d), np.uint16) for _ in range(2)]
    cache.read(out[0], out[1], s3dx.BF16, 500, ds, dt, 4, dl, 1)
    want = held.values(0, 500, np.array([[0, 1, 2, 3]], np.int32))
    assert np.array_equal(R.values(s3dx, out[0], s3dx.BF16), want[0]) and np.array_equal(R.values(s3dx, out[1], s3dx.BF16), want[1])
    q = K.rows(rng, 3, 32, d)
    qb, q64 = R.stored(s3dx, q, s3dx.BF16)
    o, lse = s3dx.DeviceArray((3, 32, d), np.uint16), s3dx.DeviceArray((3, 32), np.float32)
    ws = s3dx.DeviceArray(max(1, cache.attention_workspace_size(3, 32, 1, 500)), np.uint8)
    cache.attention(R.dev(s3dx, qb), s3dx.BF16, 3, 32, R.dev(s3dx, K.starts([3])), dt, 4, dl, 1, 500, o, lse, causal=True, workspace=ws)
    K.check(s3dx, s3dx.BF16, R.values(s3dx, o, s3dx.BF16), lse.download().astype(np.float64),
            K.attend(q64, held, np.array([[0, 1, 2, 3]], np.int32), [3], [500], d ** -0.5, True, 0, 0, True))
