"""GPU: gate, residual sum, norms and modulation in one pass against a plain 64-bit
implementation, and a decoder's step made of the library's calls."""
import numpy as np
import pytest

import attention_ref as R
import cache_ref as K

pytestmark = pytest.mark.gpu

EPS = 1e-6


def run(s3dx, x, branch, xd, bd, hd, post, pre, rs=0.5, gain=True, bias=True, gate=True, mod=True, sets=None, count=1, pad=0, place="apart",
        vectors=None, eps=EPS, rng=None):
    """Outputs, references and bounds.  place: "apart", or which inputs y and h take the place of."""
    n, c = x.shape
    rng = rng or np.random.default_rng(n + c)

    def wide(a, dtype):
        bits, a64 = R.stored(s3dx, a, dtype)
        w = np.full((n, c + pad), 0x7FC0 if dtype == s3dx.BF16 else np.nan, bits.dtype)
        w[:, :c] = bits
        return R.dev(s3dx, w), a64

    dx, x64 = wide(x, xd)
    db, b64 = wide(branch, bd)
    vec = {k: None for k in ("post_w", "post_b", "pre_w", "pre_b")}
    for k in vec:
        if (post if k.startswith("post") else pre) != K.NONE and (gain if k.endswith("w") else bias):
            vec[k] = (rng.standard_normal(c) * 0.3 + k.endswith("w")).astype(np.float32)
    mods = (rng.standard_normal((count, 3, c + 4)) * 0.4).astype(np.float32)
    dm = R.dev(s3dx, mods)
    dv = {k: None if v is None else R.dev(s3dx, v) for k, v in vec.items()}
    at = lambda j: dm.ptr + 4 * j * (c + 4)  # noqa: E731
    dsets = None if sets is None else R.dev(s3dx, np.concatenate([sets[:, None], np.full((n, 3), -7, np.int32)], 1))
    y = dx if place == "y=x" else db if place == "y=branch" else R.filled(s3dx, (n, c + pad), R.store_type(s3dx, xd), 0x5A)
    h = dx if place == "h=x" else db if place in ("h=branch", "y=x") and bd == hd else R.filled(s3dx, (n, c + pad), R.store_type(s3dx, hd), 0x5A)
    s3dx.gated_norm_rows(dx, xd, db, bd, n, c, eps, y, h, hd, post, pre, residual_scale=rs, gate=at(2) if gate else None,
                         mod_scale=at(1) if mod else None, mod_shift=at(0) if mod else None, mod_stride=3 * (c + 4), sets=dsets, set_stride=4,
                         set_count=count, x_stride=c + pad, branch_stride=c + pad, y_stride=c + pad, h_stride=c + pad, **dv)
    which = np.zeros(n, np.int64) if sets is None else sets.astype(np.int64)
    inside = (which >= 0) & (which < count)
    m = np.where(inside[:, None, None], mods[np.where(inside, which, 0)].astype(np.float64), 0.0)[:, :, :c]
    v64 = {k: None if v is None else v.astype(np.float64) for k, v in vec.items()}
    with np.errstate(all="ignore"):
        want = K.gated(x64, b64, post, v64["post_w"], v64["post_b"], float(np.float32(rs)), m[:, 2] if gate else None, pre, v64["pre_w"],
                       v64["pre_b"], m[:, 1] if mod else None, m[:, 0] if mod else None, eps)
    for a in (y, h):
        raw = a.download()
        if place == "apart":
            assert np.all(np.ascontiguousarray(raw[:, c:]).view(np.uint8) == 0x5A)
    return R.values(s3dx, y, xd)[:, :c], R.values(s3dx, h, hd)[:, :c], want


def check(s3dx, xd, hd, got_y, got_h, want, what=""):
    y, y_off, h, h_off = want
    for name, got, ref, off, dtype in (("y", got_y, y, y_off, xd), ("h", got_h, h, h_off, hd)):
        half = R.half_step(s3dx, dtype)
        bound = off + half * (np.abs(ref) + off) + 1e-37
        share = np.max(np.abs(got - ref) / bound)
        print(f"  {what} {name} worst share of the bound {share:.3f}", flush=True)
        assert share <= 1.0, (what, name)


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
@pytest.mark.parametrize("types", [(0, 0, 0), (1, 1, 1), (0, 1, 1), (1, 0, 0)])
def test_norms_and_types(s3dx, post, pre, types):
    for n, c, pad in ((1, 64, 0), (37, 256, 8), (70, 100, 0), (5, 1000, 4)):
        rng = np.random.default_rng(c)
        x, b = (rng.standard_normal((n, c)) + 0.3).astype(np.float32), (2 * rng.standard_normal((n, c)) - 0.5).astype(np.float32)
        sets = rng.integers(-1, 4, n).astype(np.int32)  # some of no set
        check(s3dx, types[0], types[2], *run(s3dx, x, b, *types, post, pre, sets=sets, count=3, pad=pad), what=str((n, c)))


@pytest.mark.parametrize("c", [1, 2, 7, 8, 9, 31, 64, 65, 96, 127, 128, 129, 511, 512, 520, 1023, 1024, 1025, 2040, 2048, 2056, 4096, 5000,
                               8192, 8193, 16383, 16384])
def test_widths(s3dx, c):
    rng = np.random.default_rng(c)
    for n in (1, 9):
        x, b = rng.standard_normal((n, c)).astype(np.float32), rng.standard_normal((n, c)).astype(np.float32)
        check(s3dx, 1, 1, *run(s3dx, x, b, 1, 1, 1, 2, 1, bias=False), what="c %d" % c)
        check(s3dx, 0, 0, *run(s3dx, x, b, 0, 0, 0, 1, 2, gain=False, gate=False, mod=False, rs=1.0), what="c %d" % c)


@pytest.mark.parametrize("types", [(0, 0, 0), (1, 1, 1)])
@pytest.mark.parametrize("place", ["y=x", "y=branch", "h=x", "h=branch"])
def test_in_place(s3dx, types, place):
    for n, c in ((300, 256), (50, 1001), (10, 4096)):
        rng = np.random.default_rng(c)
        x, b = rng.standard_normal((n, c)).astype(np.float32), rng.standard_normal((n, c)).astype(np.float32)
        check(s3dx, types[0], types[2], *run(s3dx, x, b, *types, 1, 2, place=place), what=place)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("c", [9, 333, 1025, 2601, 5003, 16381])
def test_sums_in_place_of_odd_rows(s3dx, dtype, c):
    # a row's last piece shares channels with its neighbour's, of another wave in wide rows
    rng = np.random.default_rng(c)
    for place in ("y=x", "y=branch"):
        x, b = rng.standard_normal((40, c)).astype(np.float32), rng.standard_normal((40, c)).astype(np.float32)
        dx, x64 = R.dev(s3dx, R.stored(s3dx, x, dtype)[0]), R.stored(s3dx, x, dtype)[1]
        db, b64 = R.dev(s3dx, R.stored(s3dx, b, dtype)[0]), R.stored(s3dx, b, dtype)[1]
        y = dx if place == "y=x" else db
        s3dx.gated_norm_rows(dx, dtype, db, dtype, 40, c, EPS, y)
        want = x64 + b64
        assert np.all(np.abs(R.values(s3dx, y, dtype) - want) <= (R.half_step(s3dx, dtype) + R.U32) * np.abs(want))


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("power", [-70, -40, 40, 64, 100, 120])
@pytest.mark.parametrize("c", [96, 1024, 2900])
def test_values_of_any_size(s3dx, kind, power, c):
    # squares beyond float32 and below it; beside rows of ordinary size
    rng = np.random.default_rng(c)
    n = 12
    b = rng.standard_normal((n, c)).astype(np.float32)
    b[::3] = np.ldexp(b[::3], power)
    x = rng.standard_normal((n, c)).astype(np.float32)
    check(s3dx, 0, 0, *run(s3dx, x, b, 0, 0, 0, kind, kind, mod=False), what=str(power))
    x[::3] = np.ldexp(x[::3], power - 10 if power > 0 else power)
    check(s3dx, 0, 0, *run(s3dx, x, 0.0 * b, 0, 0, 0, 0, kind, mod=False), what=str(power))


# The norms of rows whose sums pass float32.  Equal channels have a norm of 0 exactly: their mean is off by at most 39 u of them (sums of
# 38 terms in a chain, one division), so that channels less this mean are exact and alike, these differences' own mean is off by (39 u)^2 of a
# channel, far below half its last bit, and they are their mean when it is taken off them in turn.
@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("c", [7, 333, 1024, 4097, 5000, 8192, 16384])
def test_values_up_to_the_types_largest(s3dx, kind, dtype, c):
    rng = np.random.default_rng(c + kind)
    n, top = 10, 3.38e38
    b = rng.standard_normal((n, c)).astype(np.float32)
    b[1], b[2] = top * rng.choice([-1, 1], c), 1.8e38 * rng.choice([-1, 1], c)
    b[4], b[5] = top * rng.random(c), np.where(np.arange(c) % 97 == 5, -top, top)
    b[6], b[7] = 2.0 ** 120 * rng.standard_normal(c), 1e25 * rng.standard_normal(c)
    b[8] = np.where(np.arange(c) == c // 2, top, 1.0)
    x = rng.standard_normal((n, c)).astype(np.float32)
    check(s3dx, dtype, dtype, *run(s3dx, x, b, dtype, dtype, dtype, kind, kind, mod=False, gate=False), what="branch")
    check(s3dx, dtype, dtype, *run(s3dx, b, 0.0 * b, dtype, dtype, dtype, 0, kind, mod=False), what="stream")


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("c", [1, 200, 333, 1000, 1024, 2600, 5000, 16384])
def test_equal_channels_beyond_float32s_sums(s3dx, dtype, c):
    x = np.array([2.0 ** 120, -1.1e36, 3.3e38, -(2.0 ** 127), 1.7e34, 3.0], np.float32)[:, None] * np.ones((6, c), np.float32)
    zero = np.zeros_like(x)
    y, h, _ = run(s3dx, x, zero, dtype, dtype, dtype, 0, 1, bias=False, mod=False)
    assert np.array_equal(y, R.stored(s3dx, x, dtype)[1]) and not h.any()
    y, h, _ = run(s3dx, zero, x, dtype, dtype, dtype, 1, 1, bias=False, mod=False)
    assert not y.any() and not h.any()


@pytest.mark.parametrize("c", [5, 200, 333, 1000, 1024, 2600, 5000, 16384])
def test_channels_that_are_nearly_alike(s3dx, c):
    size = np.array([100.7, -3.7, 1e-3, 12345.678, -1e10, 1.3e20, 1e30, 1e-30, 1.37e-30, -1.9e-20, 7.3e-13, 1.1e-37], np.float32)
    x = size[:, None] * np.ones((len(size), c), np.float32)
    zero = np.zeros_like(x)
    for dtype in (s3dx.F32, s3dx.BF16):
        y, h, _ = run(s3dx, x, zero, dtype, dtype, dtype, 0, 1, bias=False, mod=False)
        assert np.array_equal(y, R.stored(s3dx, x, dtype)[1]) and not h.any()  # as above
    # Channels apart by a few of their last bits.  Differences from a first mean are exact, whole last bits, and what is left to round is
    # their own mean, their differences from that and the root: no more than the bound of these rows less one of their channels.
    rng = np.random.default_rng(c)
    near = np.ldexp(1.0 + 2.0 ** -23 * rng.integers(5, 12, (8, c)), rng.integers(-20, 90, (8, 1)))
    got = run(s3dx, near.astype(np.float32), zero[:8], 0, 0, 0, 0, 1, gain=False, bias=False, mod=False)[1]
    want, off = K.normed(near - near[:, :1], K.LAYER, None, None, EPS)
    assert np.all(np.abs(got - want) <= off + R.U32 * (np.abs(want) + off) + 1e-37)


@pytest.mark.parametrize("count", [0, 2])
@pytest.mark.parametrize("c", [5, 96, 1001, 3000])
def test_rows_of_no_set_fetch_no_vectors(s3dx, count, c):
    # a table of no sets holds nothing to be fetched: rows outside take gate, scale and shift as 0
    rng = np.random.default_rng(c + count)
    n = 21
    x, b = rng.standard_normal((n, c)).astype(np.float32), rng.standard_normal((n, c)).astype(np.float32)
    sets = rng.choice([-1, count, 2 ** 31 - 1, -(2 ** 31)] + list(range(count)), n).astype(np.int32)
    table = (1 + rng.random((max(count, 1), 3, c)) if count else np.ones(1)).astype(np.float32)
    dx, db, dm, ds = (R.dev(s3dx, a) for a in (x, b, table, sets))
    y, h = (s3dx.DeviceArray((n, c), np.float32) for _ in range(2))
    at = lambda j: dm.ptr + 4 * j * c if count else dm.ptr  # noqa: E731
    s3dx.gated_norm_rows(dx, 0, db, 0, n, c, EPS, y, h, 0, post=1, pre=1, gate=at(0), mod_scale=at(1), mod_shift=at(2), mod_stride=3 * c,
                         sets=ds, set_count=count)
    inside = (sets >= 0) & (sets < count)
    m = np.zeros((n, 3, c)) if not count else np.where(inside[:, None, None], table.astype(np.float64)[np.where(inside, sets, 0)], 0.0)
    want = K.gated(x.astype(np.float64), b.astype(np.float64), 1, None, None, 1.0, m[:, 0], 1, None, None, m[:, 1], m[:, 2], EPS)
    check(s3dx, 0, 0, y.download(), h.download(), want, "%d sets" % count)
    assert np.array_equal(y.download()[~inside], x[~inside])


def test_rows_that_are_alike_or_not_finite(s3dx):
    c = 200
    x, b = np.zeros((6, c), np.float32), np.ones((6, c), np.float32)
    x[1] = 3.0
    b[2] = 0.0
    b[3, 5], b[4, 6], x[5, 7] = np.nan, np.inf, np.nan
    y, h, want = run(s3dx, x, b, 0, 0, 0, 1, 1, bias=False, gate=False, mod=False)
    assert np.array_equal(y[:3], x[:3]) and not h[:3].any()  # the norm of equal channels is 0
    for r in (3, 4, 5):
        assert np.all(np.isnan(h[r]))
    assert np.all(np.isnan(y[3])) and np.all(np.isnan(y[4])) and np.isnan(y[5, 7]) and np.isfinite(np.delete(y[5], 7)).all()


def test_sum_alone_and_no_rows(s3dx):
    rng = np.random.default_rng(1)
    x, b = rng.standard_normal((33, 90)).astype(np.float32), rng.standard_normal((33, 90)).astype(np.float32)
    dx, db, y = R.dev(s3dx, x), R.dev(s3dx, b), s3dx.DeviceArray((33, 90), np.float32)
    s3dx.gated_norm_rows(dx, s3dx.F32, db, s3dx.F32, 33, 90, EPS, y, residual_scale=-2.0)
    want = x.astype(np.float64) - 2.0 * b.astype(np.float64)
    assert np.all(np.abs(y.download() - want) <= R.U32 * np.abs(want))
    s3dx.gated_norm_rows(dx, s3dx.F32, db, s3dx.F32, 0, 90, EPS, y)


def test_a_graph_and_another_stream(s3dx):
    rng = np.random.default_rng(2)
    n, c = 40, 768
    stream, other = s3dx.Stream(), s3dx.Stream()
    dx, db = s3dx.DeviceArray((n, c), np.float32), s3dx.DeviceArray((n, c), np.float32)
    outs = [[s3dx.DeviceArray((n, c), np.float32) for _ in range(2)] for _ in range(2)]
    call = lambda o, st: s3dx.gated_norm_rows(dx, 0, db, 0, n, c, EPS, o[0], o[1], post=1, pre=2, stream=st)  # noqa: E731
    graph = R.Graph(s3dx, stream, lambda: call(outs[0], stream))
    for _ in range(4):
        x, b = rng.standard_normal((n, c)).astype(np.float32), rng.standard_normal((n, c)).astype(np.float32)
        dx.upload(x, stream)
        db.upload(b, stream)
        graph.launch()
        stream.synchronize()
        call(outs[1], other)
        other.synchronize()
        want = K.gated(x.astype(np.float64), b.astype(np.float64), 1, None, None, 1.0, None, 2, None, None, None, None, EPS)
        check(s3dx, 0, 0, outs[0][0].download(), outs[0][1].download(), want)
        assert all(np.array_equal(a.download(), b.download()) for a, b in zip(*outs))
    graph.close()


# ---------------------------------------------------------------------------
# A block's step over a cache: norm and modulation, projection, norms and rotation of heads, the cache and its attention, projection, gate,
# sum and the next norm
# ---------------------------------------------------------------------------
def test_a_step_over_the_cache(s3dx, W):
    rng = np.random.default_rng(30)
    c, heads, kv, d, width, seqs = 256, 4, 2, 64, 4, 3
    qkv = (heads + 2 * kv) * d
    into = s3dx.SparseConv(c, qkv, 1, s3dx.BF16).set_weights((rng.standard_normal((qkv, 1, c)) / 16).astype(np.float32))
    out_of = s3dx.SparseConv(heads * d, c, 1, s3dx.BF16).set_weights((rng.standard_normal((c, 1, heads * d)) / 16).astype(np.float32))
    rotary = s3dx.Rotary.per_axis(d, [d // 2])
    side = s3dx.DeviceArray.from_host(np.zeros(s3dx.KvCache.size(seqs * width, kv, d, 64), np.uint8))
    cache = s3dx.KvCache(side, seqs * width, kv, d, 64)
    held = K.Held(seqs * width, kv, d, 64)
    table = rng.permutation(seqs * width).reshape(seqs, width).astype(np.int32)
    dt = R.dev(s3dx, table)
    mods = R.dev(s3dx, (0.3 * rng.standard_normal((seqs, 3, c))).astype(np.float32))
    at = lambda j: mods.ptr + 4 * j * c  # noqa: E731
    stream = s3dx.Stream()
    lens, graph = np.zeros(seqs, np.int64), None
    prompt = [70, 1, 33]
    for step in range(9):
        new = prompt if step == 0 else [1] * seqs   # a prompt, then rows one by one; from the third step on as a graph
        n = sum(new)
        lens = lens + new
        if step < 2:
            rows = s3dx.DeviceArray((n, qkv), np.uint16)
            x, y, h, zero = (s3dx.DeviceArray((n, c), np.uint16) for _ in range(4))
            nx, branch, o = s3dx.DeviceArray((n, c), np.uint16), s3dx.DeviceArray((n, c), np.uint16), s3dx.DeviceArray((n, heads, d), np.uint16)
            lse = s3dx.DeviceArray((n, heads), np.float32)
            zero.upload(np.zeros((n, c), np.uint16), stream)
            ds, dl, sets, pos = (s3dx.DeviceArray(k, np.int32) for k in ((seqs + 1,), (seqs,), (n,), (n,)))
            ws = s3dx.DeviceArray(max(1, cache.attention_workspace_size(n, heads, seqs, width * 64, 100, 2)), np.uint8)
        rb, r64 = R.stored(s3dx, rng.standard_normal((n, c)).astype(np.float32), s3dx.BF16)
        x.upload(rb, stream)
        ds.upload(K.starts(new), stream)
        dl.upload(lens.astype(np.int32), stream)
        sets.upload(np.repeat(np.arange(seqs), new).astype(np.int32), stream)
        pos.upload(np.concatenate([np.arange(m - k, m) for k, m in zip(new, lens)]).astype(np.int32), stream)
        gated = dict(sets=sets, set_count=seqs, mod_stride=3 * c, stream=stream)

        def body():
            s3dx.gated_norm_rows(x, 1, zero, 1, n, c, EPS, y, h, pre=1, mod_scale=at(1), mod_shift=at(0), **gated)
            into.run(h, n, None, n, rows, stream=stream)
            s3dx.qk_norm_rotary(rows, rows.ptr + 2 * heads * d, 1, n, heads, kv, d, EPS, rotary=rotary, positions=pos, position_stride=1,
                                q_stride=qkv, k_stride=qkv, stream=stream)
            cache.write(rows.ptr + 2 * heads * d, rows.ptr + 2 * (heads + kv) * d, 1, n, ds, dt, width, dl, seqs, qkv, qkv, stream=stream)
            cache.attention(rows, 1, n, heads, ds, dt, width, dl, seqs, width * 64, o, lse, q_stride=qkv, causal=True, window=100, sinks=2,
                            workspace=ws, stream=stream)
            out_of.run(o, n, None, n, branch, stream=stream)
            s3dx.gated_norm_rows(x, 1, branch, 1, n, c, EPS, y, nx, post=2, pre=1, gate=at(2), **gated)

        if step == 2:
            graph = R.Graph(s3dx, stream, body)
        graph.launch() if graph else body()
        stream.synchronize()
        # each call against the definition, from what the calls before it left
        m64 = mods.download().astype(np.float64)[np.repeat(np.arange(seqs), new)]
        want = K.gated(r64, np.zeros_like(r64), 0, None, None, 1.0, None, 1, None, None, m64[:, 1], m64[:, 0], EPS)
        check(s3dx, 1, 1, R.values(s3dx, y, 1) * 0 + want[0], R.values(s3dx, h, 1), want, "norm")
        parts = R.values(s3dx, rows, 1).reshape(n, heads + 2 * kv, d)
        held.write(parts[:, heads: heads + kv], parts[:, heads + kv:], new, lens, table)
        K.check(s3dx, 1, R.values(s3dx, o, 1), lse.download().astype(np.float64),
                K.attend(parts[:, :heads], held, table, new, lens, d ** -0.5, True, 100, 2, True), "step %d" % step)
        want = K.gated(r64, R.values(s3dx, branch, 1), 2, None, None, 1.0, m64[:, 2], 1, None, None, None, None, EPS)
        check(s3dx, 1, 1, R.values(s3dx, y, 1), R.values(s3dx, nx, 1), want, "gate")
    graph.close()
