"""GPU: rotary positions with several axes and the query/key norms in the same
pass, against 64-bit references, element by element."""
import numpy as np
import pytest

import attention_ref as R

pytestmark = pytest.mark.gpu

PER_AXIS = {"xyz": [10, 10, 10], "one": [16], "two": [3, 8], "four": [1, 2, 3, 4], "few": [1], "most": [31],
            "odd": [3, 4, 6]}


def inputs(rng, n, heads, stride, d):
    x = rng.standard_normal((n, stride)).astype(np.float32) * np.exp(rng.standard_normal((n, 1))).astype(np.float32)
    return x, lambda v: v[:, : heads * d].reshape(n, heads, d)


# cos and sin: 2^-23 off at most (their argument's rounding and the library function's 2 ulp, 4 u together with
# one to spare); two products and their sum: 3 u more.  Then the output's rounding.
TURN = 8 * R.U32


def compare(got, want, size, rel, out_step, what):
    off = np.abs(got - want) - rel * size - out_step * np.abs(want)
    print(f"  {what}: worst {np.max(off):.2e} above its bound, mean error {np.mean(np.abs(got - want)):.2e}", flush=True)
    assert np.all(off <= 1e-37), what  # 1e-37: results below float32's normal range


@pytest.mark.parametrize("x_dtype,y_dtype", [(0, 0), (1, 1), (0, 1), (1, 0)])
@pytest.mark.parametrize("n,heads,d,axes,adjacent,pad,span", [
    (1, 1, 64, "xyz", True, 0, 64),          # one row
    (333, 16, 64, "xyz", True, 0, 64),
    (100, 12, 64, "xyz", False, 1024, 64),   # rows within a wider projection
    (57, 5, 128, "one", False, 0, 2 ** 31 - 1),   # far positions
    (57, 3, 96, "two", True, 32, 100000),    # channels that do not turn
    (40, 2, 32, "one", True, 0, 4096),       # every channel turns
    (31, 3, 23, "four", False, 5, 64),       # odd width and stride
    (9, 2, 256, "two", True, 3, 64),
    # halves that are not whole pieces of 8 channels, many and few rows
    (40, 5, 64, "odd", False, 0, 64),
    (1500, 3, 64, "most", False, 0, 4096),
    (7, 4, 256, "odd", False, 64, 64),
    (3, 9, 32, "few", False, 0, 64),
    (11, 3, 96, "most", False, 32, 64),
    # many narrow rows
    (16500, 2, 64, "most", True, 5, 4096),
    (33001, 1, 32, "odd", False, 0, 64),
    (8300, 3, 24, "few", False, 2, 64),
])
def test_rotary(s3dx, x_dtype, y_dtype, n, heads, d, axes, adjacent, pad, span):
    rng = np.random.default_rng(n + d)
    m = PER_AXIS[axes]
    rot = s3dx.Rotary.per_axis(d, m, 10000.0, s3dx.ROTARY_ADJACENT if adjacent else s3dx.ROTARY_HALVES)
    axis = [a for a, k in enumerate(m) for _ in range(k)]
    freq = [10000.0 ** (-j / k) for k in m for j in range(k)]
    stride = heads * d + pad
    x, cut = inputs(rng, n, heads, stride, d)
    xs, xv = R.stored(s3dx, x, x_dtype)
    pos = rng.integers(-span, span, (n, 5), dtype=np.int64).astype(np.int32)
    dx, dp = R.dev(s3dx, xs), R.dev(s3dx, pos)
    for inverse in (False, True):
        y = R.filled(s3dx, (n + 1, heads * d + 7), R.store_type(s3dx, y_dtype), 0x5A)
        rot.apply(dx, x_dtype, n, heads, dp.ptr + 4, y, position_stride=5, inverse=inverse, x_stride=stride, y_dtype=y_dtype,
                  y_stride=heads * d + 7)
        want, size = R.turn(cut(xv), pos[:, 1:], axis, freq, adjacent, inverse)
        got = R.values(s3dx, y, y_dtype)
        compare(got[:n, : heads * d].reshape(n, heads, d), want, size, TURN, R.half_step(s3dx, y_dtype), f"inverse={inverse}")
        raw = y.download()  # what stands between and behind the rows
        assert np.all(raw[n].view(np.uint8) == 0x5A) and np.all(np.ascontiguousarray(raw[:, heads * d:]).view(np.uint8) == 0x5A)


def test_rotary_in_place_and_back(s3dx):
    rng = np.random.default_rng(5)
    n, heads, d = 200, 4, 64
    x = rng.standard_normal((n, 3 * heads * d)).astype(np.float32)
    pos = rng.integers(0, 64, (n, 3)).astype(np.int32)
    rot = s3dx.Rotary.per_axis(d, [10, 10, 10])
    dx, dp = R.dev(s3dx, x), R.dev(s3dx, pos)
    rot.apply(dx, s3dx.F32, n, heads, dp, x_stride=3 * heads * d)
    out = s3dx.DeviceArray((n, heads * d), np.float32)
    rot.apply(R.dev(s3dx, x), s3dx.F32, n, heads, dp, out, x_stride=3 * heads * d)
    turned = dx.download()
    assert np.array_equal(turned[:, : heads * d], out.download())
    assert np.array_equal(turned[:, heads * d:], x[:, heads * d:])
    rot.apply(dx, s3dx.F32, n, heads, dp, x_stride=3 * heads * d, inverse=True)
    # two turns: the first's error turns with the row
    size = np.abs(x[:, : heads * d]).reshape(n, heads, d // 2, 2).sum(-1, keepdims=True).repeat(2, -1).reshape(n, -1)
    assert np.all(np.abs(dx.download()[:, : heads * d] - x[:, : heads * d]) <= (3 * TURN + R.U32) * size)


def test_rotary_one_series_over_all_pairs(s3dx):
    # axes taking turns over one series, as any table may have it; zero and negative frequencies
    rng = np.random.default_rng(6)
    n, heads, d = 65, 2, 64
    axis = [j % 3 for j in range(32)]
    freq = [0.0, -1.0, -1e-9] + [500.0 ** (-j / 32) for j in range(29)]
    rot = s3dx.Rotary(d, axis, freq, 3, s3dx.ROTARY_HALVES)
    x = rng.standard_normal((n, heads, d)).astype(np.float32)
    pos = rng.integers(-2 ** 31, 2 ** 31, (n, 3)).astype(np.int32)
    y = s3dx.DeviceArray(x.shape, np.float32)
    rot.apply(R.dev(s3dx, x), s3dx.F32, n, heads, R.dev(s3dx, pos), y)
    want, size = R.turn(x.astype(np.float64), pos, axis, freq, False)
    compare(y.download(), want, size, TURN, R.U32, "table")


# the sum of d squares, whatever its order: (d + 2) u relative, halved by the root; the root's own 2 ulp (4 u), the
# gain, the scale
def norm_rel(d):
    return ((d + 2) / 2 + 8) * R.U32


@pytest.mark.parametrize("dtype,out_dtype", [(0, 0), (1, 1), (0, 1), (1, 0)])
@pytest.mark.parametrize("n,h,kv,d,axes,adjacent,gain,eps", [
    (1, 12, 12, 64, "xyz", True, "head", 1e-6),
    (501, 16, 16, 64, "xyz", True, "head", 1e-24),   # F.normalize's form: eps all but none
    (77, 10, 2, 128, "two", False, "all", 1e-5),
    (33, 3, 1, 96, None, False, "all", 1e-6),        # the norm alone
    (20, 4, 0, 32, "one", False, None, 1e-6),        # queries alone
    (13, 5, 3, 20, "one10", True, "head", 1e-6),     # odd width
    (65, 7, 7, 256, "two", True, "head", 1e-6),
    (1030, 6, 2, 64, "odd", False, "head", 1e-6),
    (9, 5, 5, 128, "most", False, "all", 1e-6),
])
def test_qk_norm_rotary(s3dx, dtype, out_dtype, n, h, kv, d, axes, adjacent, gain, eps):
    rng = np.random.default_rng(n + h + d)
    m = {"one10": [10], **PER_AXIS}.get(axes)
    rot = m and s3dx.Rotary.per_axis(d, m, 10000.0, s3dx.ROTARY_ADJACENT if adjacent else s3dx.ROTARY_HALVES)
    row = (h + 2 * max(kv, 1)) * d
    x = (rng.standard_normal((n, row)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32)
    if n > 4:
        x[3] = 0.0                  # a row of zeros stays zeros
        x[2] *= np.float32(1e-12)   # eps is what matters there
    xs, xv = R.stored(s3dx, x, dtype)
    pos = rng.integers(0, 64, (n, 4)).astype(np.int32)
    shape = {"head": lambda k: (k, d), "all": lambda k: (d,), None: None}[gain]
    gains = [None if shape is None or not k else (1 + 0.2 * rng.standard_normal(shape(k))).astype(np.float32) for k in (h, kv)]
    dx, dg = R.dev(s3dx, xs), [None if g is None else R.dev(s3dx, g) for g in gains]
    size = 2 if dtype == s3dx.BF16 else 4
    st = R.store_type(s3dx, out_dtype)
    yq, yk = R.filled(s3dx, (n + 1, h * d), st, 0x5A), R.filled(s3dx, (n + 1, max(kv, 1) * d), st, 0x5A)
    s3dx.qk_norm_rotary(dx, dx.ptr + h * d * size if kv else None, dtype, n, h, kv, d, eps, yq, yk if kv else None, rotary=rot,
                        positions=R.dev(s3dx, pos).ptr + 4 if rot else None, position_stride=4, q_gain=dg[0], k_gain=dg[1],
                        gain_per_head=gain == "head", q_stride=row, k_stride=row, out_dtype=out_dtype)
    for y, heads, at, g in ((yq, h, 0, gains[0]), (yk, kv, h * d, gains[1])):
        if not heads:
            continue
        want = R.rms(xv[:, at: at + heads * d].reshape(n, heads, d), g, eps)
        scale = np.abs(want)
        if m:
            axis = [a for a, k in enumerate(m) for _ in range(k)]
            freq = [10000.0 ** (-j / k) for k in m for j in range(k)]
            want, scale = R.turn(want, pos[:, 1:], axis, freq, adjacent)
        got = R.values(s3dx, y, out_dtype)[:n].reshape(n, heads, d)
        compare(got, want, scale, TURN + norm_rel(d), R.half_step(s3dx, out_dtype), f"{heads} heads")
        if n > 4:
            assert np.all(got[3] == 0.0)
        assert np.all(y.download()[n].view(np.uint8) == 0x5A)


def test_qk_norm_rotary_in_place_of_the_projection(s3dx):
    # as a forward would: the packed rows' queries and keys are replaced, the values stay
    rng = np.random.default_rng(8)
    n, h, kv, d = 130, 8, 4, 64
    row = (h + 2 * kv) * d
    bits, _ = R.stored(s3dx, rng.standard_normal((n, row)), s3dx.BF16)
    pos = R.dev(s3dx, rng.integers(0, 64, (n, 3)).astype(np.int32))
    rot = s3dx.Rotary.per_axis(d, [10, 10, 10])
    dx = R.dev(s3dx, bits)
    q, k = s3dx.DeviceArray((n, h * d), np.uint16), s3dx.DeviceArray((n, kv * d), np.uint16)
    s3dx.qk_norm_rotary(dx, dx.ptr + 2 * h * d, s3dx.BF16, n, h, kv, d, 1e-6, q, k, rotary=rot, positions=pos, q_stride=row, k_stride=row)
    s3dx.qk_norm_rotary(dx, dx.ptr + 2 * h * d, s3dx.BF16, n, h, kv, d, 1e-6, rotary=rot, positions=pos, q_stride=row, k_stride=row)
    got = dx.download()
    assert np.array_equal(got[:, : h * d], q.download()) and np.array_equal(got[:, h * d: (h + kv) * d], k.download())
    assert np.array_equal(got[:, (h + kv) * d:], bits[:, (h + kv) * d:])


def test_a_row_with_nan_or_infinity_stays_alone(s3dx):
    rng = np.random.default_rng(9)
    n, h, d = 12, 3, 64
    x = rng.standard_normal((n, h, d)).astype(np.float32)
    clean, dirty = s3dx.DeviceArray(x.shape, np.float32), s3dx.DeviceArray(x.shape, np.float32)
    pos = R.dev(s3dx, rng.integers(0, 64, (n, 3)).astype(np.int32))
    rot = s3dx.Rotary.per_axis(d, [10, 10, 10])
    y = x.copy()
    y[4, 1, 7], y[9, 2, 0] = np.nan, np.inf
    for a, out in ((x, clean), (y, dirty)):
        s3dx.qk_norm_rotary(R.dev(s3dx, a), None, s3dx.F32, n, h, 0, d, 1e-6, out, rotary=rot, positions=pos)
    c, e = clean.download(), dirty.download()
    keep = np.ones((n, h), bool)
    keep[4, 1] = keep[9, 2] = False
    assert np.array_equal(c[keep], e[keep])
    assert np.isnan(e[4, 1]).all() and np.isnan(e[9, 2, 0])


@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("pad", [0, 1])
def test_channels_that_do_not_turn_are_copied(s3dx, adjacent, pad):
    # NaN and infinities among them reach no other channel
    rng = np.random.default_rng(11)
    n, h, d = 9, 2, 64
    x = rng.standard_normal((n, h * d + pad)).astype(np.float32)
    x[:, 48: 64: 3] = np.inf
    x[2, 49] = np.nan
    rot = s3dx.Rotary.per_axis(d, [8, 8, 8], pairing=s3dx.ROTARY_ADJACENT if adjacent else s3dx.ROTARY_HALVES)
    y = s3dx.DeviceArray((n, h, d), np.float32)
    rot.apply(R.dev(s3dx, x), s3dx.F32, n, h, R.dev(s3dx, rng.integers(0, 64, (n, 3)).astype(np.int32)), y, x_stride=h * d + pad)
    got, want = y.download(), x[:, : h * d].reshape(n, h, d)
    assert np.array_equal(got[..., 48:], want[..., 48:], equal_nan=True) and np.isfinite(got[..., :48]).all()


def test_rotary_captured_and_replayed(s3dx):
    rng = np.random.default_rng(10)
    n, h, d = 300, 16, 64
    rot = s3dx.Rotary.per_axis(d, [10, 10, 10])
    x, y, z = (s3dx.DeviceArray((n, h, d), np.float32) for _ in range(3))
    pos = R.dev(s3dx, rng.integers(0, 64, (n, 3)).astype(np.int32))
    stream = s3dx.Stream()
    s3dx.synchronize()
    g = R.Graph(s3dx, stream, lambda: s3dx.qk_norm_rotary(x, None, s3dx.F32, n, h, 0, d, 1e-6, y, rotary=rot, positions=pos, stream=stream))
    for _ in range(3):
        x.upload(rng.standard_normal((n, h, d)).astype(np.float32))
        g.launch()
        stream.synchronize()
        s3dx.qk_norm_rotary(x, None, s3dx.F32, n, h, 0, d, 1e-6, z, rotary=rot, positions=pos)
        assert np.array_equal(y.download(), z.download())
    g.close()


def test_rotary_of_more_rows_than_a_launch_takes(s3dx):
    rng = np.random.default_rng(12)
    n = 2 ** 25 + 5
    x = np.tile(rng.standard_normal((64, 2)).astype(np.float32), (n // 64 + 1, 1))[:n]
    pos = np.arange(n, dtype=np.int32)
    y = R.filled(s3dx, (n + 1, 2), np.float32, 0x5A)
    s3dx.Rotary(2, [0], [0.3]).apply(R.dev(s3dx, x), s3dx.F32, n, 1, R.dev(s3dx, pos[:, None]), y)
    got = y.download()
    assert np.all(got[n].view(np.uint8) == 0x5A)
    at = np.r_[0:2000, rng.integers(0, n, 20000), 2 ** 25 - 2000: n]
    want, size = R.turn(x[at, None].astype(np.float64), pos[at, None], [0], [0.3], True)
    compare(got[at, None].astype(np.float64), want, size, TURN, R.half_step(s3dx, s3dx.F32), "rows")
