"""64-bit references of the attention operators over packed rows, in numpy, and
what the tests of them share.  Written from the definitions in the C header."""
import ctypes as C

import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative
UBF = 2.0 ** -8   # of bfloat16


def half_step(s3dx, dtype):
    return UBF if dtype == s3dx.BF16 else U32


# ---- device rows ----------------------------------------------------------
def stored(s3dx, a, dtype):
    """What the device holds of float32 `a` (bf16: its bits), and the values that it stands for."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == s3dx.F32:
        return a, a.astype(np.float64)
    bits = s3dx.workloads.f32_to_bf16_bits(a).reshape(a.shape)
    return bits, s3dx.workloads.bf16_bits_to_f32(bits).reshape(a.shape).astype(np.float64)


def values(s3dx, d, dtype):
    h = d.download()
    return (s3dx.workloads.bf16_bits_to_f32(h).reshape(h.shape) if dtype == s3dx.BF16 else h).astype(np.float64)


def dev(s3dx, a):
    return s3dx.DeviceArray.from_host(np.ascontiguousarray(a))


def filled(s3dx, shape, np_dtype, byte):
    """A device array of `byte`s: what a call must leave shows."""
    n = int(np.prod(shape, dtype=np.int64)) * np.dtype(np_dtype).itemsize
    return dev(s3dx, np.full(n, byte, np.uint8).view(np_dtype).reshape(shape))


def store_type(s3dx, dtype):
    return np.uint16 if dtype == s3dx.BF16 else np.float32


# ---- rotary ---------------------------------------------------------------
def turn(x, positions, axis, frequency, adjacent, inverse=False):
    """x [n][heads][d] turned, and the sum |a| + |b| of each channel's pair (the scale of its error)."""
    y, size = x.copy(), np.abs(x)
    for j, (a, f) in enumerate(zip(axis, frequency)):
        # whole turns out in long double: positions may be far
        angle = np.asarray(positions[:, a], np.longdouble) * np.longdouble(f)
        angle = (-angle if inverse else angle)[:, None]
        c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
        p, q = (2 * j, 2 * j + 1) if adjacent else (j, j + len(axis))
        y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
        size[..., p] = size[..., q] = np.abs(x[..., p]) + np.abs(x[..., q])
    return y, size


def rms(x, gain, eps):
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if gain is None else y * gain


# ---- selection ------------------------------------------------------------
def codes_of(x):
    most = np.abs(x).max()
    if not np.isfinite(x).all() or not most >= 2.0 ** -100:
        return np.zeros(x.shape, np.int64), 0.0
    e = int(np.frexp(most)[1]) - 1
    return np.clip(np.rint(np.ldexp(x, 6 - e)), -127, 127).astype(np.int64), float(np.ldexp(1.0, e - 6))


def index_of(k, lens, block):
    """codes [kv][rows][d], scale [kv][rows] and which rows are used."""
    kv, d = k.shape[1:]
    rows = k.shape[0] // block + len(lens)
    codes, scale, used = np.zeros((kv, rows, d), np.int64), np.zeros((kv, rows)), np.zeros(rows, bool)
    at = 0
    for s, n in enumerate(lens):
        for j in range(-(-n // block)):
            r = at // block + s + j
            used[r] = True
            for h in range(kv):
                codes[h, r], scale[h, r] = codes_of(k[at + j * block: at + min(n, (j + 1) * block), h].mean(0))
        at += n
    return codes, scale, used


def select(q, codes, scale, ql, kl, block, top, causal, near):
    n, heads, _ = q.shape
    kv = codes.shape[0]
    out = np.full((n, kv, top), -1, np.int64)
    q0 = k0 = 0
    for s, (lq, lk) in enumerate(zip(ql, kl)):
        base, nb = k0 // block + s, -(-lk // block)
        for i in range(lq):
            place = i + lk - lq
            seen = [b for b in range(nb) if not causal or b * block <= place]
            for h in range(kv):
                g = heads // kv
                qc, _ = codes_of(q[q0 + i, h * g: (h + 1) * g].sum(0))
                score = [float(qc @ codes[h, base + b]) * scale[h, base + b] for b in seen]
                if near and place >= 0:
                    score = [np.inf if b == place // block else v for b, v in zip(seen, score)]
                best = sorted(sorted(range(len(seen)), key=lambda t: (-score[t], t))[:top])
                out[q0 + i, h, : len(best)] = [seen[t] for t in best]
        q0, k0 = q0 + lq, k0 + lk
    return out


# ---- attention ------------------------------------------------------------
def attend(q, k, v, ql, kl, block, selected, scale, causal, bf16):
    """o, lse, and how far a right kernel's may be off, element by element.

    With u = 2^-24: a score is off by at most (d + 4) u scale sum|q k| (d products and sums, the scale), and an
    exponential by that, its argument's rounding (|score| u, twice) and 4 u of its own: `w`, relative to each weight.
    Numerator and denominator are both off by at most w and one u for each of their sums, the numerator by 2^-8 more where
    its weights are rounded to bfloat16 (and as much again where the denominator's were); lse is in 32 bits throughout.
    The output's own rounding is the caller's."""
    n, heads, d = q.shape
    g = heads // k.shape[1]
    o, lse = np.zeros((n, heads, d)), np.full((n, heads), -np.inf)
    off, lse_off = np.zeros((n, heads, d)), np.zeros((n, heads))
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        for i in range(lq):
            for h in range(heads):
                keys = np.arange(lk)
                if selected is not None:
                    mine = sorted({int(b) for b in selected[q0 + i, h // g] if 0 <= b < -(-lk // block)})
                    keys = np.concatenate([np.arange(b * block, min(lk, (b + 1) * block)) for b in mine] or [np.zeros(0, int)])
                if causal:
                    keys = keys[keys <= i + lk - lq]
                if keys.size == 0:
                    continue
                kk, vv = k[k0 + keys, h // g], v[k0 + keys, h // g]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (kk @ q[q0 + i, h])
                    m = s.max()
                    if m == -np.inf:
                        continue
                    p = np.exp(s - m)
                    total = p.sum()
                    o[q0 + i, h] = p @ vv / total
                    lse[q0 + i, h] = m + np.log(total)
                    fine = np.isfinite(s)
                    w = U32 * ((d + 4) * scale * (np.abs(kk) @ np.abs(q[q0 + i, h]))[fine].max(initial=0) + 4
                               + 2 * np.abs(s[fine]).max(initial=0))
                    most = 2 * w + 2 * U32 * (keys.size + 8) + (2 * UBF if bf16 else 0.0)
                    off[q0 + i, h] = most * (p @ np.abs(vv)) / total
                    lse_off[q0 + i, h] = w + U32 * (keys.size + 8 + abs(lse[q0 + i, h]))
        q0, k0 = q0 + lq, k0 + lk
    return o, lse, off, lse_off


# ---- graphs ---------------------------------------------------------------
class Graph:
    """What `body` enqueues on `stream`, captured; launch() replays it there."""

    def __init__(self, s3dx, stream, body):
        with open("/proc/self/maps") as f:  # the runtime that the library is linked to
            self.hip = C.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
        self.stream = C.c_void_p(stream.handle)
        self.graph, self.exec = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0
        try:
            body()
        finally:
            ended = self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph))
        assert ended == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exec)
        self.hip.hipGraphDestroy(self.graph)
