"""64-bit references of the cache in 8 bits, the attention over it and the gated
norms, in numpy, and what the tests of them share.  Written from the
definitions in the C header."""
import numpy as np

import attention_ref as R

NONE, LAYER, RMS = 0, 1, 2


def rows(rng, n, h, d, spread=0.7):
    """Normal rows whose heads and channels are of unlike sizes."""
    return (rng.standard_normal((n, h, d)) * np.exp(spread * rng.standard_normal((1, h, d)))).astype(np.float32)


def starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def step_of(most):
    return np.where(most >= 2.0 ** -100, np.ldexp(1.0, np.frexp(np.where(most > 0, most, 1.0))[1] - 7), 0.0)


class Held:
    """What a cache holds: codes [2][pages][kv][block][d] (keys, values; signed) and steps [pages][kv][2]."""

    def __init__(self, pages, kv, d, block):
        self.pages, self.kv, self.d, self.block = pages, kv, d, block
        self.codes = np.zeros((2, pages, kv, block, d), np.int64)
        self.steps = np.zeros((pages, kv, 2))

    def size(self):
        return self.pages * self.kv * (2 * self.block * self.d + 8)

    def write(self, k, v, new, lens, table):
        """Rows in 64 bits, by the definition; new and lens by sequence."""
        b, at = self.block, 0
        for s, (n, m) in enumerate(zip(new, lens)):
            m = max(0, min(int(m), table.shape[1] * b))
            first = m - n
            for j in range(first // b, -(-m // b)) if n else ():
                lo, hi = max(first, j * b), min(m, (j + 1) * b)
                page = int(table[s, j]) if 0 <= j < table.shape[1] else -1
                if not 0 <= page < self.pages or hi <= lo:
                    continue
                for w, x in enumerate((k, v)):
                    x = x[at + lo - first: at + hi - first]
                    big = np.where(np.isfinite(x), np.abs(x), 0.0).max((0, 2))
                    step = step_of(big)
                    if lo > j * b:
                        old = self.steps[page, :, w].copy()
                        grown = step > old
                        step = np.where(grown, step, old)
                        ratio = np.where(grown, old / np.where(step > 0, step, 1.0), 1.0)
                        self.codes[w, page] = np.rint(self.codes[w, page] * ratio[:, None, None])
                    self.steps[page, :, w] = step
                    with np.errstate(invalid="ignore"):
                        c = np.clip(np.rint(x / np.where(step > 0, step, np.inf)[:, None]), -127, 127)
                    c = np.where(step[:, None] > 0, c, 0.0)
                    self.codes[w, page, :, lo - j * b: hi - j * b] = np.where(np.isnan(x), 0.0, c).transpose(1, 0, 2)
            at += n

    def values(self, s, m, table):
        """Keys and values [m][kv][d] of sequence s, and which of them the cache holds."""
        b = self.block
        m = max(0, min(int(m), table.shape[1] * b))
        out, there = np.zeros((2, m, self.kv, self.d)), np.zeros(m, bool)
        for j in range(-(-m // b)):
            page, hi = int(table[s, j]), min(m, (j + 1) * b)
            if not 0 <= page < self.pages:
                continue
            there[j * b: hi] = True
            for w in (0, 1):
                out[w, j * b: hi] = (self.codes[w, page, :, : hi - j * b] * self.steps[page, :, w, None, None]).transpose(1, 0, 2)
        return out[0], out[1], there

    def buffer(self, behind=0x5A):
        """The device's bytes for it."""
        kb = (self.codes[0] + 128).astype(np.uint8).reshape(self.pages, self.kv, 1, -1)
        vb = (self.codes[1] + 128).astype(np.uint8).transpose(0, 1, 3, 2).reshape(self.pages, self.kv, 1, -1)
        return np.concatenate([np.concatenate([kb, vb], 2).reshape(-1), self.steps.astype(np.float32).view(np.uint8).reshape(-1)])

    def take(self, buffer):
        """Codes and steps as a device buffer has them."""
        n = self.pages * self.kv * 2 * self.block * self.d
        c = buffer[:n].reshape(self.pages, self.kv, 2, -1).astype(np.int64) - 128
        k = c[:, :, 0].reshape(self.pages, self.kv, self.block, self.d)
        v = c[:, :, 1].reshape(self.pages, self.kv, self.d, self.block).transpose(0, 1, 3, 2)
        return np.stack([k, v]), buffer[n:].view(np.float32).reshape(self.pages, self.kv, 2).astype(np.float64)


def filled(rng, kv, d, block, lens, room=1, spread=0.7):
    """A cache with rows of every sequence, and its table: pages in no order, some of them nobody's."""
    width = max(1, -(-max(lens) // block) + room)
    held = Held(width * len(lens) + 3, kv, d, block)
    table = rng.permutation(held.pages)[: width * len(lens)].reshape(len(lens), width).astype(np.int32)
    held.write(rows(rng, sum(lens), kv, d, spread).astype(np.float64), rows(rng, sum(lens), kv, d, spread).astype(np.float64), lens, lens, table)
    return held, table


def visible(i, n, m, causal, window, sinks):
    """Which of m keys row i of n sees."""
    key, place = np.arange(m), i + m - n
    see = key <= place if causal else np.ones(m, bool)
    return see & ((key > place - window) | (key < sinks)) if window else see


def attend(q, held, table, new, lens, scale, causal, window, sinks, bf16):
    """o, lse, and how far a right kernel's may be off, element by element.

    With u = 2^-24: a score is off by at most (d + 6) u scale sum|q k| (d products and sums, three factors), for float32
    queries by their 22 bits as well (2^-22 of each product); an exponential by that, its argument's rounding (|score| u, three
    times: base, difference, its second part) and 4 u of its own: `w`, relative to each weight.  Numerator and
    denominator are both off by at most w and one u for each of their sums; the numerator by 2^-11 of each weight more (float32
    queries: 2^-22), and by 2^-25 of a weight's unit, of which the row's largest has 2^7 at least.  lse is in 32 bits throughout.
    The output's own rounding is the caller's."""
    n_all, heads, d = q.shape
    g = heads // held.kv
    o, lse = np.zeros((n_all, heads, d)), np.full((n_all, heads), -np.inf)
    off, lse_off = np.zeros((n_all, heads, d)), np.zeros((n_all, heads))
    u = R.U32
    at = 0
    for s, (n, m) in enumerate(zip(new, lens)):
        k, v, there = held.values(s, m, table)
        m = len(there)
        see = np.array([visible(i, n, m, causal, window, sinks) & there for i in range(n)]).reshape(n, m)
        for h in range(heads if n and m else 0):
            kk, vv, qq = k[:, h // g], v[:, h // g], q[at: at + n, h]
            with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                sc = np.where(see, scale * (qq @ kk.T), -np.inf)
                top = sc.max(1, initial=-np.inf)
                p = np.where(see, np.exp(sc - np.where(top == -np.inf, 0.0, top)[:, None]), 0.0)
                total, count = p.sum(1), see.sum(1)
                some = total != 0
                y = p @ vv / np.where(some, total, 1.0)[:, None]
                o[at: at + n, h] = np.where(some[:, None], y, 0.0)
                lse[at: at + n, h] = np.where(some, top + np.log(np.where(some, total, 1.0)), -np.inf)
                size = scale * (np.abs(qq) @ np.abs(kk).T)
                size = np.where(see, size, 0.0).max(1)
                w = size * ((d + 6) * u + (0.0 if bf16 else 2.0 ** -22)) + 3 * u * np.where(see, np.abs(sc), 0.0).max(1) + 4 * u
                most = 2 * w + 2 * u * (count + 10) + (2.0 ** -11 if bf16 else 2.0 ** -22)
                big = (see[:, :, None] * np.abs(vv)[None]).max(1) if n * m * d < 3e7 else np.abs(vv).max(0)[None]
                off[at: at + n, h] = most[:, None] * (p @ np.abs(vv)) / np.where(some, total, 1.0)[:, None] + (count * 2.0 ** -32)[:, None] * big
                lse_off[at: at + n, h] = w + u * (count + 10 + np.abs(np.where(some, lse[at: at + n, h], 0.0)))
        at += n
    return o, lse, off, lse_off


def check(s3dx, dtype, got, lse, want, what=""):
    """As the definition says within its bounds; the same places NaN and infinite."""
    o, l, off, l_off = want
    fine = np.isfinite(o)
    assert np.array_equal(np.isnan(got), np.isnan(o)) and np.array_equal(got[~fine & ~np.isnan(o)], o[~fine & ~np.isnan(o)]), what
    err = np.abs(got - o)[fine]
    bound = (off + R.half_step(s3dx, dtype) * (np.abs(o) + off))[fine]
    rel = float(np.linalg.norm(err) / max(np.linalg.norm(o[fine]), 1e-300))
    print(f"  {what} worst share of the bound {np.max(err / np.maximum(bound, 1e-300), initial=0):.3f}, rel-L2 {rel:.2e}", flush=True)
    assert np.all(err <= bound), what
    # Over many elements the errors do not all reach their bounds: a rounding is off by its half step / sqrt(3) in the mean square at
    # most, the output's to bfloat16 (2^-8) and the weights' (2^-11).  A key left out of a few hundred shows.
    if dtype == s3dx.BF16 and err.size > 2000:
        assert rel <= (R.UBF + 2.0 ** -11) / np.sqrt(3) * 1.5, (what, rel)
    fine = np.isfinite(l)
    with np.errstate(invalid="ignore"):
        assert np.array_equal(lse[~fine & ~np.isnan(l)], l[~fine & ~np.isnan(l)]) and np.array_equal(np.isnan(lse), np.isnan(l)), what
        assert np.all(np.abs(lse - l)[fine] <= l_off[fine] + R.U32 * np.abs(l[fine])), what


# ---- gated norms ------------------------------------------------------------
def normed(x, kind, w, b, eps):
    """A norm of rows, and a bound on a float32 kernel's error, relative to its channels before w and b (see gated)."""
    if kind == NONE:
        return x, np.zeros_like(x)
    c = x.shape[1]
    mean = x.mean(1, keepdims=True) if kind == LAYER else np.zeros((len(x), 1))
    var = ((x - mean) ** 2).mean(1, keepdims=True) + eps
    y = (x - mean) / np.sqrt(var)
    # The mean of c terms is off by c u of their mean size (summed in trees: far less), a difference by that and its own rounding;
    # the root of c squares by (c + 8) u / 2 of it, and by the differences' errors.
    u = R.U32
    dm = (c * u * np.abs(x).mean(1, keepdims=True) if kind == LAYER else 0.0) + u * (np.abs(x) + np.abs(mean))
    dv = np.sqrt((dm ** 2).mean(1, keepdims=True)) / np.sqrt(var)
    off = dm / np.sqrt(var) + np.abs(y) * (dv + (c + 12) * u)
    if w is not None:
        y, off = y * w, off * np.abs(w) + u * np.abs(y * w)
    if b is not None:
        y, off = y + b, off + u * np.abs(y + b)
    return y, off


def gated(x, branch, post, post_w, post_b, rs, gate, pre, pre_w, pre_b, scale, shift, eps):
    """y, h and bounds on their errors before the outputs' rounding; gate, scale, shift by row or None."""
    u = R.U32
    z, off = normed(branch, post, post_w, post_b, eps)
    if gate is not None:
        z, off = z * gate, off * np.abs(gate) + u * np.abs(z * gate)
    y = x + rs * z
    y_off = off * abs(rs) + 2 * u * (np.abs(rs * z) + np.abs(y))
    h, h_off = normed(y, pre, pre_w, pre_b, eps)
    if pre != NONE:
        # y's error goes through the norm: its own channel's, the mean's and the root's
        c = y.shape[1]
        mean = y.mean(1, keepdims=True) if pre == LAYER else 0.0
        sd = np.sqrt(((y - mean) ** 2).mean(1, keepdims=True) + eps)
        most = y_off + y_off.mean(1, keepdims=True)
        through = most / sd + np.abs((y - mean) / sd) * np.sqrt((most ** 2).mean(1, keepdims=True)) / sd
        h_off = h_off + through * (1.0 if pre_w is None else np.abs(pre_w))
    else:
        h_off = y_off.copy()
    if scale is not None:
        h, h_off = h * (1 + scale), h_off * np.abs(1 + scale) + 2 * u * np.abs(h) * (1 + np.abs(scale))
    if shift is not None:
        h, h_off = h + shift, h_off + 2 * u * np.abs(h + shift)
    return y, y_off, h, h_off
