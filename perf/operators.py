"""The attention operators over voxel rows, as cases that can be timed.

Between the sparse blocks that this library runs, the flow model attends over the same rows: heads of queries and keys
are normed and turned by the voxels' (x, y, z) ("qk"; "rotary" is the turn alone), each query picks blocks of keys by a
cheap score ("select"), and attends to those, or to all keys of its sequence ("attend").

Where `own` is false run() computes each in its plain form by elementary torch operations; where it is true it makes
the library's calls. exact() is the same from the definition in 64 bits.

Features are rows of a smooth function of the row's place plus noise, normed per head, so that neighbours look alike
as they do in a model; voxel sets are unions of spherical shells on a 64^3 grid in lexicographic order.
"""
import functools
import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

EPS = 1e-6
BASE = 10000.0
RES = 64


def _lib():
    """The package: a folder whose name holds a dot, imported as `s3dx`."""
    if "s3dx" not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "sam3d.cpp_amd"
        spec = importlib.util.spec_from_file_location("s3dx", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["s3dx"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["s3dx"]


def listed():
    return [
        # the smallest call: one row of the decoder's 12 heads
        {"name": "rotary f32 1 row", "kind": "rotary", "n": 1, "heads": 12, "d": 64, "sections": "10,10,10",
         "pairing": "adjacent", "span": 64, "inverse": False, "dtype": "f32"},
        # the keys of the largest usual voxel set of the flow model, 16 heads x 64
        {"name": "rotary bf16 28k", "kind": "rotary", "n": 28265, "heads": 16, "d": 64, "sections": "10,10,10",
         "pairing": "adjacent", "span": 64, "inverse": False, "dtype": "bf16"},
        # queries and keys of one flow block on the coarse set, out of the packed qkv projection
        {"name": "qk bf16 5k 16x64", "kind": "qk", "n": 5086, "heads": 16, "kv": 16, "d": 64, "sections": "10,10,10",
         "pairing": "adjacent", "span": 64, "gain": "head", "dtype": "bf16"},
        # shared key heads, wide heads, far positions on one long axis and two short ones: the most rows the pipeline keeps
        {"name": "qk bf16 42k 16/4x128", "kind": "qk", "n": 42000, "heads": 16, "kv": 4, "d": 128, "sections": "24,20,20",
         "pairing": "halves", "span": 100000, "gain": "all", "dtype": "bf16"},
        # once per flow block: the index of the coarse set's keys, and each query's blocks
        {"name": "select bf16 5k 16x64", "kind": "select", "layout": "whole", "n": 5086, "keys": 5086, "seqs": 1,
         "heads": 16, "kv": 16, "d": 64, "block": 64, "top": 16, "index": True, "causal": False, "near": True, "dtype": "bf16"},
        # one new row for each of 8 sequences, over an index that is kept
        {"name": "select bf16 8 rows of 65k", "kind": "select", "layout": "single", "n": 8, "keys": 8 * 65536, "seqs": 8,
         "heads": 32, "kv": 8, "d": 128, "block": 64, "top": 32, "index": False, "causal": True, "near": True, "dtype": "bf16"},
        # a flow block's attention over the chosen blocks ...
        {"name": "attend bf16 5k top 16", "kind": "attend", "layout": "whole", "n": 5086, "keys": 5086, "seqs": 1,
         "heads": 16, "kv": 16, "d": 64, "block": 64, "top": 16, "causal": False, "dtype": "bf16"},
        # ... over all keys, as the reference's flow model has it ...
        {"name": "attend bf16 5k all", "kind": "attend", "layout": "whole", "n": 5086, "keys": 5086, "seqs": 1,
         "heads": 16, "kv": 16, "d": 64, "block": 64, "top": 0, "causal": False, "dtype": "bf16"},
        # ... and in the reference's own precision
        {"name": "attend f32 5k all", "kind": "attend", "layout": "whole", "n": 5086, "keys": 5086, "seqs": 1,
         "heads": 16, "kv": 16, "d": 64, "block": 64, "top": 0, "causal": False, "dtype": "f32"},
        # the decoder: windows of 8^3 voxels, each a short sequence of its own
        {"name": "attend bf16 10k windows", "kind": "attend", "layout": "windows", "n": 10366, "keys": 10366, "seqs": 0,
         "heads": 12, "kv": 12, "d": 64, "block": 64, "top": 0, "causal": False, "dtype": "bf16"},
        # one new row for each of 8 sequences over the blocks it chose
        {"name": "attend bf16 8 rows of 65k", "kind": "attend", "layout": "single", "n": 8, "keys": 8 * 65536, "seqs": 8,
         "heads": 32, "kv": 8, "d": 128, "block": 64, "top": 32, "causal": True, "dtype": "bf16"},
        # the largest: a long causal batch of ragged sequences with shared key heads
        {"name": "attend bf16 12k ragged top 32", "kind": "attend", "layout": "ragged", "n": 12001, "keys": 12001, "seqs": 2,
         "heads": 16, "kv": 4, "d": 128, "block": 64, "top": 32, "causal": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "qk", "qk", "select", "select", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    d = rng.choice([32, 64, 64, 96, 128])
    kv, group = rng.choice([(16, 1), (12, 1), (4, 4), (8, 2), (2, 5), (1, 8)])
    c = {"kind": kind, "heads": kv * group, "kv": kv, "d": d, "dtype": dtype}
    if kind in ("rotary", "qk"):
        axes = rng.randint(1, 3)
        cut = sorted(rng.randint(1, d // 2 - 1) for _ in range(axes))
        sec = [cut[0]] + [b - a for a, b in zip(cut, cut[1:])]
        c.update(n=_log(rng, 1, 40000), sections=",".join(str(max(1, s)) for s in sec) if sum(max(1, s) for s in sec) <= d // 2 else str(d // 2),
                 pairing=rng.choice(["adjacent", "halves"]), span=rng.choice([64, 64, 4096, 1000000]))
        c.update({"inverse": rng.random() < 0.3} if kind == "rotary" else {"gain": rng.choice(["head", "all", "none"])})
        return c
    layout = rng.choice(["whole", "ragged", "single", "windows"] if kind == "attend" else ["whole", "ragged", "single"])
    c.update(layout=layout, block=rng.choice([32, 64, 64, 128]), top=rng.choice([4, 8, 16, 24, 32]), causal=rng.random() < 0.4)
    if layout == "single":
        c["seqs"] = rng.randint(1, 12)
        c["n"], c["keys"] = c["seqs"], c["seqs"] * _log(rng, 100, 30000)
    else:
        c["seqs"] = {"whole": 1, "ragged": rng.randint(2, 9), "windows": 0}[layout]
        c["n"] = c["keys"] = _log(rng, 60, 6000 if dtype == "f32" else 9000)
    if kind == "select":
        c.update(index=layout != "single" or rng.random() < 0.5, near=rng.random() < 0.7)
    elif layout == "windows":
        c.update(top=0, causal=False)
    elif rng.random() < 0.3:
        c["top"] = 0
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _dev():
    return torch.device("cuda", 0)


@functools.lru_cache(maxsize=64)
def _voxels(n, seed):
    """n rows (0, x, y, z) in lexicographic order: shells of thickness 3 with centres in [12, 52]^3, radii in [6, 14];
    a set that needs more rows than the grid's shells give goes on at the next batch number."""
    r = random.Random("voxels %d %d" % (n, seed))
    ax = np.arange(RES, dtype=np.float64)
    parts, have, b = [], 0, 0
    while have < n:
        mask = np.zeros((RES, RES, RES), bool)
        for _ in range(10):
            c = [r.uniform(12.0, 52.0) for _ in range(3)]
            d = np.sqrt((ax[:, None, None] - c[0]) ** 2 + (ax[None, :, None] - c[1]) ** 2 + (ax[None, None, :] - c[2]) ** 2)
            mask |= np.abs(d - r.uniform(6.0, 14.0)) <= 1.5
            if have + int(mask.sum()) >= n:
                break
        xyz = np.argwhere(mask).astype(np.int32)
        parts.append(np.concatenate([np.full((xyz.shape[0], 1), b, np.int32), xyz], 1))
        have, b = have + xyz.shape[0], b + 1
    return np.ascontiguousarray(np.concatenate(parts, 0)[:n])


def _gen(seed, tag):
    g = torch.Generator(device=_dev())
    g.manual_seed((seed * 1000003 + tag) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, tag, shape, std=1.0):
    return torch.randn(shape, generator=_gen(seed, tag), device=_dev(), dtype=torch.float32) * std


def _tdt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _features(seed, tag, place, heads, d, smooth):
    """[n][heads][d], of unit mean square per head: waves over the rows' places (one set of waves for every tag, as
    queries and keys of a trained layer agree), and noise of the tag's own."""
    n, axes = place.shape
    x = _normal(seed, tag, (n, heads, d), math.sqrt(1.0 - smooth * smooth))
    if smooth:
        wave = _normal(seed, 901, (axes, heads * d), 0.12)
        phase = _normal(seed, 902, (heads * d,), 3.0)
        x += torch.sin(place @ wave + phase).view(n, heads, d) * (smooth * math.sqrt(2.0))
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _pairs(case):
    """(axis, frequency) of each pair: every axis its own geometric series."""
    return [(a, BASE ** (-j / s)) for a, s in enumerate(_sections(case)) for j in range(s)]


def _positions(case, seed):
    """int32 [n][4]: (batch, x, y, z) of voxels, or where the span is longer than the grid, places up to it."""
    n = case["n"]
    if case["span"] <= RES:
        return torch.from_numpy(_voxels(n, seed % 64)).to(_dev())
    g = _gen(seed, 7)
    return torch.randint(0, case["span"], (n, 4), generator=g, device=_dev(), dtype=torch.int32)


def _cuts(n, parts, word):
    """Lengths of `parts` sequences of n rows in all; of four or more, one is empty and one has one row."""
    r = random.Random("%s %d %d" % (word, n, parts))
    fixed = [0, 1] if parts >= 4 else []
    at = sorted(r.randint(0, n - sum(fixed)) for _ in range(parts - len(fixed) - 1))
    lens = [b - a for a, b in zip([0] + at, at + [n - sum(fixed)])] + fixed
    r.shuffle(lens)
    return lens


def _window_order(n):
    """Voxels of a set of n rows in the order of their 8^3 windows, and the windows' lengths."""
    v = _voxels(n, 0)
    w = v.astype(np.int64)
    key = ((w[:, 0] * 8 + w[:, 1] // 8) * 8 + w[:, 2] // 8) * 8 + w[:, 3] // 8
    order = np.argsort(key, kind="stable")
    return v[order], np.unique(key, return_counts=True)[1].tolist()


def _lens(case):
    """(query rows, key rows) of each sequence."""
    if case["layout"] == "windows":
        lens = _window_order(case["n"])[1]
        return lens, lens
    if case["layout"] == "single":
        per = case["keys"] // case["seqs"]
        return [1] * case["seqs"], [per] * case["seqs"]
    lens = _cuts(case["n"], case["seqs"], "rows") if case["seqs"] > 1 else [case["n"]]
    return lens, lens


def _starts(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=_dev())


def _turn_inputs(case, seed):
    h, kv, d, n = case["heads"], case.get("kv", 0), case["d"], case["n"]
    t = {"positions": _positions(case, seed)}
    if case["kind"] == "rotary":
        t["x"] = _normal(seed, 1, (n, h, d)).to(_tdt(case))
        return t
    # the projection's output: query, key and value heads of a row beside one another
    t["qkv"] = (_normal(seed, 1, (n, (h + 2 * kv) * d)) * torch.exp(_normal(seed, 2, (n, 1), 0.5))).to(_tdt(case))
    t["q"], t["k"] = t["qkv"][:, : h * d].unflatten(1, (h, d)), t["qkv"][:, h * d: (h + kv) * d].unflatten(1, (kv, d))
    shape = {"head": lambda heads: (heads, d), "all": lambda heads: (d,), "none": lambda heads: None}[case["gain"]]
    for name, heads in (("gq", h), ("gk", kv)):
        t[name] = None if shape(heads) is None else _normal(seed, 3 + heads, shape(heads), 0.2) + 1.0
    return t


def _token_inputs(case, seed):
    """q, k, v [rows][heads][d], the sequences' starts and, for attention over chosen blocks, the choice."""
    h, kv, d = case["heads"], case["kv"], case["d"]
    ql, kl = _lens(case)
    if case["layout"] == "windows":
        place = torch.from_numpy(_window_order(case["n"])[0][:, 1:]).to(_dev()).float()
    elif case["layout"] == "whole":
        place = torch.from_numpy(_voxels(case["n"], seed % 64)[:, 1:]).to(_dev()).float()
    else:
        place = torch.arange(case["keys"], device=_dev(), dtype=torch.float32)[:, None] / 16.0
    t = {"ql": ql, "kl": kl, "qs": _starts(ql), "ks": _starts(kl)}
    dt = _tdt(case)
    if case["layout"] == "single":
        last = t["ks"][1:].long() - 1
        t["q"] = _features(seed, 1, place[last], h, d, 0.6).to(dt)
        t["k"] = _features(seed, 2, place, kv, d, 0.6 if case["kind"] == "select" else 0.0).to(dt)
        if case["kind"] == "attend":
            t["v"] = _normal(seed, 3, (case["keys"], kv, d)).to(dt)
    else:
        qkv = torch.empty((case["n"], h + 2 * kv, d), dtype=dt, device=_dev())
        qkv[:, :h] = _features(seed, 1, place, h, d, 0.6)
        qkv[:, h: h + kv] = _features(seed, 2, place, kv, d, 0.6)
        qkv[:, h + kv:] = _normal(seed, 3, (case["n"], kv, d))
        t["q"], t["k"], t["v"] = qkv[:, :h], qkv[:, h: h + kv], qkv[:, h + kv:]
    if case["kind"] == "attend" and case["top"]:
        t["selected"] = _choice(t, case, seed)
    return t


def _choice(t, case, seed):
    """What the selection gives for these rows (for single rows, whose keys are noise: random blocks)."""
    if case["layout"] != "single":
        codes, scale = _plain_index(t, case)
        return _plain_select(t, case, codes, scale, near=True)
    nb = -(-max(t["kl"]) // case["block"])
    s = torch.rand((case["n"], case["kv"], nb), generator=_gen(seed, 11), device=_dev())
    got = s.topk(min(case["top"], nb), dim=-1).indices.sort(-1).values.to(torch.int32)
    return torch.nn.functional.pad(got, (0, case["top"] - got.shape[-1]), value=-1).contiguous()


def _index_rows(case, t):
    return t["k"].shape[0] // case["block"] + len(t["kl"])


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def prepare(case, seed):
    st = {"case": case}
    h, d, dt = case["heads"], case["d"], _tdt(case)
    new = functools.partial(torch.zeros, device=_dev())
    if case["kind"] in ("rotary", "qk"):
        st.update(_turn_inputs(case, seed))
        st["axis"] = torch.tensor([a for a, _ in _pairs(case)], device=_dev())
        st["freq"] = torch.tensor([f for _, f in _pairs(case)], device=_dev(), dtype=torch.float64)
        st["yq"] = new((case["n"], h, d), dtype=dt)
        if case["kind"] == "qk":
            st["yk"] = new((case["n"], case["kv"], d), dtype=dt)
        if own:
            s3dx = _lib()
            st["rotary"] = s3dx.Rotary(d, [a for a, _ in _pairs(case)], [f for _, f in _pairs(case)],
                                       axes=len(_sections(case)),
                                       pairing=s3dx.ROTARY_ADJACENT if case["pairing"] == "adjacent" else s3dx.ROTARY_HALVES)
    else:
        st.update(_token_inputs(case, seed))
        st["rows_q"], st["rows_k"] = max(st["ql"]), max(st["kl"])
        if case["kind"] == "select":
            st["codes"] = new((case["kv"], _index_rows(case, st), d), dtype=torch.int8)
            st["scale"] = new((case["kv"], _index_rows(case, st)), dtype=torch.float32)
            if not case["index"]:
                st["codes"], st["scale"] = _plain_index(st, case)
            st["selected"] = new((case["n"], case["kv"], case["top"]), dtype=torch.int32)
        else:
            st["o"] = new((case["n"], h, d), dtype=dt)
            st["lse"] = new((case["n"], h), dtype=torch.float32)
            if own:
                s3dx = _lib()
                st["ws"] = torch.empty(max(1, s3dx.block_attention_workspace_size(
                    case["n"], h, case["kv"], d, len(st["ql"]), case["block"], case["top"], st["rows_k"])),
                    dtype=torch.uint8, device=_dev())
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------
# run: the plain forms
# ---------------------------------------------------------------------------
def _plain_turn(x, st, inverse=False):
    """x float32 [n][heads][d]."""
    p = st["axis"].shape[0]
    pos = st["positions"][:, 1:] if len(_sections(st["case"])) == 3 else st["positions"]
    angle = pos[:, st["axis"]].double() * st["freq"]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    sin = -sin if inverse else sin
    if st["case"]["pairing"] == "adjacent":
        a, b = x[..., 0: 2 * p: 2], x[..., 1: 2 * p: 2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p: 2 * p]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * p:]], -1)


def _plain_norm(x, gain):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if gain is None else y * gain


def _padded(x, starts, lens):
    """(rows by sequence [S][L][...], their validity [S][L]) of packed rows."""
    most = max(lens)
    at = torch.arange(most, device=x.device)
    real = at < torch.diff(starts)[:, None]
    row = (starts[:-1, None] + at).clamp(max=x.shape[0] - 1)
    return x[row.long()], real


def _two_to(e):
    """2^e for whole e, exactly, in 64 bits."""
    return ((e + 1023) << 52).view(torch.float64)


def _codes(x):
    """8-bit codes of the last axis of 64-bit x at a power of two that brings the largest to [64, 128), and the power."""
    most = x.abs().amax(-1, keepdim=True)
    fine = (most >= 2.0 ** -100) & torch.isfinite(most)
    e = torch.where(fine, (most.view(torch.int64) >> 52) - 1023, 0)
    codes = torch.where(fine, torch.round(x * _two_to(6 - e)).clamp(-127, 127), 0.0)
    return codes, torch.where(fine, _two_to(e - 6), 0.0)[..., 0]


def _plain_index(st, case):
    """Codes int8 [kv][index rows][d] and scale float32 [kv][index rows] of each block's mean key."""
    b = case["block"]
    k, real = _padded(st["k"], st["ks"], st["kl"])
    s, most = real.shape
    nb = -(-most // b)
    k = torch.nn.functional.pad(k.double() * real[..., None, None], (0, 0, 0, 0, 0, nb * b - most))
    count = torch.nn.functional.pad(real, (0, nb * b - most)).view(s, nb, b).sum(-1)
    mean = k.view(s, nb, b, case["kv"], case["d"]).sum(2) / count.clamp(min=1)[..., None, None]
    c, p = _codes(mean)
    row = (st["ks"][:-1].long() // b + torch.arange(s, device=k.device))[:, None] + torch.arange(nb, device=k.device)
    used = count > 0
    codes = torch.zeros((case["kv"], _index_rows(case, st), case["d"]), dtype=torch.int8, device=k.device)
    scale = torch.zeros(codes.shape[:2], dtype=torch.float32, device=k.device)
    codes[:, row[used]] = c[used].to(torch.int8).transpose(0, 1)
    scale[:, row[used]] = p[used].float().transpose(0, 1)
    return codes, scale


def _plain_select(st, case, codes, scale, near):
    b, kv, top = case["block"], case["kv"], case["top"]
    g = case["heads"] // kv
    q, real = _padded(st["q"], st["qs"], st["ql"])
    s, lq = real.shape
    qc = _codes(q.unflatten(2, (kv, g)).double().sum(3))[0].float()      # [S][Lq][kv][d]
    nb = -(-max(st["kl"]) // b)
    block = torch.arange(nb, device=q.device)
    row = (st["ks"][:-1].long() // b + torch.arange(s, device=q.device))[:, None] + block
    row = row.clamp(max=codes.shape[1] - 1)
    dots = torch.matmul(qc.transpose(1, 2).contiguous(), codes[:, row].float().permute(1, 0, 3, 2).contiguous())
    score = dots * scale[:, row].transpose(0, 1)[:, :, None, :]          # [S][kv][Lq][nb]
    lk = torch.diff(st["ks"]).long()[:, None, None, None]
    place = (torch.arange(lq, device=q.device)[:, None] + lk - torch.diff(st["qs"]).long()[:, None, None, None])
    may = block * b < lk
    if case["causal"]:
        may = may & (block * b <= place)
    if near:
        score = torch.where((block == place.div(b, rounding_mode="floor")) & (place >= 0), math.inf, score)
    score = torch.where(may, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True)
    best = torch.where(order.values == -math.inf, nb, order.indices)[..., :top].sort(-1).values
    best = torch.where(best == nb, -1, best).to(torch.int32).permute(0, 2, 1, 3)
    best = torch.nn.functional.pad(best, (0, top - best.shape[-1]), value=-1)
    return best[real].contiguous()                                       # rows in order: [n][kv][top]


def _plain_attend(st, case):
    kv, d, g = case["kv"], case["d"], case["heads"] // case["kv"]
    q, real = _padded(st["q"], st["qs"], st["ql"])
    k, kreal = _padded(st["k"], st["ks"], st["kl"])
    v, _ = _padded(st["v"], st["ks"], st["kl"])
    s, lq = real.shape
    lk = kreal.shape[1]
    rows = q.float().unflatten(2, (kv, g)).permute(0, 2, 3, 1, 4).reshape(s, kv, g * lq, d)
    score = torch.matmul(rows, k.float().permute(0, 2, 3, 1).contiguous()).mul_(d ** -0.5).view(s, kv, g, lq, lk)
    may = kreal[:, None, None, :]
    if case["causal"]:
        place = torch.arange(lq, device=q.device)[:, None] + (torch.diff(st["ks"]) - torch.diff(st["qs"]))[:, None, None, None]
        may = may & (torch.arange(lk, device=q.device) <= place)
    if case["top"]:
        chosen = torch.full((s, lq, kv, case["top"]), -1, dtype=torch.int64, device=q.device)
        chosen[real] = st["selected"].long()
        nb = -(-lk // case["block"])
        hit = torch.zeros((s, lq, kv, nb + 1), dtype=torch.bool, device=q.device)
        hit.scatter_(3, torch.where(chosen < 0, nb, chosen), True)
        at = torch.arange(lk, device=q.device) // case["block"]
        may = may & hit[..., at].transpose(1, 2)
    score.masked_fill_(~may[:, :, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = score.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(s, kv, g * lq, lk), v.float().transpose(1, 2).contiguous()).view(s, kv, g, lq, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(s, lq, kv * g, d)
    lse = (m + total.log())[..., 0].permute(0, 3, 1, 2).reshape(s, lq, kv * g)
    return o[real].to(q.dtype), lse[real]


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    if case["kind"] == "rotary":
        return {"y": _plain_turn(st["x"].float(), st, case["inverse"]).to(st["x"].dtype)}
    if case["kind"] == "qk":
        return {"q": _plain_turn(_plain_norm(st["q"], st["gq"]), st).to(st["q"].dtype),
                "k": _plain_turn(_plain_norm(st["k"], st["gk"]), st).to(st["k"].dtype)}
    if case["kind"] == "select":
        codes, scale = _plain_index(st, case) if case["index"] else (st["codes"], st["scale"])
        got = {"selected": _plain_select(st, case, codes, scale, case["near"])}
        return {**got, "index": codes * scale[..., None]} if case["index"] else got
    o, lse = _plain_attend(st, case)
    return {"o": o, "lse": lse}


# ---------------------------------------------------------------------------
# run: the library's calls
# ---------------------------------------------------------------------------
def _run_own(st):
    s3dx, case = _lib(), st["case"]
    n, h, d = case["n"], case["heads"], case["d"]
    dt = s3dx.BF16 if case["dtype"] == "bf16" else s3dx.F32
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] in ("rotary", "qk"):
        pos = st["positions"].data_ptr() + (4 if len(_sections(case)) == 3 else 0)
        if case["kind"] == "rotary":
            st["rotary"].apply(st["x"].data_ptr(), dt, n, h, pos, st["yq"].data_ptr(), position_stride=4,
                               inverse=case["inverse"], stream=stream)
            return {"y": st["yq"]}
        s3dx.qk_norm_rotary(st["q"].data_ptr(), st["k"].data_ptr(), dt, n, h, case["kv"], d, EPS,
                            st["yq"].data_ptr(), st["yk"].data_ptr(), rotary=st["rotary"], positions=pos,
                            position_stride=4, q_gain=None if st["gq"] is None else st["gq"].data_ptr(),
                            k_gain=None if st["gk"] is None else st["gk"].data_ptr(), gain_per_head=case["gain"] == "head",
                            q_stride=st["q"].stride(0), k_stride=st["k"].stride(0), stream=stream)
        return {"q": st["yq"], "k": st["yk"]}
    qs, ks, seqs = st["qs"].data_ptr(), st["ks"].data_ptr(), len(st["ql"])
    if case["kind"] == "select":
        if case["index"]:
            s3dx.block_index(st["k"].data_ptr(), dt, st["k"].shape[0], case["kv"], d, ks, seqs, case["block"],
                             st["codes"].data_ptr(), st["scale"].data_ptr(), k_stride=st["k"].stride(0), stream=stream)
        s3dx.block_select(st["q"].data_ptr(), dt, n, st["k"].shape[0], h, case["kv"], d, qs, ks, seqs, case["block"],
                          case["top"], st["rows_k"], st["codes"].data_ptr(), st["scale"].data_ptr(), st["selected"].data_ptr(),
                          q_stride=st["q"].stride(0), causal=case["causal"], near=case["near"], stream=stream)
        got = {"selected": st["selected"]}
        return {**got, "index": st["codes"] * st["scale"][..., None]} if case["index"] else got
    s3dx.block_attention(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), dt, n, st["k"].shape[0], h, case["kv"], d,
                         qs, ks, seqs, case["block"], st["rows_k"], st["o"].data_ptr(), lse=st["lse"].data_ptr(),
                         selected=st["selected"].data_ptr() if case["top"] else None, top=case["top"],
                         q_stride=st["q"].stride(0), k_stride=st["k"].stride(0), v_stride=st["v"].stride(0),
                         causal=case["causal"], workspace=st["ws"].data_ptr(), workspace_bytes=st["ws"].numel(), stream=stream)
    return {"o": st["o"], "lse": st["lse"]}


# ---------------------------------------------------------------------------
# work, exact
# ---------------------------------------------------------------------------
def _seen(case):
    """Pairs of a query row and a key row, in all, that a head computes: chosen blocks are whole ones."""
    pairs = 0
    for lq, lk in zip(*_lens(case)):
        most = case["top"] * case["block"] if case["top"] else lk
        if not case["causal"]:
            pairs += lq * min(lk, most)
            continue
        i = np.arange(lq, dtype=np.int64) + lk - lq + 1
        pairs += int(np.clip(i, 0, min(most, lk)).sum())
    return pairs


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    n, h, d = case["n"], case["heads"], case["d"]
    if case["kind"] in ("rotary", "qk"):
        heads = h + (case["kv"] if case["kind"] == "qk" else 0)
        return {"bytes": n * (2 * heads * d * e + 4 * len(_sections(case))), "flops": n * heads * d * (3 if case["kind"] == "rotary" else 7)}
    kv = case["kv"]
    ql, kl = _lens(case)
    blocks = sum(-(-k // case["block"]) for k in kl)
    if case["kind"] == "select":
        dots = sum(q * -(-k // case["block"]) for q, k in zip(ql, kl)) * kv
        keys = case["keys"] * kv * d * e + blocks * kv * (d + 4) if case["index"] else 0
        return {"bytes": keys + blocks * kv * (d + 4) + n * h * d * e + n * kv * case["top"] * 4,
                "flops": dots * 2 * d + (case["keys"] * kv * d if case["index"] else 0)}
    pairs = _seen(case)
    keys = min(case["keys"], pairs) if case["layout"] == "single" else case["keys"]
    return {"bytes": 2 * n * h * d * e + 2 * keys * kv * d * e + n * h * 4 + (n * kv * case["top"] * 4),
            "flops": 4 * d * h * pairs}


def _exact_turn(x, t, case, sign):
    """The pairs as complex numbers, times e^(i angle)."""
    pairs = _pairs(case)
    p = len(pairs)
    pos = t["positions"][:, 1:] if len(_sections(case)) == 3 else t["positions"]
    angle = torch.stack([pos[:, a].double() * f for a, f in pairs], 1)
    first = [2 * j for j in range(p)] if case["pairing"] == "adjacent" else list(range(p))
    second = [j + 1 for j in first] if case["pairing"] == "adjacent" else [j + p for j in first]
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), sign * angle)[:, None, :]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_codes(row):
    """A 64-bit matrix' rows as 8-bit codes and powers, by numpy."""
    most = np.abs(row).max(-1)
    with np.errstate(invalid="ignore"):
        fine = np.isfinite(most) & (most >= 2.0 ** -100)
    e = np.frexp(np.where(fine, most, 1.0))[1] - 1
    c = np.clip(np.rint(np.ldexp(np.where(fine[..., None], row, 0.0), (6 - e)[..., None])), -127, 127)
    return c, np.where(fine, np.ldexp(1.0, e - 6), 0.0)


def _exact_select(t, case):
    b, kv, g, top = case["block"], case["kv"], case["heads"] // case["kv"], case["top"]
    k, q = t["k"].double().cpu().numpy(), t["q"].double().cpu().numpy()
    rows = _index_rows(case, t)
    index, powers = np.zeros((kv, rows, case["d"])), np.zeros((kv, rows))
    picked = np.full((case["n"], kv, top), -1, np.int64)
    q0 = k0 = 0
    for s, (lq, lk) in enumerate(zip(t["ql"], t["kl"])):
        nb, base = -(-lk // b), k0 // b + s
        for j in range(nb):
            mean = k[k0 + j * b: k0 + min(lk, (j + 1) * b)].mean(0)
            index[:, base + j], powers[:, base + j] = _exact_codes(mean)
        if lq and nb:
            qc = _exact_codes(q[q0: q0 + lq].reshape(lq, kv, g, -1).sum(2))[0]
            place = np.arange(lq) + lk - lq
            for a in range(kv):
                score = qc[:, a] @ index[a, base: base + nb].T * powers[a, base: base + nb]
                if case["near"]:
                    mine = np.nonzero(place >= 0)[0]
                    score[mine, place[mine] // b] = np.inf
                if case["causal"]:
                    score[np.arange(nb)[None, :] * b > place[:, None]] = -np.inf
                best = np.argsort(-score, axis=1, kind="stable")[:, :top]
                none = np.take_along_axis(score, best, 1) == -np.inf
                best = np.sort(np.where(none, nb, best), 1)
                picked[q0: q0 + lq, a, : best.shape[1]] = np.where(best == nb, -1, best)
        q0, k0 = q0 + lq, k0 + lk
    got = {"selected": torch.from_numpy(picked).to(torch.int32)}
    return {**got, "index": torch.from_numpy(index * powers[..., None])} if case["index"] else got


def _exact_attend(t, case):
    g, b, d = case["heads"] // case["kv"], case["block"], case["d"]
    o = torch.zeros((case["n"], case["heads"], d), dtype=torch.float64, device=_dev())
    lse = torch.full((case["n"], case["heads"]), -math.inf, dtype=torch.float64, device=_dev())
    q0 = k0 = 0
    for lq, lk in zip(t["ql"], t["kl"]):
        for a in range(case["kv"]) if lq and lk else ():
            see = torch.ones((lq, lk), dtype=torch.bool, device=_dev())
            if case["causal"]:
                see = see.tril(lk - lq)
            if case["top"]:
                mine = t["selected"][q0: q0 + lq, a].long()
                hit = torch.zeros((lq, -(-lk // b)), dtype=torch.bool, device=_dev())
                hit[torch.arange(lq, device=_dev())[:, None].expand_as(mine)[mine >= 0], mine[mine >= 0]] = True
                see &= hit.repeat_interleave(b, 1)[:, :lk]
            kk, vv = t["k"][k0: k0 + lk, a].double(), t["v"][k0: k0 + lk, a].double()
            for e in range(a * g, (a + 1) * g):
                s = (t["q"][q0: q0 + lq, e].double() @ kk.T / math.sqrt(d)).masked_fill(~see, -math.inf)
                lse[q0: q0 + lq, e] = torch.logsumexp(s, 1)
                o[q0: q0 + lq, e] = torch.softmax(s, 1).nan_to_num(0.0) @ vv
        q0, k0 = q0 + lq, k0 + lk
    return {"o": o, "lse": lse}


def exact(case, seed):
    if case["kind"] in ("rotary", "qk"):
        t = _turn_inputs(case, seed)
        if case["kind"] == "rotary":
            return {"y": _exact_turn(t["x"].double(), t, case, -1.0 if case["inverse"] else 1.0)}
        got = {}
        for name, gain in (("q", "gq"), ("k", "gk")):
            x = t[name].double()
            y = x / (x.square().sum(-1, keepdim=True) / case["d"] + EPS).sqrt()
            got[name] = _exact_turn(y if t[gain] is None else y * t[gain].double(), t, case, 1.0)
        return got
    t = _token_inputs(case, seed)
    return _exact_select(t, case) if case["kind"] == "select" else _exact_attend(t, case)
