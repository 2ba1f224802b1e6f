"""The operators that serve rows over a cache held in 8 bits, as cases that can be timed.

A program that answers row by row, or chunk by chunk, keeps its keys and values: "cache" writes new rows into pages of 8-bit
codes, with a scale for each block of rows and head, and reads rows back; "attend" is the attention of new rows over such a
cache, over all of it or over a window and the first keys; "norm" is what stands around each such block: the branch's
norm, its gate and the residual sum, and the next branch's norm and modulation.

Where `own` is false run() computes each in its plain form by elementary torch operations; where it is true it makes
the library's calls. exact() is the same from the definition in 64 bits.

Cached keys and values are normal, with channels of unlike sizes and heads of unlike sizes; pages lie in no order.
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
        # one new row for each of 8 sequences, into blocks that are partly full; their last 64 rows back
        {"name": "cache bf16 8 new rows", "kind": "cache", "write": True, "rows": 8, "seqs": 8, "past": 1000, "back": 512, "kv": 8,
         "d": 128, "block": 64, "dtype": "bf16"},
        # the rows of the largest usual voxel set of the flow model, five objects of unlike sizes, and all of them back
        {"name": "cache bf16 28k ragged", "kind": "cache", "write": True, "rows": 28265, "seqs": 5, "past": 0, "back": 28265, "kv": 16,
         "d": 64, "block": 64, "dtype": "bf16"},
        # the coarse set's rows behind others, in the reference's own precision
        {"name": "cache f32 5k", "kind": "cache", "write": True, "rows": 5086, "seqs": 1, "past": 777, "back": 5086, "kv": 16, "d": 64,
         "block": 64, "dtype": "f32"},
        # whole caches back as rows, for a call that wants rows
        {"name": "cache bf16 read 65k", "kind": "cache", "write": False, "rows": 0, "seqs": 8, "past": 8192, "back": 65536, "kv": 8,
         "d": 128, "block": 64, "dtype": "bf16"},
        # the smallest call: one new row over a short cache
        {"name": "attend bf16 1 row of 300", "kind": "attend", "rows": 1, "seqs": 1, "keys": 300, "ragged": False, "heads": 12, "kv": 12,
         "d": 64, "block": 64, "causal": True, "window": 0, "sinks": 0, "dtype": "bf16"},
        # one new row for each of 8 sequences over long caches
        {"name": "attend bf16 8 rows of 65k", "kind": "attend", "rows": 8, "seqs": 8, "keys": 65536, "ragged": False, "heads": 32, "kv": 8,
         "d": 128, "block": 64, "causal": True, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a larger batch of single rows over caches of unlike lengths, each seeing its last 4096 keys and the first 4
        {"name": "attend bf16 64 rows window", "kind": "attend", "rows": 64, "seqs": 64, "keys": 16384, "ragged": True, "heads": 32,
         "kv": 8, "d": 128, "block": 64, "causal": True, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # the same precision as the reference's, a head of keys for each head of queries
        {"name": "attend f32 8 rows of 16k", "kind": "attend", "rows": 8, "seqs": 8, "keys": 16384, "ragged": True, "heads": 16, "kv": 16,
         "d": 64, "block": 64, "causal": True, "window": 0, "sinks": 0, "dtype": "f32"},
        # the largest: chunks of rows behind long caches, as prompts are taken in
        {"name": "attend bf16 4 chunks of 1k", "kind": "attend", "rows": 4096, "seqs": 4, "keys": 9216, "ragged": False, "heads": 32,
         "kv": 8, "d": 128, "block": 64, "causal": True, "window": 0, "sinks": 0, "dtype": "bf16"},
        # the smallest: one row's stream and next input
        {"name": "norm f32 1 row", "kind": "norm", "n": 1, "c": 1024, "sets": 1, "post": "none", "pre": "layer", "mod": True,
         "stream": "f32", "branch": "f32"},
        # a flow block's row between its attention and its next branch: gate by forward, norm, modulation
        {"name": "norm bf16 5k x 1024", "kind": "norm", "n": 5086, "c": 1024, "sets": 2, "post": "none", "pre": "layer", "mod": True,
         "stream": "bf16", "branch": "bf16"},
        # norms on both sides of the branch, the stream kept in float32, at the most rows the pipeline keeps
        {"name": "norm f32 42k x 768", "kind": "norm", "n": 42000, "c": 768, "sets": 1, "post": "rms", "pre": "rms", "mod": False,
         "stream": "f32", "branch": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "cache", "attend", "attend", "attend", "attend", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "norm":
        return {"kind": "norm", "n": _log(rng, 1, 42000), "c": rng.choice([rng.randint(33, 2600), 8 * rng.randint(8, 300), 128 * rng.randint(1, 20)]),
                "sets": rng.randint(1, 6), "post": rng.choice(["none", "layer", "rms"]), "pre": rng.choice(["none", "layer", "rms"]),
                "mod": rng.random() < 0.5, "stream": rng.choice(["f32", "bf16"]), "branch": dtype}
    kv, group = rng.choice([(16, 1), (12, 1), (4, 4), (8, 4), (2, 5), (1, 8), (8, 1)])
    c = {"kind": kind, "kv": kv, "d": rng.choice([32, 64, 64, 96, 128, 128]), "block": rng.choice([64, 64, 128]), "dtype": dtype}
    seqs = rng.randint(1, 12)
    if kind == "cache":
        write = rng.random() < 0.7
        single = rng.random() < 0.3
        rows = 0 if not write else seqs if single else _log(rng, max(1, seqs), 20000)
        past = _log(rng, 70, 4000) if not write or single or rng.random() < 0.5 else 0
        back = rows if past == 0 else seqs * rng.randint(1, past)
        c.update(write=write, rows=rows, seqs=seqs, past=past, back=max(1, back))
        return c
    shape = rng.choice(["single", "single", "few", "chunk"])
    rows = seqs if shape == "single" else seqs * rng.randint(2, 40) if shape == "few" else _log(rng, 100, 2500)
    keys = _log(rng, 100, 6000) if shape == "chunk" else _log(rng, 70, 40000)
    causal = rng.random() < 0.8
    window = _log(rng, 20, 4000) if causal and rng.random() < 0.4 else 0
    c.update(rows=rows, seqs=seqs, keys=keys, ragged=rng.random() < 0.5, heads=kv * group, causal=causal, window=window,
             sinks=rng.choice([0, 1, 4, 70]) if window else 0)
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _dev():
    return torch.device("cuda", 0)


def _gen(seed, tag):
    g = torch.Generator(device=_dev())
    g.manual_seed((seed * 1000003 + tag) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, tag, shape, std=1.0):
    return torch.randn(shape, generator=_gen(seed, tag), device=_dev(), dtype=torch.float32) * std


def _tdt(word):
    return torch.bfloat16 if word == "bf16" else torch.float32


def _cuts(n, parts, word):
    """Lengths of `parts` pieces of n rows in all; of four or more, one is empty and one has one row (all alike where n is `parts`)."""
    if n == parts:
        return [1] * parts
    r = random.Random("%s %d %d" % (word, n, parts))
    fixed = [0, 1] if parts >= 4 and n > parts else []
    at = sorted(r.randint(0, n - sum(fixed)) for _ in range(parts - len(fixed) - 1))
    lens = [b - a for a, b in zip([0] + at, at + [n - sum(fixed)])] + fixed
    r.shuffle(lens)
    return lens


@functools.lru_cache(maxsize=256)
def _plan(kind, rows, seqs, keys, ragged, past, back):
    """(new rows, rows kept with them, rows read back) of each sequence."""
    r = random.Random("plan %s %d %d %d %d %d" % (kind, rows, seqs, keys, past, back))
    if kind == "attend":
        new = _cuts(rows, seqs, "rows") if ragged and rows > seqs else [rows // seqs + (1 if s < rows % seqs else 0) for s in range(seqs)]
        lens = [r.randint(max(1, keys // 8), keys) if ragged else keys for s in range(seqs)]
        return tuple(new), tuple(max(n, m) for n, m in zip(new, lens)), tuple([0] * seqs)
    new = _cuts(rows, seqs, "rows") if rows else [0] * seqs
    lens = [n + (past if rows == 0 or not past else r.randint(past // 2, past)) for n in new]
    if past == 0:
        return tuple(new), tuple(lens), tuple(new)
    return tuple(new), tuple(lens), tuple(min(n, back // seqs) if seqs > 1 else min(n, back) for n in lens)


def _lens(case):
    return _plan(case["kind"], case["rows"], case["seqs"], case.get("keys", 0), case.get("ragged", False), case.get("past", 0),
                 case.get("back", 0))


def _starts(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=_dev())


def _pages_of(case):
    """(pages of a sequence's table, pages in all): room for one block more than a sequence has."""
    width = max(_lens(case)[1]) // case["block"] + 1
    return width, width * case["seqs"] + 3


def _codes_room(case):
    return _pages_of(case)[1] * case["kv"] * 2 * case["block"] * case["d"]


def _split(buffer, case):
    """A cache's buffer as (codes [pages][kv][2][block * d], scale [pages][kv][2])."""
    room, pages = _codes_room(case), _pages_of(case)[1]
    return buffer[:room].view(pages, case["kv"], 2, -1), buffer[room:].view(torch.float32).view(pages, case["kv"], 2)


def _two_to(e):
    """2^e for whole e, exactly, in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _sizes(seed, case):
    """Factors of keys' and values' channels [2][kv][d]."""
    return torch.exp(_normal(seed, 21, (2, case["kv"], case["d"]), 0.4) + _normal(seed, 22, (2, case["kv"], 1), 0.5))


def _cache_inputs(case, seed):
    """A cache filled up to what was there before the call, its table, its lengths with the new rows, and the new rows."""
    b, kv, d = case["block"], case["kv"], case["d"]
    new, lens, back = _lens(case)
    width, pages = _pages_of(case)
    t = {"lens": torch.tensor(lens, dtype=torch.int32, device=_dev()), "new": _starts(new), "back": _starts(back)}
    t["table"] = torch.randperm(pages, generator=_gen(seed, 5), device=_dev())[: width * len(lens)].to(torch.int32).view(len(lens), width).contiguous()
    t["buffer"] = torch.zeros(_codes_room(case) + pages * kv * 8, dtype=torch.uint8, device=_dev())
    codes, scale = _split(t["buffer"], case)
    size = _sizes(seed, case)
    before = t["lens"] - torch.diff(t["new"]) if case["kind"] == "cache" else t["lens"]
    for which in (0, 1):
        for s in range(len(lens)):  # a sequence at a time: its rows in 32 bits are four times the cache
            x = _normal(seed, 1000 * (which + 1) + s, (width, kv, b, d)) * size[which][:, None, :]
            there = torch.arange(width * b, device=_dev()).view(width, 1, b, 1) < before[s]
            x = torch.where(there, x, 0.0)
            most = x.abs().amax((2, 3))
            step = torch.where(most > 0, _two_to(torch.frexp(most)[1] - 7), 0.0)
            c = torch.round(x.double() / torch.where(step > 0, step, 1.0)[..., None, None]).clamp(-127, 127) + 128
            c = c.to(torch.uint8)
            codes[t["table"][s].long(), :, which] = (c if which == 0 else c.transpose(2, 3)).reshape(width, kv, -1)
            scale[t["table"][s].long(), :, which] = step.float()
    dt = _tdt(case["dtype"])
    if case["kind"] == "attend":
        n, h = case["rows"], case["heads"]
        # queries beside other heads of a row, as a projection leaves them
        t["heads"] = torch.zeros((n, h + kv, d), dtype=dt, device=_dev())
        t["heads"][:, :h] = _normal(seed, 31, (n, h, d), 1.5) / size[0].repeat_interleave(h // kv, 0)
        t["q"] = t["heads"][:, :h]
    else:
        t["kv"] = (_normal(seed, 41, (max(1, case["rows"]), 2, kv, d)) * size).to(dt)
        t["k"], t["v"] = t["kv"][: case["rows"], 0], t["kv"][: case["rows"], 1]
    return t


def _norm_inputs(case, seed):
    n, c, s = case["n"], case["c"], case["sets"]
    t = {"x": (_normal(seed, 1, (n, c)) * torch.exp(_normal(seed, 2, (n, 1), 0.5)) + _normal(seed, 3, (c,), 0.5)).to(_tdt(case["stream"])),
         "branch": (_normal(seed, 4, (n, c)) + 0.25).to(_tdt(case["branch"])),
         # coordinates of voxels: the set (object) of a row stands first
         "coords": torch.randint(0, s, (n, 4), generator=_gen(seed, 5), device=_dev(), dtype=torch.int32)}
    for k, name in enumerate(("post_w", "post_b", "pre_w", "pre_b")):
        used = case[name.split("_")[0]] != "none" and (name.endswith("w") or case[name.split("_")[0]] == "layer")
        t[name] = (_normal(seed, 6 + k, (c,), 0.2) + (1.0 if name.endswith("w") else 0.0)) if used else None
    # a block's six vectors of a set as the modulation's projection leaves them: the first three are the norm's shift, its
    # scale, and the branch's gate
    t["mods"] = _normal(seed, 11, (s, 6, c), 0.3)
    return t


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def prepare(case, seed):
    st = {"case": case}
    new = functools.partial(torch.zeros, device=_dev())
    if case["kind"] == "norm":
        st.update(_norm_inputs(case, seed))
        st["y"] = new((case["n"], case["c"]), dtype=_tdt(case["stream"]))
        st["h"] = new((case["n"], case["c"]), dtype=_tdt(case["branch"]))
        torch.cuda.synchronize()
        return st
    st.update(_cache_inputs(case, seed))
    dt, kv, d = _tdt(case["dtype"]), case["kv"], case["d"]
    rows, lens, back = _lens(case)
    st["longest"], st["read_rows"] = max(lens), sum(back)
    if own:
        st["cache"] = _lib().KvCache(st["buffer"].data_ptr(), _pages_of(case)[1], kv, d, case["block"])
    if case["kind"] == "cache":
        st["rk"], st["rv"] = new((st["read_rows"], kv, d), dtype=dt), new((st["read_rows"], kv, d), dtype=dt)
    else:
        st["o"] = new((case["rows"], case["heads"], d), dtype=dt)
        st["lse"] = new((case["rows"], case["heads"]), dtype=torch.float32)
        if own:
            st["ws"] = torch.empty(max(1, st["cache"].attention_workspace_size(case["rows"], case["heads"], case["seqs"], st["longest"],
                                                                              case["window"], case["sinks"])), dtype=torch.uint8, device=_dev())
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------
# run: the plain forms
# ---------------------------------------------------------------------------
def _places(starts, lens, total):
    """(sequence, place) of packed rows: a sequence's last row stands at its last place."""
    row = torch.arange(total, device=starts.device)
    s = torch.searchsorted(starts.long(), row, right=True) - 1
    return s, row - starts.long()[s + 1] + lens.long()[s]


def _power_below(most):
    """2^(e - 6) of 2^e <= most < 2^(e + 1), exactly; 0 of what is below 2^-100."""
    e = (most.view(torch.int32) >> 23) - 127
    return torch.where(most >= 2.0 ** -100, ((e - 6 + 127).clamp(min=1) << 23).view(torch.float32), 0.0)


def _plain_write(st, case):
    b, kv, d, total = case["block"], case["kv"], case["d"], case["rows"]
    codes, scale = _split(st["buffer"], case)
    s, place = _places(st["new"], st["lens"], total)
    page = st["table"][s, place // b].long()
    x = torch.stack([st["k"], st["v"]], 2).float()                                   # [rows][kv][2][d]
    most = torch.zeros_like(scale).scatter_reduce_(0, page[:, None, None].expand(-1, kv, 2), x.abs().amax(-1), "amax")
    # the block that a sequence's rows begin in keeps what it held before
    first = st["lens"].long() - torch.diff(st["new"]).long()
    left = st["table"].gather(1, (first // b)[:, None])[:, 0].long()
    keeps = (first % b > 0)[:, None, None]
    was = torch.where(keeps, scale[left], 0.0)
    now = torch.maximum(_power_below(most[left]), was)
    kept = (codes[left].float() - 128.0) * torch.where(now > 0, was / torch.where(now > 0, now, 1.0), 0.0)[..., None]
    codes[left] = torch.where(keeps[..., None], (torch.round(kept) + 128.0).to(torch.uint8), codes[left])
    fresh = _power_below(most)
    fresh[left] = now
    scale[page] = fresh[page]
    scale[left] = torch.where(keeps, now, scale[left])
    step = scale[page][..., None]
    c = (torch.round(x / torch.where(step > 0, step, 1.0)).clamp(-127, 127) + 128.0).to(torch.uint8)
    slot = place % b
    codes[:, :, 0].view(-1, kv, b, d)[page, :, slot] = c[:, :, 0]
    codes[:, :, 1].view(-1, kv, d, b)[page, :, :, slot] = c[:, :, 1]


def _plain_read(st, case):
    b, kv, d = case["block"], case["kv"], case["d"]
    codes, scale = _split(st["buffer"], case)
    s, place = _places(st["back"], st["lens"], st["read_rows"])
    page, slot = st["table"][s, place // b].long(), place % b
    k = (codes[:, :, 0].view(-1, kv, b, d)[page, :, slot].float() - 128.0) * scale[page, :, 0, None]
    v = (codes[:, :, 1].view(-1, kv, d, b)[page, :, :, slot].float() - 128.0) * scale[page, :, 1, None]
    return {"k": k.to(_tdt(case["dtype"])), "v": v.to(_tdt(case["dtype"]))}


def _plain_attend(st, case):
    b, kv, d, g = case["block"], case["kv"], case["d"], case["heads"] // case["kv"]
    codes, scale = _split(st["buffer"], case)
    lens, n = st["lens"].long(), torch.diff(st["new"]).long()
    lq, lk = max(_lens(case)[0]), st["longest"]
    used = st["table"][:, : -(-lk // b)].long()                                      # [S][blocks]
    k = (codes[used, :, 0].unflatten(-1, (b, d)).float() - 128.0) * scale[used][..., 0, None, None]
    v = (codes[used, :, 1].unflatten(-1, (d, b)).float() - 128.0) * scale[used][..., 1, None, None]
    k = k.permute(0, 2, 4, 1, 3).flatten(3)[..., :lk].contiguous()                   # [S][kv][d][keys]
    v = v.permute(0, 2, 1, 4, 3).flatten(2, 3)[:, :, :lk].contiguous()               # [S][kv][keys][d]
    at = torch.arange(lq, device=lens.device)
    real = at < n[:, None]
    row = (st["new"][:-1, None].long() + at).clamp(max=case["rows"] - 1)
    q = st["q"][row].float().unflatten(2, (kv, g)).permute(0, 2, 3, 1, 4).reshape(len(n), kv, g * lq, d)
    score = torch.matmul(q, k).mul_(d ** -0.5).view(len(n), kv, g, lq, lk)
    place = (at + (lens - n)[:, None])[:, :, None]                                   # [S][lq][1]
    key = torch.arange(lk, device=lens.device)
    may = key < (torch.minimum(place + 1, lens[:, None, None]) if case["causal"] else lens[:, None, None])
    if case["window"]:
        may = may & ((key > place - case["window"]) | (key < case["sinks"]))
    score.masked_fill_(~may.expand(-1, lq, -1)[:, None, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = score.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(len(n), kv, g * lq, lk), v).view(len(n), kv, g, lq, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    lse = (m + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
    return {"o": o[real].to(st["q"].dtype), "lse": lse[real]}


def _plain_norm(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    y = y if w is None else y * w
    return y if b is None else y + b


def _plain_gated(st, case):
    shift, scale, gate = (st["mods"][:, j][st["coords"][:, 0].long()] for j in range(3))
    y = st["x"].float() + 0.5 * gate * _plain_norm(st["branch"].float(), case["post"], st["post_w"], st["post_b"])
    got = {"y": y.to(st["x"].dtype)}
    if case["pre"] != "none":
        h = _plain_norm(y, case["pre"], st["pre_w"], st["pre_b"])
        got["h"] = (h * (1.0 + scale) + shift if case["mod"] else h).to(st["branch"].dtype)
    return got


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    if case["kind"] == "norm":
        return _plain_gated(st, case)
    if case["kind"] == "attend":
        return _plain_attend(st, case)
    if case["write"]:
        _plain_write(st, case)
    return _plain_read(st, case)


# ---------------------------------------------------------------------------
# run: the library's calls
# ---------------------------------------------------------------------------
def _run_own(st):
    s3dx, case = _lib(), st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] == "norm":
        kinds = {"none": s3dx.NORM_NONE, "layer": s3dx.NORM_LAYER, "rms": s3dx.NORM_RMS}
        dts = {"f32": s3dx.F32, "bf16": s3dx.BF16}
        ptr = {k: None if st[k] is None else st[k].data_ptr() for k in ("post_w", "post_b", "pre_w", "pre_b")}
        pre, c = case["pre"] != "none", case["c"]
        s3dx.gated_norm_rows(st["x"].data_ptr(), dts[case["stream"]], st["branch"].data_ptr(), dts[case["branch"]], case["n"], c, EPS,
                             st["y"].data_ptr(), st["h"].data_ptr() if pre else None, dts[case["branch"]],
                             post=kinds[case["post"]], pre=kinds[case["pre"]], residual_scale=0.5,
                             gate=st["mods"].data_ptr() + 8 * c, mod_shift=st["mods"].data_ptr() if pre and case["mod"] else None,
                             mod_scale=st["mods"].data_ptr() + 4 * c if pre and case["mod"] else None, mod_stride=6 * c,
                             sets=st["coords"].data_ptr(), set_stride=4, set_count=case["sets"], stream=stream, **ptr)
        return {"y": st["y"], "h": st["h"]} if pre else {"y": st["y"]}
    dt = s3dx.BF16 if case["dtype"] == "bf16" else s3dx.F32
    where = (st["table"].data_ptr(), st["table"].shape[1], st["lens"].data_ptr(), case["seqs"])
    if case["kind"] == "attend":
        st["cache"].attention(st["q"].data_ptr(), dt, case["rows"], case["heads"], st["new"].data_ptr(), *where, st["longest"],
                              st["o"].data_ptr(), lse=st["lse"].data_ptr(), q_stride=st["q"].stride(0), causal=case["causal"],
                              window=case["window"], sinks=case["sinks"], workspace=st["ws"].data_ptr(),
                              workspace_bytes=st["ws"].numel(), stream=stream)
        return {"o": st["o"], "lse": st["lse"]}
    if case["write"]:
        st["cache"].write(st["k"].data_ptr(), st["v"].data_ptr(), dt, case["rows"], st["new"].data_ptr(), *where,
                          k_stride=st["k"].stride(0), v_stride=st["v"].stride(0), stream=stream)
    st["cache"].read(st["rk"].data_ptr(), st["rv"].data_ptr(), dt, st["read_rows"], st["back"].data_ptr(), *where, stream=stream)
    return {"k": st["rk"], "v": st["rv"]}


# ---------------------------------------------------------------------------
# work, exact
# ---------------------------------------------------------------------------
def _seen(case):
    """(pairs of a query row and a key row in all, key rows that some query row of their sequence sees)."""
    pairs = keys = 0
    for n, m in zip(*_lens(case)[:2]):
        if n == 0:
            continue
        if not case["causal"]:
            pairs, keys = pairs + n * m, keys + m
            continue
        end = np.arange(n, dtype=np.int64) + m - n + 1
        begin = np.maximum(0, end - case["window"]) if case["window"] else np.zeros_like(end)
        pairs += int((end - begin + np.minimum(begin, case["sinks"])).sum())
        keys += int(m - begin[0] + min(begin[0], case["sinks"]))
    return pairs, keys


def work(case):
    if case["kind"] == "norm":
        size = {"f32": 4, "bf16": 2}
        per = 2 * size[case["stream"]] + size[case["branch"]] * (2 if case["pre"] != "none" else 1)
        return {"bytes": case["n"] * (case["c"] * per + 4) + case["sets"] * case["c"] * 4 * (3 if case["mod"] else 1), "flops": 12 * case["n"] * case["c"]}
    e = 2 if case["dtype"] == "bf16" else 4
    row = 2 * case["kv"] * case["d"]
    if case["kind"] == "cache":
        back = sum(_lens(case)[2])
        return {"bytes": (case["rows"] + back) * row * (e + 1), "flops": (case["rows"] * 3 + back) * row}
    pairs, keys = _seen(case)
    return {"bytes": 2 * case["rows"] * case["heads"] * case["d"] * e + keys * row + case["rows"] * case["heads"] * 4,
            "flops": 4 * case["d"] * case["heads"] * pairs}


def _held(t, case, s, which):
    """The 64-bit values [places][kv][d] that sequence s' pages stand for, and their steps [blocks][kv]."""
    codes, scale = _split(t["buffer"], case)
    pages, b, d = t["table"][s].long(), case["block"], case["d"]
    c = codes[pages, :, which].double() - 128.0
    c = c.view(-1, case["kv"], b, d) if which == 0 else c.view(-1, case["kv"], d, b).transpose(2, 3)
    step = scale[pages, :, which].double()
    return (c * step[..., None, None]).transpose(1, 2).reshape(-1, case["kv"], d), step


def _exact_cache(t, case):
    """Block by block from the definition: the largest magnitude's power, every value in steps of it."""
    b, kv, got = case["block"], case["kv"], {}
    new, lens, back = _lens(case)
    for which, name in ((0, "k"), (1, "v")):
        rows, at = [], 0
        for s, (n, m, r) in enumerate(zip(new, lens, back)):
            x, step = _held(t, case, s, which)
            if n:
                x[m - n: m] = t[name][at: at + n].double()
            at += n
            for j in range((m - n) // b, -(-m // b)) if n else ():
                blk = x[j * b: min(m, (j + 1) * b)]
                fresh = blk[max(0, m - n - j * b):]
                most = fresh.abs().amax((0, 2))
                unit = torch.where(most >= 2.0 ** -100, _two_to(torch.frexp(most)[1] - 7), 0.0)
                if j * b < m - n:
                    unit = torch.maximum(unit, step[j])
                unit = unit[:, None]
                blk[:] = torch.where(unit > 0, torch.round(blk / torch.where(unit > 0, unit, 1.0)).clamp(-127, 127) * unit, 0.0)
            rows.append(x[m - r: m])
        got[name] = torch.cat(rows)
    return got


def _exact_attend(t, case):
    new, lens, _ = _lens(case)
    g, d = case["heads"] // case["kv"], case["d"]
    o = torch.zeros((case["rows"], case["heads"], d), dtype=torch.float64, device=_dev())
    lse = torch.full((case["rows"], case["heads"]), -math.inf, dtype=torch.float64, device=_dev())
    at = 0
    for s, (n, m) in enumerate(zip(new, lens)):
        if n == 0:
            continue
        k, v = (_held(t, case, s, which)[0][:m] for which in (0, 1))
        see = torch.ones((n, m), dtype=torch.bool, device=_dev())
        if case["causal"]:
            see = see.tril(m - n)
        if case["window"]:
            far = torch.ones_like(see).tril(m - n - case["window"])
            far[:, : case["sinks"]] = False
            see &= ~far
        for h in range(case["heads"]):
            x = (t["q"][at: at + n, h].double() @ k[:, h // g].T / math.sqrt(d)).masked_fill_(~see, -math.inf)
            lse[at: at + n, h] = torch.logsumexp(x, 1)
            o[at: at + n, h] = torch.softmax(x, 1) @ v[:, h // g]
        at += n
    return {"o": o, "lse": lse}


def _exact_normed(x, kind, w, b):
    if kind == "none":
        return x
    mean = x.mean(1, keepdim=True) if kind == "layer" else 0.0
    y = (x - mean) / (((x - mean) ** 2).sum(1, keepdim=True) / x.shape[1] + EPS).sqrt()
    y = y if w is None else y * w.double()
    return y if b is None else y + b.double()


def exact(case, seed):
    if case["kind"] == "norm":
        t = _norm_inputs(case, seed)
        mods = t["mods"].double()[t["coords"][:, 0].long()]
        y = t["x"].double() + mods[:, 2] / 2.0 * _exact_normed(t["branch"].double(), case["post"], t["post_w"], t["post_b"])
        if case["pre"] == "none":
            return {"y": y}
        h = _exact_normed(y, case["pre"], t["pre_w"], t["pre_b"])
        return {"y": y, "h": h + h * mods[:, 1] + mods[:, 0] if case["mod"] else h}
    t = _cache_inputs(case, seed)
    return _exact_cache(t, case) if case["kind"] == "cache" else _exact_attend(t, case)
