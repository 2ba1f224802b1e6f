"""The entry points of the cache in 8 bits, the attention over it and the gated
norms refuse bad arguments on the host, before any device work (fake addresses:
nothing here is read)."""
import ctypes as C

import numpy as np
import pytest

import cache_ref as K
from test_attention_abi import P, refused, status


@pytest.fixture(scope="module")
def cache(s3dx):
    return s3dx.KvCache(P, 100, 2, 64, 64)


SHAPES = [(dict(pages=-1), "pages"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=65537), "kv_heads"), (dict(head_dim=48), "head_dim"),
          (dict(head_dim=256), "head_dim"), (dict(block=32), "block"), (dict(block=0), "block")]


@pytest.mark.parametrize("change,word", SHAPES + [(dict(buffer=None), "buffer"), (dict(buffer=P + 8), "buffer")])
def test_create_refuses(s3dx, change, word):
    a = {**dict(buffer=P, pages=100, kv_heads=2, head_dim=64, block=64), **change}
    with pytest.raises(s3dx.S3dxError, match=word):
        s3dx.KvCache(*a.values())
    if "buffer" not in change:
        with pytest.raises(s3dx.S3dxError, match=word):
            s3dx.KvCache.size(*list(a.values())[1:])


@pytest.mark.parametrize("pages,kv,d,block", [(0, 1, 32, 64), (7, 3, 96, 128), (2 ** 31 - 1, 65536, 128, 128)])
def test_size(s3dx, pages, kv, d, block):
    assert s3dx.KvCache.size(pages, kv, d, block) == pages * kv * (2 * block * d + 8)


ROWS = dict(cache=0, k=P, k_stride=128, v=P + 4096, v_stride=128, dtype=1, total=10, starts=P, table=P, table_stride=4, lengths=P,
            sequences=1, stream=None)


@pytest.mark.parametrize("name", ["s3dx_cache_write", "s3dx_cache_read"])
@pytest.mark.parametrize("change,word", [
    (dict(cache=None), "cache"), (dict(k=None), "NULL"), (dict(v=P + 8), "aligned"), (dict(k_stride=127), "stride"),
    (dict(v_stride=64), "stride"), (dict(k_stride=132), "16-byte pieces"), (dict(v_stride=2 ** 40 + 8), "2^40"), (dict(dtype=2), "dtype"),
    (dict(total=-1), "row count"), (dict(total=2 ** 29 + 1), "row count"), (dict(starts=None), "starts"), (dict(starts=P + 2), "starts"),
    (dict(table=None), "table"), (dict(table=P + 1), "table"), (dict(table_stride=-1), "table_stride"),
    (dict(table_stride=2 ** 23 + 1), "table_stride"), (dict(lengths=None), "lengths"), (dict(lengths=P + 2), "lengths"),
    (dict(sequences=-1), "sequences"), (dict(sequences=2 ** 24 + 1), "sequences"), (dict(total=2 ** 29, sequences=2 ** 24), "too many")])
def test_rows_refuse(s3dx, cache, name, change, word):
    refused(s3dx, name, {**ROWS, "cache": cache.handle, **change}.values(), word)


ATTEND = dict(cache=0, q=P, dtype=1, total_q=10, heads=4, q_stride=256, q_starts=P, table=P, table_stride=4, lengths=P, sequences=1,
              max_k=256, window=0, sinks=0, softmax_scale=0.125, flags=1, o=2 * P, o_stride=256, lse=None, workspace=P,
              workspace_bytes=2 ** 40, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(cache=None), "cache"), (dict(q=None), "NULL"), (dict(q=P + 2), "aligned"), (dict(o=None), "NULL"), (dict(o=P + 8), "aligned"),
    (dict(q_stride=255), "stride"), (dict(o_stride=128), "stride"), (dict(q_stride=260), "16-byte pieces"), (dict(dtype=3), "dtype"),
    (dict(total_q=-1), "row count"), (dict(total_q=2 ** 29 + 1), "row count"), (dict(heads=3), "heads"), (dict(heads=0), "heads"),
    (dict(heads=65538), "heads"), (dict(total_q=2 ** 29, heads=8, q_stride=512, o_stride=512), "out of range"), (dict(q_starts=None), "starts"),
    (dict(table=None), "table"), (dict(table_stride=2 ** 30), "table_stride"), (dict(lengths=None), "lengths"),
    (dict(sequences=-1), "sequences"), (dict(max_k=-1), "max_k"), (dict(max_k=2 ** 29 + 1), "max_k"), (dict(window=-1), "window"),
    (dict(window=2 ** 29 + 1), "window"), (dict(window=5, flags=0), "CAUSAL"), (dict(sinks=4), "sinks"), (dict(window=9, sinks=-1), "sinks"),
    (dict(softmax_scale=0.0), "softmax_scale"), (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(softmax_scale=1e6), "softmax_scale"), (dict(softmax_scale=8192.0), "softmax_scale"),
    (dict(flags=2), "flags"), (dict(lse=P + 2), "lse"), (dict(total_q=1, max_k=2 ** 20, workspace=None), "workspace"),
    (dict(total_q=1, max_k=2 ** 20, workspace=P + 4), "workspace"), (dict(total_q=1, max_k=2 ** 20, workspace_bytes=64), "workspace"),
    (dict(total_q=2 ** 28, sequences=2 ** 24), "too many")])
def test_attention_refuses(s3dx, cache, change, word):
    refused(s3dx, "s3dx_cache_attention", {**ATTEND, "cache": cache.handle, **change}.values(), word)


def test_workspace_size(s3dx, cache):
    assert cache.attention_workspace_size(0, 4, 1, 100) == 0
    assert cache.attention_workspace_size(4096, 4, 1, 100) == 0
    # few rows over many keys go to several workgroups; a short window to few
    long, short = cache.attention_workspace_size(1, 4, 1, 2 ** 20), cache.attention_workspace_size(1, 4, 1, 2 ** 20, 100, 4)
    assert long > 0 and short < long and long % 256 == 0
    for bad in ((-1, 4, 1, 100), (1, 3, 1, 100), (1, 4, -1, 100), (1, 4, 1, -1), (1, 4, 1, 100, -1), (1, 4, 1, 100, 0, 3)):
        with pytest.raises(s3dx.S3dxError):
            cache.attention_workspace_size(*bad)


NORM = dict(x=P, x_dtype=1, x_stride=100, branch=P + 65536, branch_dtype=1, branch_stride=100, n=7, c=100, post=1, post_w=P, post_b=P,
            residual_scale=1.0, gate=P, pre=2, pre_w=P, pre_b=P, mod_scale=P, mod_shift=P, mod_stride=100, sets=P, set_stride=4, set_count=3,
            eps=1e-6, y=2 * P, y_stride=100, h=3 * P, h_dtype=1, h_stride=100, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(n=-1), "n is"), (dict(n=2 ** 31), "n is"), (dict(c=0), "c must"), (dict(c=16385), "c must"), (dict(post=3), "norm"),
    (dict(pre=-1), "norm"), (dict(post=0), "post_w"), (dict(pre=0), "pre_w"), (dict(h=None), "h is NULL"),
    (dict(h=None, pre=0, pre_w=None, pre_b=None), "h is NULL"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=2.0), "eps"), (dict(residual_scale=float("inf")), "residual_scale"), (dict(residual_scale=float("nan")), "residual_scale"),
    (dict(x=None), "x is NULL"), (dict(branch=P + 1), "branch"), (dict(y=P + 1), "y is"), (dict(h=P + 2, h_dtype=0), "h is"),
    (dict(x_stride=99), "x: the row stride"), (dict(branch_stride=0), "branch: the row"), (dict(y_stride=99), "y: the row"),
    (dict(h_stride=2 ** 40 + 1), "h: the row"), (dict(x_dtype=2), "dtype"), (dict(branch_dtype=2), "dtype"), (dict(h_dtype=-1), "dtype"),
    (dict(sets=P + 2), "sets"), (dict(set_stride=0), "set_stride"), (dict(set_count=-1), "set_count"), (dict(mod_stride=99), "mod_stride"),
    (dict(gate=P + 2), "vector"), (dict(pre_b=P + 1), "vector"), (dict(y=P, y_stride=128), "in place"),
    (dict(y=P + 65536, branch_dtype=0), "in place"), (dict(h=P, h_dtype=0), "in place"), (dict(h=2 * P), "the same")])
def test_gated_norm_refuses(s3dx, change, word):
    refused(s3dx, "s3dx_gated_norm_rows", {**NORM, **change}.values(), word)


def test_nothing_to_do_needs_no_buffers(s3dx, cache):
    none = dict(k=None, v=None, starts=None)
    for name, args in (("s3dx_cache_write", {**ROWS, "cache": cache.handle, "total": 0, **none}),
                       ("s3dx_cache_read", {**ROWS, "cache": cache.handle, "sequences": 0, "table": None, "lengths": None, **none}),
                       ("s3dx_cache_attention", {**ATTEND, "cache": cache.handle, "total_q": 0, "q": None, "o": None, "q_starts": None}),
                       ("s3dx_gated_norm_rows", {**NORM, "n": 0, "x": None, "branch": None, "y": None, "h": 3 * P})):
        assert status(s3dx, name, *args.values())[0] == s3dx.OK, name
    assert status(s3dx, "s3dx_cache_create", None, 0, 1, 32, 64, C.byref(C.c_void_p()))[0] == s3dx.OK


def test_the_reference_keeps_what_it_is_given():
    # rows written at once and read: half a step off at most; a few at a time: a step and a half (rounded again when a step grows)
    rng = np.random.default_rng(1)
    k, v = (K.rows(rng, 300, 2, 32).astype(np.float64) for _ in range(2))
    table = np.array([[4, 0, 2, 5, 1]], np.int32)
    one, many = K.Held(6, 2, 32, 64), K.Held(6, 2, 32, 64)
    one.write(k, v, [300], [300], table)
    for a in range(0, 300, 7):
        many.write(k[a: a + 7], v[a: a + 7], [len(k[a: a + 7])], [min(300, a + 7)], table)
    for held, halves in ((one, 1), (many, 3)):
        for w, x in enumerate((k, v)):
            got, step = held.values(0, 300, table)[w], held.steps[table[0, np.arange(300) // 64], :, w]
            # (the largest value of a block may be cut: 127.5 to 127)
            assert np.all(np.abs(got - x) <= halves * step[:, :, None] * 0.5 + 0.5 * step[:, :, None] * (np.abs(x) > 127 * step[:, :, None]))
    back = K.Held(6, 2, 32, 64)
    back.codes, back.steps = back.take(many.buffer())
    assert np.array_equal(back.codes, many.codes) and np.array_equal(back.steps, many.steps)
