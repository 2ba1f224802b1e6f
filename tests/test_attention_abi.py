"""The attention entry points refuse bad arguments on the host, before any
device work (fake addresses: nothing here is read)."""
import ctypes as C

import numpy as np
import pytest

P = 0x10000  # an aligned address


def status(s3dx, name, *args):
    buf = C.create_string_buffer(256)
    st = getattr(s3dx.lib(), name)(*args, buf, 256)
    return st, buf.value.decode()


def refused(s3dx, name, args, word):
    st, msg = status(s3dx, name, *args)
    assert st == s3dx.INVALID_ARGUMENT and word in msg, (st, msg)


@pytest.fixture(scope="module")
def rotary(s3dx):
    return s3dx.Rotary.per_axis(64, [10, 10, 10])


@pytest.mark.parametrize("head_dim,axes,axis,frequency,pairing,word", [
    (0, 1, [0], [1.0], 0, "head_dim"), (257, 1, [0], [1.0], 0, "head_dim"), (64, 0, [0], [1.0], 0, "axes"),
    (64, 9, [0], [1.0], 0, "axes"), (64, 1, [], [], 0, "pairs"), (6, 1, [0] * 4, [1.0] * 4, 0, "pairs"),
    (1, 1, [0], [1.0], 0, "pairs"), (64, 1, [1], [1.0], 0, "axis"), (64, 1, [-1], [1.0], 0, "axis"),
    (64, 1, [0], [float("nan")], 0, "frequency"), (64, 1, [0], [float("inf")], 0, "frequency"),
    (64, 1, [0], [2e6], 0, "frequency"), (64, 1, [0], [1.0], 2, "pairing")])
def test_rotary_create_refuses(s3dx, head_dim, axes, axis, frequency, pairing, word):
    with pytest.raises(s3dx.S3dxError, match=word):
        s3dx.Rotary(head_dim, axis, frequency, axes, pairing)


def test_rotary_lists_of_two_lengths(s3dx):
    with pytest.raises(ValueError):
        s3dx.Rotary(64, [0, 0], [1.0])


APPLY = dict(rotary=None, inverse=0, x=P, x_dtype=1, n=10, heads=4, x_stride=256, positions=P, position_stride=3, y=P + 65536,
             y_dtype=1, y_stride=256, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(rotary=0), "rotary"), (dict(inverse=2), "inverse"), (dict(x_dtype=2), "dtype"), (dict(y_dtype=-1), "dtype"),
    (dict(n=-1), "n is"), (dict(n=2 ** 31), "n is"), (dict(heads=0), "heads"), (dict(heads=65537), "heads"),
    (dict(x_stride=255), "stride"), (dict(y_stride=255), "stride"), (dict(x=None), "NULL"), (dict(y=None), "NULL"),
    (dict(x=P + 1), "aligned"), (dict(y=P + 2, y_dtype=0), "aligned"), (dict(positions=None), "positions"),
    (dict(positions=P + 2), "positions"), (dict(position_stride=2), "position_stride"),
    (dict(y=P, y_dtype=0), "in place"), (dict(y=P, x_stride=512), "in place"),
    (dict(n=2 ** 31 - 1, heads=5, x_stride=320, y_stride=320), "2^33")])
def test_rotary_apply_refuses(s3dx, rotary, change, word):
    a = {**APPLY, "rotary": rotary.handle, **change}
    refused(s3dx, "s3dx_rotary_apply", a.values(), word)


QK = dict(rotary=None, positions=P, position_stride=3, q=P, q_heads=8, q_stride=768, q_gain=None, k=P + 1024, k_heads=2,
          k_stride=768, k_gain=None, gain_per_head=1, dtype=1, n=5, head_dim=64, eps=1e-6, q_out=2 * P, q_out_stride=512,
          k_out=3 * P, k_out_stride=128, out_dtype=1, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=32), "another head_dim"), (dict(head_dim=0, rotary=None), "head_dim"), (dict(eps=0.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"), (dict(gain_per_head=2), "gain_per_head"),
    (dict(k_heads=0), "k without"), (dict(k=None), "NULL"), (dict(k_heads=-1), "k without"), (dict(q_heads=0), "heads"),
    (dict(dtype=5), "dtype"), (dict(out_dtype=5), "dtype"), (dict(k_stride=127), "stride"), (dict(q_gain=P + 2), "gain"),
    (dict(k_gain=P + 1), "gain"), (dict(k_out=P + 1024), "in place"), (dict(n=-3), "n is"),
    (dict(q_heads=65536, k_heads=65536, q_stride=2 ** 22, k_stride=2 ** 22, q_out_stride=2 ** 22, k_out_stride=2 ** 22,
          n=2 ** 17), "2^33")])
def test_qk_norm_rotary_refuses(s3dx, rotary, change, word):
    a = {**QK, "rotary": rotary.handle, **change}
    refused(s3dx, "s3dx_qk_norm_rotary", a.values(), word)


INDEX = dict(k=P, dtype=1, total_k=100, kv_heads=2, head_dim=64, k_stride=128, k_starts=P, sequences=1, block=64, codes=P,
             scale=P, stream=None)
SELECT = dict(q=P, dtype=1, total_q=10, total_k=100, heads=4, kv_heads=2, head_dim=64, q_stride=256, q_starts=P, k_starts=P,
              sequences=1, block=64, top=4, max_k=100, codes=P, scale=P, flags=0, selected=P, stream=None)
ATTEND = dict(q=P, k=P, v=P, dtype=1, total_q=10, total_k=100, heads=4, kv_heads=2, head_dim=64, q_stride=256, k_stride=128,
              v_stride=128, q_starts=P, k_starts=P, sequences=1, block=64, max_k=100, selected=P, top=4, softmax_scale=0.125,
              flags=0, o=P, o_stride=256, lse=None, workspace=P, workspace_bytes=2 ** 40, stream=None)
SHAPES = [(dict(dtype=2), "dtype"), (dict(head_dim=80), "head_dim"), (dict(head_dim=256), "head_dim"),
          (dict(block=16), "block"), (dict(block=0), "block"), (dict(sequences=-1), "sequences"), (dict(kv_heads=0), "heads"),
          (dict(total_k=-1), "row count"), (dict(total_k=2 ** 31), "row count"),
          (dict(total_k=2 ** 29 + 1), "row count"), (dict(k_starts=None), "starts"),
          (dict(k_starts=P + 1), "starts")]


@pytest.mark.parametrize("change,word", SHAPES + [
    (dict(k=None), "NULL"), (dict(k=P + 8), "aligned"), (dict(k_stride=127), "stride"), (dict(k_stride=132), "16-byte pieces"),
    (dict(total_k=2 ** 29, block=32), "too many"), (dict(k_stride=2 ** 22), "2^22"), (dict(codes=P + 8), "codes"), (dict(scale=None), "scale")])
def test_block_index_refuses(s3dx, change, word):
    refused(s3dx, "s3dx_block_index", {**INDEX, **change}.values(), word)


@pytest.mark.parametrize("change,word", SHAPES + [
    (dict(heads=5), "heads"), (dict(heads=1), "heads"), (dict(top=0), "top"), (dict(top=4097), "top"), (dict(flags=4), "flags"),
    (dict(max_k=-1), "max_k"), (dict(max_k=32768 * 64 + 1), "max_k"), (dict(q=None), "NULL"), (dict(q_stride=255), "stride"),
    (dict(q_starts=None), "starts"), (dict(selected=None), "selected"), (dict(selected=P + 2), "selected"),
    (dict(codes=None), "codes"), (dict(total_q=-1), "row count"),
    (dict(total_q=2 ** 29), "too many"), (dict(total_q=2 ** 29, heads=8, kv_heads=8, q_stride=512), "out of range"),
    (dict(total_q=2 ** 31 - 1, heads=8, kv_heads=8, q_stride=512), "out of range")])
def test_block_select_refuses(s3dx, change, word):
    refused(s3dx, "s3dx_block_select", {**SELECT, **change}.values(), word)


@pytest.mark.parametrize("change,word", SHAPES + [
    (dict(heads=5), "heads"), (dict(top=0), "top"), (dict(selected=None), "top"), (dict(top=4097), "top"),
    (dict(flags=2), "flags"), (dict(softmax_scale=0.0), "softmax_scale"), (dict(softmax_scale=float("nan")), "softmax_scale"),
    (dict(softmax_scale=float("inf")), "softmax_scale"), (dict(softmax_scale=-1.0), "softmax_scale"), (dict(v=None), "NULL"),
    (dict(o=None), "NULL"), (dict(o=P + 2), "aligned"), (dict(o_stride=128), "stride"), (dict(v_stride=64), "stride"),
    (dict(lse=P + 2), "lse"), (dict(selected=P + 1), "selected"), (dict(max_k=-1), "row count"), (dict(q_starts=P + 2), "starts"),
    (dict(total_q=2 ** 29, heads=2, sequences=2 ** 24), "too many"), (dict(total_q=2 ** 31 - 1), "out of range")])
def test_block_attention_refuses(s3dx, change, word):
    refused(s3dx, "s3dx_block_attention", {**ATTEND, **change}.values(), word)


def test_nothing_to_do_needs_no_buffers(s3dx, rotary):
    for name, args in (("s3dx_rotary_apply", {**APPLY, "rotary": rotary.handle, "n": 0, "x": None, "y": None, "positions": None}),
                       ("s3dx_qk_norm_rotary", {**QK, "n": 0, "q": None, "k": None, "q_out": None, "k_out": None}),
                       ("s3dx_block_index", {**INDEX, "total_k": 0, "k": None, "codes": None}),
                       ("s3dx_block_select", {**SELECT, "total_q": 0, "q": None, "selected": None}),
                       ("s3dx_block_attention", {**ATTEND, "sequences": 0, "q": None, "o": None, "workspace": None})):
        assert status(s3dx, name, *args.values())[0] == s3dx.OK, name


def test_sizes(s3dx):
    assert s3dx.block_index_rows(0, 3, 64) == 3
    assert s3dx.block_index_rows(129, 2, 32) == 6
    # every sequence's blocks have rows of their own, whatever the lengths
    rng = np.random.default_rng(1)
    for _ in range(200):
        lens = rng.integers(0, 200, rng.integers(1, 8))
        at, end = 0, 0
        for s, n in enumerate(lens):
            first = at // 32 + s
            assert first >= end
            end, at = first + -(-int(n) // 32), at + int(n)
        assert end <= s3dx.block_index_rows(at, len(lens), 32)
    for bad in ((-1, 1, 64), (10, -1, 64), (10, 1, 48)):
        with pytest.raises(s3dx.S3dxError):
            s3dx.block_index_rows(*bad)
    for bad in ((-1, 4, 2, 64, 1, 64, 4, 100), (10, 4, 3, 64, 1, 64, 4, 100), (10, 4, 2, 72, 1, 64, 4, 100),
                (10, 4, 2, 64, 1, 64, -1, 100), (10, 4, 2, 64, 1, 64, 4, -1)):
        with pytest.raises(s3dx.S3dxError):
            s3dx.block_attention_workspace_size(*bad)
    assert s3dx.block_attention_workspace_size(0, 4, 2, 64, 1, 64, 4, 100) == 0
