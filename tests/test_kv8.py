"""Refusals of the paged 8-bit cache's entry points, on the host before any launch, and the plain forms' own arithmetic."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kv8_plain as plain

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4097)
OFF8 = ctypes.c_void_p(4096 + 8)


class PlanCall(ctypes.Structure):  # include/lfm25_hip.h
    _fields_ = [(n, ctypes.c_void_p) for n in ("past", "counts", "table", "ring_at", "cursor", "starts", "slots", "next", "status")] + [
        (n, ctypes.c_int32) for n in ("requests", "width", "ring", "rows", "page")]


class AppendCall(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("keys", "values", "slots", "kc", "vc", "ksc", "vsc")] + [
        (n, ctypes.c_int64) for n in ("ks", "vs")] + [(n, ctypes.c_int32) for n in ("rows", "pages", "page", "kv", "dim", "format")]


class AttendCall(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("query", "kc", "vc", "ksc", "vsc", "table", "past", "starts", "out", "status", "ws")] + [
        ("stride", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
            "width", "requests", "rows", "heads", "max_rows", "pages", "page", "kv", "dim", "format", "reserved")] + [("scale", ctypes.c_float)]


def plan_args(**change):
    a = dict(past=P, counts=P, requests=4, table=P, width=8, ring_at=P, ring=16, cursor=P, starts=P, slots=P, rows=4, next=P,
             status=P, page=64)
    return bytes(PlanCall(**(a | change))), None


def append_args(**change):
    a = dict(keys=P, ks=512, values=P, vs=512, slots=P, rows=4, kc=P, vc=P, ksc=P, vsc=P, pages=8, page=64, kv=8, dim=64, format=0)
    return bytes(AppendCall(**(a | change))), None


def attend_args(**change):
    a = dict(query=P, stride=1024, kc=P, vc=P, ksc=P, vsc=P, table=P, width=8, past=P, starts=P, requests=4, out=P, rows=4,
             heads=16, max_rows=1, scale=0.125, pages=8, page=64, kv=8, dim=64, format=0)
    return bytes(AttendCall(**(a | change))), None


def test_packed_calls_have_the_structures_sizes(lab):
    for packed, call in ((lab.ops._PLAN, PlanCall), (lab.ops._APPEND, AppendCall), (lab.ops._ATTEND, AttendCall)):
        # (struct leaves out the padding behind the last member)
        assert 0 <= ctypes.sizeof(call) - packed.size < 8
    lib = lab.load_library()
    for f in (lib.lfm25_kv8_plan, lib.lfm25_kv8_append, lib.lfm25_kv8_attention):
        assert f(None, None) == lab._lib.LFM25_EINVAL and b"null" in lib.lfm25_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(past=None), b"null"), (dict(status=None), b"null"), (dict(page=48), b"page"), (dict(page=8), b"page"),
    (dict(page=512), b"page"), (dict(requests=0), b"requests"), (dict(requests=4097), b"requests"), (dict(width=0), b"width"),
    (dict(width=1 << 30), b"width"), (dict(ring=0), b"ring"), (dict(rows=0), b"rows"), (dict(cursor=ctypes.c_void_p(4100)), b"misaligned"),
    (dict(slots=ODD), b"misaligned")])
def test_plan_refuses(lab, change, message):
    lib = lab.load_library()
    assert lib.lfm25_kv8_plan(*plan_args(**change)) == lab._lib.LFM25_EINVAL
    assert message in lib.lfm25_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(keys=None), b"null"), (dict(vsc=None), b"null"), (dict(page=24), b"page"), (dict(pages=0), b"pages"),
    (dict(pages=1 << 25), b"pages"), (dict(kv=0), b"kv_heads"), (dict(kv=257), b"kv_heads"), (dict(dim=96), b"head_dim"),
    (dict(format=2), b"format"), (dict(rows=0), b"rows"), (dict(rows=-3), b"rows"), (dict(ks=504), b"stride"),
    (dict(vs=516), b"stride"), (dict(vs=-512), b"stride"), (dict(keys=OFF8), b"aligned"), (dict(vc=OFF8), b"aligned"),
    (dict(slots=ODD), b"misaligned")])
def test_append_refuses(lab, change, message):
    lib = lab.load_library()
    assert lib.lfm25_kv8_append(*append_args(**change)) == lab._lib.LFM25_EINVAL
    assert message in lib.lfm25_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(query=None), b"null"), (dict(starts=None), b"null"), (dict(page=0), b"page"), (dict(pages=-1), b"pages"),
    (dict(heads=12), b"heads"), (dict(heads=136), b"heads"), (dict(heads=0), b"heads"), (dict(dim=32), b"head_dim"),
    (dict(rows=0), b"rows"), (dict(rows=1 << 28), b"rows"), (dict(requests=4097), b"requests"), (dict(max_rows=0), b"max_rows"),
    (dict(width=0), b"width"), (dict(width=1 << 26), b"width"), (dict(stride=1020), b"stride"), (dict(stride=1000), b"stride"),
    (dict(query=OFF8), b"aligned"), (dict(out=OFF8), b"aligned"), (dict(past=ODD), b"misaligned"), (dict(status=ODD), b"misaligned"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(reserved=1), b"reserved"),
    (dict(width=64), b"workspace")])
def test_attention_refuses(lab, change, message):
    lib = lab.load_library()
    assert lib.lfm25_kv8_attention(*attend_args(**change)) == lab._lib.LFM25_EINVAL
    assert message in lib.lfm25_last_error()


def test_workspace_sizes(lab):
    size = lab.load_library().lfm25_kv8_attention_workspace_bytes
    column = 4 * (64 + 2)
    assert size(4, 16, 8, 64, 4, 1, 3, 64) == 0            # too few positions to divide
    assert size(64, 16, 8, 64, 0, 1, 64, 64) == 0          # a refused call
    assert size(4, 16, 8, 64, 4, 1, 64, 64) == 32 * 8 * 16 * column                # parts of 512 positions
    assert size(1, 16, 8, 64, 1, 1, 1 << 20, 64) == 8 * 65 * 16 * column          # a full chip
    assert size(512, 16, 8, 64, 2, 256, 64, 64) == 256 * 128 * column             # parts of tiles of 128 columns


def test_ops_refuse_before_any_launch(lab):
    ops = lab.ops
    f = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    cache = torch.zeros(8, 8, 64, 64, dtype=torch.int8)
    scales = torch.ones(8, 8)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="page must be"):
        ops.kv8_plan(i, i, i, i, i, i, i, i, i, page=20)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.kv8_plan(i, i, i, i, i, i, i, i, i, page=64)
    with pytest.raises(ValueError, match="lengths"):
        ops.kv8_plan(i[:0], i, i, i, i, i, i, i, i, page=64)
    with pytest.raises(ValueError, match="int8 or"):
        ops.kv8_append(f, f, i, cache.half(), cache, scales, scales)
    with pytest.raises(ValueError, match="positions"):
        ops.kv8_append(f, f, i, cache[:, :, :20], cache, scales, scales)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.kv8_append(f, f, i, cache, cache, scales, scales)
    with pytest.raises(ValueError, match="pages, kv_heads"):
        ops.kv8_attention(f, cache[0], cache, scales, scales, i, i, i, f, max_rows=1)


# ---------------------------------------------------------------- the plain forms

def test_plain_codes_are_torchs():
    v = np.concatenate([np.linspace(-500, 500, 20001), np.exp2(np.linspace(-14, 9, 4001))])
    v = v[np.abs(v) <= 448].astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(plain.round_codes(v.astype(np.float64), torch.float8_e4m3fn), want.astype(np.float64))
    assert np.array_equal(plain.round_codes(v.astype(np.float64), torch.int8), torch.from_numpy(v).round().clamp(-127, 127).numpy())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_plain_scale_is_the_smallest(dtype):
    for largest in (0.0, 2.0 ** -126, 1.0, 127.0, 127.5, 448.0, 450.0, 3.3895313892515355e38):
        s = plain.scale_for(largest, dtype)
        assert s >= 2.0 ** -120 and largest <= plain.MOST[dtype] * s
        assert s == 2.0 ** -120 or largest > plain.MOST[dtype] * s / 2


def test_plain_plan_by_hand():
    table = np.full((3, 4), -1)
    table[0, :1], table[2, :2] = [7], [8, 9]
    out = plain.plan(np.array([16, 0, 20]), np.array([1, 17, -1]), table, np.array([1, 2, 3, 4, 5, 6]), np.array([4, 7]), 20, 16)
    assert out[0].tolist() == [[7, 5, -1, -1], [6, 1, -1, -1], [8, 9, -1, -1]]
    assert out[1].tolist() == [1, 8, 9, 4, 5, 6] and out[4].tolist() == [7, 9] and out[5].tolist() == [0, 0, 0]
    assert out[2].tolist() == [0, 1, 18, 18]
    assert out[3].tolist() == [80] + list(range(96, 112)) + [16, -1, -1]


def test_plain_attention_of_one_position_is_its_value():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(1, 4, 64)), rng.integers(-9, 9, (2, 2, 16, 64)) * 1.0, rng.integers(-9, 9, (2, 2, 16, 64)) * 1.0
    out, reach = plain.attention(q, k, v, np.ones((2, 2)), np.full((2, 2), 0.5), np.array([[1]]), [0], [0, 1], 0.125)
    assert np.array_equal(out[0], np.repeat(v[1, :, 0] * 0.5, 2, axis=0)) and (reach > 0).any()
