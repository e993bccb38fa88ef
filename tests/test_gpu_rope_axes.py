"""ROPE_AXES_F32 on the GPU against rotations in 64 bits (serving_ops.py)."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
import serving_ops as ops
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def case(s, tokens, heads, kv_heads, d, sections, order=0, ladders=0, rotation=abi.ROTATE_HALF, layout="rows", batch=1, theta=0.0,
         scaling=0.0, in_place=False, positions=None, ld=0, host=False, shift=3, seed=4, change=None):
    rng = np.random.default_rng(seed)
    ld = ld or tokens
    where = rng.integers(0, 5000, (len(sections), ld)).astype(np.int32) if positions is None else positions
    gap = dict(layout="wide", gap=36, shift=shift) if layout == "wide" else dict(layout=layout, batch=batch)
    f = dict(batch=batch, tokens=tokens, head_dim=d, position_ld=ld if ld != tokens else 0, axes=len(sections),
             sections=(C.c_uint32 * 4)(*sections), order=order, ladders=ladders, rotation=rotation, theta_base=theta, scaling=scaling)
    held, sides = [], []
    for name, out, h in (("Q", "o", heads), ("K", "ko", kv_heads)):
        if not h:
            continue
        x = normal(rng, tokens, h, d)
        if change:
            change(x)
        rows = kv.Rows(x, **gap)
        to = rows if in_place else kv.Rows(np.full_like(x, 7.0), **gap)
        stride = rows.strides if rows.strides[0] else (tokens // batch * rows.strides[1], *rows.strides[1:])
        f.update({name: rows.upload(s), ("heads" if name == "Q" else "kv_heads"): h, **kv.strides(name.lower(), stride),
                  **kv.strides(out, stride)})
        f[name + "_out"] = f[name] if in_place else to.upload(s)
        sides.append((x, rows, to))
    if host:
        f["positions"] = where.ctypes.data
    else:
        held.append(s.upload(where))
        f["positions"] = held[0].ptr
    s.run(abi.OP_ROPE_AXES_F32, **f)
    results = []
    for x, rows, to in sides:
        got = to.download(s)
        want, bound = ops.rope_axes(x, where[:, :tokens], sections, order, ladders, rotation, theta or 1e4, scaling or 1.0)
        off = np.abs(got - want)
        if not change:
            assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(~(off <= bound))[:3].tolist())
        if layout == "wide":
            assert np.all(np.isnan(to.rest))
        if not in_place:
            assert np.array_equal(rows.download(s), x, equal_nan=True)
        results.append((x, got))
        kv.free(s, rows.buffer, *([] if in_place else [to.buffer]))
    kv.free(s, *held)
    return results


@pytest.mark.parametrize("d,sections", [(2, (1,)), (16, (8,)), (64, (16, 16)), (64, (8, 12, 12)), (80, (20, 20)), (80, (3, 17, 20)),
                                        (96, (5, 6, 7)), (128, (24, 20, 20)), (128, (16, 16, 16, 16)), (128, (1, 1, 1, 1)),
                                        (256, (100, 3, 24, 1)), (250, (61, 64)), (6, (1, 1))])
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("ladders", [0, 1])
@pytest.mark.parametrize("rotation", [1, 2])
def test_axes(gpu, d, sections, order, ladders, rotation):
    case(gpu, 13, 5, 2, d, sections, order, ladders, rotation)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 65535, 65535), (1, 14000, 14000), (7, 65535, 1)])
def test_as_many_heads_as_there_may_be(gpu, tokens, heads, kv_heads):
    case(gpu, tokens, heads, kv_heads, 2, (1,))


@pytest.mark.parametrize("tokens", [1, 2, 3, 63, 64, 65, 300, 1601])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (32, 8), (7, 0), (0, 3), (17, 9)])
def test_tokens_and_heads(gpu, tokens, heads, kv_heads):
    case(gpu, tokens, heads, kv_heads, 64, (8, 12, 12))


@pytest.mark.parametrize("layout", ["rows", "wide", "heads"])
@pytest.mark.parametrize("rotation", [1, 2])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("d,sections", [(64, (8, 12, 12)), (80, (9, 10, 11)), (64, (4, 8)), (72, (4, 4))])
def test_layouts(gpu, layout, rotation, in_place, d, sections):
    for shift in (3, 4):
        case(gpu, 24, 6, 3, d, sections, 1, 0, rotation, layout, batch=4, in_place=in_place, shift=shift)


def test_positions(gpu):
    """Far, negative, the borders of int32, not the same for an axis, of a longer array, in host memory; other bases."""
    rng = np.random.default_rng(1)
    far = rng.integers(-2**31, 2**31, (3, 40)).astype(np.int32)
    far[:, :3] = [[0, 2**31 - 1, -2**31]] * 3
    for theta, scaling in ((0, 0), (500000, 0.125), (100, 3)):
        case(gpu, 40, 4, 2, 128, (24, 20, 20), 1, positions=far, theta=theta, scaling=scaling)
        case(gpu, 40, 4, 2, 80, (20, 10, 10), ladders=1, rotation=2, theta=theta, scaling=scaling, ld=77, host=True)


def test_back_by_the_opposite_positions(gpu):
    """Turned there and back: two results' roundings."""
    rng = np.random.default_rng(2)
    where = rng.integers(0, 3000, (2, 50)).astype(np.int32)
    x, there = case(gpu, 50, 4, 0, 64, (16, 16), positions=where)[0]
    b, p = gpu.upload(there), gpu.upload(-where)
    gpu.run(abi.OP_ROPE_AXES_F32, Q=b, Q_out=b, positions=p, tokens=50, heads=4, head_dim=64, axes=2,
            sections=(C.c_uint32 * 4)(16, 16), rotation=abi.ROTATE_HALF)
    back = gpu.download(b, np.float32, x.shape)
    size = np.abs(x[..., :32]) + np.abs(x[..., 32:])
    assert np.all(np.abs(back - x) <= 4 * ops.EPS * np.concatenate((size, size), axis=-1))
    kv.free(gpu, b, p)


def test_one_axis_is_the_cache_s_rotation(gpu):
    """One axis of positions in a row against KV_APPEND_I8's queries, whose cosines and sines are rounded to f32."""
    rng = np.random.default_rng(3)
    c = kv.Cache(rng, 1, 1, 64, 16, 8)
    cache, bufs = kv.upload(gpu, c)
    q, k = normal(rng, 30, 4, 64), normal(rng, 30, 1, 64)
    bq, bk, bo, bt = gpu.upload(q), gpu.upload(k), gpu.alloc(q.nbytes), gpu.alloc(q.nbytes)
    past, where = gpu.upload(np.array([70], np.int32)), gpu.upload(np.arange(70, 100).astype(np.int32))
    gpu.run(abi.OP_KV_APPEND_I8, cache=cache, Q=bq, Q_out=bo, K=bk, V=bk, past=past, batch=1, tokens=30, heads=4,
            rotation=abi.ROTATE_HALF)
    gpu.run(abi.OP_ROPE_AXES_F32, Q=bq, Q_out=bt, positions=where, tokens=30, heads=4, head_dim=64, axes=1,
            sections=(C.c_uint32 * 4)(32), rotation=abi.ROTATE_HALF)
    a, b = (gpu.download(x, np.float32, q.shape) for x in (bo, bt))
    size = np.abs(q[..., :32]) + np.abs(q[..., 32:])
    assert np.all(np.abs(a - b) <= 4 * ops.EPS * np.concatenate((size, size), axis=-1))
    kv.free(gpu, bufs, bq, bk, bo, bt, past, where)


def test_values_that_are_not_finite_stay_in_their_pair(gpu):
    def change(x):
        x[2, 0, 5], x[3, 1, 60] = np.nan, np.inf
    for x, got in case(gpu, 6, 2, 2, 64, (10, 14), change=change):
        bad = ~np.isfinite(got)
        want = np.zeros(x.shape, bool)
        want[2, 0, [5, 5 + 24]] = True   # 24 pairs
        want[3, 1, 60] = True            # behind them: copied
        assert np.array_equal(bad, want) and got[3, 1, 60] == np.inf


def test_refused_calls_fail_the_stream():
    s = Session()
    try:
        x = s.alloc(4096)
        f = dict(Q=x, Q_out=x, positions=x, tokens=1, heads=1, head_dim=64, axes=1, sections=(C.c_uint32 * 4)(32), rotation=1)
        s.run(abi.OP_ROPE_AXES_F32, **f)
        assert s.submit([s.command(abi.OP_ROPE_AXES_F32, **{**f, "axes": 5})]) == abi.OK
        assert s.sync() == abi.ERR_DEVICE_ERROR
    finally:
        s.close()


def test_rows_beyond_32_bits(gpu):
    """Rows a long way apart: the last begins behind 2^32 floats."""
    stride, tokens, d = (1 << 31) + 64, 3, 64
    b = gpu.alloc(4 * (2 * stride + d))
    rng = np.random.default_rng(6)
    x = normal(rng, tokens, 1, d)
    for t in range(tokens):
        gpu.write(b, x[t], offset=4 * t * stride)
    where = rng.integers(0, 1000, (2, tokens)).astype(np.int32)
    p = gpu.upload(where)
    gpu.run(abi.OP_ROPE_AXES_F32, Q=b, Q_out=b, positions=p, tokens=tokens, heads=1, head_dim=d, axes=2, q_token_stride=stride,
            o_token_stride=stride, sections=(C.c_uint32 * 4)(12, 20), rotation=abi.ROTATE_HALF)
    want, bound = ops.rope_axes(x, where, (12, 20))
    for t in range(tokens):
        got = gpu.download(b, np.float32, (1, d), offset=4 * t * stride)
        assert np.all(np.abs(got - want[t]) <= bound[t])
    kv.free(gpu, b, p)
