"""KV_READ_F32 and KV_APPEND_I8 with f32 tensors in host memory that share one array: rows beside each other, one tensor behind
another, only one side, with a third tensor between."""
import numpy as np
import pytest

import kv_ops as kv
from vnpu_mi355x import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [0, 3, 40])
@pytest.mark.parametrize("v_first", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_read_both_sides_into_rows_of_one_array(gpu, gap, v_first, ragged):
    """Row t: K's heads, V's heads, `gap` floats that are the caller's own."""
    rng = np.random.default_rng(gap + 1)
    batch, heads, d, n = 2, 3, 32, [21, 40] if ragged else [21, 21]
    c = kv.Cache(rng, batch, heads, d, 16, 3)
    cache, bufs = kv.upload(gpu, c)
    side, T = heads * d, sum(n)
    rows = np.full((T + 2, 2 * side + gap), 7.0, np.float32)   # two rows behind the last
    start = kv.starts(n)
    k_at, v_at = (side, 0) if v_first else (0, side)
    step = rows.shape[1]
    strides = {**kv.strides("k", (n[0] * step, step, d)), **kv.strides("v", (n[0] * step, step, d))}
    assert gpu.submit([gpu.command(
        abi.OP_KV_READ_F32, cache=cache, K=rows.ctypes.data + 4 * k_at, V=rows.ctypes.data + 4 * v_at, batch=batch, tokens=T,
        seq_start=start.ctypes.data if ragged else None, **strides)]) == abi.OK and gpu.sync() == abi.OK
    at = 0
    for b, m in enumerate(n):
        for want, first in zip(c.values(b, m), (k_at, v_at)):
            want = want.transpose(1, 0, 2).reshape(m, side).astype(np.float32)
            assert np.array_equal(rows[at:at + m, first:first + side], want)
        at += m
    assert np.all(rows[:, 2 * side:] == 7) and np.all(rows[T:] == 7)
    kv.free(gpu, bufs)


@pytest.mark.parametrize("order", ["heads_of_both", "one_behind_the_other", "one_side_on_the_device"])
def test_read_both_sides_in_other_orders(gpu, order):
    rng = np.random.default_rng(8)
    heads, d, n = 4, 64, 37
    c = kv.Cache(rng, 1, heads, d, 32, 2)
    cache, bufs = kv.upload(gpu, c)
    want = [x.astype(np.float32) for x in c.values(0, n)]   # [heads][n][d]
    out = np.full(2 * heads * n * d + 5, 7.0, np.float32)
    other = gpu.upload(np.zeros(heads * n * d, np.float32))
    at, head = (n * d, 2 * n * d) if order == "heads_of_both" else (heads * n * d, n * d)
    k, v = out.ctypes.data, out.ctypes.data + 4 * at
    if order == "one_side_on_the_device":
        k = other.ptr
    assert gpu.submit([gpu.command(abi.OP_KV_READ_F32, cache=cache, K=k, V=v, batch=1, tokens=n,
                                   **kv.strides("k", (0, d, head)), **kv.strides("v", (0, d, head)))]) == abi.OK
    assert gpu.sync() == abi.OK
    body = out[:-5]
    if order == "heads_of_both":
        body = body.reshape(heads, 2, n, d).transpose(1, 0, 2, 3)
    else:
        body = body.reshape(2, heads, n, d)
    if order == "one_side_on_the_device":
        assert np.all(body[0] == 7) and np.array_equal(gpu.download(other, np.float32, want[0].shape), want[0])
    else:
        assert np.array_equal(body[0], want[0])
    assert np.array_equal(body[1], want[1]) and np.all(out[-5:] == 7)
    kv.free(gpu, bufs, other)


def test_append_from_rows_of_one_array(gpu):
    """Q, K and V of one projection in host memory, queries turned in place: K and V stay."""
    rng = np.random.default_rng(2)
    heads, kv_heads, d, n = 4, 2, 64, 23
    c = kv.Cache(rng, 1, kv_heads, d, 16, 3)
    cache, bufs = kv.upload(gpu, c)
    step = (heads + 2 * kv_heads) * d
    rows = rng.standard_normal((n, step)).astype(np.float32)
    before, past = rows.copy(), np.array([4], np.int32)
    at = [rows.ctypes.data + 4 * x for x in (0, heads * d, (heads + kv_heads) * d)]
    assert gpu.submit([gpu.command(abi.OP_KV_APPEND_I8, cache=cache, Q=at[0], Q_out=at[0], K=at[1], V=at[2],
                                   past=past.ctypes.data, batch=1, tokens=n, heads=heads, rotation=1, q_token_stride=step,
                                   o_token_stride=step, k_token_stride=step, v_token_stride=step)]) == abi.OK
    assert gpu.sync() == abi.OK
    q, k, v = (before[:, a:b].reshape(n, -1, d) for a, b in ((0, heads * d), (heads * d, (heads + kv_heads) * d),
                                                             ((heads + kv_heads) * d, step)))
    kv.append(c, k, v, [4], [n], 1)
    got = kv.download(gpu, c, bufs)
    assert all(np.array_equal(got[name], getattr(c, name)) for name in got)
    turned = kv.turned(q, 4 + np.arange(n), 1, 0).reshape(n, -1)
    # Two products with a cosine that may round the other way.
    assert np.all(np.abs(rows[:, :heads * d] - turned) <= 2.0**-24 * 2 * (np.abs(q).max() + np.abs(turned)))
    assert np.array_equal(rows[:, heads * d:], before[:, heads * d:])
    kv.free(gpu, bufs)
