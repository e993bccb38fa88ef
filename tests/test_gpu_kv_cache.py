"""KV_APPEND_I8, KV_ATTENTION_I8 and KV_READ_F32 on the GPU against the operators in 64 bits (kv_ops.py)."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu


@pytest.fixture()
def own():
    """A session of its own: an error on a stream stays."""
    s = Session()
    yield s
    s.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def run(s, *cmds):
    assert s.submit([s.command(op, **f) for op, f in cmds]) == abi.OK
    assert s.sync() == abi.OK


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------

def append_case(s, heads, kv_heads, d, page, past, n, rotation=abi.ROTATE_HALF, rope_dim=0, ragged=True, layout="rows",
                in_place=False, with_q=True, theta=0.0, scaling=0.0, extra=0, host=False, change=None, seed=5):
    rng = np.random.default_rng(seed)
    batch, T = len(n), int(np.sum(n)) + extra
    c = kv.Cache(rng, batch, kv_heads, d, page, max(-(-(a + m) // page) for a, m in zip(past, n)) + 2)
    c.forget([a + m for a, m in zip(past, n)])
    for b, (a, m) in enumerate(zip(past, n)):   # a page begun by this call has a stale scale
        for pg in range(-(-a // page), -(-(a + m) // page)):
            c.ks[c.table[b, pg]] = np.nan if pg % 2 else 1e30
    q, k, v = (normal(rng, T, h, d) for h in (heads, kv_heads, kv_heads))
    if change:
        change(c, k, v)
    cache, bufs = kv.upload(s, c)
    gap = dict(layout="wide", gap=36, shift=4) if layout == "wide" else dict(layout=layout, batch=batch)
    rq, rk, rv = kv.Rows(q, **gap), kv.Rows(k, **gap), kv.Rows(v, **gap)
    ro = rq if in_place else kv.Rows(np.full_like(q, 7.0), **gap)
    past32, start32 = np.array(past, np.int32), kv.starts(n)
    held = [] if host else [s.upload(past32), s.upload(start32)]
    pp, sp = (past32.ctypes.data, start32.ctypes.data) if host else (held[0].ptr, held[1].ptr)
    f = dict(cache=cache, K=rk.upload(s), V=rv.upload(s), past=pp, seq_start=sp if ragged else None, batch=batch,
             tokens=T, rotation=rotation, rope_dim=rope_dim, theta_base=theta, scaling=scaling,
             **kv.strides("k", rk.strides), **kv.strides("v", rv.strides))
    if with_q:
        f.update(Q=rq.upload(s), heads=heads, **kv.strides("q", rq.strides), **kv.strides("o", ro.strides))
        f["Q_out"] = f["Q"] if in_place else ro.upload(s)
    run(s, (abi.OP_KV_APPEND_I8, f))
    got = kv.download(s, c, bufs)
    used = T - extra
    kv.append(c, k[:used], v[:used], past, n, rotation, rope_dim, theta or 1e4, scaling or 1.0)
    # Steps of the same roundings: the same codes and scales, and every other slot as it was.
    for name in ("ks", "vs", "k", "v"):
        assert np.array_equal(got[name], getattr(c, name), equal_nan=name in ("ks", "vs")), name
    if with_q:
        out = ro.download(s)
        position = np.concatenate([a + np.arange(m) for a, m in zip(past, n)])
        want = kv.turned(q[:used], position, rotation, rope_dim, theta or 1e4, scaling or 1.0)
        # A cosine next to a border of f32 may round the other way: 2^-24 of it, of both terms.
        assert np.all(np.abs(out[:used] - want) <= 2.0**-24 * 2 * (np.abs(q[:used]).max() + np.abs(want)))
        if not in_place:
            assert np.all(out[used:] == 7.0)
        if layout == "wide":
            assert np.all(np.isnan(ro.rest))
        if not in_place:
            assert np.array_equal(rq.download(s), q)
    kv.free(s, bufs, *held, rk.buffer, rv.buffer, *([rq.buffer] if with_q else []),
            *([ro.buffer] if with_q and not in_place else []))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d,heads,kv_heads", [(16, 2, 1), (64, 8, 8), (80, 6, 2), (128, 8, 2), (256, 3, 3)])
def test_append_pages_and_heads(gpu, page, d, heads, kv_heads):
    """Sequences that begin a page, go on in one, end at its end, pass over several; one without tokens."""
    n = [1, page, 0, 3 * page + 5, 17, page - 3]
    append_case(gpu, heads, kv_heads, d, page, [0, 0, 9, page // 2 + 1, page - 1, 3], n)


@pytest.mark.parametrize("rotation,rope_dim", [(0, 0), (1, 0), (1, 32), (2, 0), (2, 20), (1, 2)])
@pytest.mark.parametrize("layout", ["rows", "wide", "heads"])
def test_append_rotations_and_layouts(gpu, rotation, rope_dim, layout):
    n, past = [5, 5, 5], [0, 30, 1000]
    append_case(gpu, 8, 4, 64, 32, past, n, rotation, rope_dim, ragged=False, layout=layout)
    append_case(gpu, 8, 4, 64, 32, past, n, rotation, rope_dim, ragged=layout != "heads", layout=layout, in_place=True)


@pytest.mark.parametrize("batch", [1, 3, 64, 65, 200])
def test_append_one_token_each(gpu, batch):
    past = [(37 * b) % 99 for b in range(batch)]
    append_case(gpu, 8, 2, 128, 16, past, [1] * batch, ragged=False)
    append_case(gpu, 8, 2, 128, 16, past, [1] * batch, ragged=True, with_q=False)


@pytest.mark.parametrize("d,page,n", [(64, 128, [200] + [1] * 39), (128, 256, [1] * 7 + [300] + [2] * 8),
                                      (256, 256, [300, 200]), (80, 256, [6] * 20 + [256, 0, 5])])
@pytest.mark.parametrize("rotation", [0, 1, 2])
def test_append_one_long_among_short(gpu, d, page, n, rotation):
    """Ragged sequences with many times the mean's tokens: a page's tokens are taken in several rounds."""
    append_case(gpu, 4, 2, d, page, [(53 * b) % 300 for b in range(len(n))], n, rotation=rotation)
    append_case(gpu, 4, 2, d, page, [page * (b % 2) for b in range(len(n))], n, rotation=rotation, with_q=False, layout="wide")


def test_append_far_positions_and_bases(gpu):
    append_case(gpu, 2, 1, 128, 256, [131000, 70000], [9, 300])
    append_case(gpu, 2, 1, 128, 256, [131000, 70000], [9, 300], theta=500000.0, scaling=0.125, rotation=2)


def test_append_host_lengths_and_rows_behind_the_last(gpu):
    append_case(gpu, 4, 2, 64, 16, [3, 40], [7, 21], host=True)
    append_case(gpu, 4, 2, 64, 16, [3, 40], [7, 21], extra=5, layout="wide")


@pytest.mark.parametrize("what", ["zero", "tiny", "huge", "nan", "inf", "nan_before", "zero_before"])
def test_append_scales_at_the_borders(gpu, what):
    """Zero and denormal pages, values at the end of f32, infinities and NaN, a page whose kept tokens are all zero."""
    def change(c, k, v):
        if what == "zero":
            k[:], v[:] = 0, 0
        if what == "tiny":
            k[:], v[:] = k * np.float32(1e-38), v * np.float32(1e-40)
        if what == "huge":
            k[:], v[:] = k * np.float32(5e37), v * np.float32(8e37)
        if what in ("nan", "inf"):
            k[4, 1, 3] = v[11, 0, 60] = np.nan if what == "nan" else -np.inf
        if what == "nan_before":
            c.ks[c.table[0, 0], 1] = c.vs[c.table[1, 0], 0] = np.nan
        if what == "zero_before":
            c.ks[c.table[0, 0]] = c.vs[c.table[1, 0]] = 0
    rotation = 0 if what in ("nan", "inf", "huge", "tiny") else 1
    if what in ("nan", "inf"):
        # Codes under a NaN scale are unspecified: only the scales, and every other page's codes, are compared.
        rng = np.random.default_rng(5)
        c = kv.Cache(rng, 2, 2, 64, 16, 4)
        k, v = normal(rng, 24, 2, 64), normal(rng, 24, 2, 64)
        change(c, k, v)
        cache, bufs = kv.upload(gpu, c)
        held = [gpu.upload(x) for x in (k, v, np.array([5, 2], np.int32))]
        run(gpu, (abi.OP_KV_APPEND_I8, dict(cache=cache, K=held[0].ptr, V=held[1].ptr, past=held[2].ptr, batch=2, tokens=24)))
        got = kv.download(gpu, c, bufs)
        kv.append(c, k, v, [5, 2], [12, 12], 0)
        assert np.isnan(c.ks).sum() == np.isnan(c.vs).sum() == 1
        for codes, scales in (("k", "ks"), ("v", "vs")):
            assert np.array_equal(got[scales], getattr(c, scales), equal_nan=True)
            fine = ~np.isnan(getattr(c, scales))
            assert np.array_equal(got[codes][fine], getattr(c, codes)[fine])
        kv.free(gpu, bufs, *held)
        return
    append_case(gpu, 4, 2, 64, 16, [5, 2], [12, 12], rotation, change=change)


def test_append_products_that_round_to_a_half(gpu):
    """x / scale in f32 is a whole number and a half where the exact product is not: the code goes by the f32 product."""
    largest = np.float32(3.3)
    inv = np.float32(1) / (largest * (np.float32(1) / np.float32(127)))
    x = ((np.arange(126)[:, None] + 0.5) / inv).astype(np.float32)
    x = (x.view(np.int32) + np.arange(-2, 3)).view(np.float32).reshape(-1)
    exact = x.astype(np.float64) * np.float64(inv)
    x = x[((x * inv) % 1 == 0.5) & (exact % 1 != 0.5)]
    assert x.size > 30 and (exact % 1 < 0.5).any()

    def change(c, k, v):
        v[:] = np.resize(np.concatenate([x, -x]), v.shape)
        v[:, :, 0] = largest
        k[:] = v[:, :, ::-1]
    append_case(gpu, 1, 1, 256, 16, [0, 16], [16, 3], rotation=0, change=change)


def test_append_again_and_further_back(gpu):
    """The same tokens twice give the same; a sequence taken back to an earlier length goes on from there."""
    rng = np.random.default_rng(8)
    c = kv.Cache(rng, 1, 2, 64, 16, 6)
    cache, bufs = kv.upload(gpu, c)
    for past, m in ((0, 21), (21, 7), (21, 7), (19, 3), (2, 40)):
        k, v = normal(rng, m, 2, 64), normal(rng, m, 2, 64) * 3
        held = [gpu.upload(x) for x in (k, v, np.array([past], np.int32))]
        for _ in range(2):
            run(gpu, (abi.OP_KV_APPEND_I8, dict(cache=cache, K=held[0].ptr, V=held[1].ptr, past=held[2].ptr, batch=1,
                                                tokens=m, rotation=1)))
            kv.append(c, k, v, [past], [m], 1)
            got = kv.download(gpu, c, bufs)
            for name in got:
                assert np.array_equal(got[name], getattr(c, name)), (past, name)
        kv.free(gpu, *held)
    kv.free(gpu, bufs)


# ---------------------------------------------------------------------------
# Read
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("d,kv_heads,layout", [(16, 1, "rows"), (80, 3, "wide"), (128, 8, "rows"), (256, 2, "wide")])
def test_read(gpu, page, d, kv_heads, layout):
    rng = np.random.default_rng(page + d)
    first, n = [0, page - 1, 5, 3 * page], [1, 2 * page + 3, 0, page]
    c = kv.Cache(rng, 4, kv_heads, d, page, 6).forget([a + m for a, m in zip(first, n)])
    cache, bufs = kv.upload(gpu, c)
    T = sum(n) + 3
    gap = dict(layout=layout, gap=20, shift=1)
    rk, rv = (kv.Rows(np.full((T, kv_heads, d), 7.0), **gap) for _ in range(2))
    held = [gpu.upload(np.array(first, np.int32)), gpu.upload(kv.starts(n))]
    run(gpu, (abi.OP_KV_READ_F32, dict(cache=cache, K=rk.upload(gpu), V=rv.upload(gpu), first=held[0].ptr,
                                       seq_start=held[1].ptr, batch=4, tokens=T, **kv.strides("k", rk.strides),
                                       **kv.strides("v", rv.strides))))
    k, v = rk.download(gpu), rv.download(gpu)
    at = 0
    for b, (a, m) in enumerate(zip(first, n)):
        for got, want in zip((k, v), c.values(b, a + m)):
            assert np.array_equal(got[at:at + m], want[:, a:].transpose(1, 0, 2).astype(np.float32))
        at += m
    assert np.all(k[at:] == 7) and np.all(v[at:] == 7)
    if layout == "wide":
        assert np.all(np.isnan(rk.rest)) and np.all(np.isnan(rv.rest))
    kv.free(gpu, bufs, rk.buffer, rv.buffer, *held)


def test_read_one_side_to_host_memory(gpu):
    """Uniform, from the beginning, one tensor, staged: the rest of the caller's array stays."""
    rng = np.random.default_rng(2)
    c = kv.Cache(rng, 2, 2, 64, 32, 3)
    cache, bufs = kv.upload(gpu, c)
    want = [np.stack([c.values(b, 50)[i] for b in range(2)]).astype(np.float32) for i in range(2)]
    for i, name in enumerate("KV"):
        out = np.full((2, 2, 50, 64), 5, np.float32)
        run(gpu, (abi.OP_KV_READ_F32, {"cache": cache, name: out.ctypes.data, "batch": 2, "tokens": 100,
                                       **kv.strides(name.lower(), (2 * 50 * 64, 64, 50 * 64))}))
        assert np.array_equal(out, want[i])
    kv.free(gpu, bufs)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def attention_case(s, heads, kv_heads, d, page, kv_len, n, causal=1, ragged=True, layout="rows", in_place=False, scale=0.0,
                   extra=0, hints=True, q_factor=1.0, seed=11, change=None, bounds=True):
    rng = np.random.default_rng(seed)
    batch, T = len(n), int(np.sum(n)) + extra
    c = kv.Cache(rng, batch, kv_heads, d, page, max(1, max(-(-int(x) // page) for x in kv_len)) + 1).forget(kv_len)
    q = normal(rng, T, heads, d) * np.float32(q_factor)
    if change:
        change(c, q)
    cache, bufs = kv.upload(s, c)
    gap = dict(layout="wide", gap=36, shift=3) if layout == "wide" else dict(layout=layout, batch=batch)
    rq = kv.Rows(q, **gap)
    ro = rq if in_place else kv.Rows(np.full_like(q, 7.0), **gap)
    held = [s.upload(np.array(kv_len, np.int32)), s.upload(kv.starts(n))]
    f = dict(cache=cache, Q=rq.upload(s), kv_len=held[0].ptr, seq_start=held[1].ptr if ragged else None, batch=batch,
             tokens=T, heads=heads, causal=causal, scale=scale, **kv.strides("q", rq.strides), **kv.strides("o", ro.strides))
    if hints:
        f.update(max_tokens=max(n), max_kv=max(1, max(kv_len)))
    f["O"] = f["Q"] if in_place else ro.upload(s)
    run(s, (abi.OP_KV_ATTENTION_I8, f))
    out = ro.download(s)
    used = T - extra
    want, bound = kv.attention(c, q[:used], kv_len, n, causal, scale)
    if bounds:
        off = np.abs(out[:used] - want)
        assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(off > bound)[:3].tolist())
        if not in_place:
            assert np.all(out[used:] == 7.0)
        if layout == "wide":
            assert np.all(np.isnan(ro.rest))
    kv.free(s, bufs, *held, rq.buffer, *([] if in_place else [ro.buffer]))
    return out, want


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 255, 256, 300, 1000]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d,heads,kv_heads", [(16, 1, 1), (48, 3, 3), (64, 8, 8), (80, 12, 4), (128, 8, 2), (128, 32, 2),
                                              (192, 5, 1), (256, 4, 2)])
def test_attention_one_token(gpu, page, d, heads, kv_heads):
    attention_case(gpu, heads, kv_heads, d, page, LENGTHS, [1] * len(LENGTHS), ragged=False)


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("d,heads,kv_heads,page", [(64, 4, 4, 16), (80, 6, 2, 32), (128, 8, 1, 64), (112, 20, 4, 128),
                                                   (256, 4, 4, 256), (16, 2, 1, 16)])
def test_attention_ragged(gpu, causal, d, heads, kv_heads, page):
    """A few tokens, many, none; cached lengths shorter than the tokens, so that causal rows see nothing."""
    n = [1, 5, 0, 17, 130, 2, 64, 33, 9, 1]
    kv_len = [700, 5, 33, 16, 131, 0, 1500, 10, 259, 1]
    attention_case(gpu, heads, kv_heads, d, page, kv_len, n, causal)
    attention_case(gpu, heads, kv_heads, d, page, kv_len, n, causal, hints=False, extra=4, layout="wide")


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 64, 100, 128, 129, 257])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (5, 1)])
def test_attention_row_counts(gpu, n, heads, kv_heads):
    attention_case(gpu, heads, kv_heads, 64, 32, [n + 77, n], [n, n], ragged=False)
    attention_case(gpu, heads, kv_heads, 128, 16, [n + 300], [n], ragged=False, causal=0)


@pytest.mark.parametrize("layout,in_place", [("heads", False), ("heads", True), ("wide", False), ("wide", True), ("rows", True)])
@pytest.mark.parametrize("n,kv_len", [(1, 3000), (6, 500), (70, 200)])
def test_attention_layouts_and_in_place(gpu, layout, in_place, n, kv_len):
    attention_case(gpu, 8, 2, 128, 16, [kv_len, kv_len - 100], [n, n], ragged=False, layout=layout, in_place=in_place)


@pytest.mark.parametrize("batch,n,kv_len", [(1, 1, 20000), (1, 3, 9001), (2, 40, 6000), (70, 1, 300), (3, 200, 2000),
                                            (1, 1, 70001), (130, 1, 65)])
def test_attention_long_and_many(gpu, batch, n, kv_len):
    """Keys split over workgroups, and more sequences than a wave has lanes."""
    lens = [max(n, kv_len - 37 * b % 150) for b in range(batch)]
    attention_case(gpu, 4, 1, 64, 64, lens, [n] * batch, ragged=False)
    attention_case(gpu, 4, 1, 64, 64, lens, [n] * batch, ragged=True, hints=False)


def test_attention_uneven_lengths(gpu):
    """One sequence that is far longer than the others of its batch."""
    attention_case(gpu, 8, 4, 128, 16, [12000, 3, 50, 1, 700, 16], [1] * 6, ragged=False)
    attention_case(gpu, 8, 4, 128, 16, [12000, 3, 50, 1, 700, 16], [1, 2, 30, 1, 1, 5])


@pytest.mark.parametrize("q_factor,scale", [(30.0, 0.0), (1e-3, 0.0), (1.0, 2.0), (1e20, 1e-21), (1e-30, 1e29), (0.0, 0.0)])
def test_attention_sizes_of_scores(gpu, q_factor, scale):
    """Softmax that picks one key, that is flat, queries near the ends of f32, and zero queries."""
    attention_case(gpu, 4, 2, 64, 16, [300, 40, 9], [1, 20, 9], q_factor=q_factor, scale=scale)
    attention_case(gpu, 4, 2, 64, 16, [3000], [1], q_factor=q_factor, scale=scale)


def test_attention_scales_far_apart(gpu):
    """Pages whose scales differ by 10^12 and pages of zeros: each product keeps its own weight."""
    def change(c, q):
        r = np.random.default_rng(1)
        c.vs *= (10.0 ** r.uniform(-9, 3, c.vs.shape)).astype(np.float32)
        c.ks[c.table[0, 1]] = 0
        c.vs[c.table[0, 2]] = 0
        c.vs[c.table[1, :12]] = 0   # a whole sequence's values
    attention_case(gpu, 4, 2, 64, 16, [200, 180], [1, 1], ragged=False, change=change)
    attention_case(gpu, 4, 2, 64, 16, [200, 180], [40, 7], change=change)


@pytest.mark.parametrize("n", [1, 70])
def test_attention_not_finite(gpu, n):
    """A NaN or infinite query row, and a page with such a scale, give NaN where they are seen, and only there."""
    def change(c, q):
        q[0, 1, 5] = np.nan
        q[n, 0, 0] = np.inf
        c.ks[c.table[2, 3], 0] = np.nan
        c.vs[c.table[3, 0], 1] = np.nan
    kv_len = [n + 90] * 5
    out, _ = attention_case(gpu, 4, 2, 64, 16, kv_len, [n] * 5, ragged=False, change=change, bounds=False)
    nan = np.isnan(out)
    want = np.zeros(out.shape, bool)
    want[0, 1] = want[n, 0] = True
    see = 90 + np.arange(n)
    want[2 * n:3 * n, :2] = (see >= 48)[:, None, None]
    want[3 * n:4 * n, 2:] = True
    assert np.array_equal(nan, want)


# ---------------------------------------------------------------------------
# What the host cannot check
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bad", ["page_high", "page_negative", "long", "negative", "falling", "beyond", "more_than_told"])
@pytest.mark.parametrize("op", ["append", "attention", "attention_many", "read"])
def test_bad_arrays_fail_the_stream(own, op, bad):
    """Out of range on the device: the sync says so; the guards around the outputs stay."""
    rng = np.random.default_rng(1)
    c = kv.Cache(rng, 3, 2, 64, 16, 8)
    lengths, n = np.array([40, 3, 90], np.int32), [40, 4, 40] if op == "attention_many" else [2, 1, 3]
    start = kv.starts(n)
    if bad == "page_high":
        c.table[2, 5] = c.pages
    if bad == "page_negative":
        c.table[0, 2] = -7
    if bad == "long":
        lengths[1] = 129
    if bad == "negative":
        lengths[2] = -1
    if bad == "falling":
        start[1], start[2] = 3, 2
    if bad == "beyond":
        start[3] += 1
    hints = dict(max_tokens=max(n), max_kv=128)
    if bad == "more_than_told":
        if not op.startswith("attention"):
            pytest.skip("nothing is told")
        hints = dict(max_tokens=max(n), max_kv=64)
    if op == "read" and bad in ("page_high", "page_negative"):
        lengths = np.array([32, 3, 78], np.int32)   # the bad page is read
    T = sum(n)
    cache, bufs = kv.upload(own, c)
    rows = own.upload(np.full((T + 64, 4, 64), 7, np.float32))
    x = own.upload(normal(rng, T + 64, 4, 64))
    held = [own.upload(lengths), own.upload(start)]
    f = dict(cache=cache, batch=3, tokens=T, seq_start=held[1].ptr)
    if op == "append":
        if bad.startswith("page"):   # the new tokens' own page
            lengths = np.array([38, 3, 88], np.int32)
            own.write(held[0], lengths)
        f.update(K=x.ptr, V=x.ptr, past=held[0].ptr, Q=x.ptr, Q_out=rows.ptr, heads=4, rotation=1)
        code = abi.OP_KV_APPEND_I8
    elif op == "read":
        f.update(K=rows.ptr, V=None, first=held[0].ptr)
        code = abi.OP_KV_READ_F32
    else:
        f.update(Q=x.ptr, O=rows.ptr, kv_len=held[0].ptr, heads=4, causal=0, **hints)
        code = abi.OP_KV_ATTENTION_I8
    assert own.submit([own.command(code, **f)]) == abi.OK
    assert own.sync() == abi.ERR_DEVICE_ERROR
    out = np.empty((T + 64, 4, 64), np.float32)
    other = Session()
    try:
        assert other.lib.vnpu_buffer_copy(other.stream, out.ctypes.data_as(C.c_void_p), C.c_void_p(rows.ptr), out.nbytes,
                                          abi.COPY_D2H) == abi.OK
    finally:
        other.close()
    assert np.all(out[T:] == 7)


@pytest.mark.parametrize("n,told", [([3, 1, 2], 2), ([40, 1, 2], 39), ([1, 200, 1], 1)])
def test_more_tokens_than_told_fail_the_stream(own, n, told):
    """A sequence with more tokens than max_tokens says, met by either kernel or by none."""
    c = kv.Cache(np.random.default_rng(1), 3, 2, 64, 16, 20)
    cache, _ = kv.upload(own, c)
    T = sum(n)
    q, o = own.alloc(T * 4 * 64 * 4), own.alloc(T * 4 * 64 * 4)
    lengths, start = own.upload(np.array([300, 250, 200], np.int32)), own.upload(kv.starts(n))
    f = dict(cache=cache, Q=q, O=o, kv_len=lengths.ptr, seq_start=start.ptr, batch=3, tokens=T, heads=4, causal=1)
    run(own, (abi.OP_KV_ATTENTION_I8, dict(f, max_tokens=max(n))))
    assert own.submit([own.command(abi.OP_KV_ATTENTION_I8, **dict(f, max_tokens=told))]) == abi.OK
    assert own.sync() == abi.ERR_DEVICE_ERROR


def test_refused_commands_fail_the_stream(own):
    c = kv.Cache(np.random.default_rng(1), 1, 1, 64, 16, 2)
    cache, _ = kv.upload(own, c)
    x = own.alloc(4096)
    host = np.zeros((c.pages, 1, 16, 64), np.int8)
    args = abi.KvReadArgs(cache=cache, K=x.ptr, batch=1, tokens=4)
    assert own.lib.vnpu_kv_read_f32(own.stream, C.byref(args)) == abi.OK
    args.cache.k = host.ctypes.data   # the cache is not staged
    assert own.lib.vnpu_kv_read_f32(own.stream, C.byref(args)) == abi.ERR_DEVICE_ERROR
