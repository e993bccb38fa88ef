"""KV_ATTENTION_I8 where weights and value scales lie far apart: each row against 64 bits within a bound of its own, made of
what the row sees and weighs."""
import numpy as np
import pytest

import kv_ops as kv
from vnpu_mi355x import abi

pytestmark = pytest.mark.gpu

EPS = 2.0**-24   # half a step of f32


def rows_of(c, b, h, kv_head, q, kv_len, causal, scale, last):
    """Query head h of one sequence, q [tokens][D]: (o, bound) [tokens][D] in 64 bits.

    A score's error, in what its weight is off by: the query's whole numbers (half a step of 2^-23 of its largest element,
    one f32 rounding of as much), and 8 roundings of the score and the same of the largest.  A weight: twice that, 4
    roundings of exponential and products, 2^-22 as digits or halves.  Sums over keys, of numerator and denominator:
    a rounding for every 16 keys of each, 16 more for waves, parts and the division.  All of them relative to the row's own
    sum of p |v|.  Behind these the last place of the weights' parts: `last` of the largest p * scale among the same 64 keys
    for each; and exponentials below 2^-126 are 0."""
    k, v = (x[kv_head] for x in c.values(b, kv_len))
    m, n, D = q.shape[0], kv_len, c.head_dim
    s = q.astype(np.float64) @ k.T * scale
    see = np.arange(n)[None, :] < (n - m + 1 + np.arange(m)[:, None] if causal else n)
    s = np.where(see, s, -np.inf)
    top = s.max(axis=1, keepdims=True)
    some = np.isfinite(top[:, 0])
    p = np.exp(s - np.where(np.isfinite(top), top, 0))
    seen = np.where(see, p, 0)
    total = seen.sum(axis=1, keepdims=True)
    total = np.where(total > 0, total, 1)
    p = seen / total
    # Rows that see a scale that is no number are compared elsewhere; to the others it is 0 times nothing.
    vs = c.vs[c.table[b, np.arange(n) // c.page], kv_head].astype(np.float64)
    v, vs = np.where(np.isfinite(v), v, 0), np.where(np.isfinite(vs), vs, 0)
    o, mass = p @ v, p @ np.abs(v)
    ks = np.where(see, np.abs(k).sum(axis=1)[None, :], 0).max(axis=1)
    off = scale * ks * np.abs(q).max(axis=1) * 2.0**-23
    off += 8 * EPS * np.where(see, np.abs(np.where(see, s, 0)), 0).max(axis=1)
    rel = 2 * off + 4 * EPS + 2.0**-22 + 2 * (-(-n // 16) + 16) * EPS
    pad = -n % 64
    w = np.pad(p * vs, ((0, 0), (0, pad))).reshape(m, -1, 64).max(axis=2)
    codes = np.abs(np.where(vs[:, None] > 0, v / np.where(vs > 0, vs, 1)[:, None], 0))
    codes = np.pad(codes, ((0, pad), (0, 0))).reshape(-1, 64, D).sum(axis=1)
    bound = rel[:, None] * mass + last * (w @ codes) + 2.0**-126 * (see @ np.abs(v))
    return np.where(some[:, None], o, 0), bound


def check(s, c, q, kv_len, n, heads, causal=1, scale=0.0, nan=None, last=None, **more):
    """Runs one call over uniform or ragged sequences and compares every row; returns the largest share of its bound."""
    D, G, batch = c.head_dim, c.kv_heads, len(n)
    used = scale if scale > 0 else float(np.float32(1.0) / np.sqrt(np.float32(D)))
    cache, bufs = kv.upload(s, c)
    start, lens = s.upload(kv.starts(n)), s.upload(np.array(kv_len, np.int32))
    x, y = s.upload(q), s.upload(np.full_like(q, 7.0))
    ragged = len(set(n)) > 1
    assert s.submit([s.command(abi.OP_KV_ATTENTION_I8, cache=cache, Q=x, O=y, kv_len=lens, seq_start=start.ptr if ragged else None,
                               batch=batch, tokens=sum(n), heads=heads, max_tokens=max(n), max_kv=max(kv_len), causal=causal,
                               scale=scale, **more)]) == abi.OK
    assert s.sync() == abi.OK
    out = s.download(y, np.float32, q.shape)
    kv.free(s, bufs, start, lens, x, y)
    # Four digits and four of the remainder for up to 16 rows of a kv head (8 above 128 dimensions).  Else two f16 parts in a
    # unit that the largest product is at most 2^12 below: half of 2^-24 of 2^14.
    last = last or (2.0**-56 if not ragged and n[0] * heads // G <= (16 if D <= 128 else 8) else 2.0**-27)
    at, worst = 0, 0.0
    for b, m in enumerate(n):
        for h in range(heads):
            got = out[at:at + m, h]
            want, bound = rows_of(c, b, h, h // (heads // G), q[at:at + m, h], int(kv_len[b]), causal, used, last)
            rows = np.ones(m, bool) if nan is None else ~nan[at:at + m, h]
            assert np.all(np.isnan(got[~rows]))
            if not rows.any():
                continue
            off = np.abs(got[rows] - want[rows])
            over = ~(off <= bound[rows])
            assert not over.any(), (b, h, np.argwhere(over)[:3].tolist(), float((off / bound[rows]).max()),
                                    float(np.abs(off).max() / np.abs(want[rows]).max()))
            worst = max(worst, float((off / np.where(bound[rows] > 0, bound[rows], 1)).max()))
        at += m
    return worst


def lean(rng, c, n, heads, weight, at, kv_len, noise=0.02):
    """Queries near one direction, keys of small random codes, but key at(b) of each sequence along it: with the scale that
    is returned it has `weight` of the softmax over kv_len keys."""
    D = c.head_dim
    u = rng.choice([-1.0, 1.0], D)
    q = (u + noise * rng.standard_normal((sum(n), heads, D))).astype(np.float32)
    c.k[:] = rng.integers(-6, 7, c.k.shape)
    c.ks[:] = np.float32(0.01)
    for b, length in enumerate(kv_len):
        j = at(length)
        c.k[c.table[b, j // c.page], :, j % c.page] = 100 * u
    return q, float(np.log(weight / (1 - weight) * max(kv_len)) / D)   # its score is D * 100 * 0.01


PLACES = {"first": lambda n: 0, "second_chunk": lambda n: min(n - 1, 70), "last": lambda n: n - 1,
          "middle": lambda n: n // 2}


@pytest.mark.parametrize("weight", [0.5, 0.96, 0.9999, 0.9999999])
@pytest.mark.parametrize("place", list(PLACES))
@pytest.mark.parametrize("silent", [True, False])
@pytest.mark.parametrize("n,heads,kv_heads,d", [(1, 2, 2, 128), (1, 8, 2, 64), (2, 8, 2, 80), (3, 8, 2, 128), (1, 4, 1, 256),
                                                (2, 4, 1, 192), (4, 4, 1, 128), (5, 2, 1, 112),
                                                (70, 2, 1, 64), (130, 1, 1, 128), (33, 2, 2, 80), (40, 2, 2, 256)])
def test_one_key_with_most_of_the_weight(gpu, n, heads, kv_heads, d, silent, place, weight):
    """The others, before and behind it, keep what their own small weights give, also where its values are all zero."""
    rng = np.random.default_rng(9)
    kv_len = [1500, 700, 130 + n, 61 + n, n]
    c = kv.Cache(rng, len(kv_len), kv_heads, d, 16, -(-max(kv_len) // 16))
    q, scale = lean(rng, c, [n] * len(kv_len), heads, weight, PLACES[place], kv_len)
    if silent:
        for b, length in enumerate(kv_len):
            j = PLACES[place](length)
            c.v[c.table[b, j // 16], :, :, j % 16] = 0
    check(gpu, c, q, kv_len, [n] * len(kv_len), heads, scale=scale, causal=0)


@pytest.mark.parametrize("weight", [0.96, 0.99999])
@pytest.mark.parametrize("silent", [True, False])
def test_one_key_with_most_of_the_weight_of_a_long_sequence(gpu, silent, weight):
    """A workgroup a sequence and head, 16 chunks a wave, and values that all have one sign behind the first key."""
    rng = np.random.default_rng(4)
    kv_len, d = [4096] * 16, 128
    c = kv.Cache(rng, 16, 8, d, 256, 16)
    c.v[:] = np.abs(c.v)
    q, scale = lean(rng, c, [1] * 16, 8, weight, PLACES["first"], kv_len)
    c.k[np.abs(c.k) != 100] = 0   # equal scores: every weight rounds the same way
    if silent:
        c.v[c.table[:, 0], :, :, 0] = 0
    check(gpu, c, q, kv_len, [1] * 16, 8, scale=scale)


@pytest.mark.parametrize("power", range(20, 33, 2))
@pytest.mark.parametrize("n,heads,kv_heads,d", [(1, 2, 2, 128), (70, 2, 1, 64), (70, 1, 1, 128), (33, 1, 1, 256)])
def test_the_chunk_of_a_key_without_values(gpu, n, heads, kv_heads, d, power):
    """The first key has all but 2^-power of the weight and no values; the few others, all alike, round the same way.  In
    tiles the unit has the largest product between 2^14 and 2^15 then: half of 2^-24 is 2^-39 of it."""
    rng = np.random.default_rng(power)
    kv_len = [64, 30, 200]
    c = kv.Cache(rng, 3, kv_heads, d, 16, 13)
    c.v[:] = np.maximum(np.abs(c.v), 1)
    q, scale = lean(rng, c, [n] * 3, heads, 1 - 2.0**-power, PLACES["first"], kv_len, noise=0)
    c.k[np.abs(c.k) != 100] = 0
    c.v[c.table[:, 0], :, :, 0] = 0
    check(gpu, c, q, kv_len, [n] * 3, heads, scale=scale, causal=0, last=2.0**-39 if n > 1 else None)


@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6, 1e8, 1e20])
@pytest.mark.parametrize("n,heads,kv_heads,d,page", [(1, 4, 2, 128, 16), (3, 4, 1, 64, 64), (1, 4, 4, 256, 16),
                                                     (4, 4, 1, 80, 32), (70, 2, 1, 64, 16), (70, 2, 1, 128, 64), (33, 1, 1, 256, 16)])
def test_quiet_pages_beside_loud_ones(gpu, n, heads, kv_heads, d, page, ratio):
    """Pages of large values with next to no weight leave the others theirs, in the same 64 keys and in others."""
    rng = np.random.default_rng(3)
    kv_len = [700, 64 + n]
    c = kv.Cache(rng, 2, kv_heads, d, page, -(-max(kv_len) // page))
    u = rng.choice([-1.0, 1.0], d)
    q = (u + 0.02 * rng.standard_normal((2 * n, heads, d))).astype(np.float32)
    c.k[:] = rng.integers(-6, 7, c.k.shape)
    c.ks[:] = np.float32(0.01)
    for loud in (c.table[0, 1], c.table[0, 400 // page], c.table[1, 0]):
        c.vs[loud] *= np.float32(ratio)
        c.k[loud] = (-100 * u).astype(np.int8)
    check(gpu, c, q, kv_len, [n, n], heads, scale=90.0 / d, causal=0)   # about e^-90 of the others
    check(gpu, c, q, kv_len, [n, n], heads, scale=20.0 / d, causal=0)


@pytest.mark.parametrize("what,value", [("vs", 1e6), ("vs", 1e30), ("vs", np.inf), ("vs", np.nan), ("ks", 1e20), ("ks", np.nan), ("ks", np.inf)])
@pytest.mark.parametrize("n,heads,kv_heads,d,page", [(2, 4, 2, 64, 16), (7, 2, 1, 128, 16), (16, 1, 1, 80, 16), (8, 2, 2, 256, 16),
                                                     (70, 2, 1, 64, 16), (200, 1, 1, 128, 64), (70, 1, 1, 256, 16)])
def test_pages_that_a_row_does_not_see(gpu, n, heads, kv_heads, d, page, what, value):
    """Earlier tokens of a causal call have nothing of a later one's scales; infinite ones give NaN to those that see them."""
    rng = np.random.default_rng(6)
    kv_len = [16 * page + 1, 2 * page + n - n % page + 1, page * (-(-n // page))]
    kv_len = [max(x, n) for x in kv_len]
    c = kv.Cache(rng, 3, kv_heads, d, page, -(-max(kv_len) // page))
    q = rng.standard_normal((3 * n, heads, d)).astype(np.float32)
    nan = np.zeros((3 * n, heads), bool)
    for b, length in enumerate(kv_len):
        last = (length - 1) // page
        getattr(c, what)[c.table[b, last]] = value
        sees = length - n + np.arange(n) >= last * page
        if not np.isfinite(value):
            nan[b * n:(b + 1) * n] = sees[:, None]
        elif what == "ks":   # scores as they are elsewhere for the rows that see it
            q[b * n:(b + 1) * n][sees] *= np.float32(1e-20)
    with np.errstate(all="ignore"):
        check(gpu, c, q, kv_len, [n] * 3, heads, nan=nan)


@pytest.mark.parametrize("n", [1, 3, 12, 70])
@pytest.mark.parametrize("spread", [2, 6, 14])
def test_scales_and_scores_over_orders_of_magnitude(gpu, n, spread):
    """Random scales of both sides, scores from flat to picking one key."""
    for seed, factor in enumerate((0.3, 3.0, 20.0)):
        rng = np.random.default_rng(seed)
        kv_len = [900, 65 + n, n]
        c = kv.Cache(rng, 3, 2, 64, 32, 29)
        c.vs *= (10.0 ** rng.uniform(-spread, 1, c.vs.shape)).astype(np.float32)
        c.ks *= (2.0 ** rng.uniform(-3, 1, c.ks.shape)).astype(np.float32)
        q = (factor * rng.standard_normal((3 * n, 4, 64))).astype(np.float32)
        check(gpu, c, q, kv_len, [n] * 3, 4)
        check(gpu, c, q[:sum([n, n, 1])], kv_len, [n, n, 1], 4)


@pytest.mark.parametrize("weight", [0.9, 0.99, 0.9945, 0.9999])
@pytest.mark.parametrize("batch,n,kv_heads,d,kv_len", [
    (16, 1, 8, 128, 131072),   # a workgroup a sequence and head
    (1, 4, 8, 64, 131072),     # keys split over workgroups
    (96, 64, 8, 64, 16384),    # tiles, whole
    (2, 70, 1, 256, 30000)])   # tiles, keys split
def test_weights_that_only_count_together(gpu, batch, n, kv_heads, d, kv_len, weight):
    """Weights of less than half a step of the largest each, and together a part of the sum.  Only the heaviest key has
    values, so that the result shows the sum of weights alone: relative error a rounding for each of 64 steps
    (exponentials, products, the kept sums of lanes, waves and parts, the division) and the score's 8 roundings.  All sequences share
    two pages, the second is used again and again."""
    page = 256
    k, v = np.zeros((2, kv_heads, page, d), np.int8), np.zeros((2, kv_heads, d, page), np.int8)
    u = np.random.default_rng(5).choice([-1, 1], d)
    k[0, :, 0], v[0, :, :, 0] = 100 * u, -50
    table = np.ones((batch, -(-kv_len // page)), np.int32)
    table[:, 0] = 0
    scales, q = np.full((2, kv_heads), 2.0**-7, np.float32), np.broadcast_to(u, (batch * n, kv_heads, d)).astype(np.float32)
    scale = np.float32(np.log(weight / (1 - weight) * kv_len) / (d * 100 * 2.0**-7))
    bufs = [gpu.upload(x) for x in (k, v, scales, table, q, np.full(batch, kv_len, np.int32))]
    cache = abi.KvCache(k=bufs[0].ptr, v=bufs[1].ptr, k_scales=bufs[2].ptr, v_scales=bufs[2].ptr, table=bufs[3].ptr, pages=2,
                        page_size=page, kv_heads=kv_heads, head_dim=d, table_ld=table.shape[1])
    out = gpu.alloc(q.nbytes)
    gpu.run(abi.OP_KV_ATTENTION_I8, cache=cache, Q=bufs[4], O=out, kv_len=bufs[5], batch=batch, tokens=batch * n,
            heads=kv_heads, scale=scale)
    got = gpu.download(out, np.float32, q.shape)
    score = float(scale) * d * 100 * 2.0**-7
    want = -50 * 2.0**-7 / (1 + (kv_len - 1) * np.exp(-score))
    off = float(np.abs(got / want - 1).max())
    assert off <= EPS * (64 + 2 * 8 * score), off
    kv.free(gpu, *bufs, out)
