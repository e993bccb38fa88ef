"""KV_PREFIX_ATTENTION_I8 on the GPU against attention over the whole sequences in 64 bits (serving_ops.py)."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
import serving_ops as ops
from gpu_ops import route
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


class Call:
    """A cache with a shared prefix, queries and the command over them."""

    def __init__(self, s, heads, kv_heads, d, page, prefix, mine, n, causal=1, ragged=True, layout="rows", in_place=False, scale=0.0,
                 extra=0, before=0, hints=True, q_factor=1.0, seed=11, change=None, forget=True):
        rng = np.random.default_rng(seed)
        self.s, self.n, self.causal, self.scale, self.before = s, n, causal, scale, before
        batch, T = len(n), before + int(np.sum(n)) + extra
        self.kv_len = [prefix + m for m in mine]
        self.c, self.table = ops.shared_cache(rng, batch, kv_heads, d, page, prefix, max(mine))
        c = self.c
        if forget:   # what no sequence has; the rows' entries for the prefix are not read
            used = np.zeros(c.pages, bool)
            used[self.table] = True
            for b, m in enumerate(mine):
                used[c.table[b, :-(-self.kv_len[b] // page)]] = True
                c.table[b, -(-self.kv_len[b] // page):] = [-1, 2**31 - 1, -2**31][b % 3]
            c.ks[~used], c.vs[~used] = np.nan, np.nan
        self.q = normal(rng, T, heads, d) * np.float32(q_factor)
        if change:
            change(self)
        self.cache, self.bufs = kv.upload(s, c)
        if forget and prefix:
            hidden = c.table.copy()
            hidden[:, :prefix // page] = -5
            s.write(self.bufs["table"], hidden)
        self.layout, self.in_place = layout, in_place
        gap = dict(layout="wide", gap=36, shift=3) if layout == "wide" else dict(layout=layout, batch=batch)
        self.rq = kv.Rows(self.q, **gap)
        self.ro = self.rq if in_place else kv.Rows(np.full_like(self.q, 7.0), **gap)
        start = before + kv.starts(n)
        self.held = [s.upload(np.array(self.kv_len, np.int32)), s.upload(start.astype(np.int32)),
                     s.upload(np.append(self.table, -9).astype(np.int32))]
        q = self.rq.upload(s)
        self.args = dict(cache=self.cache, Q=q, O=q if in_place else self.ro.upload(s), kv_len=self.held[0].ptr,
                         seq_start=self.held[1].ptr if ragged else None, batch=batch, tokens=T, heads=heads, causal=causal, scale=scale,
                         **kv.strides("q", self.rq.strides), **kv.strides("o", self.ro.strides))
        if hints:
            self.args.update(max_tokens=max(n), max_kv=max(1, max(self.kv_len)))
        self.prefix = prefix

    def command(self, **more):
        a = abi.KvAttentionArgs(**{**self.args, **more})
        return self.s.command(abi.OP_KV_PREFIX_ATTENTION_I8, attention=a, prefix_table=self.held[2].ptr, prefix_len=self.prefix)

    def run(self, **more):
        assert self.s.submit([self.command(**more)]) == abi.OK
        assert self.s.sync() == abi.OK
        return self.ro.download(self.s)

    def want(self):
        used = slice(self.before, self.before + int(np.sum(self.n)))
        return ops.prefix_attention(self.c, self.q[used], self.kv_len, self.n, self.causal, self.scale)

    def check(self, out):
        used = slice(self.before, self.before + int(np.sum(self.n)))
        want, bound = self.want()
        off = np.abs(out[used] - want)
        assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(~(off <= bound))[:3].tolist())
        if not self.in_place:
            assert np.all(out[:used.start] == 7.0) and np.all(out[used.stop:] == 7.0)
        if self.layout == "wide":
            assert np.all(np.isnan(self.ro.rest))

    def free(self):
        kv.free(self.s, self.bufs, *self.held, self.rq.buffer, *([] if self.in_place else [self.ro.buffer]))


def case(s, *a, **kw):
    x = Call(s, *a, **kw)
    x.check(x.run())
    x.free()


MINE = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 256, 300]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d,heads,kv_heads", [(16, 1, 1), (48, 3, 3), (64, 8, 8), (80, 12, 4), (128, 8, 2), (128, 32, 2),
                                              (192, 5, 1), (256, 4, 2)])
def test_one_token_each(gpu, page, d, heads, kv_heads):
    case(gpu, heads, kv_heads, d, page, 2 * page, MINE, [1] * len(MINE), ragged=False)
    case(gpu, heads, kv_heads, d, page, 5 * page, MINE[:2], [1] * 2)


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("d,heads,kv_heads,page", [(64, 4, 4, 16), (80, 6, 2, 32), (128, 8, 1, 64), (112, 20, 4, 128),
                                                   (256, 4, 4, 256), (16, 2, 1, 16)])
def test_ragged(gpu, causal, d, heads, kv_heads, page):
    """A few tokens, many, none; sequences that are all new tokens; rows before the first and behind the last."""
    n = [1, 5, 0, 17, 130, 2, 64, 33, 9, 1]
    mine = [400, 5, 0, 17, 131, 2, 500, 40, 259, 1]
    case(gpu, heads, kv_heads, d, page, 512, mine, n, causal)
    case(gpu, heads, kv_heads, d, page, 256, mine, n, causal, hints=False, before=3, extra=4, layout="wide")


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 16, 17, 31, 33, 64, 129])
@pytest.mark.parametrize("batch", [1, 2, 7])
def test_row_counts(gpu, batch, n):
    case(gpu, 8, 2, 64, 16, 208, [n + 20] * batch, [n] * batch, ragged=batch == 2)


# One pass over the prefix and what lies behind it, by tiles of 64 and 128 rows, each in one and in several ranges of
# keys; the ranges are joined where they are several.
@pytest.mark.parametrize("d", range(16, 257, 16))
@pytest.mark.parametrize("batch,n,prefix,parts", [(40, 33, 64, False), (2, 150, 1024, True)])
def test_through_the_prefix(gpu, d, batch, n, prefix, parts):
    x = Call(gpu, 8, 4, d, 16, prefix, [n + 45 + b % 7 for b in range(batch)], [n - b % 3 for b in range(batch)])
    way = route(abi.OP_KV_PREFIX_ATTENTION_I8, attention=abi.KvAttentionArgs(**x.args), prefix_table=x.held[2].ptr, prefix_len=prefix)
    assert way.startswith("through: tile=64") and (way.split()[2] != "parts=1") == parts, way
    x.check(x.run())
    x.check(x.run(causal=1, max_tokens=n, max_kv=prefix + n + 60))
    x.free()


# And by a workgroup for each sequence and kv head where rows are few and the prefix is short.
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("heads,n", [(2, 1), (2, 2), (6, 2), (2, 5), (8, 2)])
def test_through_the_prefix_by_few_rows(gpu, page, d, heads, n):
    mine = [n, n + 1, n + 15, n + 63, n + 70, n + 130, n]
    for prefix, causal, ragged in ((page, 1, True), (256, 0, False), (512, 1, True)):
        tokens = [n - b % 2 for b in range(7)] if ragged else [n] * 7
        x = Call(gpu, heads, 2 if heads == 6 else 1, d, page, prefix, mine, tokens, causal, ragged=ragged)
        way = route(abi.OP_KV_PREFIX_ATTENTION_I8, attention=abi.KvAttentionArgs(**x.args), prefix_table=x.held[2].ptr, prefix_len=prefix)
        if prefix == 16:
            assert (way == "through: few ws=0") == (n * heads // (2 if heads == 6 else 1) <= (8 if d > 128 else 16)), way
        x.check(x.run())
        x.free()


@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads,kv_heads,batch,n,prefix,parts", [(16, 16, 6, 500, 320, False), (8, 2, 6, 257, 4000, True)])
def test_through_the_prefix_by_large_tiles(gpu, d, heads, kv_heads, batch, n, prefix, parts):
    x = Call(gpu, heads, kv_heads, d, 32, prefix, [n + 50 - b % 3 for b in range(batch)], [n - 2 * b for b in range(batch)])
    way = route(abi.OP_KV_PREFIX_ATTENTION_I8, attention=abi.KvAttentionArgs(**x.args), prefix_table=x.held[2].ptr, prefix_len=prefix)
    assert way.startswith("through: tile=128") and (way.split()[2] != "parts=1") == parts, way
    x.check(x.run())
    x.free()


@pytest.mark.parametrize("layout", ["rows", "wide", "heads"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [1, 6, 70])
def test_layouts_and_in_place(gpu, layout, in_place, n):
    case(gpu, 4, 2, 64, 16, 160, [n + 30] * 3, [n] * 3, ragged=False, layout=layout, in_place=in_place)


@pytest.mark.parametrize("batch,n,prefix,mine", [(1, 1, 4096, 100), (64, 1, 4096, 60), (65, 1, 1024, 1000), (130, 2, 512, 40),
                                                 (3, 300, 2048, 400), (1, 1, 16, 5000), (2, 40, 16, 3000), (33, 1, 8192, 1)])
def test_long_and_many(gpu, batch, n, prefix, mine):
    case(gpu, 8, 2, 64, 16, prefix, [max(n, mine - 3 * b) for b in range(batch)], [n] * batch, ragged=False)
    case(gpu, 4, 4, 128, 16, prefix, [max(n, mine - 2 * b) for b in range(batch)], [n] * batch)


@pytest.mark.parametrize("mine", [0, 1, 100])
def test_without_keys_of_their_own(gpu, mine):
    """Not causal: sequences that are the prefix and nothing else."""
    case(gpu, 4, 2, 64, 32, 96, [mine, 0, 0], [1, 3, 40], causal=0)


def test_no_prefix(gpu):
    case(gpu, 4, 2, 64, 32, 0, [40, 3, 200], [1, 3, 40])


@pytest.mark.parametrize("q_factor,scale", [(8.0, 0.0), (64.0, 0.0), (1e-20, 0.0), (1.0, 3.0), (0.0, 0.0)])
def test_sizes_of_scores(gpu, q_factor, scale):
    for n in (1, 30):
        case(gpu, 8, 4, 64, 16, 320, [n + 77] * 3, [n] * 3, q_factor=q_factor, scale=scale)


@pytest.mark.parametrize("side", ["prefix", "own"])
@pytest.mark.parametrize("n", [1, 30])
def test_one_side_with_all_the_weight(gpu, side, n):
    """Scores of one side so far above the other's that nothing of that is left, and values of the other 1000 times as large."""
    def change(x):
        ids = x.table if side == "prefix" else np.setdiff1d(np.arange(x.c.pages), x.table)
        other = np.setdiff1d(np.arange(x.c.pages), ids)
        x.c.ks[ids] *= 40
        x.c.vs[other] *= 1000
    case(gpu, 4, 2, 64, 16, 160, [n + 50] * 3, [n] * 3, q_factor=4.0, change=change)


@pytest.mark.parametrize("n", [1, 70])
def test_not_finite(gpu, n):
    """A NaN or infinite query row and a sequence's page with such a scale give NaN there only; in the prefix, everywhere."""
    def bad(x):
        x.q[0, 1, 5] = np.nan
        x.q[n, 0, 0] = np.inf
        x.c.ks[x.c.table[2, 4 + 3], 0] = np.nan   # own tokens 48 to 63
    x = Call(gpu, 4, 2, 64, 16, 64, [n + 90] * 4, [n] * 4, ragged=False, change=bad)
    nan = np.isnan(x.run())
    want = np.zeros(nan.shape, bool)
    want[0, 1] = want[n, 0] = want[2 * n:3 * n, :2] = True
    assert np.array_equal(nan, want)
    x.free()

    def worse(x):
        x.c.vs[x.table[1], 1] = np.inf
    x = Call(gpu, 4, 2, 64, 16, 64, [n + 90] * 4, [n] * 4, ragged=False, change=worse)
    nan = np.isnan(x.run())
    assert np.all(nan[:, 2:]) and not np.any(nan[:, :2])
    x.free()


@pytest.mark.parametrize("n", [1, 40])
def test_against_the_plain_attention(gpu, n):
    """The same sequences through KV_ATTENTION_I8: within both bounds of each other."""
    x = Call(gpu, 8, 2, 128, 32, 992, [n + 200, n, n + 31], [n] * 3, forget=False)
    got = x.run()
    want, bound = x.want()
    assert gpu.submit([gpu.command(abi.OP_KV_ATTENTION_I8, **x.args)]) == abi.OK and gpu.sync() == abi.OK
    plain = x.ro.download(gpu)
    assert np.all(np.abs(got - plain) <= 2 * bound)
    x.free()


def test_host_tables_and_lengths(gpu):
    x = Call(gpu, 4, 2, 64, 16, 96, [30, 7], [2, 5])
    lengths, table, start = np.array(x.kv_len, np.int32), x.table.astype(np.int32), kv.starts(x.n)
    a = abi.KvAttentionArgs(**{**x.args, "kv_len": lengths.ctypes.data, "seq_start": start.ctypes.data})
    gpu.run(abi.OP_KV_PREFIX_ATTENTION_I8, attention=a, prefix_table=table.ctypes.data, prefix_len=96)
    x.check(x.ro.download(gpu))
    x.free()


@pytest.mark.parametrize("bad", ["page_high", "page_negative", "own_page", "long", "inside", "negative", "falling", "beyond",
                                 "more_than_told", "more_tokens"])
@pytest.mark.parametrize("many", [False, True])
def test_bad_arrays_fail_the_stream(own, bad, many):
    """Out of range on the device: the sync says so; nothing behind the outputs is touched."""
    n = [40, 4, 40] if many else [2, 1, 3]
    x = Call(own, 4, 2, 64, 16, 64, [60, 50, 45], n, forget=False)
    table, lengths, start, more = np.append(x.table, -9).astype(np.int32), np.array(x.kv_len, np.int32), kv.starts(n), {}
    if bad == "page_high":
        table[2] = x.c.pages
    if bad == "page_negative":
        table[0] = -1
    if bad == "own_page":
        t = x.c.table.copy()
        t[1, 5] = x.c.pages + 3
        own.write(x.bufs["table"], t)
    if bad == "long":
        lengths[1] = x.c.table_ld * 16 + 1
    if bad == "inside":   # a new token in the prefix
        lengths[2] = 64 + n[2] - 1
    if bad == "negative":
        lengths[0] = -5
    if bad == "falling":
        start[1], start[2] = start[2], start[1]
    if bad == "beyond":
        start[3] += 1
    if bad == "more_than_told":
        more = dict(max_kv=64 + 59)
    if bad == "more_tokens":
        more = dict(max_tokens=max(n) - 1)
    for b, v in zip(x.held, (lengths, start, table)):
        own.write(b, v)
    guard = own.upload(np.full((sum(n) + 64, 4, 64), 7, np.float32))
    assert own.submit([x.command(O=guard.ptr, **more)]) == abi.OK
    assert own.sync() == abi.ERR_DEVICE_ERROR
    out = np.empty((sum(n) + 64, 4, 64), np.float32)
    other = Session()
    try:
        assert other.lib.vnpu_buffer_copy(other.stream, out.ctypes.data_as(C.c_void_p), C.c_void_p(guard.ptr), out.nbytes,
                                          abi.COPY_D2H) == abi.OK
    finally:
        other.close()
    assert np.all(out[sum(n):] == 7)


def test_a_sequence_without_tokens_may_have_any_length(gpu):
    """Idle places of a batch: no tokens, a length and a table that mean nothing."""
    x = Call(gpu, 4, 2, 64, 16, 64, [60, 0, 45], [2, 0, 3])
    for length in (-7, 0, 63, 2**31 - 1, -2**31):
        gpu.write(x.held[0], np.array([124, length, 109], np.int32))
        gpu.write(x.ro.buffer, np.full_like(x.q, 7.0))
        x.check(x.run())
    x.free()


@pytest.mark.parametrize("batch,n,prefix", [(4, 1, 4096), (3, 30, 1024), (40, 1, 4096)])
def test_workspace_of_the_size_asked_for(own, batch, n, prefix):
    x = Call(own, 8, 2, 64, 16, prefix, [n + 100] * batch, [n] * batch, ragged=False)
    want = x.run()
    cmd = x.command()
    need = own.lib.vnpu_kv_prefix_attention_workspace(own.dev, C.byref(cmd.args.kv_prefix_attention))
    assert need > 0 and need % 4 == 0
    ws = own.upload(np.full(need // 4 + 64, 5.0, np.float32))
    own.write(x.ro.buffer, np.zeros_like(want))
    assert np.array_equal(x.run(workspace=ws.ptr, workspace_bytes=need), want)
    held = own.download(ws, np.float32, (need // 4 + 64,))
    assert np.all(held[need // 4:] == 5.0) and not np.all(held[:need // 4] == 5.0)
    x.check(want)
    kv.free(own, ws)
    x.free()
    s = Session()
    try:
        small = s.alloc(need)
        y = Call(s, 8, 2, 64, 16, prefix, [n + 100] * batch, [n] * batch, ragged=False)
        assert s.submit([y.command(workspace=small.ptr, workspace_bytes=need - 1)]) == abi.OK
        assert s.sync() == abi.ERR_DEVICE_ERROR
    finally:
        s.close()


def tiles_of(x):
    """Rows of a tile of the prefix's and the own part; slots of few rows of the own part."""
    way = route(abi.OP_KV_PREFIX_ATTENTION_I8, attention=abi.KvAttentionArgs(**x.args), prefix_table=x.held[2].ptr, prefix_len=x.prefix)
    assert way.startswith("shared: "), way
    shared, own = (dict(w.split("=") for w in part.split()[:4]) for part in way[8:].split("own: "))
    return int(shared["tile"]), int(own["tile"]), int(own["few"])


# In two parts behind a long prefix: few rows of both, and tiles of the prefix beside few rows.
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("batch,n", [(2, 1), (3, 2), (24, 1), (24, 3)])
def test_few_rows_of_both_parts(gpu, page, d, batch, n):
    x = Call(gpu, 2, 1, d, page, 4096, [n + 50 * b % 170 for b in range(batch)], [n] * batch, ragged=n == 3)
    shared, own, few = tiles_of(x)
    assert own == 0 and few > 0 and (shared > 0) == (batch == 24)
    x.check(x.run())
    x.free()


# In two parts by tiles: a long prefix and too few rows for one pass; beside them sequences of few rows.
@pytest.mark.parametrize("d", [16, 64, 80, 128, 256])
def test_tiles_of_both_parts(gpu, d):
    x = Call(gpu, 8, 2, d, 16, 8192, [60, 20, 41], [20] * 3, ragged=False)
    assert tiles_of(x) == (64, 64, 0)
    x.check(x.run())
    x.free()
    n = [40 if b % 8 == 3 else 1 + b % 5 for b in range(40)]
    x = Call(gpu, 8, 4, d, 16, 8192, [m + 7 * b % 60 for b, m in enumerate(n)], n)
    assert tiles_of(x)[:2] == (64, 64) and tiles_of(x)[2] > 0
    x.check(x.run())
    x.free()


@pytest.mark.parametrize("d", [16, 128])
def test_large_tiles_of_both_parts(gpu, d):
    x = Call(gpu, 4, 4, d, 16, 2304, [65 + b % 16 for b in range(256)], [65] * 256, ragged=False)
    assert tiles_of(x) == (128, 128, 0)
    x.check(x.run())
    x.free()


# 64-row tiles in one range write their results themselves and need no workspace; several ranges need one.
@pytest.mark.parametrize("batch,n,prefix,parts", [(40, 33, 64, False), (2, 150, 1024, True)])
def test_through_the_prefix_without_allocation(own, batch, n, prefix, parts):
    x = Call(own, 8, 4, 64, 16, prefix, [n + 45] * batch, [n] * batch)
    want = x.run()
    cmds = (abi.Command * 1)(x.command())
    need = own.lib.vnpu_kv_prefix_attention_workspace(own.dev, C.byref(cmds[0].args.kv_prefix_attention))
    assert (need > 0) == parts
    own.write(x.ro.buffer, np.full_like(want, 7.0))
    assert own.lib.vnpu_kv_enqueue_noalloc(own.stream, cmds, 1) == (abi.ERR_INVALID_ARGUMENT if parts else abi.OK)
    if parts:
        ws = own.alloc(need)
        cmds[0] = x.command(workspace=ws.ptr, workspace_bytes=need)
        assert own.lib.vnpu_kv_enqueue_noalloc(own.stream, cmds, 1) == abi.OK
    assert own.sync() == abi.OK
    assert np.array_equal(x.ro.download(own), want)
    x.check(want)


def test_the_same_call_gives_the_same_bits(gpu):
    for n in (1, 33):
        x = Call(gpu, 8, 2, 128, 16, 2048, [n + 300] * 9, [n] * 9)
        first = x.run()
        for _ in range(3):
            assert np.array_equal(x.run(), first)
        x.free()
