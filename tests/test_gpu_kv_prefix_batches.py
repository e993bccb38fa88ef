"""KV_PREFIX_ATTENTION_I8 of large batches and of prefixes that fill a table, against attention in 64 bits (serving_ops.py)."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
import serving_ops as ops
from gpu_ops import route
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu


class Batch:
    """A batch behind one prefix over a small pool, whose pages behind the prefix several sequences have; its command.

    table_ld: pages of a sequence in the table (None: as many as the longest needs)."""

    def __init__(self, s, heads, kv_heads, d, page, prefix, mine, n, causal=1, ragged=True, table_ld=None, seed=5):
        rng = np.random.default_rng(seed)
        batch, first = len(n), prefix // page
        ld = table_ld or -(-(prefix + max(mine)) // page)
        self.s, self.n, self.causal, self.prefix = s, n, causal, prefix
        self.c = c = kv.Cache(rng, 1, kv_heads, d, page, first + 40)
        ids, c.batch, c.table_ld = c.table[0], batch, ld
        c.table = np.empty((batch, ld), np.int32)
        c.table[:, :first] = ids[:first]
        c.table[:, first:] = ids[first + rng.integers(0, 40, (batch, ld - first))]
        self.kv_len = [prefix + m for m in mine]
        self.q = rng.standard_normal((int(np.sum(n)), heads, d)).astype(np.float32)
        self.cache, self.bufs = kv.upload(s, c)
        self.held = [s.upload(np.array(self.kv_len, np.int32)), s.upload(kv.starts(n)), s.upload(ids[:first].copy()),
                     s.upload(self.q), s.upload(np.full_like(self.q, 7.0))]
        self.args = dict(cache=self.cache, Q=self.held[3], O=self.held[4], kv_len=self.held[0], batch=batch, tokens=self.q.shape[0],
                         seq_start=self.held[1] if ragged else None, heads=heads, causal=causal, max_tokens=max(n),
                         max_kv=max(self.kv_len))
        self.args = {k: C.c_void_p(v.ptr) if hasattr(v, "ptr") else v for k, v in self.args.items()}

    def fields(self, **more):
        a = abi.KvAttentionArgs(**{**self.args, **more})
        return dict(attention=a, prefix_table=self.held[2].ptr, prefix_len=self.prefix)

    def route(self, **more):
        return route(abi.OP_KV_PREFIX_ATTENTION_I8, **self.fields(**more))

    def sync(self, s=None, **more):
        """The sync's status of the call on s's stream."""
        s = s or self.s
        assert s.submit([s.command(abi.OP_KV_PREFIX_ATTENTION_I8, **self.fields(**more))]) == abi.OK
        return s.sync()

    def fails(self, **more):
        """Whether the call fails its stream, one of its own: an error stays there."""
        s = Session()
        try:
            return self.sync(s, **more) == abi.ERR_DEVICE_ERROR
        finally:
            s.close()

    def check(self, **more):
        assert self.sync(**more) == abi.OK
        out = self.s.download(self.held[4], np.float32, self.q.shape)
        want, bound = ops.prefix_attention(self.c, self.q, self.kv_len, self.n, self.causal)
        off = np.abs(out - want)
        assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(~(off <= bound))[:3].tolist())

    def free(self):
        kv.free(self.s, self.bufs, *self.held)


@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_bad_arrays_of_a_large_batch_fail_the_stream(gpu, d):
    """Prefix tiles and few rows in one launch, whose workgroups may have more threads than the waves of few rows: every
    sequence is looked over."""
    n = [1] * 250
    x = Batch(gpu, 4, 2, d, 16, 4096, [1 + b % 30 for b in range(250)], n)
    way = x.route()
    assert way.startswith("shared: few=0 rows=0 tile=64 ") and "own: few=250 rows=2 tile=0" in way, way
    x.check()
    lengths, start = np.array(x.kv_len, np.int32), kv.starts(n)
    accepted = []
    for at in (0, 127, 130, 200, 249):
        for bad, length in (("long", x.c.table_ld * 16 + 1), ("inside", 4096), ("negative", -5)):
            changed = lengths.copy()
            changed[at] = length
            gpu.write(x.held[0], changed)
            if not x.fails():
                accepted.append((bad, at))
        gpu.write(x.held[0], lengths)
        changed = start.copy()
        changed[at] += 2   # behind the next sequence's; the one before has more tokens than told
        gpu.write(x.held[1], changed)
        if not x.fails():
            accepted.append(("falling", at))
        gpu.write(x.held[1], start)
    assert not accepted
    x.check()
    x.free()


# A prefix that is all that a sequence may have, because the table ends with it or because max_kv says so.  Few rows and
# tiles in one pass; few rows twice, tiles and few rows, tiles twice.
@pytest.mark.parametrize("room", [0, 2])
@pytest.mark.parametrize("way,batch,n,page,prefix", [
    ("through: few", 4, 1, 16, 64), ("through: tile=64", 5, 40, 16, 64), ("through: tile=64", 2, 150, 16, 1024),
    ("shared: few=", 2, 1, 64, 4096), ("shared: few=0", 24, 1, 64, 4096), ("shared: few=0", 3, 20, 256, 16384)])
@pytest.mark.parametrize("ragged", [False, True])
def test_a_prefix_without_room_behind_it(gpu, way, batch, n, page, prefix, room, ragged):
    x = Batch(gpu, 8, 2, 64, page, prefix, [0] * batch, [n] * batch, causal=0, ragged=ragged, table_ld=prefix // page + room)
    assert x.route().startswith(way), x.route()
    x.check()
    accepted = []
    for at in (0, batch - 1):
        lengths = np.array(x.kv_len, np.int32)
        lengths[at] = prefix + 1
        gpu.write(x.held[0], lengths)
        if not x.fails():
            accepted.append(at)
        if not room and not x.fails(max_kv=0):   # the table's room
            accepted.append(("table", at))
    assert not accepted
    gpu.write(x.held[0], np.array(x.kv_len, np.int32))
    assert x.fails(causal=1)   # new tokens would be keys of their own
    x.check()
    x.free()


# Prefix tiles beside few rows of four waves and of two, with 4, 8 and 16 rows a workgroup; of up to 128 dimensions and 4 rows
# four waves where the launch has no more than two workgroups a CU (512 here) and two where it has more.
@pytest.mark.parametrize("waves,d,heads,kv_heads,batch,n,prefix", [
    (4, 80, 8, 2, 120, 1, 2048), (4, 128, 8, 2, 120, 1, 2048), (4, 128, 8, 8, 30, 2, 2048),
    (2, 80, 8, 2, 250, 1, 2048), (2, 128, 8, 2, 250, 1, 2048), (2, 128, 16, 8, 64, 1, 2048), (2, 112, 8, 8, 60, 3, 2048),
    (2, 128, 8, 2, 120, 2, 2048), (2, 128, 8, 2, 48, 3, 2048), (2, 80, 8, 2, 48, 4, 2048),
    (2, 144, 8, 2, 120, 1, 1024), (2, 256, 8, 2, 64, 2, 1024), (2, 256, 4, 4, 64, 1, 1024),
    (4, 64, 8, 2, 64, 2, 2048), (4, 48, 8, 2, 64, 4, 2048)])
@pytest.mark.parametrize("ragged", [False, True])
def test_tiles_beside_few_rows(gpu, waves, d, heads, kv_heads, batch, n, prefix, ragged):
    tokens = [n - (b % n if ragged else 0) for b in range(batch)]
    x = Batch(gpu, heads, kv_heads, d, 64, prefix, [m + 11 * b % 150 for b, m in enumerate(tokens)], tokens, ragged=ragged)
    way = x.route()
    assert way.startswith("shared: few=0 rows=0 tile=64 ") and f" tile=0 parts=0 waves={waves} " in way, way
    x.check()
    x.free()
