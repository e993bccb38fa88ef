"""The KV commands as a serving loop uses them: together, captured into graphs, on several streams, traced, far into large
buffers.  Attention is compared with kv_ops.attention within its bound, codes and scales with kv_ops.append exactly."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, D, PAGE = 8, 2, 64, 16


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def close(got, want_bound):
    want, bound = want_bound
    off = np.abs(got - want)
    assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(off > bound)[:3].tolist())


class Loop:
    """A cache on a session with the buffers of one step of up to `room` tokens: append the step's tokens, turn its queries
    in place, attend to what is cached."""

    def __init__(self, s, batch, table_ld, room, heads=HEADS, kv_heads=KV_HEADS, d=D, page=PAGE, seed=3, workspace=False):
        self.s, self.heads, self.batch, self.rng = s, heads, batch, np.random.default_rng(seed)
        self.c = kv.Cache(self.rng, batch, kv_heads, d, page, table_ld)
        self.cache, self.bufs = kv.upload(s, self.c)
        self.q, self.k, self.v, self.o = (s.alloc(room * h * d * 4) for h in (heads, kv_heads, kv_heads, heads))
        self.past, self.len = s.alloc(4 * batch), s.alloc(4 * batch)
        self.start = s.alloc(4 * batch + 4)
        self.lengths = np.zeros(batch, np.int32)
        self.workspace = None
        if workspace:
            self.workspace = s.alloc(self.workspace_bytes(batch, False, 1))

    def commands(self, tokens, ragged, most):
        strides = dict(batch=self.batch, tokens=tokens, seq_start=self.start.ptr if ragged else None, cache=self.cache)
        more = {}
        if self.workspace and tokens == self.batch:   # a workspace for steps of a token each
            more = dict(workspace=self.workspace.ptr, workspace_bytes=self.workspace.nbytes)
        return [self.s.command(abi.OP_KV_APPEND_I8, Q=self.q, Q_out=self.q, K=self.k, V=self.v, past=self.past,
                               heads=self.heads, rotation=abi.ROTATE_HALF, **strides),
                self.s.command(abi.OP_KV_ATTENTION_I8, Q=self.q, O=self.o, kv_len=self.len, heads=self.heads,
                               max_tokens=most, causal=1, **strides, **more)]

    def workspace_bytes(self, tokens, ragged, most):
        args = self.commands(tokens, ragged, most)[1].args.kv_attention
        return self.s.lib.vnpu_kv_attention_workspace(self.s.dev, C.byref(args))

    def draw(self, n):
        """New tokens for each sequence, on the device and in the 64-bit cache."""
        t = int(np.sum(n))
        q, k, v = (normal(self.rng, t, h, self.c.head_dim) for h in (self.heads, self.c.kv_heads, self.c.kv_heads))
        for b, x in ((self.q, q), (self.k, k), (self.v, v), (self.past, self.lengths), (self.start, kv.starts(n)),
                     (self.len, self.lengths + np.array(n, np.int32))):
            self.s.write(b, x)
        kv.append(self.c, k, v, self.lengths, n, abi.ROTATE_HALF)
        position = np.concatenate([a + np.arange(m) for a, m in zip(self.lengths, n)])
        self.turned = kv.turned(q, position, abi.ROTATE_HALF, 0)
        self.lengths = self.lengths + np.array(n, np.int32)
        self.n = n

    def result(self):
        return self.s.download(self.o, np.float32, (int(np.sum(self.n)), self.heads, self.c.head_dim))

    def check(self):
        t = int(np.sum(self.n))
        q = self.s.download(self.q, np.float32, (t, self.heads, self.c.head_dim))
        # Two products with a cosine that may round the other way.
        assert np.all(np.abs(q - self.turned) <= 2.0**-24 * 2 * (np.abs(q).max() + np.abs(q)))
        got = kv.download(self.s, self.c, self.bufs)
        for name in ("ks", "vs", "k", "v"):
            assert np.array_equal(got[name], getattr(self.c, name)), name
        close(self.result(), kv.attention(self.c, q, self.lengths, self.n, 1))

    def free(self):
        kv.free(self.s, self.bufs, self.q, self.k, self.v, self.o, self.past, self.len, self.start, self.workspace)


@pytest.mark.parametrize("heads,kv_heads,d,page", [(8, 2, 64, 16), (4, 4, 128, 64), (6, 2, 80, 32), (4, 1, 256, 256)])
def test_prompts_then_tokens(gpu, heads, kv_heads, d, page):
    """Ragged prompts, tokens one by one, a draft of four verified and partly taken back, a prompt that joins tokens."""
    x = Loop(gpu, 3, 400 // page + 2, 300, heads, kv_heads, d, page)
    steps = [[37, 1, 130]] + [[1, 1, 1]] * 6 + [[4, 4, 4]] + [[1, 90, 0]] + [[1, 1, 1]] * 3
    for i, n in enumerate(steps):
        ragged = len(set(n)) > 1 or i % 2 == 0
        x.draw(n)
        assert gpu.submit(x.commands(sum(n), ragged, max(n))) == abi.OK and gpu.sync() == abi.OK
        x.check()
        if n[0] == 4:
            x.lengths = x.lengths - np.array([3, 0, 2], np.int32)
    x.free()


def test_the_f32_attention_over_what_is_read(gpu):
    """One submission: append, attend, read everything in [head][token] order, ATTENTION_F32 over it.  Both attentions are
    sums of the same values: theirs, in f32, adds D products to a score and n weighted values, one rounding each."""
    heads, d, n = 4, 64, 90
    x = Loop(gpu, 1, 8, n, heads, heads, d, PAGE)
    x.draw([n])
    rows = dict(token=d, head=n * d)
    kf, vf, qf, of = (gpu.alloc(heads * n * d * 4) for _ in range(4))
    cmds = x.commands(n, False, n)
    for side in "qo":
        setattr(cmds[0].args.kv_append, f"{side}_token_stride", 0)
    cmds.append(gpu.command(abi.OP_KV_READ_F32, cache=x.cache, K=kf, V=vf, batch=1, tokens=n, k_token_stride=rows["token"],
                            k_head_stride=rows["head"], v_token_stride=rows["token"], v_head_stride=rows["head"]))
    assert gpu.submit(cmds) == abi.OK and gpu.sync() == abi.OK
    x.check()
    q = gpu.download(x.q, np.float32, (n, heads, d))
    gpu.write(qf, np.ascontiguousarray(q.transpose(1, 0, 2)))
    gpu.run(abi.OP_ATTENTION_F32, Q=qf, K=kf, V=vf, O=of, batch=1, heads=heads, seq_q=n, seq_k=n, head_dim=d, causal=1)
    f32 = gpu.download(of, np.float32, (heads, n, d)).transpose(1, 0, 2)
    want, bound = kv.attention(x.c, q, [n], [n], 1)
    k, v = x.c.values(0, n)
    score = np.abs(q.astype(np.float64)).max() * np.abs(k).sum(axis=2).max() / np.sqrt(d)
    theirs = np.abs(v).max() * 2.0**-24 * (2 * (d + 8) * score + 2 * n + 16)
    assert np.all(np.abs(f32 - want) <= theirs)
    assert np.all(np.abs(f32 - x.result()) <= theirs + bound)
    x.free()
    kv.free(gpu, kf, vf, qf, of)


# ---------------------------------------------------------------------------
# Graphs
# ---------------------------------------------------------------------------

def hip():
    """The HIP runtime that the backend has loaded."""
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    return C.CDLL(path)


class Graph:
    """vnpu_kv_enqueue_noalloc of some commands, captured on the session's stream."""

    def __init__(self, s, cmds):
        self.h, self.stream = hip(), C.c_void_p(s.lib.vnpu_stream_hip_handle(s.stream))
        graph, self.exec = C.c_void_p(), C.c_void_p()
        arr = (abi.Command * len(cmds))(*cmds)
        assert self.h.hipStreamBeginCapture(self.stream, 1) == 0
        rc = s.lib.vnpu_kv_enqueue_noalloc(s.stream, arr, len(cmds))
        assert self.h.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        assert rc == abi.OK
        assert self.h.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        assert self.h.hipGraphDestroy(graph) == 0

    def launch(self):
        assert self.h.hipGraphLaunch(self.exec, self.stream) == 0

    def free(self):
        assert self.h.hipGraphExecDestroy(self.exec) == 0


def eager(s, x, cmds):
    assert s.submit(cmds) == abi.OK and s.sync() == abi.OK
    return x.result()


@pytest.mark.parametrize("batch,table_ld", [(1, 300), (3, 300), (5, 4)])
def test_captured_steps(own, batch, table_ld):
    """A captured decode step, replayed over growing lengths (some past a page, some in tiles of their own), with eager
    steps of another cache between: each replay is the eager step's bits, and the oracle's."""
    x = Loop(own, batch, table_ld, 64 * batch, seed=1, workspace=True)
    y = Loop(own, batch, table_ld, 64 * batch, seed=1)
    g = None
    for step in range(9):
        n = [40] * batch if step == 0 else [1] * batch
        if step in (3, 6) and table_ld > 100:   # as if many tokens had come
            grow = 700 * (1 + np.arange(batch, dtype=np.int32))
            for z in (x, y):
                z.lengths = z.lengths + grow
        for z in (x, y):
            z.draw(n)
        want = eager(own, y, y.commands(sum(n), False, max(n)))
        if step == 0:
            eager(own, x, x.commands(sum(n), False, max(n)))
            continue
        if g is None:
            g = Graph(own, x.commands(batch, False, 1))
            before = x.result()
            assert not np.array_equal(before, want)   # captured, not run
        g.launch()
        assert own.sync() == abi.OK
        assert np.array_equal(x.result(), want)
        x.check()
    g.free()
    x.free()
    y.free()


def test_two_graphs_at_once(own):
    """Two captured steps on two streams, each with its own workspace, replayed without a wait between them."""
    other = Session()
    try:
        loops = [Loop(s, 1, 300, 32, seed=i, workspace=True) for i, s in enumerate((own, other))]
        assert all(x.workspace.nbytes > 0 for x in loops)
        graphs = []
        for x in loops:
            x.lengths = x.lengths + np.int32(4000)
            x.draw([1])
            graphs.append(Graph(x.s, x.commands(1, False, 1)))
        for step in range(6):
            if step:
                for x in loops:
                    x.draw([1])
            for _ in range(3):   # the step again: the same codes, queries turned further
                for x, g in zip(loops, graphs):
                    x.s.write(x.q, x.turned)   # turned again from here
                    g.launch()
            for x in loops:
                assert x.s.sync() == abi.OK
            for x in loops:
                q = x.s.download(x.q, np.float32, (1, HEADS, D))
                close(x.result(), kv.attention(x.c, q, x.lengths, [1], 1))
                got = kv.download(x.s, x.c, x.bufs)
                assert all(np.array_equal(got[name], getattr(x.c, name)) for name in got)
        for x, g in zip(loops, graphs):
            g.free()
        loops[1].free()
    finally:
        other.close()


# ---------------------------------------------------------------------------
# Workspaces and what is refused
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("batch,tokens,max_kv,causal", [(1, 1, 4800, 1), (2, 5, 4000, 1), (1, 60, 4800, 0), (1, 150, 4800, 1)])
def test_workspace_of_the_size_asked_for(own, batch, tokens, max_kv, causal):
    """Enough, and not a byte behind it is touched; the result is that of the stream's own workspace."""
    x = Loop(own, batch, 300, batch * tokens)
    x.lengths = x.lengths + np.int32(max_kv - tokens)
    x.draw([tokens] * batch)
    cmds = x.commands(batch * tokens, False, tokens)
    args = cmds[1].args.kv_attention
    args.causal = causal
    want = eager(own, x, cmds)
    need = own.lib.vnpu_kv_attention_workspace(own.dev, C.byref(args))
    assert need > 0 and need % 4 == 0
    ws = own.upload(np.full(need // 4 + 64, 5.0, np.float32))
    args.workspace, args.workspace_bytes = ws.ptr, need
    own.write(x.o, np.zeros_like(want))
    assert own.submit([cmds[1]]) == abi.OK and own.sync() == abi.OK
    assert np.array_equal(x.result(), want)
    held = own.download(ws, np.float32, (need // 4 + 64,))
    assert np.all(held[need // 4:] == 5.0) and not np.all(held[:need // 4] == 5.0)
    kv.free(own, ws)
    x.free()


def test_noalloc_refusals_enqueue_nothing(own):
    """Host memory, a missing, small, unaligned or host workspace, other opcodes, a bad command behind a good one."""
    x = Loop(own, 1, 300, 4)
    x.lengths = x.lengths + np.int32(4000)
    x.draw([1])
    before = x.result()
    need = x.workspace_bytes(1, False, 1)
    ws = own.alloc(need + 32)
    host = np.zeros(max(need, 4096), np.uint8)

    def call(*cmds):
        arr = (abi.Command * len(cmds))(*cmds)
        return own.lib.vnpu_kv_enqueue_noalloc(own.stream, arr, len(cmds))

    def attention(**kw):
        cmd = x.commands(1, False, 1)[1]
        for name, value in {**dict(workspace=ws.ptr, workspace_bytes=need), **kw}.items():
            setattr(cmd.args.kv_attention, name, value)
        return cmd

    bad = [attention(workspace=None), attention(workspace_bytes=need - 1), attention(workspace=ws.ptr + 4),
           attention(workspace=host.ctypes.data), attention(Q=host.ctypes.data), attention(O=host.ctypes.data),
           attention(kv_len=host.ctypes.data), attention(heads=HEADS + 1),
           own.command(abi.OP_ADD_F32, A=x.o, B=x.o, Y=x.o, count=4), own.command(abi.OP_BARRIER)]
    for cmd in bad:
        assert call(cmd) == abi.ERR_INVALID_ARGUMENT
        assert call(attention(), cmd) == abi.ERR_INVALID_ARGUMENT
    for name in ("K", "V", "past", "Q", "Q_out"):
        cmd = x.commands(1, False, 1)[0]
        setattr(cmd.args.kv_append, name, host.ctypes.data)
        assert call(cmd) == abi.ERR_INVALID_ARGUMENT
    read = own.command(abi.OP_KV_READ_F32, cache=x.cache, K=host.ctypes.data, batch=1, tokens=4)
    assert call(read) == abi.ERR_INVALID_ARGUMENT
    assert own.sync() == abi.OK and np.array_equal(x.result(), before)
    assert call() == abi.OK
    assert call(x.commands(1, False, 1)[0], attention()) == abi.OK and own.sync() == abi.OK
    x.check()
    kv.free(own, ws)
    x.free()


# ---------------------------------------------------------------------------
# Streams, traces, memory
# ---------------------------------------------------------------------------

@pytest.fixture()
def own():
    s = Session()
    yield s
    s.close()


def test_two_streams_at_once(own):
    """The commands of two streams that run at the same time, each with its stream's workspace."""
    other = Session()
    try:
        loops = [Loop(s, 2, 300, 8, seed=7 + i) for i, s in enumerate((own, other))]
        for x in loops:
            x.lengths = x.lengths + np.int32(3500)
        for _ in range(4):
            for x in loops:
                x.draw([1, 1])
            for x in loops:
                assert x.s.submit(x.commands(2, False, 1)) == abi.OK
            for x in loops:
                assert x.s.submit(x.commands(2, False, 1)[1:] * 8) == abi.OK
            for x in loops:
                assert x.s.sync() == abi.OK
            for x in loops:
                x.check()
        loops[1].free()
    finally:
        other.close()


def test_traces_and_counters(own):
    """Each command is an event with its name, and counts what it reads, writes and computes."""
    x = Loop(own, 2, 20, 64)
    x.draw([30, 30])
    lib = own.lib
    assert lib.vnpu_device_reset(own.dev) == abi.OK and lib.vnpu_trace_enable(own.dev, 1) == abi.OK
    out = own.alloc(60 * KV_HEADS * D * 4)
    read = own.command(abi.OP_KV_READ_F32, cache=x.cache, K=out, batch=2, tokens=60)
    assert own.submit([*x.commands(60, False, 30), read]) == abi.OK and own.sync() == abi.OK
    st, summary = own.status(), abi.TraceSummary()
    assert lib.vnpu_trace_get_summary(own.dev, C.byref(summary)) == abi.OK
    assert summary.events == 3 and st.commands_completed == 3 and st.last_opcode == abi.OP_KV_READ_F32
    assert abi.OP_KV_APPEND_I8 <= summary.hot_opcode <= abi.OP_KV_READ_F32 and summary.hot_time_ns > 0
    q, k = 60 * HEADS * D, 60 * KV_HEADS * D
    assert st.bytes_written == (4 * q + 2 * k) + 4 * q + 4 * k == summary.bytes_written
    assert lib.vnpu_trace_enable(own.dev, 0) == abi.OK
    kv.free(own, out)
    x.free()


def test_codes_and_rows_beyond_32_bits(own):
    """Pages beyond 4 GiB of codes, f32 rows beyond 2^32 elements."""
    kv_heads, d, page, n = 8, 256, 256, 600
    pages = (1 << 32) // (kv_heads * d * page) + 9
    rng = np.random.default_rng(4)
    small = kv.Cache(rng, 1, kv_heads, d, page, 3, spare=0)   # the same pages under small numbers
    small.table[:] = [[1, 2, 0]]
    ids = np.array([[pages - 1, 3, pages - 6]], np.int32)
    size = pages * kv_heads * page * d
    assert size > 1 << 32
    k, v, ks, vs = own.alloc(size), own.alloc(size), own.alloc(4 * pages * kv_heads), own.alloc(4 * pages * kv_heads)
    table, past, length = own.upload(ids), own.upload(np.zeros(1, np.int32)), own.upload(np.array([n], np.int32))
    cache = abi.KvCache(k=k.ptr, v=v.ptr, k_scales=ks.ptr, v_scales=vs.ptr, table=table.ptr, pages=pages, page_size=page,
                        kv_heads=kv_heads, head_dim=d, table_ld=3)
    x, y = normal(rng, n, kv_heads, d), normal(rng, n, kv_heads, d)
    bx, by, q, o = own.upload(x), own.upload(y), own.upload(x[:4]), own.alloc(4 * 4 * kv_heads * d)
    out = own.alloc(n * kv_heads * d * 4)
    assert own.submit([
        own.command(abi.OP_KV_APPEND_I8, cache=cache, K=bx, V=by, past=past, batch=1, tokens=n, rotation=abi.ROTATE_HALF),
        own.command(abi.OP_KV_ATTENTION_I8, cache=cache, Q=q, O=o, kv_len=length, batch=1, tokens=4, heads=kv_heads, causal=1),
        own.command(abi.OP_KV_READ_F32, cache=cache, V=out, batch=1, tokens=n)]) == abi.OK and own.sync() == abi.OK
    kv.append(small, x, y, [0], [n], abi.ROTATE_HALF)
    want = small.values(0, n)
    assert np.array_equal(own.download(out, np.float32, (n, kv_heads, d)), want[1].transpose(1, 0, 2).astype(np.float32))
    close(own.download(o, np.float32, (4, kv_heads, d)), kv.attention(small, x[:4], [n], [4], 1))
    for b in (k, v, out):
        own.free(b)
    # Five rows, 2^30 floats from one to the next.
    step = 1 << 30
    far = own.alloc(4 * (4 * step + kv_heads * d))
    c = kv.Cache(rng, 1, kv_heads, d, 16, 1)
    cache, bufs = kv.upload(own, c)
    own.run(abi.OP_KV_READ_F32, cache=cache, K=far, batch=1, tokens=5, k_token_stride=step)
    rows = np.stack([own.download(far, np.float32, (kv_heads, d), offset=4 * step * t) for t in range(5)])
    want = c.values(0, 5)[0].transpose(1, 0, 2).astype(np.float32)
    assert np.array_equal(rows, want)
    # Appended from there and attended to from there, each row in its place.
    own.run(abi.OP_KV_APPEND_I8, cache=cache, K=far, V=far, past=past, batch=1, tokens=5, k_token_stride=step, v_token_stride=step)
    kv.append(c, want, want, [0], [5], 0)
    got = kv.download(own, c, bufs)
    assert all(np.array_equal(got[name], getattr(c, name)) for name in got)
    own.write(length, np.array([5], np.int32))
    own.run(abi.OP_KV_ATTENTION_I8, cache=cache, Q=far, O=far, kv_len=length, batch=1, tokens=5, heads=kv_heads, causal=1,
            q_token_stride=step, o_token_stride=step)
    rows = np.stack([own.download(far, np.float32, (kv_heads, d), offset=4 * step * t) for t in range(5)])
    close(rows, kv.attention(c, want, [5], [5], 1))
