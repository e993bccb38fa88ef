"""MATMUL_I4, ROPE_AXES_F32, KV_APPEND_I8 and KV_PREFIX_ATTENTION_I8 as a serving loop uses them: a layer's attention with
4-bit projections behind a shared prompt, in one batch of commands, captured into graphs, on several streams, traced."""
import ctypes as C

import numpy as np
import pytest

import kv_ops as kv
import serving_ops as ops
from test_gpu_kv_decode import Graph
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, D, PAGE, WIDTH, PREFIX = 8, 2, 64, 16, 256, 160
SECTIONS = (8, 12, 12)
ROW = (HEADS + 2 * KV_HEADS) * D


@pytest.fixture()
def own():
    s = Session()
    yield s
    s.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def within(got, want_bound):
    want, bound = want_bound
    off = np.abs(got - want)
    assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(~(off <= bound))[:3].tolist())


class Layer:
    """x -> QKV (4 bits) -> turned by three axes -> cache -> attention behind the prefix -> projection (4 bits)."""

    def __init__(self, s, batch, room, seed=1, workspace=0, projections=None, prefix=PREFIX):
        self.s, self.batch, self.room, self.prefix, self.rng = s, batch, room, prefix, np.random.default_rng(seed)
        rng = np.random.default_rng(99)   # the model
        self.w_qkv, self.w_o = ops.Weights(rng, WIDTH, ROW, 64), ops.Weights(rng, HEADS * D, WIDTH, 128, zeros=False, trans=True)
        self.bias = normal(rng, ROW)
        self.qkv_packed, self.o_packed = projections or (self.w_qkv.pack(s), self.w_o.pack(s))
        self.c, table = ops.shared_cache(self.rng, batch, KV_HEADS, D, PAGE, prefix, 400)
        self.cache, self.bufs = kv.upload(s, self.c)
        size = dict(x=room * WIDTH, qkv=room * ROW, q=room * HEADS * D, o=room * HEADS * D, y=room * WIDTH, positions=3 * room,
                    past=batch, len=batch, start=batch + 1, bias=ROW)
        self.b = {n: s.alloc(4 * v) for n, v in size.items()}
        self.b["table"] = s.upload(table)
        s.write(self.b["bias"], self.bias)
        self.lengths = np.full(batch, prefix, np.int32)
        self.ws = []
        if workspace:
            for i, cmd in enumerate(self.commands(workspace, 1, False)):
                need = self.need(cmd)
                self.ws.append((i, s.alloc(need), need) if need else None)

    def need(self, cmd):
        lib, dev = self.s.lib, self.s.dev
        if cmd.opcode == abi.OP_MATMUL_I4:
            return lib.vnpu_matmul_i4_workspace(dev, C.byref(cmd.args.matmul_i4))
        if cmd.opcode == abi.OP_KV_PREFIX_ATTENTION_I8:
            return lib.vnpu_kv_prefix_attention_workspace(dev, C.byref(cmd.args.kv_prefix_attention))
        return 0

    def commands(self, tokens, most, ragged=True):
        b, s = self.b, self.s
        start = b["start"].ptr if ragged else None
        qkv = b["qkv"].ptr
        attention = abi.KvAttentionArgs(cache=self.cache, Q=b["q"].ptr, O=b["o"].ptr, kv_len=b["len"].ptr, seq_start=start,
                                        batch=self.batch, tokens=tokens, heads=HEADS, max_tokens=most, causal=1)
        # Keys are turned where the projection left them, queries into rows of their own.
        cmds = [
            s.command(abi.OP_MATMUL_I4, A=b["x"], B=self.qkv_packed, bias=b["bias"], C=b["qkv"], M=tokens, K=WIDTH, N=ROW),
            s.command(abi.OP_ROPE_AXES_F32, Q=qkv, Q_out=b["q"], K=qkv + 4 * HEADS * D, K_out=qkv + 4 * HEADS * D,
                      positions=b["positions"], tokens=tokens, heads=HEADS, kv_heads=KV_HEADS, head_dim=D, position_ld=self.room,
                      axes=3, sections=(C.c_uint32 * 4)(*SECTIONS), order=abi.AXES_TURNS, rotation=abi.ROTATE_HALF,
                      q_token_stride=ROW, k_token_stride=ROW, ko_token_stride=ROW),
            s.command(abi.OP_KV_APPEND_I8, cache=self.cache, K=qkv + 4 * HEADS * D, V=qkv + 4 * (HEADS + KV_HEADS) * D,
                      past=b["past"], seq_start=start, batch=self.batch, tokens=tokens, rotation=abi.ROTATE_NONE,
                      k_token_stride=ROW, v_token_stride=ROW),
            s.command(abi.OP_KV_PREFIX_ATTENTION_I8, attention=attention, prefix_table=b["table"], prefix_len=self.prefix),
            s.command(abi.OP_MATMUL_I4, A=b["o"], B=self.o_packed, C=b["y"], M=tokens, K=HEADS * D, N=WIDTH),
        ]
        for held in self.ws:
            if held:
                i, buf, need = held
                args = cmds[i].args.matmul_i4 if cmds[i].opcode == abi.OP_MATMUL_I4 else cmds[i].args.kv_prefix_attention.attention
                args.workspace, args.workspace_bytes = buf.ptr, need
        return cmds

    def draw(self, n):
        t = int(np.sum(n))
        self.x = normal(self.rng, t, WIDTH)
        self.positions = np.zeros((3, self.room), np.int32)
        self.positions[:, :t] = self.rng.integers(0, 4000, (3, t))
        for name, v in (("x", self.x), ("positions", self.positions), ("past", self.lengths), ("start", kv.starts(n)),
                        ("len", self.lengths + np.array(n, np.int32))):
            self.s.write(self.b[name], v)
        self.n, self.before = n, self.lengths.copy()
        self.lengths = self.lengths + np.array(n, np.int32)

    def get(self, name, *shape):
        return self.s.download(self.b[name], np.float32, shape)

    def check(self):
        """Each command against its definition in 64 bits, from what the one before left."""
        t = int(np.sum(self.n))
        projected, bound = ops.matmul(self.x, self.w_qkv, self.bias)
        qkv = self.get("qkv", t, ROW)   # its keys are turned by now
        plain = np.r_[0:HEADS * D, (HEADS + KV_HEADS) * D:ROW]
        within(qkv[:, plain], (projected[:, plain], bound[:, plain]))
        q = self.get("q", t, HEADS, D)
        within(q, ops.rope_axes(qkv[:, :HEADS * D].reshape(t, HEADS, D), self.positions[:, :t], SECTIONS, abi.AXES_TURNS))
        at = slice(HEADS * D, (HEADS + KV_HEADS) * D)
        want, off = ops.rope_axes(projected[:, at].reshape(t, KV_HEADS, D), self.positions[:, :t], SECTIONS, abi.AXES_TURNS)
        k = qkv[:, at].reshape(t, KV_HEADS, D)
        # A pair's two errors, turned: at most their sum for either; and a rounding more than from an f32 value.
        pair = bound[:, at].reshape(t, KV_HEADS, 2, D // 2).sum(axis=2)
        within(k, (want, off + np.concatenate((pair, pair), axis=-1) + ops.EPS * np.abs(want)))
        v = qkv[:, (HEADS + KV_HEADS) * D:].reshape(t, KV_HEADS, D)
        kv.append(self.c, k, v, self.before, self.n, abi.ROTATE_NONE)
        got = kv.download(self.s, self.c, self.bufs)
        for name in ("ks", "vs", "k", "v"):
            assert np.array_equal(got[name], getattr(self.c, name)), name
        o = self.get("o", t, HEADS, D)
        within(o, ops.prefix_attention(self.c, q, self.lengths, self.n, 1))
        within(self.get("y", t, WIDTH), ops.matmul(o.reshape(t, -1), self.w_o))

    def result(self):
        return self.get("y", int(np.sum(self.n)), WIDTH)

    def free(self):
        kv.free(self.s, self.bufs, self.b, *[w[1] for w in self.ws if w])


def test_chunks_of_prompts_then_tokens(gpu):
    """Ragged chunks, single tokens, a sequence that waits, a draft of three."""
    x = Layer(gpu, 4, 120)
    for n in ([30, 1, 70, 5], [1, 1, 1, 1], [1, 1, 0, 1], [3, 3, 3, 3], [1, 40, 1, 1], [1, 1, 1, 1]):
        x.draw(n)
        assert gpu.submit(x.commands(sum(n), max(n))) == abi.OK and gpu.sync() == abi.OK
        x.check()
    x.free()


@pytest.mark.parametrize("prefix", [PREFIX, 4096])   # without and with workspaces
@pytest.mark.parametrize("batch", [1, 5, 24])
def test_captured_steps(own, batch, prefix):
    """A captured step of a token each, replayed over growing sequences with eager steps of another layer between: each
    replay is the eager step's bits, and within the oracle's bounds."""
    x, y = Layer(own, batch, 8 * batch, workspace=batch, prefix=prefix), Layer(own, batch, 8 * batch, prefix=prefix)
    assert any(x.ws) == (prefix > PREFIX)
    g = None
    for step in range(6):
        n = [7] * batch if step == 0 else [1] * batch
        for z in (x, y):
            z.draw(n)
        assert own.submit(y.commands(sum(n), max(n), False)) == abi.OK and own.sync() == abi.OK
        if step == 0:
            held, x.ws = x.ws, []
            assert own.submit(x.commands(sum(n), max(n), False)) == abi.OK and own.sync() == abi.OK
            x.ws = held
        else:
            if g is None:
                g = Graph(own, x.commands(batch, 1, False))
            g.launch()
            assert own.sync() == abi.OK
            assert np.array_equal(x.result(), y.result())
        x.check()
        y.check()
    g.free()
    x.free()
    y.free()


@pytest.mark.parametrize("prefix", [PREFIX, 4096])
def test_two_graphs_at_once(own, prefix):
    """Two streams of one device share the weights; each graph has its own workspaces; replayed without a wait between."""
    other = Session()
    try:
        a = Layer(own, 6, 12, seed=3, workspace=6, prefix=prefix)
        b = Layer(other, 6, 12, seed=4, workspace=6, projections=(a.qkv_packed, a.o_packed), prefix=prefix)
        graphs = []
        for z in (a, b):
            z.draw([1] * 6)
            graphs.append(Graph(z.s, z.commands(6, 1, False)))
        for step in range(5):
            if step:
                for z in (a, b):
                    z.draw([1] * 6)
            for g in graphs:
                g.launch()
            for z in (a, b):
                assert z.s.sync() == abi.OK
                z.check()
        for g in graphs:
            g.free()
        b.free()
    finally:
        other.close()


def test_two_streams_at_once(own):
    """Eager steps of two streams, both submitted before either is waited for."""
    other = Session()
    try:
        a, b = Layer(own, 3, 60, seed=5), Layer(other, 3, 60, seed=6)
        for n in ([20, 1, 30], [1, 1, 1], [2, 2, 2]):
            for z in (a, b):
                z.draw(n)
            for z in (a, b):
                assert z.s.submit(z.commands(sum(n), max(n))) == abi.OK
            for z in (a, b):
                assert z.s.sync() == abi.OK
                z.check()
        b.free()
    finally:
        other.close()


def test_noalloc_refusals_enqueue_nothing(own):
    """Host memory, a missing, small or unaligned workspace, another opcode, a bad command behind a good one."""
    x = Layer(own, 24, 24, workspace=24, prefix=4096)
    x.draw([1] * 24)

    def rc(cmds):
        arr = (abi.Command * len(cmds))(*cmds)
        return own.lib.vnpu_kv_enqueue_noalloc(own.stream, arr, len(cmds))

    good = x.commands(24, 1, False)
    own.write(x.b["y"], np.full((24, WIDTH), 7, np.float32))
    host = np.zeros((24, WIDTH), np.float32)
    bad = []
    c = x.commands(24, 1, False)
    c[0].args.matmul_i4.A = host.ctypes.data
    bad.append(c)
    c = x.commands(24, 1, False)
    c[1].args.rope_axes.positions = host.ctypes.data
    bad.append(c)
    for change in (dict(workspace=None), dict(workspace_bytes=4)):
        c = x.commands(24, 1, False)
        for k, v in change.items():
            setattr(c[3].args.kv_prefix_attention.attention, k, v)
        bad.append(c)
    c = x.commands(24, 1, False)
    c[3].args.kv_prefix_attention.attention.workspace += 4
    bad.append(c)
    c = x.commands(24, 1, False)
    c[3].args.kv_prefix_attention.prefix_table = host.ctypes.data
    bad.append(c)
    c = x.commands(24, 1, False)
    c[4].args.matmul_i4.K = 7
    bad.append(c)
    bad.append(good + [own.command(abi.OP_NOP)])
    for c in bad:
        assert rc(c) == abi.ERR_INVALID_ARGUMENT
    assert own.sync() == abi.OK and np.all(x.result() == 7)
    assert rc(good) == abi.OK and own.sync() == abi.OK
    x.check()
    x.free()


def test_a_graph_s_workspace_for_products(own):
    """A product whose ranges of K need a workspace, captured: nothing behind the workspace is touched."""
    rng = np.random.default_rng(8)
    w = ops.Weights(rng, 8192, 64, 128)
    packed = w.pack(own)
    for M in (8, 70):
        a = normal(rng, M, 8192)
        ba, bc = own.upload(a), own.alloc(M * 64 * 4)
        f = dict(A=ba, B=packed, C=bc, M=M, K=8192, N=64)
        cmd = own.command(abi.OP_MATMUL_I4, **f)
        need = own.lib.vnpu_matmul_i4_workspace(own.dev, C.byref(cmd.args.matmul_i4))
        assert need > 0 and need % 4 == 0
        ws = own.upload(np.full(need // 4 + 64, 5.0, np.float32))
        cmd.args.matmul_i4.workspace, cmd.args.matmul_i4.workspace_bytes = ws.ptr, need
        g = Graph(own, [cmd])
        for _ in range(3):
            own.run(abi.OP_MATMUL_I4, **f)
            want = own.download(bc, np.float32, (M, 64))
            own.write(bc, np.zeros((M, 64), np.float32))
            g.launch()
            assert own.sync() == abi.OK
            got = own.download(bc, np.float32, (M, 64))
            assert np.array_equal(got, want)
        within(got, ops.matmul(a, w))
        held = own.download(ws, np.float32, (need // 4 + 64,))
        assert np.all(held[need // 4:] == 5.0)
        g.free()
        kv.free(own, ba, bc, ws)


def test_wrappers_traces_and_counters(own):
    x = Layer(own, 2, 10)
    x.draw([4, 1])
    cmds = x.commands(5, 4)
    lib = own.lib
    assert lib.vnpu_trace_enable(own.dev, 1) == abi.OK
    before = own.status()
    calls = [(lib.vnpu_matmul_i4, "matmul_i4"), (lib.vnpu_rope_axes_f32, "rope_axes"), (lib.vnpu_kv_append_i8, "kv_append"),
             (lib.vnpu_kv_prefix_attention_i8, "kv_prefix_attention"), (lib.vnpu_matmul_i4, "matmul_i4")]
    for cmd, (fn, name) in zip(cmds, calls):
        assert fn(own.stream, C.byref(getattr(cmd.args, name))) == abi.OK
    after = own.status()
    summary = abi.TraceSummary()
    assert lib.vnpu_trace_get_summary(own.dev, C.byref(summary)) == abi.OK
    assert lib.vnpu_trace_enable(own.dev, 0) == abi.OK
    assert summary.events == 5 and summary.total_time_ns > 0 and summary.flops == after.flops - before.flops
    assert after.commands_completed - before.commands_completed == 5
    flops = 2 * 5 * (WIDTH * ROW + HEADS * D * WIDTH) + 3 * 5 * (HEADS + KV_HEADS) * D + 4 * 5 * KV_HEADS * D
    flops += 4 * 5 * HEADS * D * x.c.table_ld * PAGE   # max_kv is not given: all that the table holds
    assert after.flops - before.flops == flops
    x.check()
    x.free()
