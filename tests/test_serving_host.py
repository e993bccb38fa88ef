"""MATMUL_I4, ROPE_AXES_F32 and KV_PREFIX_ATTENTION_I8 without a GPU: what is refused, and how the work is laid out."""
import ctypes as C

import pytest

from vnpu_mi355x import Session, abi, load_backend

P = 1 << 20   # an address that is never used here


def route(opcode, fields):
    """The dispatch rules' answer, None for a call that is refused."""
    lib = load_backend()
    lib.vnpu_debug_route.restype = C.c_int32
    lib.vnpu_debug_route.argtypes = [C.c_void_p, C.c_uint32, C.c_char_p, C.c_uint32]
    out = C.create_string_buffer(256)
    cmd = Session.command(opcode, **fields)
    return out.value.decode() if lib.vnpu_debug_route(C.byref(cmd), 0, out, 256) == abi.OK else None


def matmul(**kw):
    return abi.OP_MATMUL_I4, {**dict(A=P, B=P, C=2 * P, M=3, K=100, N=50), **kw}


def rope(sections=(8, 12, 12), **kw):
    f = dict(Q=P, Q_out=2 * P, K=P, K_out=3 * P, positions=P, batch=2, tokens=6, heads=8, kv_heads=2, head_dim=64,
             axes=len(sections), rotation=abi.ROTATE_HALF)
    return abi.OP_ROPE_AXES_F32, {**f, "sections": (C.c_uint32 * 4)(*sections[:4]), **kw}


def prefix(c=None, prefix_len=64, prefix_table=P, **kw):
    f = dict(k=P, v=P, k_scales=P, v_scales=P, table=P, pages=40, page_size=16, kv_heads=4, head_dim=64, table_ld=8)
    cache = abi.KvCache(**{**f, **(c or {})})
    a = abi.KvAttentionArgs(**{**dict(cache=cache, Q=P, O=2 * P, kv_len=P, batch=2, tokens=6, heads=8, causal=1), **kw})
    return abi.OP_KV_PREFIX_ATTENTION_I8, dict(attention=a, prefix_table=prefix_table, prefix_len=prefix_len)


@pytest.mark.parametrize("bad", [
    dict(A=None), dict(B=None), dict(C=None), dict(M=0), dict(K=0), dict(N=0), dict(lda=99), dict(ldc=49), dict(epilogue=5),
    dict(K=(1 << 30) + 1), dict(N=(1 << 30) + 1), dict(M=1 << 31),
])
def test_bad_products_are_refused(bad):
    assert route(*matmul()) is not None
    assert route(*matmul(**bad)) is None


@pytest.mark.parametrize("bad", [
    dict(Q=None), dict(Q_out=None), dict(K=None), dict(K_out=None), dict(Q=None, Q_out=None, K=None, K_out=None),
    dict(positions=None), dict(tokens=0), dict(tokens=7), dict(heads=0), dict(kv_heads=0), dict(heads=1 << 16), dict(head_dim=0),
    dict(head_dim=62), dict(head_dim=65), dict(head_dim=258), dict(axes=0), dict(axes=5), dict(rotation=0), dict(rotation=3),
    dict(order=2), dict(ladders=2), dict(position_ld=5), dict(sections=(8, 0, 8)), dict(sections=(8, 12, 13)),
    dict(sections=(0xffffffff, 2, 2)), dict(Q_out=P, q_token_stride=512, o_token_stride=520), dict(o_token_stride=500),
    dict(ko_head_stride=60), dict(o_batch_stride=1000), dict(tokens=(1 << 28) + 2), dict(tokens=1 << 28, batch=1, head_dim=256),
])
def test_bad_rotations_are_refused(bad):
    assert route(*rope()) is not None
    assert route(*rope(**bad)) is None


@pytest.mark.parametrize("fine", [
    dict(Q=None, Q_out=None, heads=0), dict(K=None, K_out=None, kv_heads=0), dict(Q_out=P), dict(batch=0, tokens=7),
    dict(sections=(32,)), dict(sections=(1, 1, 1, 1)), dict(position_ld=1000), dict(order=1, ladders=1, rotation=2),
    dict(q_token_stride=1, q_head_stride=1), dict(sections=(64, 64), head_dim=256), dict(sections=(1,), head_dim=2),
    dict(o_batch_stride=64 * 24, o_token_stride=64, o_head_stride=192),
])
def test_rotations_that_are_taken(fine):
    assert route(*rope(**fine)) is not None


@pytest.mark.parametrize("bad", [
    dict(prefix_table=None), dict(prefix_len=65), dict(prefix_len=144), dict(prefix_len=64, max_kv=63),
    dict(Q=None), dict(O=None), dict(kv_len=None), dict(heads=0), dict(heads=7), dict(tokens=5), dict(o_token_stride=500),
    dict(c=dict(k=None)), dict(c=dict(table=None)), dict(c=dict(page_size=0)), dict(c=dict(page_size=24)), dict(c=dict(head_dim=72)),
    dict(c=dict(k=P + 4)), dict(O=P, q_head_stride=64, o_head_stride=80),
    dict(batch=1, tokens=1 << 26, heads=64, c=dict(kv_heads=64)),
])
def test_bad_prefix_calls_are_refused(bad):
    assert route(*prefix()) is not None
    assert route(*prefix(**bad)) is None


@pytest.mark.parametrize("fine", [
    dict(prefix_len=0, prefix_table=None), dict(prefix_len=128), dict(max_kv=64), dict(tokens=5, seq_start=P), dict(O=P),
    dict(q_batch_stride=4096, q_token_stride=64, q_head_stride=192),
])
def test_prefix_calls_that_are_taken(fine):
    assert route(*prefix(**fine)) is not None


def test_a_prefix_of_no_tokens_is_the_plain_attention():
    _, f = prefix(prefix_len=0)
    a = f["attention"]
    plain = {n: getattr(a, n) for n, _ in abi.KvAttentionArgs._fields_}
    assert route(*prefix(prefix_len=0)) == route(abi.OP_KV_ATTENTION_I8, plain)


def test_names_and_null_arguments():
    lib = load_backend()
    assert [lib.vnpu_opcode_name(i) for i in (80, 81, 82)] == [b"MATMUL_I4", b"ROPE_AXES_F32", b"KV_PREFIX_ATTENTION_I8"]
    assert [lib.vnpu_opcode_name(i) for i in (67, 79, 83)] == [b"UNKNOWN"] * 3
    for fn in (lib.vnpu_matmul_i4, lib.vnpu_rope_axes_f32, lib.vnpu_kv_prefix_attention_i8):
        assert fn(None, None) == abi.ERR_INVALID_ARGUMENT
    assert lib.vnpu_matmul_i4_workspace(None, None) == 0 and lib.vnpu_kv_prefix_attention_workspace(None, None) == 0
    out = C.c_void_p()
    assert lib.vnpu_pack_weights_i4(None, None, None, None, 1, 1, 0, 0, 0, C.byref(out)) == abi.ERR_INVALID_ARGUMENT
    assert lib.vnpu_packed_weights_i4_info(None, None, None, None, None) == abi.ERR_INVALID_ARGUMENT
    lib.vnpu_packed_weights_i4_destroy(None)


def test_every_kernel_of_the_products_is_some_call_s():
    """Strips and waves of few rows, rows and strips of tens of rows, tiles of four shapes; with and without ranges of K."""
    seen = set()
    for M in (1, 2, 4, 5, 8, 9, 16, 17, 48, 96, 128, 256, 600, 2048):
        for K in (64, 300, 1000, 2048, 4096, 8192, 16384):
            for N in (16, 500, 1001, 2048, 4096, 6000, 11008, 16000, 32000):
                name, rows, strips, waves, splits, _ = route(*matmul(M=M, K=K, N=N)).split()
                seen.add((name, int(rows[5:]), int(strips[7:]), int(waves[6:])))
                assert 1 <= int(splits[7:]) <= 8
                assert name == "few" or M > 4
                assert name != "few" or M <= 8
    few = {("few", r, t, w) for r in (1, 2) for t, w in ((1, 16), (2, 16), (2, 8), (3, 8), (4, 8))}
    mid = {("mid", 1, t, 8) for t in (1, 2, 3, 4)} | {("mid", 2, t, 8) for t in (3, 4)}
    assert seen == few | mid | {("tile", r, t, 4) for r, t in ((2, 1), (2, 2), (4, 2), (4, 4))}


def test_rows_too_far_apart_for_32_bits_go_in_tiles():
    assert route(*matmul(M=1, K=64, N=64, lda=1 << 31)).startswith("few")   # one row
    assert route(*matmul(M=2, K=64, N=64, lda=1 << 30)).startswith("tile")
    assert route(*matmul(M=2, K=64, N=64, lda=1 << 20)).startswith("few")


def test_routes_of_a_shared_prefix():
    """Few rows against the prefix and own keys, tiles against the prefix, tiles on both sides; one pass over both."""
    def words(batch, n, prefix_len, mine):
        c = dict(page_size=16, kv_heads=8, head_dim=128, table_ld=1 << 14)
        return route(*prefix(c=c, prefix_len=prefix_len, batch=batch, tokens=batch * n, heads=32, max_kv=prefix_len + mine)).split()

    def text(*call):
        w = words(*call)
        at = w.index("own:")
        return [dict(x.split("=") for x in w[a:b]) for a, b in ((1, at), (at + 1, at + 5))]

    shared, own = text(2, 1, 4096, 40)
    assert shared["few"] != "0" and own["few"] != "0" and shared["tile"] == own["tile"] == "0"
    shared, own = text(32, 1, 4096, 500)
    assert shared["tile"] == "64" and int(shared["parts"]) > 4 and own["few"] == "32" and own["tile"] == "0"
    shared, own = text(3, 20, 16384, 440)
    assert shared["tile"] != "0" and own["tile"] != "0" and own["few"] == "0"
    assert words(4, 300, 2048, 700)[0] == "through:"
    assert words(4, 1, 320, 20)[:2] == ["through:", "few"]
    assert words(4, 17, 64, 64)[0] == "through:" and words(4, 17, 32768, 64)[0] == "shared:"


def test_waves_of_few_rows_beside_tiles():
    """Four where the launch has no more than two workgroups a CU, for up to 4 rows of 65 to 128 dimensions; always for less."""
    def waves(d, heads, kv_heads, batch, n=1, prefix_len=4096):
        c = dict(page_size=16, kv_heads=kv_heads, head_dim=d, table_ld=1 << 14)
        way = route(*prefix(c=c, prefix_len=prefix_len, batch=batch, tokens=batch * n, heads=heads, max_kv=prefix_len + 64))
        return next((int(w[6:]) for w in way.split() if w.startswith("waves=")), None)

    assert waves(128, 32, 8, 32) == 4 and waves(128, 32, 8, 64, prefix_len=32768) == 2
    assert waves(80, 8, 2, 120) == 4 and waves(80, 8, 2, 250) == 2
    assert waves(64, 8, 2, 250) == 4 and waves(128, 8, 2, 30, n=2) == 2 and waves(256, 8, 2, 30) == 2
    assert waves(128, 32, 8, 2) is None   # few rows twice
