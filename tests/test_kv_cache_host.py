"""KV_APPEND_I8, KV_ATTENTION_I8 and KV_READ_F32 without a GPU: what is refused, and how the work is laid out."""
import ctypes as C

import pytest

from gpu_ops import route
from vnpu_mi355x import Session, abi, load_backend

P = 1 << 20   # an address that is never used here


def cache(**kw):
    f = dict(k=P, v=P, k_scales=P, v_scales=P, table=P, pages=40, page_size=16, kv_heads=4, head_dim=64, table_ld=8)
    return abi.KvCache(**{**f, **kw})


def append(c=None, **kw):
    f = dict(cache=c or cache(), Q=P, Q_out=2 * P, K=P, V=P, past=P, batch=2, tokens=6, heads=8, rotation=1)
    return abi.OP_KV_APPEND_I8, {**f, **kw}


def attention(c=None, **kw):
    f = dict(cache=c or cache(), Q=P, O=2 * P, kv_len=P, batch=2, tokens=6, heads=8, causal=1)
    return abi.OP_KV_ATTENTION_I8, {**f, **kw}


def read(c=None, **kw):
    f = dict(cache=c or cache(), K=P, V=2 * P, batch=2, tokens=6)
    return abi.OP_KV_READ_F32, {**f, **kw}


def taken(opcode, fields):
    lib = load_backend()
    lib.vnpu_debug_route.restype = C.c_int32
    lib.vnpu_debug_route.argtypes = [C.c_void_p, C.c_uint32, C.c_char_p, C.c_uint32]
    out = C.create_string_buffer(128)
    cmd = Session.command(opcode, **fields)
    return lib.vnpu_debug_route(C.byref(cmd), 0, out, 128) == abi.OK


@pytest.mark.parametrize("make", [append, attention, read])
@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(k_scales=None), dict(v_scales=None), dict(table=None), dict(pages=0),
    dict(table_ld=0), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0), dict(page_size=8), dict(page_size=24),
    dict(page_size=512), dict(head_dim=8), dict(head_dim=72), dict(head_dim=272), dict(k=P + 4), dict(v=P + 8),
    dict(pages=1 << 31), dict(table_ld=1 << 27, page_size=16), dict(kv_heads=1 << 16),
])
def test_bad_caches_are_refused(make, bad):
    assert taken(*make())
    assert not taken(*make(cache(**bad)))


@pytest.mark.parametrize("make,bad", [
    (append, dict(K=None)), (append, dict(V=None)), (append, dict(past=None)), (append, dict(Q=None)),
    (append, dict(Q_out=None)), (append, dict(heads=6)), (append, dict(heads=0)), (append, dict(rotation=3)),
    (append, dict(rope_dim=63)), (append, dict(rope_dim=66)), (append, dict(batch=0)), (append, dict(tokens=0)),
    (append, dict(tokens=7)), (append, dict(Q_out=P, q_token_stride=512, o_token_stride=520)),
    (append, dict(o_token_stride=500)), (append, dict(o_head_stride=60)), (append, dict(o_batch_stride=1000)),
    (append, dict(batch=(1 << 24) + 1, tokens=(1 << 24) + 1)),
    (attention, dict(Q=None)), (attention, dict(O=None)), (attention, dict(kv_len=None)), (attention, dict(heads=0)),
    (attention, dict(heads=7)), (attention, dict(tokens=5)), (attention, dict(o_token_stride=500)),
    (attention, dict(O=P, q_head_stride=64, o_head_stride=80)), (attention, dict(heads=4 << 16)),
    (attention, dict(seq_start=P, o_token_stride=64, o_head_stride=64 * 5)),
    (read, dict(K=None, V=None)), (read, dict(k_token_stride=200)), (read, dict(v_head_stride=32)),
    (read, dict(tokens=9)), (read, dict(tokens=(1 << 28) + 2)),
])
def test_bad_calls_are_refused(make, bad):
    assert not taken(*make(**bad))


@pytest.mark.parametrize("make,fine", [
    (append, dict(Q=None, Q_out=None, heads=0)), (append, dict(Q_out=P)), (append, dict(rope_dim=16)),
    (append, dict(tokens=7, seq_start=P)), (append, dict(o_batch_stride=64 * 24, o_token_stride=64, o_head_stride=192)),
    (append, dict(k_token_stride=1, k_head_stride=1)),   # an input's rows may overlap
    (attention, dict(O=P)), (attention, dict(heads=4)), (attention, dict(tokens=5, seq_start=P)),
    (attention, dict(o_batch_stride=512, o_token_stride=1024)),   # [token][batch][head]
    (attention, dict(seq_start=P, o_token_stride=64, o_head_stride=64 * 6)), (attention, dict(max_tokens=9, max_kv=999)),
    (read, dict(K=None)), (read, dict(V=None)), (read, dict(first=P)), (read, dict(V=None, v_token_stride=1)),
])
def test_calls_that_are_taken(make, fine):
    assert taken(*make(**fine))


def test_opcode_names():
    lib = load_backend()
    assert [lib.vnpu_opcode_name(i) for i in (64, 65, 66)] == [b"KV_APPEND_I8", b"KV_ATTENTION_I8", b"KV_READ_F32"]
    assert [lib.vnpu_opcode_name(i) for i in (17, 63, 67)] == [b"UNKNOWN"] * 3


def test_null_arguments():
    lib = load_backend()
    for fn in (lib.vnpu_kv_append_i8, lib.vnpu_kv_attention_i8, lib.vnpu_kv_read_f32):
        assert fn(None, None) == abi.ERR_INVALID_ARGUMENT
    assert lib.vnpu_kv_enqueue_noalloc(None, None, 1) == abi.ERR_INVALID_ARGUMENT
    assert lib.vnpu_kv_attention_workspace(None, None) == 0


def test_route_of_a_call():
    assert route(*attention()[:1], **attention()[1]).endswith("ws=0")


@pytest.mark.parametrize("make,bad,fine", [
    (append, dict(batch=1 << 20, tokens=1 << 20, Q=None, Q_out=None, cache=cache(kv_heads=16)), dict(cache=cache(kv_heads=2))),
    (append, dict(batch=1, tokens=1 << 28, heads=64, cache=cache(kv_heads=1, head_dim=256)), dict(heads=8, tokens=1 << 20)),
    (attention, dict(batch=1 << 24, tokens=1 << 24, heads=1, cache=cache(kv_heads=1)), dict(batch=1 << 22, tokens=1 << 22)),
    (attention, dict(batch=1, tokens=1 << 26, heads=64, cache=cache(kv_heads=64)), dict(tokens=1 << 24)),
    (read, dict(batch=1 << 24, tokens=1 << 24), dict(batch=1 << 20, tokens=1 << 20)),
])
def test_grids_that_cannot_be_launched_are_refused(make, bad, fine):
    """2^32 threads and more in one dimension: pages of a call, sequences, tiles of rows."""
    opcode, fields = make(**bad)
    assert not taken(opcode, fields)
    assert taken(opcode, {**fields, **fine})


@pytest.mark.parametrize("make", [append, attention, read])
@pytest.mark.parametrize("page", [16, 256])
def test_rooms_of_more_than_a_billion_tokens_are_refused(make, page):
    assert taken(*make(cache(page_size=page, table_ld=(1 << 30) // page)))
    assert not taken(*make(cache(page_size=page, table_ld=(1 << 30) // page + 1)))


def test_routes_over_sizes():
    """One workgroup for a sequence and head, keys split over workgroups, tiles, tiles with split keys, both."""
    def text(max_kv, batch=1, tokens=1, seq_start=None):
        c = cache(kv_heads=8, head_dim=128, table_ld=1 << 16)
        opcode, f = attention(c, batch=batch, tokens=tokens, max_kv=max_kv, seq_start=seq_start)
        return dict(x.split("=") for x in route(opcode, **f).split())

    assert text(500)["few"] == "1" and text(500)["ws"] == "0"
    assert int(text(100000)["few"]) > 1 and int(text(100000)["ws"]) > 0
    assert text(4096, batch=64, tokens=64)["few"] == "64" and text(4096, batch=64, tokens=64)["ws"] == "0"
    assert text(4096, tokens=64)["few"] == "0" and text(4096, tokens=64)["tile"] == "64"
    assert text(4096, tokens=4096)["tile"] == "64" and text(4096, tokens=4096)["parts"] == "1"
    assert text(1 << 14, tokens=1 << 14)["tile"] == "128" and text(1 << 14, tokens=1 << 14)["parts"] == "1"
    assert int(text(4096, tokens=100)["parts"]) > 1 and int(text(4096, tokens=100)["ws"]) > 0
    mixed = text(4096, batch=64, tokens=300, seq_start=P)
    assert mixed["few"] != "0" and mixed["tile"] != "0"
