"""Operators of a serving step with 4-bit weights and a shared prompt, as cases that can be timed and checked: MATMUL_I4
(products with 4-bit weights and group scales), ROPE_AXES_F32 (rotary positions with several axes) and
KV_PREFIX_ATTENTION_I8 (attention of a batch whose sequences share the first pages of the paged int8 KV cache).

With `own` false, `run` computes each operator in plain torch operations; with `own` true it submits the command packets
of this repository's stream, built once as a C program builds them.  Both work on the same tensors.

4-bit weights: codes two a byte, low half first, as [K][N / 2] ("kn") or [N][K / 2] ("nk"); a weight is (code - zero) *
scale, scale and zero [ceil(K / group)][N], zero 8 where there are none.
The cache: as KV_ATTENTION_I8 has it; the first `prefix` tokens of every sequence are the pages of one table.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA = 10000.0


def _matmul(name, rows, k, n, group, zeros=False, layout="nk", bias=False, epilogue="none"):
    return {"name": name, "kind": "matmul", "rows": rows, "k": k, "n": n, "group": group, "zeros": zeros,
            "layout": layout, "bias": bias, "epilogue": epilogue}


def _rope(name, tokens, heads, kv_heads, head_dim, sections, order="blocks", ladders="one", rotation="half",
          layout="rows", batch=1):
    """sections: pairs of each axis, as text; layout: rows of a fused projection, or [batch][heads][tokens][head_dim]."""
    return {"name": name, "kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sections": sections, "order": order, "ladders": ladders, "rotation": rotation, "layout": layout,
            "batch": batch}


def _prefix(name, batch, tokens, prefix, mine, heads, kv_heads, head_dim, page, ragged=False, causal=True):
    """tokens: (most) new tokens of a sequence; mine: (most) tokens of a sequence behind the prefix, the new ones among
    them; ragged: sequences differ."""
    return {"name": name, "kind": "prefix", "batch": batch, "tokens": tokens, "prefix": prefix, "mine": mine,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "ragged": ragged, "causal": causal}


def listed():
    return [
        # One token through a square projection of a 4096-wide model: latency and the stream of codes.
        _matmul("i4_token", 1, 4096, 4096, 128),
        # One token's logits over a vocabulary of 32000, with zero points.
        _matmul("i4_vocabulary", 1, 4096, 32000, 128, zeros=True),
        # Eight sequences decoding through the down projection, smaller groups, weights stored by rows of K.
        _matmul("i4_batch", 8, 11008, 4096, 64, zeros=True, layout="kn"),
        # The gate of a small model for a few drafted tokens of several sequences: odd sizes, a bias, an activation.
        _matmul("i4_odd", 37, 1000, 1001, 32, zeros=True, bias=True, epilogue="silu"),
        # A prompt of 2048 tokens through the up projection: the matrix cores.
        _matmul("i4_prompt", 2048, 4096, 11008, 128, zeros=True),
        # Eight sequences decoding, three axes of a text and image model: latency.
        _rope("rope_token", 8, 32, 8, 128, "16 24 24"),
        # The patches of some images in an image encoder, 16 heads of 80: height and width, a ladder of frequencies each,
        # pairs side by side.
        _rope("rope_image", 1601, 16, 16, 80, "20 20", ladders="own", rotation="interleaved"),
        # Prompts of 4096 tokens in all with time, height and width in turns, head-major as ATTENTION_F32 takes them.
        _rope("rope_prompt", 4096, 32, 8, 128, "24 20 20", order="turns", layout="heads", batch=2),
        # Four short chats behind one instruction, a small model: latency.
        _prefix("prefix_small", 4, 1, 320, 20, 8, 8, 64, 16),
        # A serving batch behind a shared prompt of 4096 tokens, four query heads to a key head.
        _prefix("prefix_decode", 32, 1, 4096, 500, 32, 8, 128, 32, ragged=True),
        # Many short answers about one long document.
        _prefix("prefix_long", 64, 1, 32768, 1000, 32, 8, 128, 64, ragged=True),
        # Chunks of questions and single tokens behind a shared prompt, head size 80, odd lengths.
        _prefix("prefix_mixed", 6, 331, 2000, 777, 16, 4, 80, 16, ragged=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _draw_matmul(rng):
    while True:
        rows = rng.choice((1, 1, rng.randint(2, 8), rng.randint(9, 64), _log_int(rng, 65, 2048)))
        k, n = _log_int(rng, 48, 16384), _log_int(rng, 16, 32000)
        if rng.random() < 0.5:   # half of the projections of real models are whole multiples of 128
            k, n = max(128, k // 128 * 128), max(128, n // 128 * 128)
        c = _matmul("", rows, k, n, rng.choice((32, 64, 128, 128)), rng.random() < 0.6, rng.choice(("nk", "kn")),
                    rng.random() < 0.3, rng.choice(("none", "none", "silu", "gelu", "relu")))
        if k * n <= 4096 * 32000 and work(c)["flops"] <= 1.8e11:
            return c


def _draw_rope(rng):
    while True:
        head_dim = rng.choice((64, 80, 96, 128, 128, 256))
        axes, pairs = rng.choice((1, 2, 3, 3, 4)), head_dim // 2
        if rng.random() < 0.2:
            pairs = rng.randint(axes, pairs)   # the rest of a head is not turned
        cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if pairs > axes else list(range(1, axes))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        kv_heads = rng.choice((1, 2, 4, 8, 8, 16))
        batch = rng.choice((1, 1, 2, 3, 8))
        c = _rope("", batch * _log_int(rng, 1, 4096), kv_heads * rng.choice((1, 2, 4, 5, 8)), kv_heads, head_dim,
                  " ".join(str(x) for x in sections), rng.choice(("blocks", "turns")), rng.choice(("one", "own")),
                  rng.choice(("half", "interleaved")), rng.choice(("rows", "heads")), batch)
        if c["heads"] <= 64 and work(c)["bytes"] <= 1.6e8:
            return c


def _draw_prefix(rng):
    while True:
        kv_heads = rng.choice((1, 2, 4, 8, 8, 32))
        heads = kv_heads * rng.choice((1, 2, 4, 4, 5, 8))
        batch = rng.choice((1, 2, 3, 5, 8, 17, 33, 64))
        page = rng.choice((16, 16, 32, 64, 128, 256))
        tokens = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1000)))
        prefix = max(1, _log_int(rng, 16, 32768) // page) * page
        mine = tokens + (0 if rng.random() < 0.2 else _log_int(rng, 1, 2000))
        c = _prefix("", batch, tokens, prefix, mine, heads, kv_heads, rng.choice((64, 64, 80, 96, 128, 128, 256)), page,
                    batch > 1 and rng.random() < 0.7, rng.random() < 0.8)
        if heads <= 64 and work(c)["flops"] <= 3.5e10 and batch * heads * tokens * (prefix + mine) <= 1 << 28:
            return c


def draw(rng):
    c = rng.choice((_draw_matmul, _draw_matmul, _draw_rope, _draw_prefix, _draw_prefix))(rng)
    del c["name"]
    return c


def _lengths(c):
    """New tokens and tokens behind the prefix, of each sequence: from the case alone."""
    batch, tokens, mine = c["batch"], c["tokens"], c["mine"]
    if not c["ragged"]:
        return [tokens] * batch, [mine] * batch
    r = random.Random(batch * 1000003 + tokens * 1009 + mine)
    n, lens = [tokens], [mine]
    for i in range(1, batch):
        m = 1 if tokens == 1 or i % 3 == 2 else r.randint(1, tokens)
        n.append(m)
        lens.append(m + int((mine - tokens) * r.random()))
    return n, lens


def _sections(c):
    return [int(x) for x in c["sections"].split()]


def _groups(c):
    return -(-c["k"] // c["group"])


def work(case):
    c = case
    if c["kind"] == "matmul":
        weights = c["k"] * c["n"] / 2 + _groups(c) * c["n"] * (5 if c["zeros"] else 4)
        return {"bytes": weights + 4 * c["rows"] * (c["k"] + c["n"]) + 4 * c["n"] * c["bias"],
                "flops": 2 * c["rows"] * c["k"] * c["n"]}
    if c["kind"] == "rope":
        turned = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": 8 * turned + 4 * c["tokens"] * len(_sections(c)), "flops": 3 * turned}
    n, mine = _lengths(c)
    H, G, D, T, P = c["heads"], c["kv_heads"], c["head_dim"], sum(n), c["prefix"]
    pairs = T * P + sum(a * (b - a) + a * (a + 1) // 2 if c["causal"] else a * b for a, b in zip(n, mine))
    pages = P // c["page"] + sum(-(-b // c["page"]) for b in mine)
    return {"bytes": 8 * T * H * D + 2 * (P + sum(mine)) * G * D + 8 * pages * G, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

class _State:
    packed = None

    def __del__(self):
        if self.packed is not None:
            _session().lib.vnpu_packed_weights_i4_destroy(self.packed)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 29)
    return g


def _inputs(c, seed):
    """What both forms and the values in 64 bits start from, on the GPU; the same for the same seed."""
    return globals()["_inputs_" + c["kind"]](c, _generator(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _inputs_matmul(c, g):
    s = _State()
    K, N = c["k"], c["n"]
    # Activations of a model: a few of the channels are much larger than the others.
    loud = 1.0 + 30.0 * (torch.rand(K, generator=g, device="cuda") < 0.004)
    s.a = _normal(g, c["rows"], K) * loud
    rows, cols = (K, N) if c["layout"] == "kn" else (N, K)
    low, high = ((_normal(g, rows, -(-cols // 2)) * 2.7).round().add(8).clamp(0, 15).to(torch.uint8) for _ in range(2))
    s.codes = low | high << 4
    s.scales = 0.004 + 0.004 * torch.rand(_groups(c), N, generator=g, device="cuda")
    s.zeros = (torch.randint(5, 12, (_groups(c), N), generator=g, device="cuda").to(torch.uint8) if c["zeros"] else None)
    s.bias = _normal(g, N) if c["bias"] else None
    return s


def _inputs_rope(c, g):
    s = _State()
    T, H, G, D, B = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], c["batch"]
    if c["layout"] == "heads":
        s.q, s.k = _normal(g, B, H, T // B, D), _normal(g, B, G, T // B, D)
    else:   # the rows that one projection to queries, keys and values leaves
        rows = _normal(g, T, (H + 2 * G) * D)
        s.q, s.k = rows[:, :H * D], rows[:, H * D:(H + G) * D]
    # Text runs along all axes alike, images from a corner of their own along height and width.
    axes = len(_sections(c))
    at = torch.arange(T, device="cuda", dtype=torch.int32) + torch.randint(0, 100000, (1,), generator=g, device="cuda").int()
    grid = torch.randint(0, 64, (axes, T), generator=g, device="cuda").int()
    image = (torch.arange(T, device="cuda") // 97) % 3 != 0
    s.positions = at + torch.where(image, grid, torch.zeros_like(grid))
    return s


def _inputs_prefix(c, g):
    s = _State()
    n, mine = _lengths(c)
    B, H, G, D, ps, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["prefix"]
    s.n, s.mine, T = n, mine, sum(n)
    shared, ld = P // ps, max(-(-b // ps) for b in mine)
    pages = shared + B * ld + 3
    # Pages lie anywhere in the pool; every sequence's table begins with the shared ones.
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s.prefix = order[:shared].contiguous()
    s.table = torch.cat((s.prefix.expand(B, shared), order[shared:shared + B * ld].reshape(B, ld)), dim=1).contiguous()
    # Codes and scales of normal values quantized by block: the largest of some hundred values is 127.
    s.k8 = (_normal(g, pages, G, ps, D) * 38).round().clamp(-127, 127).to(torch.int8)
    s.v8 = (_normal(g, pages, G, D, ps) * 38).round().clamp(-127, 127).to(torch.int8)
    s.ks = 0.024 + 0.012 * torch.rand(pages, G, generator=g, device="cuda")
    s.vs = 0.024 + 0.012 * torch.rand(pages, G, generator=g, device="cuda")
    s.start = torch.tensor([sum(n[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda")
    s.kv_len = torch.tensor([P + b for b in mine], dtype=torch.int32, device="cuda")
    s.q = _normal(g, T, H * D)
    return s


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s.case = c
    if c["kind"] == "matmul":
        s.out = torch.empty(c["rows"], c["n"], device="cuda")
    elif c["kind"] == "rope":
        s.q_out, s.k_out = (torch.empty(x.shape, device="cuda") for x in (s.q, s.k))
    else:
        s.out = torch.empty(s.q.shape, device="cuda")
    torch.cuda.synchronize()
    if own:
        _packet(s)
    return s


# ---------------------------------------------------------------------------
# The framework's commands
# ---------------------------------------------------------------------------

_sessions = []


def _session():
    if not _sessions:
        path = os.path.join(ROOT, "npuxl-improved_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from vnpu_mi355x import Session
        _sessions.append(Session())
    return _sessions[0]


def _strides(prefix, layout, tokens, heads, head_dim, row=0):
    """Strides in elements: rows of tokens (0: packed), or [batch][heads][tokens][head_dim]."""
    values = (heads * tokens * head_dim, head_dim, tokens * head_dim) if layout == "heads" else (
        tokens * (row or heads * head_dim), row or heads * head_dim, head_dim)
    return dict(zip((prefix + "_batch_stride", prefix + "_token_stride", prefix + "_head_stride"), values))


def _packet(s):
    """The command packet of a pass, built once, as a program that submits it at every step keeps it; the weights packed."""
    session = _session()
    from vnpu_mi355x import abi
    c = s.case

    def pointer(t):
        return None if t is None else t.data_ptr()

    if c["kind"] == "matmul":
        s.packed = ctypes.c_void_p()
        session.check("vnpu_pack_weights_i4", session.lib.vnpu_pack_weights_i4(
            session.dev, pointer(s.codes), pointer(s.scales), pointer(s.zeros), c["k"], c["n"], c["group"], 0,
            int(c["layout"] == "nk"), ctypes.byref(s.packed)))
        epilogue = {"none": abi.EPI_NONE, "relu": abi.EPI_RELU, "silu": abi.EPI_SILU, "gelu": abi.EPI_GELU_TANH}
        command = session.command(abi.OP_MATMUL_I4, A=pointer(s.a), B=s.packed, bias=pointer(s.bias), C=pointer(s.out),
                                  M=c["rows"], K=c["k"], N=c["n"], epilogue=epilogue[c["epilogue"]])
    elif c["kind"] == "rope":
        H, G, D, n = c["heads"], c["kv_heads"], c["head_dim"], c["tokens"] // c["batch"]
        row, sections = (H + 2 * G) * D, _sections(c)
        command = session.command(
            abi.OP_ROPE_AXES_F32, Q=pointer(s.q), Q_out=pointer(s.q_out), K=pointer(s.k), K_out=pointer(s.k_out),
            positions=pointer(s.positions), batch=c["batch"], tokens=c["tokens"], heads=H, kv_heads=G, head_dim=D,
            axes=len(sections), sections=(ctypes.c_uint32 * 4)(*sections),
            order={"blocks": abi.AXES_BLOCKS, "turns": abi.AXES_TURNS}[c["order"]],
            ladders={"one": abi.AXES_ONE_LADDER, "own": abi.AXES_OWN_LADDERS}[c["ladders"]],
            rotation={"half": abi.ROTATE_HALF, "interleaved": abi.ROTATE_INTERLEAVED}[c["rotation"]], theta_base=THETA,
            **_strides("q", c["layout"], n, H, D, row), **_strides("o", c["layout"], n, H, D),
            **_strides("k", c["layout"], n, G, D, row), **_strides("ko", c["layout"], n, G, D))
    else:
        cache = abi.KvCache(k=pointer(s.k8), v=pointer(s.v8), k_scales=pointer(s.ks), v_scales=pointer(s.vs),
                            table=pointer(s.table), pages=s.k8.shape[0], page_size=c["page"], kv_heads=c["kv_heads"],
                            head_dim=c["head_dim"], table_ld=s.table.shape[1])
        attention = abi.KvAttentionArgs(
            cache=cache, Q=pointer(s.q), O=pointer(s.out), kv_len=pointer(s.kv_len),
            seq_start=pointer(s.start) if c["ragged"] else None, batch=c["batch"], tokens=sum(s.n), heads=c["heads"],
            max_tokens=max(s.n), max_kv=c["prefix"] + max(s.mine), causal=int(c["causal"]))
        command = session.command(abi.OP_KV_PREFIX_ATTENTION_I8, attention=attention, prefix_table=pointer(s.prefix),
                                  prefix_len=c["prefix"])
    s.commands = (abi.Command * 1)(command)


def _outputs(s):
    return {"q": s.q_out, "k": s.k_out} if s.case["kind"] == "rope" else {"out": s.out}


def run(state):
    s = state
    if own:
        session = _session()
        session.check("vnpu_stream_submit", session.lib.vnpu_stream_submit(session.stream, s.commands, 1, None))
    else:
        globals()["_plain_" + s.case["kind"]](s)
    return _outputs(s)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _codes(s, c):
    """[K][N], whole numbers."""
    rows, cols = (c["k"], c["n"]) if c["layout"] == "kn" else (c["n"], c["k"])
    codes = torch.stack((s.codes & 15, s.codes >> 4), dim=2).reshape(rows, -1)[:, :cols]
    return codes if c["layout"] == "kn" else codes.t()


def _plain_matmul(s):
    c = s.case
    group = torch.arange(c["k"], device="cuda") // c["group"]
    zeros = 8.0 if s.zeros is None else s.zeros.float()[group]
    x = torch.matmul(s.a, (_codes(s, c).float() - zeros) * s.scales[group])
    if s.bias is not None:
        x = x + s.bias
    if c["epilogue"] == "relu":
        x = torch.maximum(x, torch.zeros_like(x))
    elif c["epilogue"] == "silu":
        x = x / (1.0 + torch.exp(-x))
    elif c["epilogue"] == "gelu":
        x = 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    s.out.copy_(x)


def _pairs(c):
    """Of each pair that is turned: its axis and its exponent of theta."""
    left, used, axis, place = _sections(c), [0] * len(_sections(c)), [], []
    a = 0
    for _ in range(sum(left)):
        while not left[a]:
            a = (a + 1) % len(left)
        axis.append(a)
        place.append(used[a])
        left[a] -= 1
        used[a] += 1
        if c["order"] == "turns":
            a = (a + 1) % len(left)
    if c["ladders"] == "own":
        exponent = [i / used[a] for a, i in zip(axis, place)]
    else:
        exponent = [j / len(axis) for j in range(len(axis))]
    return axis, exponent


def _by_token(x, heads, head_dim):
    """[tokens][heads][head_dim] of packed rows or of [batch][heads][tokens][head_dim]."""
    if x.dim() == 4:
        return x.transpose(1, 2).reshape(-1, heads, head_dim)
    return x.reshape(-1, heads, head_dim)


def _from_tokens(y, like):
    if like.dim() == 4:
        b, h, n, d = like.shape
        return y.reshape(b, n, h, d).transpose(1, 2)
    return y.reshape(like.shape)


def _halves(c):
    """Elements of the pairs of a head."""
    pairs = sum(_sections(c))
    return (slice(0, pairs), slice(pairs, 2 * pairs)) if c["rotation"] == "half" else (
        slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))


def _plain_rope(s):
    c = s.case
    axis, exponent = _pairs(c)
    rate = THETA ** -torch.tensor(exponent, device="cuda", dtype=torch.float64)
    angle = s.positions[torch.tensor(axis, device="cuda")].t().double() * rate
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    first, second = _halves(c)
    for x, heads, out in ((s.q, c["heads"], s.q_out), (s.k, c["kv_heads"], s.k_out)):
        x = _by_token(x, heads, c["head_dim"])
        y, a, b = x.clone(), x[..., first].double(), x[..., second].double()
        y[..., first], y[..., second] = (a * cos - b * sin).float(), (a * sin + b * cos).float()
        out.copy_(_from_tokens(y, out))


def _keys_values(s, pages):
    """f32 [...][kv_heads][tokens][head_dim] of tables [...][pages]."""
    pages = pages.long()
    k = s.k8[pages].float() * s.ks[pages][..., None, None]
    v = (s.v8[pages].float() * s.vs[pages][..., None, None]).transpose(-1, -2)
    return tuple(x.transpose(-4, -3).flatten(-3, -2) for x in (k, v))


def _plain_prefix(s):
    c = s.case
    B, H, G, D, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["prefix"]
    n, T = max(s.n), sum(s.n)
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(s.start[1:].long(), t, right=True)
    i = t - s.start.long()[seq]
    q = torch.zeros(B, n, H, D, device="cuda")
    q[seq, i] = s.q.reshape(T, H, D)
    q = q.reshape(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, D) * (1.0 / math.sqrt(D))
    k0, v0 = _keys_values(s, s.prefix)
    k1, v1 = _keys_values(s, s.table[:, P // c["page"]:])
    shared = torch.matmul(q.transpose(0, 1).reshape(G, -1, D), k0.transpose(1, 2).contiguous())
    mine = torch.matmul(q, k1.transpose(2, 3).contiguous()).reshape(B, G, H // G, n, -1)
    key = torch.arange(k1.shape[2], device="cuda")
    length = s.kv_len.long() - P
    limit = length[:, None].expand(B, n)
    if c["causal"]:
        new = s.start[1:].long() - s.start[:-1].long()
        limit = torch.minimum(limit, (length - new)[:, None] + torch.arange(n, device="cuda") + 1)
    mine = mine.masked_fill_(key >= limit[:, None, None, :, None], -math.inf).reshape(B, G, H // G * n, -1)
    shared = shared.reshape(G, B, H // G * n, P).transpose(0, 1)
    top = torch.maximum(shared.amax(dim=-1, keepdim=True), mine.amax(dim=-1, keepdim=True))
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    total = shared.sum(dim=-1, keepdim=True) + mine.sum(dim=-1, keepdim=True)
    o = torch.matmul(shared.transpose(0, 1).reshape(G, -1, P), v0.contiguous()).reshape(G, B, H // G * n, D).transpose(0, 1)
    o = (o + torch.matmul(mine, v1.contiguous())) / total
    o = o.reshape(B, G, H // G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    s.out.copy_(o[seq, i].reshape(T, H * D))


# ---------------------------------------------------------------------------
# The values from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, _inputs(case, seed))


def _exact_matmul(c, s):
    K, N = c["k"], c["n"]
    bytes_ = s.codes.int()
    if c["layout"] == "kn":
        w = torch.empty(K, N + N % 2, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (bytes_ % 16).double(), (bytes_ // 16).double()
        w = w[:, :N]
    else:
        w = torch.empty(K + K % 2, N, dtype=torch.float64, device="cuda")
        w[0::2], w[1::2] = (bytes_ % 16).double().t(), (bytes_ // 16).double().t()
        w = w[:K]
    out = torch.zeros(c["rows"], N, dtype=torch.float64, device="cuda")
    for i in range(_groups(c)):
        at = slice(i * c["group"], min(K, (i + 1) * c["group"]))
        zero = 8.0 if s.zeros is None else s.zeros[i].double()
        out += (s.a[:, at].double() @ (w[at] - zero)) * s.scales[i].double()
    if s.bias is not None:
        out += s.bias.double()
    if c["epilogue"] == "relu":
        out = out.clamp(min=0.0)
    elif c["epilogue"] == "silu":
        out = out * torch.sigmoid(out)
    elif c["epilogue"] == "gelu":
        # 1/2 (1 + tanh u) = 1 / (1 + exp(-2 u))
        out = out * torch.sigmoid(math.sqrt(8.0 / math.pi) * (out + 0.044715 * out ** 3))
    return {"out": out}


def _exact_rope(c, s):
    """Pairs turned as complex numbers, axis by axis."""
    sections = _sections(c)
    total = sum(sections)
    if c["order"] == "turns":
        rounds = [(r, a) for r in range(max(sections)) for a in range(len(sections)) if r < sections[a]]
    else:
        rounds = [(r, a) for a in range(len(sections)) for r in range(sections[a])]
    unit = torch.empty(c["tokens"], total, dtype=torch.complex128, device="cuda")
    for j, (r, a) in enumerate(rounds):
        power = r / sections[a] if c["ladders"] == "own" else j / total
        angle = s.positions[a].double() * math.exp(-power * math.log(THETA))
        unit[:, j] = torch.polar(torch.ones_like(angle), angle)
    out = {}
    for name, x, heads in (("q", s.q, c["heads"]), ("k", s.k, c["kv_heads"])):
        y = _by_token(x, heads, c["head_dim"]).double()
        if c["rotation"] == "half":
            z = torch.complex(y[..., :total], y[..., total:2 * total]) * unit[:, None]
            turned = torch.cat((z.real, z.imag), dim=-1)
        else:
            z = torch.view_as_complex(y[..., :2 * total].reshape(*y.shape[:2], total, 2).contiguous()) * unit[:, None]
            turned = torch.view_as_real(z).flatten(-2)
        out[name] = _from_tokens(torch.cat((turned, y[..., 2 * total:]), dim=-1), x)
    return out


def _exact_prefix(c, s):
    """Sequence by sequence over the whole of its table."""
    H, G, D, ps, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["prefix"]
    out, at = [], 0
    for b, (n, mine) in enumerate(zip(s.n, s.mine)):
        kv = P + mine
        pages = s.table[b, :-(-kv // ps)].long()
        k = (s.k8[pages].double() * s.ks[pages].double()[:, :, None, None]).transpose(0, 1).reshape(G, -1, D)[:, :kv]
        v = (s.v8[pages].double() * s.vs[pages].double()[:, :, None, None]).permute(1, 0, 3, 2).reshape(G, -1, D)[:, :kv]
        q = s.q[at:at + n].reshape(n, H, D).double()
        o = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
        hidden = None
        if c["causal"]:
            hidden = torch.arange(kv, device="cuda")[None, :] > kv - n + torch.arange(n, device="cuda")[:, None]
        for h in range(H):
            score = (q[:, h] @ k[h // (H // G)].T) / math.sqrt(D)
            if hidden is not None:
                score = score.masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(score, dim=1) @ v[h // (H // G)]
        out.append(o.reshape(n, H * D))
        at += n
    return {"out": torch.cat(out)}
