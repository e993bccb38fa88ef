"""The operators of the paged int8 KV cache as cases that can be timed and checked: KV_APPEND_I8 (rotate, quantize and
append keys and values), KV_ATTENTION_I8 (attention over the cache) and KV_READ_F32 (the cache's values in f32).

With `own` false, `run` computes each operator in plain torch operations; with `own` true it submits the command packets
of this repository's stream, built once as a C program builds them.  Both work on the same tensors.

The cache: pages of `page` tokens; k codes [pages][kv_heads][page][head_dim], v codes [pages][kv_heads][head_dim][page],
one f32 scale for each (page, kv head) and side; table [batch][table_ld] names the pages of each sequence in order.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA = 10000.0


def _case(name, kind, batch, tokens, kv, heads, kv_heads, head_dim, page, ragged=False, causal=True, rotation="half",
          layout="rows"):
    """tokens: (most) new tokens of a sequence, or tokens read; kv: (longest) length with them; ragged: sequences differ."""
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "kv": kv, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "ragged": ragged, "causal": causal,
            "rotation": rotation, "layout": layout}


def listed():
    return [
        # Eight sequences decoding: one new token each, taken from the rows of a fused QKV projection. Latency.
        _case("append_decode", "append", 8, 1, 4096, 32, 8, 128, 16),
        # Sequences of different lengths adding parts of their prompts, pages that begin and end anywhere, head size 80,
        # pairs interleaved.
        _case("append_ragged", "append", 7, 149, 1500, 12, 4, 80, 32, ragged=True, rotation="interleaved"),
        # A prompt of 2048 tokens enters an empty cache: bandwidth.
        _case("append_prompt", "append", 1, 2048, 2048, 32, 8, 128, 64),
        # One token of a small model (8 heads of 64) over 128 cached states that all may be seen: latency.
        _case("attn_token_small", "attention", 1, 1, 128, 8, 8, 64, 16, causal=False),
        # Batched decode of a 4096-wide model, 32 heads of 128, 4096 tokens each: the stream of codes.
        _case("attn_decode", "attention", 8, 1, 4096, 32, 32, 128, 16),
        # A serving batch: 64 sequences of 100 to 8000 tokens, four query heads to a key head.
        _case("attn_decode_ragged", "attention", 64, 1, 8000, 32, 8, 128, 32, ragged=True),
        # One sequence with a long document: one row for each head, work only along the keys.
        _case("attn_long", "attention", 1, 1, 131072, 32, 8, 128, 64),
        # Five drafted tokens verified for four sequences.
        _case("attn_verify", "attention", 4, 5, 3001, 32, 8, 128, 16, ragged=True),
        # Chunks of prompts and single tokens in one batch, head size 80, sixteen heads to four, odd lengths.
        _case("attn_mixed", "attention", 6, 331, 1831, 16, 4, 80, 32, ragged=True),
        # A prompt of 4096 tokens attends to itself: the matrix cores.
        _case("attn_prompt", "attention", 1, 4096, 4096, 32, 8, 128, 64, layout="heads"),
        # The first 300 tokens or fewer of a few sequences in f32, for a peer: latency.
        _case("read_ragged", "read", 5, 300, 777, 12, 4, 80, 16, ragged=True),
        # A whole cached prompt of eight sequences in f32, head-major as ATTENTION_F32 takes it: bandwidth.
        _case("read_prompt", "read", 8, 2048, 2048, 8, 8, 128, 16, layout="heads"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    while True:
        kind = rng.choice(("append", "attention", "attention", "attention", "read"))
        kv_heads = rng.choice((1, 2, 4, 8, 8, 32))
        heads = kv_heads * rng.choice((1, 2, 4, 4, 5, 8))
        batch = rng.choice((1, 1, 2, 3, 5, 8, 17, 33, 64))
        ragged = batch > 1 and rng.random() < 0.6
        tokens = rng.choice((1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)))
        if kind == "read":
            tokens = _log_int(rng, 1, 4096)
        past = 0 if rng.random() < 0.2 else _log_int(rng, 1, 131072)
        c = _case("", kind, batch, tokens, past + tokens, heads, kv_heads, rng.choice((64, 64, 80, 96, 112, 128, 128, 256)),
                  rng.choice((16, 16, 32, 64, 128, 256)), ragged, rng.random() < 0.8,
                  rng.choice(("half", "half", "interleaved", "none")), "heads" if not ragged and rng.random() < 0.4 else "rows")
        del c["name"]
        n, kv = _lengths(c)
        codes = 2 * sum(kv) * kv_heads * c["head_dim"]
        padded = batch * max(kv) * kv_heads * c["head_dim"]
        if heads > 64 or codes > 300 << 20 or padded > 1 << 29:
            continue
        if kind == "attention":
            scores = batch * heads * max(n) * max(kv)
            if work(c)["flops"] <= 1.4e11 and scores <= 1 << 29:
                return c
        elif work(c)["bytes"] <= 1.6e8:
            return c


def _lengths(c):
    """New (or read) tokens and cached length with them, of each sequence: from the case alone."""
    batch, tokens, kv = c["batch"], c["tokens"], c["kv"]
    if not c["ragged"]:
        return [tokens] * batch, [kv] * batch
    r = random.Random(batch * 1000003 + tokens * 1009 + kv)
    n, lens = [tokens], [kv]
    for i in range(1, batch):
        m = 1 if tokens == 1 or i % 3 == 2 else r.randint(1, tokens)
        n.append(m)
        lens.append(m + int((kv - tokens) * (0.0125 + 0.9875 * r.random())))
    return n, lens


def _pairs(c):
    n, kv = _lengths(c)
    return sum(a * (b - a) + a * (a + 1) // 2 if c["causal"] else a * b for a, b in zip(n, kv))


def work(case):
    c = case
    n, kv = _lengths(c)
    H, G, D, T, S = c["heads"], c["kv_heads"], c["head_dim"], sum(n), sum(kv)
    if c["kind"] == "append":
        # q, k, v read and rotated q written in f32, two bytes of codes; then the touched pages' tokens are read in f32.
        back = sum(b - (b - a) // c["page"] * c["page"] for a, b in zip(n, kv))
        return {"bytes": 4 * T * (2 * H + 2 * G) * D + 2 * T * G * D + 10 * back * G * D,
                "flops": T * (3 * (H + G) + 2 * G) * D + 2 * back * G * D}
    pages = sum(-(-b // c["page"]) for b in kv)
    if c["kind"] == "read":
        return {"bytes": 10 * T * G * D + 8 * sum(-(-a // c["page"]) for a in n) * G, "flops": 2 * T * G * D}
    return {"bytes": 8 * T * H * D + 2 * S * G * D + 8 * pages * G, "flops": 4 * _pairs(c) * H * D}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

class _State:
    pass


def _strides(layout, tokens, heads, head_dim, row=0):
    """(batch, token, head) strides in elements: packed token rows, or [batch][heads][tokens][head_dim]."""
    if layout == "heads":
        return heads * tokens * head_dim, head_dim, tokens * head_dim
    return 0, row or heads * head_dim, head_dim


def _inputs(c, seed):
    """What both forms and the values in 64 bits start from, on the GPU; the same for the same seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    n, kv = _lengths(c)
    B, H, G, D, ps = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    s, T = _State(), sum(n)
    s.n, s.kv = n, kv
    ld = max(-(-b // ps) for b in kv)
    pages = B * ld + 3
    # Pages lie anywhere in the pool; entries behind a sequence's last page are never read.
    s.table = torch.randperm(pages, generator=g, device="cuda")[:B * ld].to(torch.int32).reshape(B, ld)
    # Codes and scales of normal values quantized by block: the largest of some hundred values is 127.
    s.k8 = (normal(pages, G, ps, D) * 38).round().clamp(-127, 127).to(torch.int8)
    s.v8 = (normal(pages, G, D, ps) * 38).round().clamp(-127, 127).to(torch.int8)
    s.ks = 0.024 + 0.012 * torch.rand(pages, G, generator=g, device="cuda")
    s.vs = 0.024 + 0.012 * torch.rand(pages, G, generator=g, device="cuda")
    s.start = torch.tensor([sum(n[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda")
    s.kv_len = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s.past = torch.tensor([b - a for a, b in zip(n, kv)], dtype=torch.int32, device="cuda")
    if c["kind"] == "append":
        if c["layout"] == "heads":
            s.q, s.k, s.v = normal(B, H, n[0], D), normal(B, G, n[0], D), normal(B, G, n[0], D)
        else:  # the rows that one projection to queries, keys and values leaves
            rows = normal(T, (H + 2 * G) * D)
            s.q, s.k, s.v = rows[:, :H * D], rows[:, H * D:(H + G) * D], rows[:, (H + G) * D:]
        # What is read back: the tokens of every page that the call touched.
        s.first = s.past // ps * ps
        back = [b - (b - a) // ps * ps for a, b in zip(n, kv)]
        s.read_n, s.read_start = back, torch.tensor([sum(back[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda")
    elif c["kind"] == "attention":
        s.q = normal(B, H, n[0], D) if c["layout"] == "heads" else normal(T, H * D)
    else:
        s.first, s.read_n, s.read_start = torch.zeros_like(s.past), n, s.start
    return s


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s.case = c
    G, D = c["kv_heads"], c["head_dim"]
    if c["kind"] in ("append", "attention"):
        s.out = torch.empty(s.q.shape, dtype=torch.float32, device="cuda")
    if c["kind"] in ("append", "read"):
        heads = c["kind"] == "read" and c["layout"] == "heads"
        shape = (c["batch"], G, s.read_n[0], D) if heads else (sum(s.read_n), G * D)
        s.k32, s.v32 = (torch.empty(shape, dtype=torch.float32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    if own:
        _packets(s)
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


def _packets(s):
    """The command packets of one pass, built once, as a program that submits them at every step keeps them."""
    session = _session()
    from vnpu_mi355x import abi
    c = s.case
    B, H, G, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    T, layout = sum(s.n), c["layout"]
    cache = abi.KvCache(k=s.k8.data_ptr(), v=s.v8.data_ptr(), k_scales=s.ks.data_ptr(), v_scales=s.vs.data_ptr(),
                        table=s.table.data_ptr(), pages=s.k8.shape[0], page_size=c["page"], kv_heads=G, head_dim=D,
                        table_ld=s.table.shape[1])
    start = s.start.data_ptr() if c["ragged"] else None

    def strides(prefix, values):
        return dict(zip((prefix + "_batch_stride", prefix + "_token_stride", prefix + "_head_stride"), values))

    commands = []
    if c["kind"] == "append":
        row = 0 if layout == "heads" else (H + 2 * G) * D
        rotation = {"none": abi.ROTATE_NONE, "half": abi.ROTATE_HALF, "interleaved": abi.ROTATE_INTERLEAVED}
        commands.append(session.command(
            abi.OP_KV_APPEND_I8, cache=cache, Q=s.q.data_ptr(), Q_out=s.out.data_ptr(), K=s.k.data_ptr(), V=s.v.data_ptr(),
            past=s.past.data_ptr(), seq_start=start, batch=B, tokens=T, heads=H, rotation=rotation[c["rotation"]],
            theta_base=THETA, **strides("q", _strides(layout, s.n[0], H, D, row)),
            **strides("o", _strides(layout, s.n[0], H, D)), **strides("k", _strides(layout, s.n[0], G, D, row)),
            **strides("v", _strides(layout, s.n[0], G, D, row))))
    if c["kind"] == "attention":
        at = _strides(layout, s.n[0], H, D)
        commands.append(session.command(
            abi.OP_KV_ATTENTION_I8, cache=cache, Q=s.q.data_ptr(), O=s.out.data_ptr(), kv_len=s.kv_len.data_ptr(),
            seq_start=start, batch=B, tokens=T, heads=H, max_tokens=max(s.n), max_kv=max(s.kv), causal=int(c["causal"]),
            **strides("q", at), **strides("o", at)))
    else:
        uniform = c["kind"] == "read" and not c["ragged"]
        at = _strides(layout if c["kind"] == "read" else "rows", s.read_n[0], G, D)
        commands.append(session.command(
            abi.OP_KV_READ_F32, cache=cache, K=s.k32.data_ptr(), V=s.v32.data_ptr(), first=s.first.data_ptr(),
            seq_start=None if uniform else s.read_start.data_ptr(), batch=B, tokens=sum(s.read_n),
            **strides("k", at), **strides("v", at)))
    s.commands = (abi.Command * len(commands))(*commands)


def _outputs(s):
    kind = s.case["kind"]
    if kind == "attention":
        return {"o": s.out}
    if kind == "read":
        return {"k": s.k32, "v": s.v32}
    return {"q": s.out, "k": s.k32, "v": s.v32, "k_scales": s.ks, "v_scales": s.vs}


def run(state):
    s = state
    if own:
        session = _session()
        session.check("vnpu_stream_submit",
                      session.lib.vnpu_stream_submit(session.stream, s.commands, len(s.commands), None))
        return _outputs(s)
    if s.case["kind"] == "append":
        s.out.copy_(_plain_append(s))
    if s.case["kind"] == "attention":
        s.out.copy_(_plain_attention(s))
    else:
        k, v = _plain_read(s)
        s.k32.copy_(k)
        s.v32.copy_(v)
    return _outputs(s)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _token_index(start, first, total):
    """Of packed token rows: the sequence and the position in it."""
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(start[1:].long(), t, right=True)
    return seq, first.long()[seq] + t - start.long()[seq]


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


def _rotate(x, position, rotation):
    """x [tokens][heads][head_dim]: angles and products in 64 bits, cosines, sines and results in 32."""
    if rotation == "none":
        return x
    d = x.shape[2]
    rate = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = position.double()[:, None] * rate
    cos, sin = angle.cos().float().double()[:, None, :], angle.sin().float().double()[:, None, :]
    if rotation == "half":
        a, b = x[..., :d // 2].double(), x[..., d // 2:].double()
        return torch.cat(((a * cos - b * sin).float(), (a * sin + b * cos).float()), dim=-1)
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack(((a * cos - b * sin).float(), (a * sin + b * cos).float()), dim=-1).reshape(x.shape)


def _round(x):
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.5), x))


def _append_side(codes, scales, x, page, slot, kept, page_axis):
    """Appends x [tokens][kv_heads][head_dim] at (page, slot); kept [pages]: slots of a page that hold older tokens."""
    touched = torch.zeros(codes.shape[0], dtype=torch.bool, device="cuda")
    touched[page] = True
    largest = torch.zeros_like(scales)
    largest.scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(dim=2), "amax")
    wanted = largest / 127.0
    wanted = torch.where(wanted < 2.0 ** -126, torch.zeros_like(wanted), wanted)
    scale = torch.where(kept[:, None] > 0, torch.maximum(scales, wanted), wanted)
    grown = touched[:, None] & (kept[:, None] > 0) & (scale > scales)
    ratio = torch.where(grown, scales / scale, torch.ones_like(scale))
    ids = page.unique()
    codes[ids] = _round(codes[ids].float() * ratio[ids][:, :, None, None]).to(torch.int8)
    scales[ids] = scale[ids]
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))[page][:, :, None]
    new = _round(x * inv).clamp(-127, 127).to(torch.int8)
    if page_axis == 2:
        codes[page, :, slot] = new
    else:
        codes[page, :, :, slot] = new


def _plain_append(s):
    c = s.case
    ps, D = c["page"], c["head_dim"]
    seq, position = _token_index(s.start, s.past, sum(s.n))
    page = s.table[seq, position // ps].long()
    kept = torch.zeros(s.k8.shape[0], dtype=torch.int64, device="cuda")
    head = s.table[torch.arange(c["batch"], device="cuda"), s.past.long() // ps].long()
    kept[head] = s.past.long() % ps
    k = _rotate(_by_token(s.k, c["kv_heads"], D), position, c["rotation"])
    _append_side(s.k8, s.ks, k, page, position % ps, kept, 2)
    _append_side(s.v8, s.vs, _by_token(s.v, c["kv_heads"], D), page, position % ps, kept, 3)
    return _from_tokens(_rotate(_by_token(s.q, c["heads"], D), position, c["rotation"]), s.out)


def _plain_read(s):
    ps = s.case["page"]
    seq, position = _token_index(s.read_start, s.first, sum(s.read_n))
    page, slot = s.table[seq, position // ps].long(), position % ps
    k = s.k8[page, :, slot].float() * s.ks[page][:, :, None]
    v = s.v8[page, :, :, slot].float() * s.vs[page][:, :, None]
    return _from_tokens(k, s.k32), _from_tokens(v, s.v32)


def _plain_attention(s):
    c = s.case
    B, H, G, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    n, T = max(s.n), sum(s.n)
    seq, i = _token_index(s.start, torch.zeros_like(s.past), T)
    q = torch.zeros(B, n, H, D, device="cuda")
    q[seq, i] = _by_token(s.q, H, D)
    q = q.reshape(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, D)
    pages = s.table.long()
    k = (s.k8[pages].float() * s.ks[pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D)
    v = (s.v8[pages].float() * s.vs[pages][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, G, -1, D)
    scores = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    key = torch.arange(k.shape[2], device="cuda")
    limit = s.kv_len.long()[:, None].expand(B, n)
    if c["causal"]:
        limit = s.past.long()[:, None] + torch.arange(n, device="cuda") + 1
    hidden = key >= torch.minimum(limit, s.kv_len.long()[:, None])[:, None, None, :, None]
    scores = scores.reshape(B, G, H // G, n, -1).masked_fill_(hidden, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(B, G, H // G * n, -1), v).reshape(B, G, H // G, n, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    return _from_tokens(o[seq, i], s.out)


# ---------------------------------------------------------------------------
# The values from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, _inputs(case, seed))


def _sequence(s, c, b, length):
    """The codes' values of the first `length` tokens of sequence b, [kv_heads][length][head_dim] each."""
    pages = s.table[b, :-(-length // c["page"])].long()
    k = (s.k8[pages].double() * s.ks[pages].double()[:, :, None, None]).transpose(0, 1)
    v = (s.v8[pages].double() * s.vs[pages].double()[:, :, None, None]).permute(1, 0, 3, 2)
    G, D = c["kv_heads"], c["head_dim"]
    return k.reshape(G, -1, D)[:, :length], v.reshape(G, -1, D)[:, :length]


def _exact_attention(c, s):
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    out, at = [], 0
    for b, (n, kv) in enumerate(zip(s.n, s.kv)):
        q = (s.q[b].transpose(0, 1) if s.q.dim() == 4 else s.q[at:at + n].reshape(n, H, D)).double()
        k, v = _sequence(s, c, b, kv)
        o = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
        see = torch.arange(kv, device="cuda")[None, :]
        for h in range(H):
            score = (q[:, h] @ k[h // (H // G)].T) / math.sqrt(D)
            if c["causal"]:
                score = score.masked_fill(see > kv - n + torch.arange(n, device="cuda")[:, None], -math.inf)
            o[:, h] = torch.softmax(score, dim=1) @ v[h // (H // G)]
        out.append(o.transpose(0, 1) if s.q.dim() == 4 else o.reshape(n, H * D))
        at += n
    return {"o": torch.stack(out) if s.q.dim() == 4 else torch.cat(out)}


def _exact_read(c, s):
    k, v = zip(*(_sequence(s, c, b, n) for b, n in enumerate(s.n)))
    if c["layout"] == "heads":
        return {"k": torch.stack(k), "v": torch.stack(v)}
    return {n: torch.cat([t.transpose(0, 1).reshape(t.shape[1], -1) for t in x]) for n, x in (("k", k), ("v", v))}


def _exact_turn(x, first, rotation):
    """x [tokens][heads][head_dim] of one sequence from position `first` on, turned as complex numbers."""
    x = x.double()
    if rotation == "none":
        return x
    t, h, d = x.shape
    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) if rotation == "half" else torch.view_as_complex(
        x.reshape(t, h, d // 2, 2).contiguous())
    angle = torch.outer(torch.arange(first, first + t, device="cuda").double(),
                        torch.exp(torch.arange(d // 2, device="cuda").double() * (-2.0 * math.log(THETA) / d)))
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    return torch.cat((z.real, z.imag), dim=-1) if rotation == "half" else torch.view_as_real(z).reshape(t, h, d)


def _turned_in_32(x, first, rotation):
    """The keys that are quantized: with the cosines and sines of the format's own 32 bits."""
    if rotation == "none":
        return x.float()
    d = x.shape[2]
    at = (slice(0, d // 2), slice(d // 2, d)) if rotation == "half" else (slice(0, d, 2), slice(1, d, 2))
    angle = torch.outer(torch.arange(first, first + x.shape[0], device="cuda").double(),
                        THETA ** (-torch.arange(0, d, 2, device="cuda").double() / d))
    cos, sin = (f(angle).float().double()[:, None] for f in (torch.cos, torch.sin))
    y, a, b = torch.empty_like(x, dtype=torch.float32), x[..., at[0]].double(), x[..., at[1]].double()
    y[..., at[0]], y[..., at[1]] = (a * cos - b * sin).float(), (a * sin + b * cos).float()
    return y


def _exact_append(c, s):
    """Codes are whole numbers of the format's own 32-bit scales: the same steps, page by page."""
    G, H, D, ps = c["kv_heads"], c["heads"], c["head_dim"], c["page"]
    ks, vs, out, at = s.ks.double(), s.vs.double(), {"q": [], "k": [], "v": []}, 0

    def half_away(t):
        return torch.sign(t) * torch.floor(t.abs() + 0.5)

    def side(x, old, scales, past):
        """x [new][kv_heads][head_dim], old: values' codes [kv_heads][ps][head_dim] of the first page."""
        got, i = [], 0
        for first in range(past // ps * ps, past + x.shape[0], ps):
            kept, end = max(0, past - first), min(x.shape[0], first + ps - past)
            page = pages[first // ps]
            new = x[i:end]
            scale = (new.abs().amax(dim=(0, 2)) / 127.0).double()
            if kept:
                before = scales[page].clone()
                scale = torch.maximum(scale, before)
                ratio = (before / scale).float()
                codes = half_away((old[:, :kept].float() * ratio[:, None, None]).double())
                got.append((codes * scale[:, None, None]).transpose(0, 1))
            inv = (1.0 / scale).float()
            got.append(half_away((new * inv[None, :, None]).double()).clamp(-127, 127) * scale[None, :, None])
            scales[page] = scale
            i = end
        return torch.cat(got).reshape(-1, G * D)

    for b, (n, kv) in enumerate(zip(s.n, s.kv)):
        past, pages = kv - n, s.table[b].tolist()
        q, k, v = ((t[b].transpose(0, 1) if t.dim() == 4 else t[at:at + n].reshape(n, -1, D)) for t in (s.q, s.k, s.v))
        q = _exact_turn(q, past, c["rotation"])
        out["q"].append(q.transpose(0, 1) if s.q.dim() == 4 else q.reshape(n, H * D))
        out["k"].append(side(_turned_in_32(k, past, c["rotation"]), s.k8[pages[past // ps]], ks, past))
        out["v"].append(side(v, s.v8[pages[past // ps]].transpose(1, 2), vs, past))
        at += n
    return {"q": torch.stack(out["q"]) if s.q.dim() == 4 else torch.cat(out["q"]), "k": torch.cat(out["k"]),
            "v": torch.cat(out["v"]), "k_scales": ks, "v_scales": vs}
