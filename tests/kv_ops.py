"""The paged int8 KV cache for the tests: its commands on a Session with numpy in and out, and the operators in 64 bits.

The format's own roundings (the turned key in f32, the scale, the reciprocal and the ratio of two scales in f32, codes
half away from zero) are part of the operators' definition, so the 64-bit forms make them too."""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

from vnpu_mi355x import abi


@dataclass
class Cache:
    """Codes, scales and table of a cache; pages in a random order, every slot filled with something."""
    rng: np.random.Generator
    batch: int
    kv_heads: int
    head_dim: int
    page: int
    table_ld: int
    spare: int = 2
    k: np.ndarray = field(init=False)
    v: np.ndarray = field(init=False)
    ks: np.ndarray = field(init=False)
    vs: np.ndarray = field(init=False)
    table: np.ndarray = field(init=False)

    def __post_init__(self):
        r, g, d, ps = self.rng, self.kv_heads, self.head_dim, self.page
        self.pages = self.batch * self.table_ld + self.spare
        self.k = r.integers(-127, 128, (self.pages, g, ps, d)).astype(np.int8)
        self.v = r.integers(-127, 128, (self.pages, g, d, ps)).astype(np.int8)
        self.ks = (0.01 + 0.02 * r.random((self.pages, g))).astype(np.float32)
        self.vs = (0.01 + 0.02 * r.random((self.pages, g))).astype(np.float32)
        self.table = r.permutation(self.pages)[:self.batch * self.table_ld].astype(np.int32)
        self.table = self.table.reshape(self.batch, self.table_ld)

    def forget(self, lengths):
        """What lies behind each sequence's length: pages that do not exist, scales that are NaN."""
        used = np.zeros(self.pages, bool)
        for b, n in enumerate(lengths):
            own = -(-int(n) // self.page)
            used[self.table[b, :own]] = True
            self.table[b, own:] = np.array([-1, 2**31 - 1, -2**31])[np.arange(self.table_ld - own) % 3]
        self.ks[~used] = np.nan
        self.vs[~used] = np.nan
        return self

    def values(self, b, n):
        """Sequence b's first n tokens in 64 bits, [kv_heads][n][head_dim] each."""
        ids = self.table[b, :-(-n // self.page)]
        k = self.k[ids].astype(np.float64) * self.ks[ids].astype(np.float64)[:, :, None, None]
        v = self.v[ids].astype(np.float64) * self.vs[ids].astype(np.float64)[:, :, None, None]
        k = k.transpose(1, 0, 2, 3).reshape(self.kv_heads, -1, self.head_dim)
        v = v.transpose(1, 0, 3, 2).reshape(self.kv_heads, -1, self.head_dim)
        return k[:, :n], v[:, :n]


def half_away(x):
    return np.sign(x) * np.floor(np.abs(x) + 0.5)


def turned(x, position, rotation, rope_dim, theta=10000.0, scaling=1.0):
    """x [tokens][heads][head_dim] turned: cosines and sines in f32, results rounded to f32."""
    if not rotation:
        return x.astype(np.float32)
    r = rope_dim or x.shape[2]
    y = x.astype(np.float32).copy()
    angle = np.outer(np.asarray(position, np.float64) * scaling, np.float64(theta) ** (-2.0 * np.arange(r // 2) / r))
    cos, sin = (f(angle).astype(np.float32).astype(np.float64)[:, None, :] for f in (np.cos, np.sin))
    at = (slice(0, r // 2), slice(r // 2, r)) if rotation == abi.ROTATE_HALF else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., at[0]].astype(np.float64), x[..., at[1]].astype(np.float64)
    y[..., at[0]], y[..., at[1]] = (a * cos - b * sin).astype(np.float32), (a * sin + b * cos).astype(np.float32)
    return y


def append_side(codes, scales, x, ids, past):
    """Appends x [tokens][kv_heads][head_dim] (f32) to one sequence; codes [pages][kv_heads][page][head_dim]."""
    ps = codes.shape[2]
    for first in range(past // ps * ps, past + x.shape[0], ps):
        lo, hi = max(past, first), min(past + x.shape[0], first + ps)
        page = ids[first // ps]
        for h in range(x.shape[1]):
            new = x[lo - past:hi - past, h]
            before = scales[page, h] if lo > first else None
            s = np.float32(np.abs(new).max()) * (np.float32(1) / np.float32(127))
            s = np.float32(0) if s < np.float32(2.0**-126) else s
            if not np.all(np.isfinite(new)) or (before is not None and np.isnan(before)):
                s = np.float32(np.nan)
            elif before is not None:
                s = max(s, before)
                if s > before:
                    old = codes[page, h, :lo - first].astype(np.float32) * (before / s)
                    codes[page, h, :lo - first] = half_away(old.astype(np.float64))
            scales[page, h] = s
            if s > 0:
                new = (new * (np.float32(1) / s)).astype(np.float64)
                codes[page, h, lo - first:hi - first] = np.clip(half_away(new), -127, 127)
            elif s == 0:
                codes[page, h, lo - first:hi - first] = 0


def append(c: Cache, k, v, past, n, rotation, rope_dim=0, theta=10000.0, scaling=1.0):
    """k, v [tokens][kv_heads][head_dim], the sequences' rows one after another; changes c."""
    at = 0
    for b, m in enumerate(n):
        if m:
            rows = turned(k[at:at + m], past[b] + np.arange(m), rotation, rope_dim, theta, scaling)
            append_side(c.k, c.ks, rows, c.table[b], past[b])
            vt = np.ascontiguousarray(c.v.transpose(0, 1, 3, 2))
            append_side(vt, c.vs, v[at:at + m].astype(np.float32), c.table[b], past[b])
            c.v[:] = vt.transpose(0, 1, 3, 2)
        at += m


def attention(c: Cache, q, kv_len, n, causal, scale=0.0):
    """(o, bound) [tokens][heads][head_dim] in 64 bits.

    The bound, from the kernels' arithmetic (eps = 2^-24, half a step of f32): a query enters its products as a whole
    number of up to 2^23 - 2^15 steps of its largest element, half a step off and one f32 rounding of as much again, so a score
    (a sum exact in whole numbers) is off by scale * max_j sum_d |k_jd| * max|q| * 2^-22 / 2 * 2 and then by 8 roundings
    of its size; a weight is off by twice that (its own and the maximum's) and 4 roundings, weights enter the product
    with V with 2^-22 of the largest, and sums over keys by tiles of 16 or more round once for each."""
    D, G, H = c.head_dim, c.kv_heads, q.shape[1]
    scale = scale if scale > 0 else float(np.float32(1.0) / np.sqrt(np.float32(D)))
    out, bound, at, eps = np.zeros(q.shape), np.zeros(q.shape[:2]), 0, 2.0**-24
    for b, m in enumerate(n):
        k, v = c.values(b, int(kv_len[b]))
        for h in range(H):
            kh = h // (H // G)
            s = q[at:at + m, h].astype(np.float64) @ k[kh].T * scale
            if causal:
                see = int(kv_len[b]) - m + np.arange(m)[:, None]
                s = np.where(np.arange(int(kv_len[b]))[None, :] <= see, s, -np.inf)
            some = np.isfinite(s).any(axis=1) if s.shape[1] else np.zeros(m, bool)
            if not some.any():
                continue
            t = s[some]
            p = np.exp(t - t.max(axis=1, keepdims=True))
            out[at:at + m, h][some] = (p / p.sum(axis=1, keepdims=True)) @ v[kh]
            off = scale * np.abs(k[kh]).sum(axis=1).max() * np.abs(q[at:at + m, h][some]).max(axis=1) * 2.0**-22
            off += 8 * eps * np.abs(np.where(np.isfinite(t), t, 0)).max(axis=1)
            tiles = -(-k.shape[1] // 16)
            bound[at:at + m, h][some] = np.abs(v[kh]).max() * (2 * off + 8 * eps + 2.0**-21 + 2 * tiles * eps)
        at += m
    return out, bound[..., None]


# ---------------------------------------------------------------------------
# The commands
# ---------------------------------------------------------------------------

def upload(s, c: Cache):
    """(cache struct, buffers by name)"""
    bufs = {n: s.upload(getattr(c, n)) for n in ("k", "v", "ks", "vs", "table")}
    return abi.KvCache(k=bufs["k"].ptr, v=bufs["v"].ptr, k_scales=bufs["ks"].ptr, v_scales=bufs["vs"].ptr,
                       table=bufs["table"].ptr, pages=c.pages, page_size=c.page, kv_heads=c.kv_heads,
                       head_dim=c.head_dim, table_ld=c.table_ld), bufs


def download(s, c: Cache, bufs):
    return {n: s.download(bufs[n], getattr(c, n).dtype, getattr(c, n).shape) for n in ("k", "v", "ks", "vs")}


def free(s, *bufs):
    for b in bufs:
        for x in (b.values() if isinstance(b, dict) else (b,)):
            if x is not None:
                s.free(x)


def starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def strides(prefix, values):
    return dict(zip((f"{prefix}_batch_stride", f"{prefix}_token_stride", f"{prefix}_head_stride"), values))


class Rows:
    """[tokens][heads][head_dim] as the memory of a strided tensor, and back.

    layout: "rows" packed; "wide" packed rows with `gap` floats behind each and `shift` before the first; "heads"
    [batch][heads][n][head_dim] (all n alike)."""

    def __init__(self, x, layout="rows", batch=1, gap=0, shift=0, fill=np.nan):
        t, h, d = x.shape
        self.shape, self.layout, self.batch = x.shape, layout, batch
        if layout == "heads":
            n = t // batch
            self.strides, self.offset = (h * n * d, d, n * d), 0
            self.memory = np.ascontiguousarray(x.reshape(batch, n, h, d).transpose(0, 2, 1, 3)).reshape(-1)
        else:
            gap = gap if layout == "wide" else 0
            self.offset = shift if layout == "wide" else 0
            self.strides = (0, h * d + gap, d)
            self.memory = np.full(self.offset + t * (h * d + gap), fill, np.float32)
            self.memory[self.offset:].reshape(t, -1)[:, :h * d] = x.reshape(t, h * d)
        self.memory = np.ascontiguousarray(self.memory, np.float32)

    def upload(self, s):
        self.buffer = s.upload(self.memory)
        return self.buffer.ptr + 4 * self.offset

    def download(self, s):
        m = s.download(self.buffer, np.float32, self.memory.shape)
        t, h, d = self.shape
        if self.layout == "heads":
            return m.reshape(self.batch, h, t // self.batch, d).transpose(0, 2, 1, 3).reshape(self.shape)
        body = m[self.offset:].reshape(t, -1)
        self.rest = np.concatenate([m[:self.offset], body[:, h * d:].reshape(-1)])
        return body[:, :h * d].reshape(self.shape)
