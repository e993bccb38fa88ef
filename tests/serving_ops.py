"""MATMUL_I4, ROPE_AXES_F32 and KV_PREFIX_ATTENTION_I8 in 64 bits for the tests, and what they start from."""
from __future__ import annotations

import numpy as np
from scipy.special import erfc

import kv_ops as kv
from vnpu_mi355x import abi

EPS = 2.0**-24   # half a step of f32


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

class Weights:
    """Codes, scales and zeros of K x N weights and their values in 64 bits."""

    def __init__(self, rng, K, N, group, zeros=True, trans=False, pad=0):
        self.K, self.N, self.group, self.trans = K, N, group, trans
        self.size = group or K
        self.groups = -(-K // self.size)
        self.codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
        self.scales = (0.01 + 0.02 * rng.random((self.groups, N))).astype(np.float32)
        self.scales *= np.where(rng.random((self.groups, N)) < 0.1, -1, 1).astype(np.float32)
        self.zeros = rng.integers(0, 16, (self.groups, N)).astype(np.uint8) if zeros else None
        rows, cols = (N, K) if trans else (K, N)
        self.ldb = -(-cols // 2) + pad
        self.bytes = rng.integers(0, 256, (rows, self.ldb)).astype(np.uint8)   # what pads a row is anything
        c = self.codes.T if trans else self.codes
        self.bytes[:, :cols // 2] = c[:, 0:cols // 2 * 2:2] | c[:, 1::2] << 4
        if cols % 2:
            self.bytes[:, cols // 2] = c[:, -1] | (self.bytes[:, cols // 2] & 0xf0)

    def differences(self):
        at = np.arange(self.K) // self.size
        return self.codes - (8.0 if self.zeros is None else self.zeros[at].astype(np.float64))

    def values(self):
        return self.differences() * self.scales[np.arange(self.K) // self.size].astype(np.float64)

    def pack(self, s):
        return s.pack_i4(self.bytes, self.scales, self.K, self.N, self.group, zeros=self.zeros, ldb=self.ldb,
                         trans_b=int(self.trans))


def finished(x, epilogue):
    if epilogue == abi.EPI_RELU:
        return np.maximum(x, 0)
    if epilogue == abi.EPI_SILU:
        return x / (1 + np.exp(-x))
    if epilogue == abi.EPI_GELU_TANH:
        return x / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x**3)))
    if epilogue == abi.EPI_GELU_ERF:
        return 0.5 * x * erfc(-x / np.sqrt(2))
    return x


def matmul(a, w: Weights, bias=None, epilogue=0):
    """(C, bound) in 64 bits.

    The bound, from the kernels' arithmetic.  An element of A enters to 2^-23 of itself (two f16) and 2^-39 of the largest of
    its row, or to 2^-30 of the largest of its row among the same 128 (whole numbers of 29 bits at least); differences of
    codes are exact.  A group's sum goes to f32 with an error of 2^-27 of that largest (the lower two of four digit
    sums, below 2^26, are converted by themselves), is multiplied by its scale (2 roundings) and added; sums in f32 round
    at most once for 16 products, once a group, once for each of up to 16 waves and 64 ranges of K, and the bias.  An epilogue's
    slope is at most 1.13, and its own 16 roundings are of its argument and of its result.  Below 2^-126 a step of f32 is
    2^-149 whatever the value, so each of those roundings of sums is off by up to 2^-150 there."""
    a64, values = a.astype(np.float64), w.values()
    want = a64 @ values
    size = np.abs(a64) @ np.abs(values)
    largest = np.zeros_like(a64)
    for k in range(0, w.K, 128):
        largest[:, k:k + 128] = np.abs(a64[:, k:k + 128]).max(axis=1, keepdims=True)
    roundings = w.K / 16 + w.groups + 90
    bound = (2.0**-23 + roundings * EPS) * size + roundings * 2.0**-150 + 2.0**-30 * (largest @ np.abs(values))
    bound += 2.0**-39 * np.abs(a64).max(axis=1, keepdims=True) * np.abs(values).sum(axis=0)
    step = min(w.size, 128)
    for k in range(0, w.K, step):
        bound += 2.0**-27 * largest[:, k:k + 1] * np.abs(w.scales[k // w.size])
    if bias is not None:
        want = want + bias.astype(np.float64)
        bound += EPS * np.abs(want)
    if epilogue:
        x = want
        want = finished(x, epilogue)
        bound = 1.13 * (bound + 16 * EPS * np.abs(x)) + 16 * EPS * np.abs(want)
    return want, bound


# ---------------------------------------------------------------------------
# Positions with several axes
# ---------------------------------------------------------------------------

def pairs_of(sections, order):
    """(axis, place in the axis) of each pair."""
    if order == abi.AXES_BLOCKS:
        return [(a, i) for a, n in enumerate(sections) for i in range(n)]
    return [(a, i) for i in range(max(sections)) for a, n in enumerate(sections) if i < n]


def rope_axes(x, positions, sections, order=0, ladders=0, rotation=abi.ROTATE_HALF, theta=10000.0, scaling=1.0):
    """(turned, bound) of x [tokens][heads][head_dim], positions [axes][tokens].

    The bound: an angle is off by 4 roundings of 64 bits of its size, the series by 2e-14, the result is rounded to f32."""
    pairs = pairs_of(sections, order)
    P = len(pairs)
    power = np.array([i / sections[a] if ladders == abi.AXES_OWN_LADDERS else j / P for j, (a, i) in enumerate(pairs)])
    angle = positions[[a for a, _ in pairs]].T.astype(np.float64) * (scaling * np.float64(theta) ** -power)
    at = (slice(0, P), slice(P, 2 * P)) if rotation == abi.ROTATE_HALF else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y, bound = x.astype(np.float64), np.zeros(x.shape)
    a, b = x[..., at[0]].astype(np.float64), x[..., at[1]].astype(np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, a * sin + b * cos
    off = (np.abs(angle)[:, None] * 2.0**-51 + 5e-14) * (np.abs(a) + np.abs(b))
    for side in at:
        bound[..., side] = off + EPS * (1 + 2.0**-20) * np.abs(y[..., side]) + 2.0**-150
    return y, bound


# ---------------------------------------------------------------------------
# A shared prefix
# ---------------------------------------------------------------------------

def shared_cache(rng, batch, kv_heads, d, page, prefix, most, spare=2):
    """A kv.Cache whose sequences all begin with the pages of sequence 0's first `prefix` tokens; prefix_table."""
    c = kv.Cache(rng, batch, kv_heads, d, page, (prefix + most) // page + 2, spare)
    first = c.table[0, :prefix // page].copy()
    c.table[:, :prefix // page] = first
    return c, first


def prefix_attention(c, q, kv_len, n, causal, scale=0.0):
    """kv.attention with the join of the two parts: each is divided by its sum, weighed (an exponential to 2 roundings, a
    product) and divided again: 16 roundings of the largest value more."""
    want, bound = kv.attention(c, q, kv_len, n, causal, scale)
    most = max(float(np.abs(c.values(b, int(kv_len[b]))[1]).max(initial=0.0)) for b in range(len(n)) if n[b]) if any(n) else 0.0
    return want, bound + 16 * EPS * most
