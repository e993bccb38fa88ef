// kv_cache.hip - KV_APPEND_I8 and KV_READ_F32: what writes the paged int8 KV
// cache and what reads it back, on gfx950.
//
// Append, for new token i of sequence b at position p = past[b] + i:
//   angle_j = p * scaling * theta^(-2j / R), j < R / 2 (R = rope_dim)
//   (x, y) -> (f32(x cos - y sin), f32(x sin + y cos)), cos and sin in f32,
//   the products exact in f64, so each result is rounded once;
//   per (page, kv head): a = max |x| of the page's new tokens,
//   s = max(n0 ? s0 : 0, f32(a * f32(1 / 127))) for n0 tokens kept from before,
//   kept codes -> round(code * f32(s0 / s)) where s > s0,
//   new codes = round(x * f32(1 / s)), half away from zero, in +-127.
// One page and kv head of K or V is one workgroup: it alone reads and writes
// those codes and their scale, so nothing is atomic and results do not depend on
// order.  The new tokens' f32 values are read once and stay in registers between
// the largest magnitude and the codes.  Q's rows are workgroups of their own behind
// them: the three used to be one, 62 us for 2048 tokens of 32 and 8 heads of
// 128, now 24 us, 4.2 TB/s of rows in and out and codes (a large copy: 4.9 TB/s).
// A token each for 8 sequences takes 4.4 us, a launch and its latency.
//
// Read: one page and kv head of K or V is one workgroup; f32 rows, four times the
// codes, bound it: 8 x 2048 tokens of 8 heads of 128 in 27.7 us, 6.1 TB/s.
#include "device_math.hpp"
#include "kv_common.hpp"

#include <cmath>
#include <map>
#include <mutex>
#include <tuple>

namespace vnpu {
namespace k {
namespace {

// Turns (angle / 2 pi) per position of each pair, computed on the host.
struct Rates {
    double turns[128];
};

// cos and sin of 2 pi t in f32.  Their error grows with the position: of the f32
// results 1 in 10^5 is not the correctly rounded one up to position 10000, 1 in 14000 at
// 100000, 1 in 2000 at 10^6 (theta 10000, 64 and 128 dimensions), all within half a step
// and 2^-10 of one to there.
__device__ __forceinline__ void cos_sin_turns(double t, float &c, float &s)
{
    double cd, sd;
    dev::cos_sin_turns(t, cd, sd);
    c = static_cast<float>(cd);
    s = static_cast<float>(sd);
}

__device__ __forceinline__ float2 turned(float2 x, float c, float s)
{
    const double a = x.x, b = x.y, cd = c, sd = s;
    return make_float2(static_cast<float>(fma(a, cd, -(b * sd))), static_cast<float>(fma(a, sd, b * cd)));
}

// Round half away from zero into +-127.  The product is rounded by itself:
// fused into the rounding's subtraction it would decide ties from more bits.
__device__ __forceinline__ int code_of(float x, float by)
{
    return static_cast<int>(fminf(fmaxf(roundf(dev::mul_rn(x, by)), -127.0f), 127.0f));
}
__device__ __forceinline__ uint32_t rescaled4(uint32_t codes, float ratio)
{
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= (static_cast<uint32_t>(code_of(static_cast<float>(static_cast<int8_t>(codes >> (8 * i))), ratio)) & 255u) << (8 * i);
    return r;
}

// Largest bits of |x| over the workgroup: orders magnitudes, infinity and NaN.
template <int T>
__device__ __forceinline__ uint32_t block_largest(uint32_t v, uint32_t *red)
{
    for (int o = 32; o; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t r = red[0];
    for (int w = 1; w < T / 64; ++w) r = max(r, red[w]);
    return r;
}

// A product with f32(1 / 127), not a division: that is what a division by a constant
// becomes in torch on a GPU, so that a program there makes the same codes from the same
// values.  It is within a step of largest / 127, which QUANTIZE_I8 takes: its scale of the same values
// may differ in the last bit.
struct PageScale {
    float scale, ratio, inv;
};
__device__ __forceinline__ PageScale page_scale(uint32_t largest, bool kept, float before)
{
    float s = dev::mul_rn(__uint_as_float(largest), 1.0f / 127.0f);
    if (s < 1.17549435e-38f) s = 0.0f;   // no reciprocal in f32
    if (largest >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
    PageScale r;
    r.scale = !kept ? s : before != before || s != s ? __uint_as_float(0x7fc00000u) : fmaxf(before, s);
    r.ratio = kept && r.scale > before ? __fdiv_rn(before, r.scale) : 1.0f;
    r.inv = r.scale > 0.0f ? __fdiv_rn(1.0f, r.scale) : 0.0f;
    return r;
}

// Elements of pair j of a row, in the first half of the turned ones or beside each other.
__device__ __forceinline__ uint2 pair_at(const KvAppend &p, uint32_t j)
{
    const uint32_t turns = p.rope_dim / 2;
    return p.rotation == 1 && j < turns ? make_uint2(j, j + turns) : make_uint2(2 * j, 2 * j + 1);
}

// Workgroups of a call: 2 units * kv_heads that append (even: K, odd: V of a
// page and head), then those that turn Q, which are cut as their number asks.
struct AppendGrid {
    uint32_t units, q_splits, half_magic;
};

// One page and head of K or V.  Thread e of m * D / 2 pairs has pair e % (D /
// 2) of token e / (D / 2); PAIRS of a thread, and where that may not be enough
// (ROUNDS: the host does not know how many tokens a ragged sequence has) rounds of
// as many, of which all but the last are read again for their codes (64 sequences of
// 1 to 6 tokens, pages of 256: 10 us instead of 41 with room for whole pages;
// 2048 tokens of one sequence: 24 us without rounds, 26 with).  Codes go through LDS
// (dynamic, page_size * D bytes) so that the cache is written 16 bytes at a time.
template <int T, int PAIRS, bool ROUNDS, bool V>
__device__ __forceinline__ void append_page(const KvAppend &p, const Rates &rates, uint32_t magic, uint32_t b, const kv::Piece &pc,
                                            uint32_t h, int8_t *tile, uint32_t *red)
{
    const KvCall &c = p.call;
    const uint32_t tid = threadIdx.x, D = c.c.head_dim, half = D / 2, ps = c.c.page_size, pairs = pc.m * half;
    const uint64_t unit = static_cast<uint64_t>(pc.page) * c.c.kv_heads + h;
    const KvRows &rows = V ? p.v : p.k;
    const float *in = (V ? p.V : p.K) + kv::rows_base(c, rows, b, pc.seq) + pc.first * rows.token + h * rows.head;
    float *scales = V ? c.c.vs : c.c.ks;
    const float before = scales[unit];
    const uint64_t position = static_cast<uint64_t>(c.lengths[b]) + pc.first;
    const uint32_t turns = !V && p.rotation ? p.rope_dim / 2 : 0;

    float2 x[PAIRS];
    auto load = [&](uint32_t from) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const uint32_t e = from + tid + i * T;
            x[i] = make_float2(0.0f, 0.0f);
            if (e >= pairs) continue;
            const uint32_t t = __umulhi(e, magic), j = e - t * half;
            const uint2 d = V ? make_uint2(2 * j, 2 * j + 1) : pair_at(p, j);
            const float *row = in + t * rows.token;
            x[i] = make_float2(row[d.x], row[d.y]);
        }
        if (V) return;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const uint32_t e = from + tid + i * T, t = __umulhi(e, magic), j = e - t * half;
            if (e < pairs && j < turns) {
                float cs, sn;
                cos_sin_turns(static_cast<double>(position + t) * rates.turns[j], cs, sn);
                x[i] = turned(x[i], cs, sn);
            }
        }
    };
    uint32_t most = 0, from = 0;
    for (;; from += PAIRS * T) {
        load(from);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
            most = max(most, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu));
        if (!ROUNDS || from + PAIRS * T >= pairs) break;
    }
    const PageScale s = page_scale(block_largest<T>(most, red), pc.slot > 0, before);
    if (tid == 0) scales[unit] = s.scale;
    if (s.scale != s.scale) return;   // under a NaN scale the codes stay

    for (;;) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const uint32_t e = from + tid + i * T;
            if (e >= pairs) continue;
            const uint32_t t = __umulhi(e, magic), j = e - t * half;
            const int8_t c0 = static_cast<int8_t>(code_of(x[i].x, s.inv)), c1 = static_cast<int8_t>(code_of(x[i].y, s.inv));
            if (V) {
                tile[2 * j * ps + pc.slot + t] = c0;
                tile[(2 * j + 1) * ps + pc.slot + t] = c1;
            } else {
                const uint2 d = pair_at(p, j);
                tile[t * D + d.x] = c0;
                tile[t * D + d.y] = c1;
            }
        }
        if (!ROUNDS || !from) break;
        from -= PAIRS * T;
        load(from);
    }
    __syncthreads();
    const uint4 *tp = reinterpret_cast<const uint4 *>(tile);
    uint4 *to = reinterpret_cast<uint4 *>((V ? c.c.v : c.c.k) + unit * ps * D);
    if (!V) {   // [slot][D]: the new tokens' bytes are one run
        const uint32_t row16 = D / 16;
        for (uint32_t e = tid; e < pc.m * row16; e += T) to[pc.slot * row16 + e] = tp[e];
        if (s.ratio != 1.0f)
            for (uint32_t e = tid; e < pc.slot * row16; e += T) {
                const uint4 o = to[e];
                to[e] = make_uint4(rescaled4(o.x, s.ratio), rescaled4(o.y, s.ratio), rescaled4(o.z, s.ratio), rescaled4(o.w, s.ratio));
            }
        return;
    }
    // [D][slot]: rows of page_size bytes of which the new tokens are a part.
    const uint32_t log16 = c.c.log_page - 4, end = pc.slot + pc.m;
    const uint32_t from16 = s.ratio != 1.0f ? 0 : pc.slot / 16, n16 = (end + 15) / 16 - from16;
    for (uint32_t e = tid; e < D * n16; e += T) {
        const uint32_t d = e / n16, s16 = from16 + e % n16, s0 = 16 * s16, at = (d << log16) + s16;
        const uint4 fresh = tp[at];
        if (s0 >= pc.slot && s0 + 16 <= end) {
            to[at] = fresh;
            continue;
        }
        const uint4 old = to[at];
        const uint32_t o4[4] = {old.x, old.y, old.z, old.w}, f4[4] = {fresh.x, fresh.y, fresh.z, fresh.w};
        uint32_t r4[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t moved = s.ratio != 1.0f ? rescaled4(o4[w], s.ratio) : o4[w];
            r4[w] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t slot = s0 + 4 * w + i, m = 255u << (8 * i);
                r4[w] |= (slot < pc.slot ? moved : slot < end ? f4[w] : o4[w]) & m;
            }
        }
        to[at] = make_uint4(r4[0], r4[1], r4[2], r4[3]);
    }
}

// Queries: a thread has one pair of a token and turns it in some of the heads.
template <int T>
__device__ __forceinline__ void turn_queries(const KvAppend &p, const Rates &rates, uint32_t magic, uint32_t block, uint32_t splits)
{
    const KvCall &c = p.call;
    const uint32_t half = c.c.head_dim / 2, per = (p.heads + splits - 1) / splits;
    const uint64_t e = static_cast<uint64_t>(block / splits) * T + threadIdx.x;
    uint32_t row, j;
    if (e < 65536) {
        row = __umulhi(static_cast<uint32_t>(e), magic);
        j = static_cast<uint32_t>(e) - row * half;
    } else {
        row = static_cast<uint32_t>(e / half);
        j = static_cast<uint32_t>(e % half);
    }
    if (row >= c.tokens) return;
    uint32_t b;
    if (!c.seq_start) {
        b = row / (c.tokens / c.batch);
    } else {   // the last sequence that begins here or before
        uint32_t lo = 0, hi = c.batch;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (static_cast<uint32_t>(c.seq_start[mid]) <= row) lo = mid + 1;
            else hi = mid;
        }
        if (!lo) return;
        b = lo - 1;
    }
    const kv::Seq seq = kv::sequence(c, b);
    const int64_t past = c.lengths[b];
    const uint32_t i = row - seq.row;
    if (!seq.ok || i >= seq.n || past < 0 || past + seq.n > static_cast<int64_t>(kv::capacity(c))) return;   // check_all told
    const uint2 d = pair_at(p, j);
    float cs = 1.0f, sn = 0.0f;
    const bool turn = p.rotation && j < p.rope_dim / 2;
    if (turn) cos_sin_turns(static_cast<double>(past + i) * rates.turns[j], cs, sn);
    const uint32_t h0 = block % splits * per, h1 = min(p.heads, h0 + per);
    const float *in = p.Q + kv::rows_base(c, p.q, b, seq) + i * p.q.token;
    float *out = p.Q_out + kv::rows_base(c, p.o, b, seq) + i * p.o.token;
    for (uint32_t h = h0; h < h1; h += 8) {
        float2 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (h + k < h1) x[k] = make_float2(in[(h + k) * p.q.head + d.x], in[(h + k) * p.q.head + d.y]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (h + k >= h1) continue;
            if (turn) x[k] = turned(x[k], cs, sn);
            out[(h + k) * p.o.head + d.x] = x[k].x;
            out[(h + k) * p.o.head + d.y] = x[k].y;
        }
    }
}

template <int T, int PAIRS, bool ROUNDS>
__global__ __launch_bounds__(T) void kv_append_kernel(KvAppend p, Rates rates, AppendGrid grid)
{
    extern __shared__ __align__(16) int8_t tile[];
    __shared__ uint32_t red[T / 64];
    const KvCall &c = p.call;
    if (blockIdx.x == 0) kv::check_all(c, blockDim.x, true, kv::capacity(c), c.tokens);
    const uint32_t appends = 2 * grid.units * c.c.kv_heads;
    if (blockIdx.x >= appends) {
        turn_queries<T>(p, rates, grid.half_magic, blockIdx.x - appends, grid.q_splits);
        return;
    }
    const uint32_t rest = blockIdx.x / 2, h = rest % c.c.kv_heads;
    uint32_t b;
    kv::Piece pc;
    if (!kv::find_piece(c, rest / c.c.kv_heads, b, pc)) return;
    if (blockIdx.x & 1) append_page<T, PAIRS, ROUNDS, true>(p, rates, grid.half_magic, b, pc, h, tile, red);
    else append_page<T, PAIRS, ROUNDS, false>(p, rates, grid.half_magic, b, pc, h, tile, red);
}

constexpr int kReadThreads = 256;

// One page and head of K or V to f32 rows.  V's codes pass through LDS (dynamic,
// page_size rows of D + 4 bytes) to turn [D][slot] into rows.  VEC: rows that
// begin at 16 bytes.
using f32x4 = __attribute__((ext_vector_type(4))) float;

template <bool VEC>
__device__ __forceinline__ void store4(float *to, uint32_t w, float scale)
{
    float4 x;
    x.x = static_cast<float>(static_cast<int8_t>(w)) * scale;
    x.y = static_cast<float>(static_cast<int8_t>(w >> 8)) * scale;
    x.z = static_cast<float>(static_cast<int8_t>(w >> 16)) * scale;
    x.w = static_cast<float>(static_cast<int8_t>(w >> 24)) * scale;
    if (VEC) {
        // Past the caches: the rows are more than they hold where time counts.
        __builtin_nontemporal_store(f32x4{x.x, x.y, x.z, x.w}, reinterpret_cast<f32x4 *>(to));
    } else {
        to[0] = x.x;
        to[1] = x.y;
        to[2] = x.z;
        to[3] = x.w;
    }
}

template <bool VEC>
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(KvRead p, uint32_t magic)
{
    extern __shared__ __align__(16) int8_t tile[];
    const KvCall &c = p.call;
    const bool values = blockIdx.z || !p.K;
    const uint32_t h = blockIdx.y, tid = threadIdx.x;
    if (blockIdx.x == 0 && h == 0 && blockIdx.z == 0) kv::check_all(c, blockDim.x, true, kv::capacity(c), c.tokens);
    uint32_t b;
    kv::Piece pc;
    if (!kv::find_piece(c, blockIdx.x, b, pc)) return;
    const uint32_t D = c.c.head_dim, ps = c.c.page_size, quads = D / 4;
    const uint64_t unit = static_cast<uint64_t>(pc.page) * c.c.kv_heads + h;
    if (!values) {
        const float scale = c.c.ks[unit];
        const uint32_t *codes = reinterpret_cast<const uint32_t *>(c.c.k + (unit * ps + pc.slot) * D);
        float *out = p.K + kv::rows_base(c, p.k, b, pc.seq) + pc.first * p.k.token + h * p.k.head;
#pragma unroll 4
        for (uint32_t e = tid; e < pc.m * quads; e += kReadThreads) {
            const uint32_t t = __umulhi(e, magic);
            store4<VEC>(out + t * p.k.token + 4 * (e - t * quads), codes[e], scale);
        }
        return;
    }
    const float scale = c.c.vs[unit];
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(c.c.v + unit * ps * D);
    const uint32_t from4 = pc.slot / 4, n4 = (pc.slot + pc.m + 3) / 4 - from4, row = D + 4;
#pragma unroll 4
    for (uint32_t e = tid; e < D * n4; e += kReadThreads) {
        const uint32_t d = e / n4, s4 = from4 + e % n4, w = codes[d * (ps / 4) + s4];
#pragma unroll
        for (int i = 0; i < 4; ++i) tile[(4 * s4 + i) * row + d] = static_cast<int8_t>(w >> (8 * i));
    }
    __syncthreads();
    float *out = p.V + kv::rows_base(c, p.v, b, pc.seq) + pc.first * p.v.token + h * p.v.head;
#pragma unroll 4
    for (uint32_t e = tid; e < pc.m * quads; e += kReadThreads) {
        const uint32_t t = __umulhi(e, magic), d = 4 * (e - t * quads);
        store4<VEC>(out + t * p.v.token + d, *reinterpret_cast<const uint32_t *>(tile + (pc.slot + t) * row + d), scale);
    }
}

// Kept by value for a (theta, rope_dim, scaling): 128 powers are microseconds on the host.
Rates rates_of(float theta, uint32_t dim, float scaling)
{
    static std::mutex mutex;
    static auto *known = new std::map<std::tuple<float, uint32_t, float>, Rates>();
    std::lock_guard<std::mutex> lock(mutex);
    const auto key = std::make_tuple(theta, dim, scaling);
    auto it = known->find(key);
    if (it != known->end()) return it->second;
    Rates r{};
    for (uint32_t j = 0; j < dim / 2; ++j)
        r.turns[j] = static_cast<double>(scaling) * std::pow(static_cast<double>(theta), -2.0 * j / dim) / (2.0 * M_PI);
    if (known->size() >= 64) known->clear();
    known->emplace(key, r);
    return r;
}

// Pages of 256 tokens and heads of 256 take more LDS than a kernel has unasked.
template <typename Kernel>
void allow_lds(Kernel kernel, size_t bytes)
{
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(bytes));
}

// Pairs of a page's new tokens: at most (page_size * D / 2 = 32768 or less), and
// what to make room for: of ragged sequences what a page has if they have up to
// twice as many tokens as the mean, where all would be more than 4 of a thread.
uint32_t append_most(const KvCall &c)
{
    return std::min(c.seq_start ? c.tokens : c.tokens / c.batch, c.c.page_size) * (c.c.head_dim / 2);
}
uint32_t append_pairs(const KvCall &c)
{
    const uint32_t most = append_most(c);
    if (!c.seq_start || most <= 1024) return most;
    const uint64_t twice = 2ull * ((c.tokens + c.batch - 1) / c.batch) * (c.c.head_dim / 2);
    return static_cast<uint32_t>(std::min<uint64_t>(most, twice));
}
uint32_t append_threads(const KvCall &c) { return append_pairs(c) <= 4096 ? 256 : 1024; }

uint64_t append_blocks(const KvAppend &p, AppendGrid &g)
{
    const uint64_t T = append_threads(p.call);
    g.units = kv::unit_count(p.call);
    g.q_splits = 1;
    uint64_t blocks = 2ull * g.units * p.call.c.kv_heads;
    if (p.heads) {
        const uint64_t q = (static_cast<uint64_t>(p.call.tokens) * (p.call.c.head_dim / 2) + T - 1) / T;
        // Enough workgroups for two a CU, of one head each at least.
        g.q_splits = static_cast<uint32_t>(std::min<uint64_t>(p.heads, (511 + q) / q));
        blocks += q * g.q_splits;
    }
    return blocks;
}

template <int T, int PAIRS, bool ROUNDS>
void launch_append(hipStream_t s, const KvAppend &p, uint32_t blocks, const AppendGrid &grid)
{
    const size_t lds = static_cast<size_t>(p.call.c.page_size) * p.call.c.head_dim;
    allow_lds(kv_append_kernel<T, PAIRS, ROUNDS>, lds);
    const Rates rates = p.rotation ? rates_of(p.theta, p.rope_dim, p.scaling) : Rates{};
    kv_append_kernel<T, PAIRS, ROUNDS><<<blocks, T, lds, s>>>(p, rates, grid);
}
}  // namespace

// A grid's work-items count in 32 bits.
bool kv_append_fits(const KvAppend &p)
{
    AppendGrid g;
    return append_blocks(p, g) * append_threads(p.call) < (1ull << 32);
}
bool kv_read_fits(const KvRead &p) { return static_cast<uint64_t>(kv::unit_count(p.call)) * kReadThreads < (1ull << 32); }

void kv_append(hipStream_t s, const KvAppend &p)
{
    AppendGrid g;
    const uint32_t blocks = static_cast<uint32_t>(append_blocks(p, g)), half = p.call.c.head_dim / 2, most = append_pairs(p.call);
    g.half_magic = static_cast<uint32_t>((0x100000000ull + half - 1) / half);   // exact below 2^16
    const bool fit = append_most(p.call) <= (most <= 256 ? 256u : most <= 1024 ? 1024u : most <= 4096 ? 4096u : 16384u);
    if (most <= 256 && fit) launch_append<256, 1, false>(s, p, blocks, g);
    else if (most <= 1024 && fit) launch_append<256, 4, false>(s, p, blocks, g);
    else if (most <= 1024) launch_append<256, 4, true>(s, p, blocks, g);
    else if (most <= 4096 && fit) launch_append<256, 16, false>(s, p, blocks, g);
    else if (most <= 4096) launch_append<256, 16, true>(s, p, blocks, g);
    else if (fit) launch_append<1024, 16, false>(s, p, blocks, g);
    else launch_append<1024, 16, true>(s, p, blocks, g);
}

void kv_read(hipStream_t s, const KvRead &p)
{
    const KvCall &c = p.call;
    const size_t lds = p.V ? static_cast<size_t>(c.c.page_size) * (c.c.head_dim + 4) : 0;
    auto vectors = [](const float *at, const KvRows &r) {
        return !at || !((reinterpret_cast<uintptr_t>(at) & 15) | (r.batch & 3) | (r.token & 3) | (r.head & 3));
    };
    const auto kernel = vectors(p.K, p.k) && vectors(p.V, p.v) ? kv_read_kernel<true> : kv_read_kernel<false>;
    allow_lds(kernel, lds);
    const uint32_t quads = c.c.head_dim / 4;
    const uint32_t magic = static_cast<uint32_t>((0x100000000ull + quads - 1) / quads);   // exact below 2^16
    kernel<<<dim3(kv::unit_count(c), c.c.kv_heads, p.K && p.V ? 2 : 1), kReadThreads, lds, s>>>(p, magic);
}

}  // namespace k
}  // namespace vnpu
