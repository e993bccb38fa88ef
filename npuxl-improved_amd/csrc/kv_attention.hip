// kv_attention.hip - KV_ATTENTION_I8: attention over the paged int8 KV cache
// on gfx950.
//
//   o = sum_j softmax_j(scale * q . k_j) v_j,  k_j = code * k_scale(page, head)
// over the keys j that the query sees, in one pass over the keys with the
// running maximum m and sum l of the softmax.  The rows of a (sequence, kv
// head) are its tokens times the query heads of the group, row r = token r / g,
// head r % g, so grouped heads share every code that is read.
//
// Both products run on the matrix cores with the codes as they are:
//   Q . K   int8: a query row is the whole number rint(q * S), S = 8355700 /
//           max|q|, in three balanced base-256 digits (24 bits), so three
//           v_mfma_i32_16x16x64_i8 give the sum without a rounding;
//   P . V   f16: a code is exact in f16, a weight times its page's scale over a
//           power of two N >= all scales so far is hi + lo, two f16 (22 bits),
//           and two v_mfma_f32_16x16x32_f16 sum in f32.
// The scores are computed transposed (keys x rows) with the keys of a 64-key
// chunk dealt to the tiles so that lane (group g, row) ends with keys 16g ..
// 16g + 15 of its row: those are the operand of P . V as they stand, and their
// V codes are 16 consecutive bytes of a page.  No value crosses a lane in the
// loop but the row's maximum.
#include "device_math.hpp"
#include "kv_common.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <cstdio>

namespace vnpu {
namespace k {
namespace {

using v4i = int __attribute__((ext_vector_type(4)));
using v4f = float __attribute__((ext_vector_type(4)));
using v2f = float __attribute__((ext_vector_type(2)));
using v2h = _Float16 __attribute__((ext_vector_type(2)));
using v8h = _Float16 __attribute__((ext_vector_type(8)));

constexpr uint32_t kChunk = 64;      // keys of a step
constexpr float kDigits = 8355700.0f;   // three digits hold 127 * (65536 + 256 + 1) = 8355711; q * S may round up
constexpr float kNegInf = -__builtin_inff();

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48: the four groups of a row.
__device__ __forceinline__ float groups_max(float x)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float x)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Bytes i of four words in one.
__device__ __forceinline__ void planes_of(const uint32_t u[4], int &p0, int &p1, int &p2)
{
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0602u);
    p0 = static_cast<int>(__builtin_amdgcn_perm(b, a, 0x05040100u));
    p1 = static_cast<int>(__builtin_amdgcn_perm(b, a, 0x07060302u));
    p2 = static_cast<int>(__builtin_amdgcn_perm(d, c, 0x05040100u));
}

// Four codes to f16, exact: 0x6400 | (code ^ 0x80) is 1024 + (code + 128).
__device__ __forceinline__ void halves_of(int codes, v2h &a, v2h &b)
{
    const uint32_t x = static_cast<uint32_t>(codes) ^ 0x80808080u;
    const v2h bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
    b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
}

// A power of two >= the scale (from 2^-100, to 2^127); NaN counts as none.
__device__ __forceinline__ float power_above(float scale)
{
    const uint32_t bits = __float_as_uint(scale == scale ? scale : 0.0f);
    return fminf(fmaxf(__uint_as_float((bits + 0x7fffffu) & 0x7f800000u), 7.888609052210118e-31f), 1.7014118346046923e38f);
}
// 2^14 / N, exact.
__device__ __forceinline__ float up_over(float n) { return __uint_as_float((268u << 23) - __float_as_uint(n)); }

// ---------------------------------------------------------------------------
// Which workgroup does what.  kv_len is on the device, so the host gives a
// grid of `target + batch` slots for each kv head and the workgroups share the
// keys out themselves: `per` chunks each, so that all sequences together take
// `target` slots and their ragged ends at most one more each.
// ---------------------------------------------------------------------------

struct Split {
    uint32_t target, min_per;    // slots aimed at; least chunks of a slot
    uint32_t low_rows, high_rows;   // sequences with rows in (low, high] are this kernel's
};
struct Slot {
    uint32_t b, part, parts, per, chunks;
};

__device__ __forceinline__ uint32_t wave_total(uint32_t v)
{
    for (int o = 1; o < 64; o <<= 1) v += static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o));
    return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)   // inclusive
{
    const uint32_t lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = static_cast<uint32_t>(__shfl_up(static_cast<int>(v), o));
        if (lane >= static_cast<uint32_t>(o)) v += x;
    }
    return v;
}
// Chunks of sequence b; none where it is not this kernel's or out of range
// (check_all tells); one for a sequence without keys, whose rows are zeros.
__device__ __forceinline__ uint32_t chunks_of(const KvAttn &p, const Split &sp, uint32_t b)
{
    if (b >= p.call.batch) return 0;
    const kv::Seq s = kv::sequence(p.call, b);
    const int32_t len = p.call.lengths[b];
    const uint64_t rows = static_cast<uint64_t>(s.n) * (p.heads / p.call.c.kv_heads);
    if (!s.ok || len < 0 || static_cast<uint32_t>(len) > p.max_kv || s.n > p.max_tokens || rows <= sp.low_rows ||
        rows > sp.high_rows)
        return 0;
    return max(1u, (static_cast<uint32_t>(len) + kChunk - 1) / kChunk);
}
// The slot's share, or (of_b) sequence b's parts and first slot; by each wave.
__device__ __forceinline__ bool find_slot(const KvAttn &p, const Split &sp, bool of_b, uint32_t &slot, Slot &r)
{
    const uint32_t lane = threadIdx.x & 63, batch = p.call.batch;
    uint64_t total = 0;
    for (uint32_t i = 0; i < batch; i += 64) total += wave_total(chunks_of(p, sp, i + lane));
    const uint64_t share = (total + sp.target - 1) / sp.target;
    r.per = max(sp.min_per, static_cast<uint32_t>(share));
    uint32_t before = 0;
    for (uint32_t i = 0; i < batch; i += 64) {
        const uint32_t c = chunks_of(p, sp, i + lane), parts = (c + r.per - 1) / r.per;
        const uint32_t upto = wave_scan(parts);
        const uint64_t hit = of_b ? (r.b - i < 64 ? 1ull << (r.b - i) : 0) : __ballot(before + upto > slot);
        if (hit) {
            const int at = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            const uint32_t first = before + static_cast<uint32_t>(__shfl(static_cast<int>(upto - parts), at));
            r.b = i + at;
            r.parts = static_cast<uint32_t>(__shfl(static_cast<int>(parts), at));
            r.chunks = static_cast<uint32_t>(__shfl(static_cast<int>(c), at));
            if (of_b) slot = first;
            r.part = slot - first;
            return r.parts > 0;
        }
        before += static_cast<uint32_t>(__shfl(static_cast<int>(upto), 63));
    }
    return false;
}

// A row's query as digits for the matrix cores: lane (group g, row) holds
// elements 64 s + 16 g .. + 15 of its row.
template <int DS>
struct Query {
    v4i digit[3][DS];
    float factor;   // score in powers of two = sum of digits * factor * k_scale
    __device__ __forceinline__ void load(const float *row, bool here, uint32_t D, float scale, bool aligned)
    {
        const uint32_t g = (threadIdx.x & 63) >> 4;
        float x[DS * 16];
        uint32_t most = 0;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            const uint32_t d = 64 * s + 16 * g;
            const bool in = here && d < D;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (in) {
                    const float *at = row + d + 4 * w;
                    v = aligned ? *reinterpret_cast<const float4 *>(at) : make_float4(at[0], at[1], at[2], at[3]);
                }
                x[16 * s + 4 * w] = v.x;
                x[16 * s + 4 * w + 1] = v.y;
                x[16 * s + 4 * w + 2] = v.z;
                x[16 * s + 4 * w + 3] = v.w;
            }
        }
#pragma unroll
        for (int i = 0; i < DS * 16; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
        // Bits of magnitudes order as floats do, infinity and NaN above all.
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        const float up = most < 0x0f800000u ? 7.922816251426434e28f : 1.0f;   // below 2^-96: 2^96, S stays finite
        const float largest = __uint_as_float(most) * up;
        const float S = most ? kDigits / largest : 1.0f;
        factor = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : scale * 1.4426950408889634f / S / up;
#pragma unroll
        for (int s = 0; s < DS; ++s)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = static_cast<int>(rintf(x[16 * s + 4 * w + i] * up * S));
                    u[i] = (static_cast<uint32_t>(t) + 0x808080u) ^ 0x808080u;   // bytes: balanced digits
                }
                int p0, p1, p2;
                planes_of(u, p0, p1, p2);
                digit[0][s][w] = p2;
                digit[1][s][w] = p1;
                digit[2][s][w] = p0;
            }
    }
};

// The running softmax of a lane's row and its part of O^T: dimensions 16 t +
// 4 g + i.  o counts in N / 2^14; l is this lane's part of the sum.
template <int DT>
struct State {
    v4f o[DT];
    float m, l;
    __device__ __forceinline__ void clear()
    {
        m = kNegInf;
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// Scores f (sums of digits, keys 16 g + 4 t + i) to weights: the softmax step
// and the two f16 parts of p * v_scale.  seen: this lane's keys below it count.
// beta: N before over N now.
template <int DT, bool MASK>
__device__ __forceinline__ void weigh(State<DT> &st, v4f f[4], float ck, float fv, float beta, int seen, v8h hi[2], v8h lo[2])
{
    float top = kNegInf;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, !MASK || 4 * t + i < seen ? f[t][i] : kNegInf);
    // k scales are not negative: the largest sum is the largest score of the lane.
    top = MASK && seen <= 0 ? kNegInf : top * ck;
    const float now = fmaxf(st.m, groups_max(top));
    const float base = now == kNegInf ? 0.0f : now;
    const float alpha = __builtin_amdgcn_exp2f(st.m - base);
    // 1 for rows whose maximum stays; o is left alone where all do.
    if (__any(now > st.m) || beta != 1.0f) {
        const float a = now > st.m ? alpha : 1.0f;
        st.l *= a;
#pragma unroll
        for (int t = 0; t < DT; ++t) st.o[t] *= a * beta;
        st.m = now;
    }
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        v4f p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(f[t][i], ck, -base));
            if (MASK && 4 * t + i >= seen) p[i] = 0.0f;
            sum += p[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            v2f x = {p[i] * fv, p[i + 1] * fv};
            if (MASK) {   // a scale that is NaN reaches seen keys only
                x[0] = 4 * t + i < seen ? x[0] : 0.0f;
                x[1] = 4 * t + i + 1 < seen ? x[1] : 0.0f;
            }
            const v2h h = __builtin_convertvector(x, v2h);
            const v2h r = __builtin_convertvector(x - __builtin_convertvector(h, v2f), v2h);
            hi[t / 2][4 * (t & 1) + i] = h[0];
            hi[t / 2][4 * (t & 1) + i + 1] = h[1];
            lo[t / 2][4 * (t & 1) + i] = r[0];
            lo[t / 2][4 * (t & 1) + i + 1] = r[1];
        }
    }
    st.l += sum;
}

// ---------------------------------------------------------------------------
// Few rows: a workgroup of four waves takes up to 16 RT rows and a range of
// the keys, its waves every fourth chunk, codes straight from memory into the
// operands.  K of the next chunk is on its way while the softmax and P . V
// of this one run, V while the next scores do.
// ---------------------------------------------------------------------------

template <int DP, int RT>
__global__ __launch_bounds__(256, DP * RT <= 128 ? 2 : 1) void kv_attention_stream(KvAttn p, Split sp, float *ws, uint32_t ws_rows)
{
    constexpr int DS = DP / 64, DT = DP / 16, R = 16 * RT;
    __shared__ float sh_o[4][R][68];
    __shared__ float sh_m[4][R], sh_l[4][R];
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const uint32_t h = blockIdx.y, D = c.c.head_dim, ps = c.c.page_size, group = p.heads / c.c.kv_heads;
    if (blockIdx.x == 0 && h == 0) kv::check_all(c, false, p.max_kv);
    uint32_t slot = blockIdx.x;
    Slot sl;
    if (!find_slot(p, sp, false, slot, sl)) return;
    const kv::Seq seq = kv::sequence(c, sl.b);
    const uint32_t len = static_cast<uint32_t>(c.lengths[sl.b]), rows = seq.n * group;
    const uint32_t begin = sl.part * sl.per, end = min(sl.chunks, begin + sl.per);

    Query<DS> q[RT];
    State<DT> st[RT];
    int limit[RT];   // keys that the lane's row sees
    int least = static_cast<int>(len);
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.Q) & 15) | (p.q.batch & 3) | (p.q.token & 3) | (p.q.head & 3)) == 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t row = 16 * r + col, i = row / group;
        const bool here = row < rows;
        const float *at = p.Q + kv::rows_base(c, p.q, sl.b, seq) + (here ? i * p.q.token + (h * group + row % group) * p.q.head : 0);
        q[r].load(at, here, D, p.scale, aligned);
        st[r].clear();
        limit[r] = p.causal && here ? max(0, static_cast<int>(len) - static_cast<int>(seq.n) + static_cast<int>(i) + 1)
                                    : static_cast<int>(len);
    }
    if (p.causal) least = max(0, static_cast<int>(len) - static_cast<int>(seq.n) + 1);

    // Page of the 16 keys that this lane loads K from (kb) and V and the scales (g).
    const uint32_t kb = col >> 2;
    const uint32_t last16 = len ? (len - 1) / 16 : 0, log16 = c.c.log_page - 4;
    const int32_t *table = c.c.table + static_cast<uint64_t>(sl.b) * c.c.table_ld;
    auto page_at = [&](uint32_t block) -> int32_t { return table[min(block, last16) >> log16]; };
    auto checked = [&](int32_t id) -> uint32_t {
        if (static_cast<uint32_t>(id) < c.c.pages) return static_cast<uint32_t>(id);
        kv::fail(c.err);
        return 0;
    };
    v4i kf[4][DS], vf[DT];
    float ks = 0.0f, vs = 0.0f, N = power_above(0.0f);
    int32_t k_id = 0, v_id = 0;
    auto load_k = [&](uint32_t chunk) {   // and the scales
        const uint32_t in = (16 * min(4 * chunk + kb, last16)) & (ps - 1);
        const int8_t *at = c.c.k + ((static_cast<uint64_t>(checked(k_id)) * c.c.kv_heads + h) * ps + in + (col & 3)) * D;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            const uint32_t d = 64 * s + 16 * g;
            const int8_t *from = at + (d < D ? d : 0);   // times digits that are zero
#pragma unroll
            for (int t = 0; t < 4; ++t) kf[t][s] = *reinterpret_cast<const v4i *>(from + 4 * t * D);
        }
        const uint64_t unit = static_cast<uint64_t>(checked(v_id)) * c.c.kv_heads + h;
        ks = c.c.ks[unit];
        vs = c.c.vs[unit];
    };
    auto load_v = [&](uint32_t chunk) {
        const uint32_t in = (16 * min(4 * chunk + g, last16)) & (ps - 1);
        const int8_t *at = c.c.v + ((static_cast<uint64_t>(checked(v_id)) * c.c.kv_heads + h) * D + col) * ps + in;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (16 * t < static_cast<int>(D)) vf[t] = *reinterpret_cast<const v4i *>(at + static_cast<uint64_t>(16 * t) * ps);
    };
    auto ids = [&](uint32_t chunk) {
        k_id = page_at(4 * chunk + kb);
        v_id = page_at(4 * chunk + g);
    };

    auto step = [&](uint32_t chunk, auto more) {
        v4f f[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                v4i a0 = {}, a1 = {}, a2 = {};
#pragma unroll
                for (int s = 0; s < DS; ++s) {
                    a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[0][s], a0, 0, 0, 0);
                    a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[1][s], a1, 0, 0, 0);
                    a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[2][s], a2, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)   // |a0| <= 256 * 127 * 127: a0 * 256 + a1 fits
                    f[r][t][i] = fmaf(static_cast<float>(a0[i] * 256 + a1[i]), 256.0f, static_cast<float>(a2[i]));
            }
        const float ck = ks, v_scale = vs;
        const float above = groups_max(power_above(v_scale)), N_now = fmaxf(N, above);
        const float beta = N / N_now, fv = v_scale * up_over(N_now);
        N = N_now;
        if (more) load_k(chunk + 4);   // v_id is the next chunk's already
        v8h hi[RT][2], lo[RT][2];
        const int first = static_cast<int>(kChunk * chunk + 16 * g);
        if (static_cast<int>(kChunk * chunk + kChunk) <= least) {
#pragma unroll
            for (int r = 0; r < RT; ++r) weigh<DT, false>(st[r], f[r], q[r].factor * ck, fv, beta, 16, hi[r], lo[r]);
        } else {
#pragma unroll
            for (int r = 0; r < RT; ++r) weigh<DT, true>(st[r], f[r], q[r].factor * ck, fv, beta, limit[r] - first, hi[r], lo[r]);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (16 * t >= static_cast<int>(D)) continue;
            v8h a[2];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                v2h x, y;
                halves_of(vf[t][w], x, y);
                a[w / 2][4 * (w & 1)] = x[0];
                a[w / 2][4 * (w & 1) + 1] = x[1];
                a[w / 2][4 * (w & 1) + 2] = y[0];
                a[w / 2][4 * (w & 1) + 3] = y[1];
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[k], lo[r][k], st[r].o[t], 0, 0, 0);
                    st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[k], hi[r][k], st[r].o[t], 0, 0, 0);
                }
        }
        if (more) {
            load_v(chunk + 4);
            ids(min(chunk + 8, end - 1));
        }
    };
    uint32_t chunk = begin + wave;
    if (len && chunk < end) {
        ids(chunk);
        load_k(chunk);
        load_v(chunk);
        ids(min(chunk + 4, end - 1));
        for (; chunk + 4 < end; chunk += 4) step(chunk, std::true_type{});
        step(chunk, std::false_type{});
    }

    // The waves' parts together: each is o / l, weighed by l 2^(m - max m).
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        st[r].l = groups_sum(st[r].l);
        if (g == 0) {
            sh_m[wave][16 * r + col] = st[r].m;
            sh_l[wave][16 * r + col] = st[r].l;
        }
    }
    const uint64_t part_at = (static_cast<uint64_t>(slot) * c.c.kv_heads + h) * ws_rows;
    const bool whole = sl.parts == 1;
    float *ws_o = ws + part_at * (D + 2);
#pragma unroll
    for (int d0 = 0; d0 < DP; d0 += 64) {
        if (d0 >= static_cast<int>(D)) continue;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float by = st[r].l != 0.0f ? N * 6.103515625e-05f / st[r].l : 0.0f;   // 2^-14
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *reinterpret_cast<v4f *>(&sh_o[wave][16 * r + col][16 * t + 4 * g]) = st[r].o[d0 / 16 + t] * by;
        }
        __syncthreads();
        const uint32_t d = d0 + lane;
        for (uint32_t row = wave; row < min(rows, static_cast<uint32_t>(R)); row += 4) {
            float M = kNegInf, L = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, sh_m[w][row]);
            const float base = M == kNegInf ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float x = sh_l[w][row] * __builtin_amdgcn_exp2f(sh_m[w][row] - base);
                L += x;
                o = fmaf(x, sh_o[w][row][lane], o);
            }
            o = L != 0.0f ? o / L : 0.0f;
            if (d < D) {
                if (whole)
                    p.O[kv::rows_base(c, p.o, sl.b, seq) + row / group * p.o.token + (h * group + row % group) * p.o.head + d] = o;
                else
                    ws_o[row * (D + 2) + d] = o;
            }
            if (!whole && d0 == 0 && lane < 2) ws_o[row * (D + 2) + D + lane] = lane ? L : M;
        }
    }
}

// Parts of a row, `step` floats apart, each o / l with its m and l behind it:
// weighed by l 2^(m - max m).  One wave.
__device__ __forceinline__ void join_parts(const float *at, uint64_t step, uint32_t parts, uint32_t D, uint32_t lane, float *out)
{
    float M = kNegInf, L = 0.0f, o[4] = {};
    for (uint32_t i = lane; i < parts; i += 64) M = fmaxf(M, at[i * step + D]);
    for (int x = 32; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    const float base = M == kNegInf ? 0.0f : M;
    for (uint32_t i = 0; i < parts; ++i) {
        const float x = at[i * step + D + 1] * __builtin_amdgcn_exp2f(at[i * step + D] - base);
        L += x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (lane + 64 * r < D) o[r] = fmaf(x, at[i * step + lane + 64 * r], o[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (lane + 64 * r < D) out[lane + 64 * r] = L != 0.0f ? o[r] / L : 0.0f;
}

// A sequence's parts together, one wave for a row.
__global__ __launch_bounds__(64) void kv_attention_merge(KvAttn p, Split sp, const float *ws, uint32_t ws_rows)
{
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x, h = blockIdx.y, row = blockIdx.z, D = c.c.head_dim, group = p.heads / c.c.kv_heads;
    Slot sl;
    sl.b = blockIdx.x;
    uint32_t slot = 0;
    if (!find_slot(p, sp, true, slot, sl) || sl.parts < 2) return;
    const kv::Seq seq = kv::sequence(c, sl.b);
    if (row >= seq.n * group) return;
    const uint64_t step = static_cast<uint64_t>(c.c.kv_heads) * ws_rows * (D + 2);
    const float *at = ws + ((static_cast<uint64_t>(slot) * c.c.kv_heads + h) * ws_rows + row) * (D + 2);
    join_parts(at, step, sl.parts, D, lane,
               p.O + kv::rows_base(c, p.o, sl.b, seq) + row / group * p.o.token + (h * group + row % group) * p.o.head);
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of four waves takes 64 RT rows, each wave 16 RT of
// them, and its part of the keys 64 at a time.  The chunk's K codes are copied
// into LDS in operand order, its V codes pass through registers to be turned into
// f16 once for the four waves; both of the next chunk are on their way while
// this one is computed, and one barrier a chunk hands the buffers over.
// ---------------------------------------------------------------------------

struct Tiles {
    uint32_t per_seq;      // tiles a sequence (without seq_start)
    uint32_t count;        // room for tiles a kv head
    uint32_t parts;        // key ranges of a tile
    uint32_t low_rows;     // sequences with more rows are this kernel's
};

// Tile -> sequence and its tile, as find_unit does: ceil(rows / M) tiles of a
// sequence fit between floor(first row / M) + b and the next sequence's.
template <uint32_t M>
__device__ __forceinline__ bool find_tile(const KvAttn &p, const Tiles &tl, uint32_t group, uint32_t unit, uint32_t &b, uint32_t &tile)
{
    const KvCall &c = p.call;
    if (!c.seq_start) {
        b = unit / tl.per_seq;
        tile = unit % tl.per_seq;
        return b < c.batch;
    }
    uint32_t before = 0;
    for (uint32_t i = 0; i < c.batch; i += 64) {
        const uint32_t at = i + (threadIdx.x & 63);
        const bool here = at < c.batch &&
                          static_cast<uint64_t>(static_cast<uint32_t>(c.seq_start[at])) * group / M + at <= unit;
        before += __popcll(__ballot(here));
    }
    if (!before) return false;
    b = before - 1;
    tile = unit - (static_cast<uint32_t>(static_cast<uint64_t>(static_cast<uint32_t>(c.seq_start[b])) * group / M) + b);
    return true;
}
// The sequence of a tile and whether it is this kernel's.
__device__ __forceinline__ bool tile_sequence(const KvAttn &p, const Tiles &tl, uint32_t group, uint32_t b, kv::Seq &seq, uint32_t &len)
{
    seq = kv::sequence(p.call, b);
    const int32_t n = p.call.lengths[b];
    len = static_cast<uint32_t>(n);
    return seq.ok && n >= 0 && len <= p.max_kv && seq.n <= p.max_tokens && static_cast<uint64_t>(seq.n) * group > tl.low_rows;
}

template <int DP, int RT>
__global__ __launch_bounds__(256, 2) void kv_attention_tile(KvAttn p, Tiles tl, float *ws)
{
    constexpr int DS = DP / 64, DT = DP / 16;
    constexpr uint32_t M = 64 * RT;
    constexpr uint32_t kK = 4 * DS * 1024, kV = DT * 2048, kBuf = kK + kV;   // bytes of a chunk's operands
    extern __shared__ __align__(1024) int8_t lds[];
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t G = c.c.kv_heads, h = blockIdx.x % G, D = c.c.head_dim, ps = c.c.page_size, group = p.heads / G;
    if (blockIdx.x == 0 && blockIdx.y == 0) kv::check_all(c, false, p.max_kv);
    // The last tiles of a causal sequence have the most keys: they come first.
    uint32_t b, tile, len;
    kv::Seq seq;
    const uint32_t unit = tl.count - 1 - blockIdx.x / G;
    if (!find_tile<M>(p, tl, group, unit, b, tile) || !tile_sequence(p, tl, group, b, seq, len)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    len = __builtin_amdgcn_readfirstlane(len);
    const uint32_t rows = __builtin_amdgcn_readfirstlane(seq.n) * group, n = __builtin_amdgcn_readfirstlane(seq.n);
    if (static_cast<uint64_t>(tile) * M >= rows) return;
    const uint32_t row0 = tile * M + wave * 16 * RT;   // the wave's first
    auto sees = [&](uint32_t row) -> int {
        return p.causal ? max(0, static_cast<int>(len) - static_cast<int>(n) + static_cast<int>(row / group) + 1) : static_cast<int>(len);
    };
    // Keys of the tile, of the wave; below `least` every row of the wave sees all.
    const int tile_keys = sees(min(rows, tile * M + M) - 1);
    const int wave_keys = row0 < rows ? sees(min(rows, row0 + 16 * RT) - 1) : 0, least = row0 < rows ? sees(row0) : 0;
    const uint32_t chunks = (static_cast<uint32_t>(tile_keys) + kChunk - 1) / kChunk;
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * blockIdx.y / tl.parts);
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (blockIdx.y + 1) / tl.parts);

    Query<DS> q[RT];
    State<DT> st[RT];
    int limit[RT];
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.Q) & 15) | (p.q.batch & 3) | (p.q.token & 3) | (p.q.head & 3)) == 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t row = row0 + 16 * r + col;
        const bool here = row < rows;
        const float *at = p.Q + kv::rows_base(c, p.q, b, seq) + (here ? (row / group) * p.q.token + (h * group + row % group) * p.q.head : 0);
        q[r].load(at, here, D, p.scale, aligned);
        st[r].clear();
        limit[r] = here ? sees(row) : static_cast<int>(len);
    }

    const uint32_t kb = col >> 2, last16 = len ? (len - 1) / 16 : 0, log16 = c.c.log_page - 4;
    const int32_t *table = c.c.table + static_cast<uint64_t>(b) * c.c.table_ld;
    auto checked = [&](int32_t id) -> uint32_t {
        if (static_cast<uint32_t>(id) < c.c.pages) return static_cast<uint32_t>(id);
        kv::fail(c.err);
        return 0;
    };
    int32_t k_id = 0, v_id = 0;
    auto ids = [&](uint32_t chunk) {
        k_id = table[min(4 * chunk + kb, last16) >> log16];
        v_id = table[min(4 * chunk + g, last16) >> log16];
    };
    constexpr int VW = (DT + 3) / 4;   // tiles of V that a wave brings in
    v4i vf[VW];
    float ks = 0.0f, vs = 0.0f, N = power_above(0.0f);
    auto fetch = [&](uint32_t chunk, int8_t *buf) {
        const uint32_t in_k = (16 * min(4 * chunk + kb, last16)) & (ps - 1);
        const int8_t *kat = c.c.k + ((static_cast<uint64_t>(checked(k_id)) * G + h) * ps + in_k + (col & 3)) * D;
#pragma unroll
        for (int i = 0; i < DS; ++i) {   // operand (tile t, step s) is piece t * DS + s
            const uint32_t piece = wave + 4 * i, t = piece / DS, s = piece % DS, d = 64 * s + 16 * g;
            lds::dma16(kat + 4 * t * D + (d < D ? d : 0), buf + piece * 1024);
        }
        const uint64_t unit_v = static_cast<uint64_t>(checked(v_id)) * G + h;
        const uint32_t in_v = (16 * min(4 * chunk + g, last16)) & (ps - 1);
        const int8_t *vat = c.c.v + (unit_v * D + col) * ps + in_v;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const uint32_t t = wave + 4 * i;
            if (16 * t < D) vf[i] = *reinterpret_cast<const v4i *>(vat + static_cast<uint64_t>(16 * t) * ps);
        }
        ks = c.c.ks[unit_v];
        vs = c.c.vs[unit_v];
    };
    auto turn_v = [&](int8_t *buf) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const uint32_t t = wave + 4 * i;
            if (16 * t >= D) continue;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v2h x[4];
                halves_of(vf[i][2 * k], x[0], x[1]);
                halves_of(vf[i][2 * k + 1], x[2], x[3]);
                const v8h a = {x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
                *reinterpret_cast<v8h *>(buf + kK + (2 * t + k) * 1024 + lane * 16) = a;
            }
        }
    };
    if (begin < end) {
        ids(begin);
        fetch(begin, lds);
        turn_v(lds);
        ids(min(begin + 1, end - 1));
        lds::wait_vmcnt<0>();
        __syncthreads();
    }
    for (uint32_t chunk = begin; chunk < end; ++chunk) {
        int8_t *now = lds + ((chunk - begin) & 1) * kBuf, *next = lds + ((chunk - begin + 1) & 1) * kBuf;
        const float ck = ks, v_scale = vs;
        const bool more = chunk + 1 < end;
        if (more) {
            fetch(chunk + 1, next);
            ids(min(chunk + 2, end - 1));
        }
        const bool work = static_cast<int>(kChunk * chunk) < wave_keys;
        v8h hi[RT][2], lo[RT][2];
        if (work) {
            v4i kf[4][DS];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int s = 0; s < DS; ++s) kf[t][s] = *reinterpret_cast<const v4i *>(now + (t * DS + s) * 1024 + lane * 16);
            const float above = groups_max(power_above(v_scale)), N_now = fmaxf(N, above);
            const float beta = N / N_now, fv = v_scale * up_over(N_now);
            N = N_now;
            const int first = static_cast<int>(kChunk * chunk + 16 * g);
            const bool all = static_cast<int>(kChunk * chunk + kChunk) <= least;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                v4f f[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    v4i a0 = {}, a1 = {}, a2 = {};
#pragma unroll
                    for (int s = 0; s < DS; ++s) {
                        a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[0][s], a0, 0, 0, 0);
                        a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[1][s], a1, 0, 0, 0);
                        a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][s], q[r].digit[2][s], a2, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        f[t][i] = fmaf(static_cast<float>(a0[i] * 256 + a1[i]), 256.0f, static_cast<float>(a2[i]));
                }
                if (all) weigh<DT, false>(st[r], f, q[r].factor * ck, fv, beta, 16, hi[r], lo[r]);
                else weigh<DT, true>(st[r], f, q[r].factor * ck, fv, beta, limit[r] - first, hi[r], lo[r]);
            }
        }
        if (more) turn_v(next);
        if (work) {
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (16 * t >= static_cast<int>(D)) continue;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const v8h a = *reinterpret_cast<const v8h *>(now + kK + (2 * t + k) * 1024 + lane * 16);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo[r][k], st[r].o[t], 0, 0, 0);
                        st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi[r][k], st[r].o[t], 0, 0, 0);
                    }
                }
            }
        }
        lds::wait_vmcnt<0>();
        __syncthreads();
    }

    const bool out_aligned = ((reinterpret_cast<uintptr_t>(p.O) & 15) | (p.o.batch & 3) | (p.o.token & 3) | (p.o.head & 3)) == 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t row = row0 + 16 * r + col;
        const float l = groups_sum(st[r].l);
        const float by = l != 0.0f ? N * 6.103515625e-05f / l : 0.0f;   // 2^-14
        if (row >= rows) continue;
        if (tl.parts == 1) {
            float *at = p.O + kv::rows_base(c, p.o, b, seq) + (row / group) * p.o.token + (h * group + row % group) * p.o.head + 4 * g;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (16 * t >= static_cast<int>(D)) continue;
                const v4f x = st[r].o[t] * by;
                if (out_aligned) *reinterpret_cast<v4f *>(at + 16 * t) = x;
                else
                    for (int i = 0; i < 4; ++i) at[16 * t + i] = x[i];
            }
        } else {
            float *at = ws + (((static_cast<uint64_t>(unit) * G + h) * tl.parts + blockIdx.y) * M + (row - tile * M)) * (D + 4);
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t < static_cast<int>(D)) *reinterpret_cast<v4f *>(at + 4 * g + 16 * t) = st[r].o[t] * by;
            if (g == 0) {
                at[D] = st[r].m;
                at[D + 1] = l;
            }
        }
    }
}

// A tile's key ranges together, one wave for a row.
template <uint32_t M>
__global__ __launch_bounds__(256) void kv_attention_join(KvAttn p, Tiles tl, const float *ws)
{
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x & 63, G = c.c.kv_heads, h = blockIdx.x % G, unit = blockIdx.x / G, D = c.c.head_dim;
    const uint32_t group = p.heads / G;
    uint32_t b, tile, len;
    kv::Seq seq;
    if (!find_tile<M>(p, tl, group, unit, b, tile) || !tile_sequence(p, tl, group, b, seq, len)) return;
    const uint32_t in = blockIdx.y * 4 + (threadIdx.x >> 6), row = tile * M + in;
    if (static_cast<uint64_t>(tile) * M + in >= static_cast<uint64_t>(seq.n) * group) return;
    const uint64_t step = static_cast<uint64_t>(M) * (D + 4);
    const float *at = ws + ((static_cast<uint64_t>(unit) * G + h) * tl.parts * M + in) * (D + 4);
    float *out = p.O + kv::rows_base(c, p.o, b, seq) + (row / group) * p.o.token + (h * group + row % group) * p.o.head;
    join_parts(at, step, tl.parts, D, lane, out);
}

constexpr uint32_t kStreamRows = 32;

struct Plan {
    bool stream = false, tiled = false;   // kernels of the call: sequences of few rows, of many
    Split split{};
    uint32_t slots = 0, rows = 0;   // of the stream kernel: slots a kv head, rows a slot at most
    Tiles tiles{};
    uint32_t tile_rows = 0;
    size_t stream_ws = 0, ws = 0;
};
Plan plan_of(const KvAttn &p)
{
    Plan r;
    const KvCall &c = p.call;
    const uint32_t G = c.c.kv_heads, group = p.heads / G, D = c.c.head_dim;
    const uint64_t most = static_cast<uint64_t>(p.max_tokens) * group;
    r.tiled = most > kStreamRows;
    // Without seq_start all sequences have max_tokens.
    r.stream = !r.tiled || c.seq_start;
    if (r.stream) {
        r.rows = static_cast<uint32_t>(std::min<uint64_t>(most, kStreamRows));
        r.split.target = (2 * p.cus + G - 1) / G;
        r.split.min_per = 4;
        r.split.low_rows = 0;
        r.split.high_rows = kStreamRows;
        r.slots = r.split.target + c.batch;
        if (p.max_kv <= r.split.min_per * kChunk) r.slots = c.batch;   // none splits
        else r.stream_ws = (static_cast<size_t>(r.slots) * G * r.rows * (D + 2) * sizeof(float) + 15) / 16 * 16;
    }
    r.ws = r.stream_ws;
    if (r.tiled) {
        r.tile_rows = most <= 64 || D > 128 ? 64 : 128;
        r.tiles.low_rows = r.stream ? kStreamRows : 0;
        r.tiles.per_seq = static_cast<uint32_t>((most + r.tile_rows - 1) / r.tile_rows);
        r.tiles.count = c.seq_start ? static_cast<uint32_t>(static_cast<uint64_t>(c.tokens) * group / r.tile_rows) + c.batch
                                    : r.tiles.per_seq * c.batch;
        const uint64_t grid = static_cast<uint64_t>(r.tiles.count) * G;
        const uint32_t chunks = (p.max_kv + kChunk - 1) / kChunk;
        r.tiles.parts = grid >= p.cus ? 1 : std::max<uint32_t>(1, std::min<uint64_t>(2 * p.cus / grid, chunks / 8));
        if (r.tiles.parts > 1) r.ws += static_cast<size_t>(grid) * r.tiles.parts * r.tile_rows * (D + 4) * sizeof(float);
    }
    return r;
}

template <int DP, int RT>
void launch_stream(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    kv_attention_stream<DP, RT><<<dim3(pl.slots, p.call.c.kv_heads), 256, 0, s>>>(p, pl.split, ws, pl.rows);
}
template <int DP, int RT>
void launch_tile(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    constexpr uint32_t bytes = 2 * (4 * (DP / 64) * 1024 + (DP / 16) * 2048);
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kv_attention_tile<DP, RT>),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const uint32_t grid = pl.tiles.count * p.call.c.kv_heads;
    kv_attention_tile<DP, RT><<<dim3(grid, pl.tiles.parts), 256, bytes, s>>>(p, pl.tiles, ws);
    if (pl.tiles.parts > 1) kv_attention_join<64 * RT><<<dim3(grid, 16 * RT), 256, 0, s>>>(p, pl.tiles, ws);
}
template <int DP>
void launch(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    if (pl.stream) {
        if (pl.rows <= 16) launch_stream<DP, 1>(s, p, pl, ws);
        else launch_stream<DP, 2>(s, p, pl, ws);
        if (pl.stream_ws)
            kv_attention_merge<<<dim3(p.call.batch, p.call.c.kv_heads, pl.rows), 64, 0, s>>>(p, pl.split, ws, pl.rows);
    }
    if (pl.tiled) {
        float *rest = ws + pl.stream_ws / sizeof(float);
        if constexpr (DP > 128) launch_tile<DP, 1>(s, p, pl, rest);
        else if (pl.tile_rows == 64) launch_tile<DP, 1>(s, p, pl, rest);
        else launch_tile<DP, 2>(s, p, pl, rest);
    }
}

}  // namespace

std::string kv_attention_route(const KvAttn &p)
{
    const Plan pl = plan_of(p);
    char text[96];
    std::snprintf(text, sizeof(text), "stream=%u rows=%u tile=%u parts=%u", pl.stream ? pl.slots : 0, pl.rows,
                  pl.tile_rows, pl.tiles.parts);
    return text;
}

size_t kv_attention_ws_bytes(const KvAttn &p) { return plan_of(p).ws; }

void kv_attention(hipStream_t s, const KvAttn &p, void *ws)
{
    const Plan pl = plan_of(p);
    float *part = static_cast<float *>(ws);
    if (p.call.c.head_dim <= 64) launch<64>(s, p, pl, part);
    else if (p.call.c.head_dim <= 128) launch<128>(s, p, pl, part);
    else launch<256>(s, p, pl, part);
}

}  // namespace k
}  // namespace vnpu
