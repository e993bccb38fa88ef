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
    float M = kNegInf, L = 0.0f, o[4] = {};
    for (uint32_t i = lane; i < sl.parts; i += 64) M = fmaxf(M, at[i * step + D]);
    for (int x = 32; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    const float base = M == kNegInf ? 0.0f : M;
    for (uint32_t i = 0; i < sl.parts; ++i) {
        const float x = at[i * step + D + 1] * __builtin_amdgcn_exp2f(at[i * step + D] - base);
        L += x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (lane + 64 * r < D) o[r] = fmaf(x, at[i * step + lane + 64 * r], o[r]);
    }
    float *out = p.O + kv::rows_base(c, p.o, sl.b, seq) + row / group * p.o.token + (h * group + row % group) * p.o.head;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (lane + 64 * r < D) out[lane + 64 * r] = L != 0.0f ? o[r] / L : 0.0f;
}

constexpr uint32_t kStreamRows = 32;

struct Plan {
    Split stream;
    uint32_t slots = 0, rows = 0;   // of the stream kernel: slots a kv head, rows a slot at most
    size_t ws = 0;
};
Plan plan_of(const KvAttn &p)
{
    Plan r;
    const uint32_t G = p.call.c.kv_heads, group = p.heads / G;
    const uint64_t most = static_cast<uint64_t>(p.max_tokens) * group;
    r.rows = static_cast<uint32_t>(std::min<uint64_t>(most, kStreamRows));
    r.stream.target = (2 * p.cus + G - 1) / G;
    r.stream.min_per = 4;
    r.stream.low_rows = 0;
    r.stream.high_rows = kStreamRows;
    r.slots = r.stream.target + p.call.batch;
    const bool splits = p.max_kv > r.stream.min_per * kChunk;
    if (!splits) r.slots = p.call.batch;
    else r.ws = static_cast<size_t>(r.slots) * G * r.rows * (p.call.c.head_dim + 2) * sizeof(float);
    return r;
}

template <int DP, int RT>
void launch_stream(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    kv_attention_stream<DP, RT><<<dim3(pl.slots, p.call.c.kv_heads), 256, 0, s>>>(p, pl.stream, ws, pl.rows);
}
template <int DP>
void launch_stream_rows(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    if (pl.rows <= 16) launch_stream<DP, 1>(s, p, pl, ws);
    else launch_stream<DP, 2>(s, p, pl, ws);
}

// One wave per token and query head; lane = key for the scores, lane = head
// dimension for the products with V.  Sequences of more rows than low_rows.
__global__ __launch_bounds__(64) void kv_attention_simple(KvAttn p, uint32_t low_rows)
{
    __shared__ float q[256], w[64], ws[64];
    __shared__ uint32_t pages[64];
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x, h = blockIdx.y;
    if (blockIdx.x == 0 && h == 0) kv::check_all(c, false, p.max_kv);
    uint32_t b, i;
    if (!c.seq_start) {
        const uint32_t n = c.tokens / c.batch;
        b = blockIdx.x / n;
        i = blockIdx.x % n;
    } else {
        uint32_t before = 0;
        for (uint32_t k = 0; k < c.batch; k += 64)
            before += __popcll(__ballot(k + lane < c.batch && static_cast<uint32_t>(c.seq_start[k + lane]) <= blockIdx.x));
        if (!before) return;
        b = before - 1;
        i = blockIdx.x - static_cast<uint32_t>(c.seq_start[b]);
    }
    const kv::Seq s = kv::sequence(c, b);
    const int32_t len = c.lengths[b];
    if (!s.ok || i >= s.n || len < 0 || static_cast<uint32_t>(len) > p.max_kv || s.n * (p.heads / c.c.kv_heads) <= low_rows) return;
    const int64_t see = p.causal ? static_cast<int64_t>(len) - s.n + i + 1 : len;
    const uint32_t keys = see > 0 ? static_cast<uint32_t>(see) : 0;
    const uint32_t D = c.c.head_dim, ps = c.c.page_size, kh = h / (p.heads / c.c.kv_heads);
    const float *qr = p.Q + kv::rows_base(c, p.q, b, s) + i * p.q.token + h * p.q.head;
    for (uint32_t d = lane; d < D; d += 64) q[d] = qr[d];
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, o[4] = {};
    const float factor = p.scale * 1.4426950408889634f;   // the softmax in powers of two
    for (uint32_t k0 = 0; k0 < keys; k0 += 64) {
        const uint32_t key = k0 + lane;
        float score = -__builtin_inff();
        w[lane] = 0.0f;
        if (key < keys) {
            const uint32_t page = kv::page_of(c, b, key >> c.c.log_page);
            const uint64_t unit = static_cast<uint64_t>(page) * c.c.kv_heads + kh;
            pages[lane] = page;
            const uint32_t *row = reinterpret_cast<const uint32_t *>(c.c.k + (unit * ps + (key & (ps - 1))) * D);
            float dot = 0.0f;
            for (uint32_t d = 0; d < D; d += 4) {
                const uint32_t x = row[d / 4];
                for (int e = 0; e < 4; ++e) dot = fmaf(q[d + e], static_cast<float>(static_cast<int8_t>(x >> (8 * e))), dot);
            }
            score = dot * c.c.ks[unit] * factor;
            ws[lane] = c.c.vs[unit];
        }
        float top = score;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float now = fmaxf(m, top);
        const float a = now == -__builtin_inff() ? 0.0f : now;   // no finite score yet
        const float e = key < keys ? exp2f(score - a) : 0.0f, keep = exp2f(m - a);
        float sum = e;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * keep + sum;
        m = now;
        if (key < keys) w[lane] = e * ws[lane];
        __syncthreads();
        const uint32_t n = min(64u, keys - k0);
        for (int r = 0; r < 4; ++r) {
            const uint32_t d = lane + 64 * r;
            if (d >= D) continue;
            float acc = o[r] * keep;
            for (uint32_t k = 0; k < n; ++k) {
                const uint64_t unit = static_cast<uint64_t>(pages[k]) * c.c.kv_heads + kh;
                acc = fmaf(w[k], static_cast<float>(c.c.v[(unit * D + d) * ps + ((k0 + k) & (ps - 1))]), acc);
            }
            o[r] = acc;
        }
        __syncthreads();
    }
    float *out = p.O + kv::rows_base(c, p.o, b, s) + i * p.o.token + h * p.o.head;
    for (int r = 0; r < 4; ++r) {
        const uint32_t d = lane + 64 * r;
        if (d < D) out[d] = keys ? o[r] / l : 0.0f;
    }
}

}  // namespace

std::string kv_attention_route(const KvAttn &p)
{
    const Plan pl = plan_of(p);
    char text[96];
    std::snprintf(text, sizeof(text), "stream slots=%u rows=%u", pl.slots, pl.rows);
    return text;
}

size_t kv_attention_ws_bytes(const KvAttn &p) { return plan_of(p).ws; }

void kv_attention(hipStream_t s, const KvAttn &p, void *ws)
{
    const Plan pl = plan_of(p);
    float *part = static_cast<float *>(ws);
    const uint32_t D = p.call.c.head_dim;
    if (D <= 64) launch_stream_rows<64>(s, p, pl, part);
    else if (D <= 128) launch_stream_rows<128>(s, p, pl, part);
    else launch_stream_rows<256>(s, p, pl, part);
    if (pl.ws) kv_attention_merge<<<dim3(p.call.batch, p.call.c.kv_heads, pl.rows), 64, 0, s>>>(p, pl.stream, part, pl.rows);
    if (static_cast<uint64_t>(p.max_tokens) * (p.heads / p.call.c.kv_heads) > kStreamRows)
        kv_attention_simple<<<dim3(p.call.tokens, p.heads), 64, 0, s>>>(p, kStreamRows);
}

}  // namespace k
}  // namespace vnpu
