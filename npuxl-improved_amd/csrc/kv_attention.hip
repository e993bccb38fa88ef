// kv_attention.hip - KV_ATTENTION_I8: attention over the paged int8 KV cache
// on gfx950.
//
//   o = sum_j softmax_j(scale * q . k_j) v_j,  k_j = code * k_scale(page, head)
// over the keys j that the query sees, in one pass over the keys with the
// running maximum m and sum l of the softmax.  The rows of a (sequence, kv
// head) are its tokens times the query heads of the group, row r = token r / g,
// head r % g, so grouped heads share every code that is read.
//
// Both products run on the matrix cores with the codes as they are.  Calls of
// many rows (the kernel of few rows has its own forms, see there):
//   Q . K   int8: a query row is the whole number rint(q * S), S = 8355700 /
//           max|q|, in three balanced base-256 digits (24 bits), so three
//           v_mfma_i32_16x16x64_i8 give the sum without a rounding;
//   P . V   f16: a code is exact in f16, a weight times its page's scale over the
//           row's unit U is hi + lo, two f16 (22 bits, and 2^-25 where those end),
//           and two v_mfma_f32_16x16x32_f16 sum in f32.  U is a power of two that
//           follows the largest product of the row in each chunk, up and down.
// The scores are computed transposed (keys x rows) with the keys of a 64-key
// chunk dealt to the tiles so that lane (group g, row) ends with keys 16g ..
// 16g + 15 of its row: those are the operand of P . V as they stand, and their
// V codes are 16 consecutive bytes of a page.  No value crosses a lane in the
// loop but where a row's maximum or unit moves.
#include "device_math.hpp"
#include "kv_common.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <type_traits>
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
// a / b of two powers of two with a <= b; 0 below 2^-126.
__device__ __forceinline__ float power_ratio(float a, float b)
{
    return __int_as_float(max(0, 0x3f800000 + __float_as_int(a) - __float_as_int(b)));
}
// sum + rest += x, x a chunk's: rest keeps what sum's rounding loses.  Weights below
// 2^-24 of the largest would add nothing to a sum that holds it, however many they
// are (16384 keys, 99.99 % of the weight on one: 2.5e-5 of the result; 131072: 8.5e-5).
__device__ __forceinline__ void add_kept(float &sum, float &rest, float x)
{
    const float now = sum + x;
    rest += x - (now - sum);
    sum = now;
}
// 1 / N of a power of two from 2^-126 to 2^126, exact.
__device__ __forceinline__ float over_power(float n) { return __uint_as_float((254u << 23) - __float_as_uint(n)); }

// ---------------------------------------------------------------------------
// Which workgroup does what.  kv_len is on the device.  With enough sequences
// and heads a slot is a sequence (whole); else the host gives a grid of
// `target + batch` slots for each kv head and the workgroups share the keys out
// themselves: `per` chunks each, so that all sequences together take
// `target` slots and their ragged ends at most one more each.
// ---------------------------------------------------------------------------

struct Split {
    uint32_t whole;                 // slot = sequence
    uint32_t target, min_per;       // slots aimed at; least chunks of a slot
    uint32_t low_rows, high_rows;   // sequences with rows in (low, high] are this kernel's
};
struct Slot {
    uint32_t b, part, parts, per, chunks;
};

// Inclusive sums over the first `count` lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t count)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t o = 1; o < 64 && o < count; o <<= 1) {
        const uint32_t x = static_cast<uint32_t>(__shfl_up(static_cast<int>(v), o));
        if (lane >= o) v += x;
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
// The slot's share, or (of_b) sequence r.b's parts and first slot; by each wave.
__device__ __forceinline__ bool find_slot(const KvAttn &p, const Split &sp, bool of_b, uint32_t &slot, Slot &r)
{
    const uint32_t lane = threadIdx.x & 63, batch = p.call.batch;
    if (sp.whole || batch == 1) {
        if (sp.whole) r.b = slot;
        else r.b = 0;
        r.chunks = chunks_of(p, sp, r.b);
        r.per = sp.whole ? r.chunks : max(sp.min_per, (r.chunks + sp.target - 1) / sp.target);
        r.parts = r.chunks ? (r.chunks + r.per - 1) / r.per : 0;
        if (of_b) slot = 0;
        r.part = sp.whole ? 0 : slot;
        return r.part < r.parts;
    }
    uint64_t total = 0;
    for (uint32_t i = 0; i < batch; i += 64) {
        const uint32_t n = min(64u, batch - i);
        total += static_cast<uint32_t>(__shfl(static_cast<int>(wave_scan(chunks_of(p, sp, i + lane), n)), n - 1));
    }
    const uint64_t share = (total + sp.target - 1) / sp.target;
    r.per = max(sp.min_per, static_cast<uint32_t>(share));
    uint32_t before = 0;
    for (uint32_t i = 0; i < batch; i += 64) {
        const uint32_t n = min(64u, batch - i);
        const uint32_t c = chunks_of(p, sp, i + lane), parts = (c + r.per - 1) / r.per;
        const uint32_t upto = wave_scan(parts, n);
        const uint64_t hit = of_b ? (r.b - i < 64 ? 1ull << (r.b - i) : 0) : __ballot(lane < n && before + upto > slot);
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
        before += static_cast<uint32_t>(__shfl(static_cast<int>(upto), n - 1));
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
        // Loads under a condition would be waited for one by one.
        auto at = [&](int s) { return row + (64 * s + 16 * g < D ? 64 * s + 16 * g : 0); };
        if (aligned) {
#pragma unroll
            for (int s = 0; s < DS; ++s)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float4 v = *reinterpret_cast<const float4 *>(at(s) + 4 * w);
                    x[16 * s + 4 * w] = v.x;
                    x[16 * s + 4 * w + 1] = v.y;
                    x[16 * s + 4 * w + 2] = v.z;
                    x[16 * s + 4 * w + 3] = v.w;
                }
        } else {
#pragma unroll
            for (int s = 0; s < DS; ++s)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[16 * s + i] = at(s)[i];
        }
#pragma unroll
        for (int s = 0; s < DS; ++s)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[16 * s + i] = here && 64 * s + 16 * g < D ? x[16 * s + i] : 0.0f;
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
// 4 g + i.  o counts in 2^-shift = U / 2^14; l is this lane's part of the sum.
// The largest p * v_scale of the row's chunk lies between 2^-12 U and 2 U: below, U
// comes down after it, so that its smaller weights keep their bits, unless o, which
// holds what was summed before, would pass 2^100.  The reference m is one that
// scores may pass by kAhead, as for few rows.  (Scores of normal numbers: one chunk in
// 40 moves something for one of a wave's 32 rows, 243 us for 4096 tokens against 237 with a
// U that only grew; 8 times as far apart every chunk does, 280 against 228.  Within 2^-6
// a fifth of the chunks did for ordinary scores: 259.)
constexpr float kAhead = 4.0f, kMostShift = 114.0f, kFar = 12.0f, kJump = 8.0f;
template <int DT>
struct State {
    v4f o[DT];
    float m, l, l_rest, shift;
    __device__ __forceinline__ void clear()
    {
        m = kNegInf;
        l = l_rest = 0.0f;
        shift = kMostShift;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// The largest of a lane's scores f (sums of digits, keys 16 g + 4 t + i).
// seen: this lane's keys below it count.
template <bool MASK>
__device__ __forceinline__ float largest(const v4f f[4], float ck, int seen)
{
    float top = kNegInf;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, !MASK || 4 * t + i < seen ? f[t][i] : kNegInf);
    // k scales are not negative: the largest sum is the largest score.
    return MASK && seen <= 0 ? kNegInf : top * ck;
}

// Scores of tiles 2 half and 2 half + 1 to weights: the two f16 parts of
// p * v_scale, p added to the lane's sum.
template <bool MASK>
__device__ __forceinline__ void weigh(float &sum, const v4f f[4], int half, float ck, float base, float fv, int seen, v8h &hi, v8h &lo)
{
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t = 2 * half + u;
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
            hi[4 * u + i] = h[0];
            hi[4 * u + i + 1] = h[1];
            lo[4 * u + i] = r[0];
            lo[4 * u + i + 1] = r[1];
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows (a token or a few of grouped heads): the codes are read once and
// bound the kernel.  A workgroup takes the rows and a range of the keys, its
// waves every WAVES-th chunk of 64.  Each wave copies a chunk's K and V codes
// into LDS of its own with 64-byte runs for every four lanes (read straight into
// operands, where neighbouring lanes hold different keys, the same loads took
// four times the cycles of the address unit: 10 TB/s even from cache), and asks for
// the next chunk as soon as the operands have left LDS, so 16 KiB a wave are
// under way; pages and scales come through scalar loads and disturb no count.
// Both products run on the int8 matrix cores, no code converted: the 16
// operand rows of a product are 4 rows times 4 base-256 digits, row 4 r + d,
// so one product gives a lane the four digit sums of one result:
//   q digits x K codes   lane (r = g, c): row r, key 4 c + t of tile t;
//   p digits x V codes   lane (r = g, c): row r, dimension 16 t + c of tile t.
// A weight w = p * v_scale / N, p = 2^(s - m) for a reference m that s may pass by
// 4, N a power of two that no v_scale seen by the row passes, becomes the whole
// number rint(w * 2^k), k such that the largest of the row's weights in these 64
// keys has 31 bits: a chunk's sums are whole numbers of their own unit, then added to f32 sums.  What
// the rounding left is four digits more, under 2^-31 of the unit, and goes through
// the product again where it is more than 2^-22 of some weight: one key with nearly
// all of the weight, or a page of large values, takes nothing from the others.
// (In one unit for all chunks, that of the largest weight so far, whole sums could
// stay on the matrix cores, 3 to 6 % faster, with 16 rows 52 us instead of 68 for 16
// sequences of 4096 keys, but weights 2^-26 below it were lost: 7 % of a result
// whose first of 4096 keys has 99.99 % of the weight and zeros for values.)
// Bound by the codes from HBM where there are enough of them (32 heads of 128, 8
// sequences of 4096 keys: 42 us, 6.3 TB/s of codes; a large read reaches 6.2 to
// 6.7; 64 sequences of 100 to 8000 keys, 32 heads to 8: 110 us, 5.4 TB/s; one of
// 131072 keys: 43 us and 4.5 us of join), by the latency of launch, page,
// copy and join where not (one sequence of 128 keys 5.4 us, of 4096 11.3 us).
// Not temporal copies: 67 -> 56 us at the first size, which nothing reads twice.
// ---------------------------------------------------------------------------

constexpr float kDigits4 = 2139060000.0f;   // four digits hold 127 * (2^24 + 2^16 + 2^8 + 1) = 2139062143
// Biased exponent e for whole numbers of up to 31 bits: x * 2^(157 - e), x at most
// `largest`, fits four digits (2139062143 / 2^30 is 2 less 65793 / 2^23; 0x10400 is 66560).
// Below 2^-96 e stays, so that 2^(e - 157) is a normal number.
__device__ __forceinline__ uint32_t digits_exponent(float largest)
{
    return max((__float_as_uint(largest) + 0x10400u) >> 23, 31u);
}

// Maximum / sum over the 16 lanes of a row.
template <int CTRL>
__device__ __forceinline__ float dpp_row(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_max(float x)
{
    x = fmaxf(x, dpp_row<0x128>(x));   // row_ror:8
    x = fmaxf(x, dpp_row<0x124>(x));
    x = fmaxf(x, dpp_row<0x122>(x));
    return fmaxf(x, dpp_row<0x121>(x));
}
__device__ __forceinline__ float row_sum(float x)
{
    x += dpp_row<0x128>(x);
    x += dpp_row<0x124>(x);
    x += dpp_row<0x122>(x);
    return x + dpp_row<0x121>(x);
}
// Sum of four digit sums over 64 keys or 256 dimensions, digit i counting 256^i.
__device__ __forceinline__ float digits_sum(const v4i &a)
{
    return fmaf(static_cast<float>(a[3] * 256 + a[2]), 65536.0f, static_cast<float>(a[1] * 256 + a[0]));
}

template <typename T>
__device__ __forceinline__ T scalar_load(const T *at)   // a wave's address, memory that the kernel does not write
{
    return *(const __attribute__((address_space(4))) T *)at;
}
// At most n copies under way; n is one of the tile counts of DP.
template <int DP, bool FULL>
__device__ __forceinline__ void wait_copies(uint32_t n)
{
    if constexpr (FULL) lds::wait_vmcnt<DP / 16>();
    else if constexpr (DP == 64) lds::wait_vmcnt<1>();
    else if constexpr (DP == 128) {
        if (n >= 6) lds::wait_vmcnt<6>();
        else lds::wait_vmcnt<5>();
    } else {
        if (n >= 12) lds::wait_vmcnt<12>();
        else lds::wait_vmcnt<9>();
    }
}

// Bytes of dynamic LDS: a chunk's K and V a wave, its digits and its f32
// sums; the queries.
template <int DP, int RT, int WAVES>
constexpr uint32_t few_lds()
{
    return WAVES * (128 * DP + 1024 + RT * DP * 16) + RT * (DP / 64) * 1024;
}

template <int DP, int RT, bool FULL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP * RT <= 256 && DP <= 128 ? 2 : 1) void kv_attention_few(KvAttn p, Split sp, float *ws, uint32_t ws_rows)
{
    constexpr int DS = DP / 64, DT = DP / 16, R = 4 * RT;
    extern __shared__ __align__(1024) int8_t lds[];
    __shared__ float sh_m[WAVES][R], sh_l[WAVES][R], sh_f[R];
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t h = blockIdx.y, G = c.c.kv_heads, D = FULL ? DP : c.c.head_dim, ps = c.c.page_size, group = p.heads / G;
    int8_t *k_lds = lds + wave * 128 * DP, *v_lds = k_lds + 64 * DP;
    uint32_t *sh_p = reinterpret_cast<uint32_t *>(lds + WAVES * 128 * DP) + wave * 256;
    float *sh_o_all = reinterpret_cast<float *>(lds + WAVES * (128 * DP + 1024)), *sh_o = sh_o_all + wave * RT * DT * 64;
    if (blockIdx.x == 0 && h == 0) kv::check_all(c, false, p.max_kv, p.max_tokens);
    uint32_t slot = blockIdx.x;
    Slot sl;
    if (!find_slot(p, sp, false, slot, sl)) return;
    const uint32_t b = __builtin_amdgcn_readfirstlane(sl.b), parts = __builtin_amdgcn_readfirstlane(sl.parts);
    const kv::Seq seq = kv::sequence(c, b);
    const uint32_t n = __builtin_amdgcn_readfirstlane(seq.n), rows = n * group, row0 = blockIdx.z * R;
    if (row0 >= rows) return;
    const int len = __builtin_amdgcn_readfirstlane(c.lengths[b]);
    // Even parts of the keys.
    const uint32_t chunks = __builtin_amdgcn_readfirstlane(sl.chunks), part = __builtin_amdgcn_readfirstlane(sl.part);
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * part / parts);
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (part + 1) / parts);

    // Pages of a chunk's four blocks of 16 keys (blocks behind the last are
    // the last) and, of the chunk in LDS, their scales.
    const uint32_t last16 = len ? (len - 1) / 16 : 0, log16 = c.c.log_page - 4, tiles = D / 16;
    const int32_t *table = c.c.table + static_cast<uint64_t>(b) * c.c.table_ld;
    bool strange = false;   // a page outside the pool: page 0 is read in its place
    int32_t id[4] = {};
    uint64_t unit[4] = {};
    float ks4[4], vs4[4];
    // Asked for a chunk ahead: `pages` waits for nothing, `units` for them.
    auto pages = [&](uint32_t chunk) {
#pragma unroll
        for (int j = 0; j < 4; ++j) id[j] = scalar_load(table + (min(4 * chunk + j, last16) >> log16));
    };
    auto units = [&]() {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = static_cast<uint32_t>(id[j]) < c.c.pages;
            strange |= !in;
            unit[j] = static_cast<uint64_t>(static_cast<uint32_t>(in ? id[j] : 0)) * G + h;
        }
    };
    auto scales = [&]() {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ks4[j] = scalar_load(c.c.ks + unit[j]);
            vs4[j] = scalar_load(c.c.vs + unit[j]);
        }
    };
    auto of_block = [&](uint32_t j, const auto &x) {
        const auto a = x[0], b = x[1], c = x[2], d = x[3];   // values: an index would put the array into memory
        return j & 2 ? (j & 1 ? d : c) : (j & 1 ? b : a);
    };
    // K: a block's 16 keys are 16 D bytes in a row.  The 16-byte pieces of a key
    // are swapped by its place, so that the operands' reads, at keys 4 apart, spread over the banks.
    constexpr uint32_t kSwap = FULL ? DP / 16 - 1 : 0;
    auto copy_k = [&](uint32_t chunk) {
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            if (!FULL && i >= static_cast<int>(tiles)) break;
            if constexpr (FULL) {
                constexpr int kPer = DP / 64;   // copies of a block
                const uint32_t j = i / kPer, in = (16 * min(4 * chunk + j, last16)) & (ps - 1);
                const uint32_t piece = 64 * (i % kPer) + lane, key = piece / (DP / 16), at = piece % (DP / 16);
                lds::dma16_nt(c.c.k + (unit[j] * ps + in + key) * DP + 16 * (at ^ ((4 * j + key / 4) & kSwap)), k_lds + 1024 * i);
            } else {
                const uint32_t piece = 64 * i + lane, j = piece / D, in = (16 * min(4 * chunk + j, last16)) & (ps - 1);
                lds::dma16_nt(c.c.k + (of_block(j, unit) * ps + in) * D + 16 * (piece - j * D), k_lds + 1024 * i);
            }
        }
    };
    // V: a dimension's keys of a page are a row; where a page is 16 or 32 keys,
    // rows of neighbouring dimensions follow each other.  Lane -> dimension
    // and block of 16 keys so that lanes in a row read bytes in a row; the blocks of a
    // row are swapped for the banks too.
    const uint32_t low = min(c.c.log_page, 6u) - 4, low_mask = (1u << low) - 1;
    const uint32_t v_dim = (lane >> low) & 15;
    const uint32_t v_block = (lane >> (4 + low)) << low | ((lane & low_mask) ^ ((v_dim >> (4 - low)) & low_mask));
    const uint32_t v_at = 16 * ((g >> low) << (4 + low) | col << low | ((g & low_mask) ^ ((col >> (4 - low)) & low_mask)));
    auto copy_v = [&](uint32_t chunk) {
        const uint32_t in = (16 * min(4 * chunk + v_block, last16)) & (ps - 1);
        const int8_t *from = c.c.v + (of_block(v_block, unit) * D + v_dim) * ps + in;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (FULL || t < static_cast<int>(tiles)) lds::dma16_nt(from + static_cast<uint64_t>(16 * t) * ps, v_lds + 1024 * t);
    };
    uint32_t chunk = begin + wave;
    const bool any = len && chunk < end;
    if (any) pages(chunk);
    // The rows' queries to LDS (where the f32 sums will be), all loads at once.
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.Q) & 15) | (p.q.batch & 3) | (p.q.token & 3) | (p.q.head & 3)) == 0;
    constexpr int kLoads = (R * DP / 4 + 64 * WAVES - 1) / (64 * WAVES);
    float4 *sh_x = reinterpret_cast<float4 *>(sh_o_all);
    const float *q_base = p.Q + kv::rows_base(c, p.q, b, seq) + h * group * p.q.head;
    float4 raw[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
        // Loads under a condition would be waited for one by one.
        const uint32_t e = threadIdx.x + k * 64 * WAVES, r = e / (DP / 4), d = 4 * (e % (DP / 4));
        const uint32_t row = min(row0 + r, rows - 1), i = row / group;
        const float *at = q_base + i * p.q.token + (row - i * group) * p.q.head + min(d, D - 4);
        raw[k] = aligned ? *reinterpret_cast<const float4 *>(at) : make_float4(at[0], at[1], at[2], at[3]);
        if (row0 + r >= rows || d >= D) raw[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (any) units();
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
        const uint32_t e = threadIdx.x + k * 64 * WAVES;
        if (e < R * DP / 4) sh_x[e] = raw[k];
    }
    if (any) {
        copy_k(chunk);
        copy_v(chunk);
        scales();
        pages(min(chunk + WAVES, end - 1));
    }
    __syncthreads();

    // Queries: lane (operand row 4 r + d, group g) holds digit d of row r's
    // elements 64 s + 16 g .. + 15.  The waves share the (r, s) out and hand
    // them over in LDS.
    v4i *sh_q = reinterpret_cast<v4i *>(lds + WAVES * (128 * DP + 1024 + RT * DP * 16));
#pragma unroll 1
    for (uint32_t task = wave; task < RT * DS; task += WAVES) {
        const uint32_t r = task / DS, s = task % DS;
        const float4 *at = sh_x + (4 * r + (col >> 2)) * (DP / 4) + 4 * g;
        uint32_t most = 0;
        float x[16];
#pragma unroll 1
        for (uint32_t k = 1; k <= DS; ++k) {   // the task's own step last
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 v = at[16 * ((s + k) % DS) + w];
                x[4 * w] = v.x;
                x[4 * w + 1] = v.y;
                x[4 * w + 2] = v.z;
                x[4 * w + 3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
        }
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        const float up = most < 0x0f800000u ? 7.922816251426434e28f : 1.0f;   // below 2^-96: times 2^96
        const float S = most ? kDigits4 / (__uint_as_float(most) * up) : 1.0f;
        if (s == 0 && g == 0 && (col & 3) == 0)
            sh_f[4 * r + (col >> 2)] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : p.scale * 1.4426950408889634f / S / up;
        const uint32_t d = col & 3, pick = 0x0c0c0000u | (4 + d) << 8 | d;
        v4i digits;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                u[e] = (static_cast<uint32_t>(static_cast<int>(rintf(x[4 * w + e] * up * S))) + 0x80808080u) ^ 0x80808080u;
            digits[w] = static_cast<int>(__builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], pick),
                                                               __builtin_amdgcn_perm(u[1], u[0], pick), 0x05040100u));
        }
        sh_q[task * 64 + lane] = digits;
    }
    __syncthreads();
    // With 16 rows the queries stay in LDS: a register spilled in the loop would
    // wait for the copies under way.
    constexpr bool kHeld = RT < 4;
    v4i q[kHeld ? RT : 1][DS];
    float o[RT][DT];                  // row g, dimension 16 t + col, in N
    float factor[RT], m[RT], l[RT], l_rest[RT], N[RT];   // of row g: score in powers of two = sum * factor * k_scale
    int limit[RT];                    // keys that row g sees
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int s = 0; s < DS; ++s)
            if (kHeld) q[r][s] = sh_q[(r * DS + s) * 64 + lane];
        factor[r] = sh_f[4 * r + g];
        const uint32_t mine = row0 + 4 * r + g;
        limit[r] = p.causal && mine < rows ? max(0, len - static_cast<int>(n) + static_cast<int>(mine / group) + 1) : len;
        m[r] = kNegInf;
        l[r] = l_rest[r] = 0.0f;
        N[r] = power_above(0.0f);
#pragma unroll
        for (int t = 0; t < DT; ++t) o[r][t] = 0.0f;
    }
    const int least = p.causal ? max(0, len - static_cast<int>(n) + static_cast<int>(row0 / group) + 1) : len;   // every row sees the keys below
    // Four whole numbers of this lane's keys as digits through LDS: operand row 4 r + d
    // of the product with V.
    auto operand = [&](const int x[4]) {
        uint32_t u[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) u[t] = (static_cast<uint32_t>(x[t]) + 0x80808080u) ^ 0x80808080u;
        const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), e = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
        const uint32_t d = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), k = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
        uint32_t *to = sh_p + 64 * g + col;
        to[0] = __builtin_amdgcn_perm(e, a, 0x05040100u);
        to[16] = __builtin_amdgcn_perm(e, a, 0x07060302u);
        to[32] = __builtin_amdgcn_perm(k, d, 0x05040100u);
        to[48] = __builtin_amdgcn_perm(k, d, 0x07060302u);
        __builtin_amdgcn_wave_barrier();
        const v4i got = *reinterpret_cast<const v4i *>(sh_p + 16 * col + 4 * g);
        __builtin_amdgcn_wave_barrier();
        return got;
    };

    for (bool more = any; more;) {
        more = chunk + WAVES < end;
        const uint32_t kb = col >> 2;
        const float ks = of_block(kb, ks4), scale = of_block(kb, vs4);
        const int first = static_cast<int>(kChunk * chunk + 4 * col);
        const bool all = static_cast<int>(kChunk * chunk + kChunk) <= least;
        auto seen = [&](int r) { return all || first < limit[r]; };   // keys of this lane's page
        wait_copies<DP, FULL>(tiles);   // V's may be under way
        v4i kf[4][DS];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const uint32_t piece = FULL ? (4 * s + g) ^ (col & kSwap) : 4 * s + g < tiles ? 4 * s + g : 0;   // times zeros
                kf[t][s] = *reinterpret_cast<const v4i *>(k_lds + (4 * col + t) * D + 16 * piece);
            }
        __builtin_amdgcn_s_waitcnt(lds::waitcnt_imm(63, 7, 0));
        if (more) {
            units();
            copy_k(chunk + WAVES);
        }
        float f[RT][4], top[RT];
        bool move = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            top[r] = kNegInf;
            constexpr int H = kHeld ? 1 : 0;
            if (!kHeld)
#pragma unroll
                for (int s = 0; s < DS; ++s) q[0][s] = sh_q[(r * DS + s) * 64 + lane];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                v4i a = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < DS; ++s) a = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[H * r][s], kf[t][s], a, 0, 0, 0);
                f[r][t] = digits_sum(a);
            }
            const float ck = factor[r] * ks;
#pragma unroll
            for (int t = 0; t < 4; ++t) f[r][t] *= ck;
            if (all) {
                top[r] = fmaxf(fmaxf(f[r][0], f[r][1]), fmaxf(f[r][2], f[r][3]));
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) top[r] = fmaxf(top[r], first + t < limit[r] ? f[r][t] : kNegInf);
            }
            // A page that the row does not see counts for nothing.
            move |= top[r] > m[r] + kAhead || (seen(r) && scale > N[r]);
        }
        if (__any(move)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                // With a factor of two to spare, up to 2^126.
                const float need = row_max(power_above(seen(r) ? scale : 0.0f));
                const float N_now = need > N[r] ? fminf(2.0f * need, 8.507059173023462e37f) : N[r];
                const float beta = power_ratio(N[r], N_now);
                N[r] = N_now;
                const float now = fmaxf(m[r], row_max(top[r]));
                const float alpha = now > m[r] ? __builtin_amdgcn_exp2f(m[r] - now) : 1.0f;
                l[r] *= alpha;
                l_rest[r] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[r][t] *= alpha * beta;
                m[r] = now;
            }
        }
        v4i pd[RT];
        float unit[RT];   // of the chunk's whole numbers, in N; f becomes what their rounding left
        bool again[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float base = m[r] == kNegInf ? 0.0f : m[r], fv = scale * over_power(N[r]);
            float w[4], sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float e = __builtin_amdgcn_exp2f(f[r][t] - base);
                w[t] = e * fv;
                if (!all && first + t >= limit[r]) e = w[t] = 0.0f;
                sum += e;
            }
            // A scale that is infinite or no number shows in l: whole numbers and weights of 0 cannot.
            if (seen(r)) sum = fmaf(fv + ks, 0.0f, sum);
            add_kept(l[r], l_rest[r], sum);
            const uint32_t e = digits_exponent(row_max(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))));
            const float up = __uint_as_float((284u - e) << 23);
            unit[r] = __uint_as_float((e - 30u) << 23);
            int x[4];
            bool lost = false;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float y = w[t] * up, whole = rintf(y);
                x[t] = static_cast<int>(whole);
                f[r][t] = y - whole;
                lost |= fabsf(f[r][t]) > y * 2.384185791015625e-07f;   // 2^-22
            }
            again[r] = __any(lost);
            pd[r] = operand(x);
        }
        if (more) wait_copies<DP, FULL>(tiles);   // the next K's may be under way
        else lds::wait_vmcnt<0>();
        v4i vf[DT];
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (FULL || t < static_cast<int>(tiles)) vf[t] = *reinterpret_cast<const v4i *>(v_lds + 1024 * t + v_at);
        __builtin_amdgcn_s_waitcnt(lds::waitcnt_imm(63, 7, 0));
        if (more) {
            copy_v(chunk + WAVES);
            scales();
            pages(min(chunk + 2 * WAVES, end - 1));
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (!FULL && t >= static_cast<int>(tiles)) continue;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const v4i sums = __builtin_amdgcn_mfma_i32_16x16x64_i8(pd[r], vf[t], v4i{0, 0, 0, 0}, 0, 0, 0);
                o[r][t] = fmaf(digits_sum(sums), unit[r], o[r][t]);
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (!again[r]) continue;
            int x[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) x[t] = static_cast<int>(rintf(f[r][t] * 2147483648.0f));   // 2^31; f is 1/2 at most
            const v4i rest = operand(x);
            const float below = unit[r] * 4.656612873077393e-10f;   // 2^-31
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (!FULL && t >= static_cast<int>(tiles)) continue;
                const v4i sums = __builtin_amdgcn_mfma_i32_16x16x64_i8(rest, vf[t], v4i{0, 0, 0, 0}, 0, 0, 0);
                o[r][t] = fmaf(digits_sum(sums), below, o[r][t]);
            }
        }
        chunk += WAVES;
    }
    if (strange) kv::fail(c.err);

    // The waves' parts together: each is o / l, weighed by l 2^(m - max m).
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const float sum = row_sum(l[r] + l_rest[r]);
        const float by = sum != 0.0f ? N[r] / sum : 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (FULL || 16 * t < static_cast<int>(D)) sh_o[(r * DT + t) * 64 + lane] = o[r][t] * by;
        if (col == 0) {
            sh_m[wave][4 * r + g] = m[r];
            sh_l[wave][4 * r + g] = sum;
        }
    }
    __syncthreads();
    float *ws_o = ws + (static_cast<uint64_t>(slot) * G + h) * ws_rows * (D + 2);
    const uint32_t count = min(rows - row0, static_cast<uint32_t>(R));
    for (uint32_t e = threadIdx.x; e < count * DP; e += 64 * WAVES) {
        const uint32_t row = e / DP, d = e % DP;
        if (!FULL && d >= D) continue;
        float M = kNegInf, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M = fmaxf(M, sh_m[w][row]);
        const float base = M == kNegInf ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float x = sh_l[w][row] * __builtin_amdgcn_exp2f(sh_m[w][row] - base);
            L += x;
            o = fmaf(x, sh_o_all[((w * RT + row / 4) * DT + d / 16) * 64 + 16 * (row & 3) + (d & 15)], o);
        }
        o = L != 0.0f ? o / L : 0.0f;
        const uint32_t at = row0 + row;
        if (parts == 1) {
            p.O[kv::rows_base(c, p.o, b, seq) + at / group * p.o.token + (h * group + at % group) * p.o.head + d] = o;
        } else {
            ws_o[at * (D + 2) + d] = o;
            if (d < 2) ws_o[at * (D + 2) + D + d] = d ? L : M;
        }
    }
}

// Parts of a row, `step` floats apart, each o / l with its m and l behind it:
// weighed by l 2^(m - max m).  A workgroup a row: the weights first, a part a
// thread, then the sums, threads over the dimensions and every few parts.  The
// latency of what other dies have just written bounds it: 4.6 us for 65 parts of 32 rows,
// 7.6 us with the sums asked for after the weights.
constexpr uint32_t kJoinThreads = 512, kMostParts = 1024;
__device__ __forceinline__ void join_parts(const float *at, uint64_t step, uint32_t parts, uint32_t D, float *out)
{
    __shared__ float weight[kMostParts], sums[kJoinThreads], red[2][kJoinThreads / 64];
    const uint32_t tid = threadIdx.x, wave = tid >> 6;
    // The statistics and each thread's first parts are asked for together; what
    // is behind the last part is that one again, its weight 0.
    constexpr uint32_t kFirst = 16;
    const uint32_t width = D <= 64 ? 64 : D <= 128 ? 128 : 256, every = kJoinThreads / width, d = min(tid % width, D - 1);
    float m[kMostParts / kJoinThreads], l[kMostParts / kJoinThreads], x[kFirst], M = kNegInf, L = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kMostParts / kJoinThreads; ++k) {
        const float *part = at + min(tid + k * kJoinThreads, parts - 1) * step + D;
        m[k] = part[0];
        l[k] = part[1];
    }
#pragma unroll
    for (uint32_t k = 0; k < kFirst; ++k) x[k] = at[min(tid / width + k * every, parts - 1) * step + d];
#pragma unroll
    for (uint32_t k = 0; k < kMostParts / kJoinThreads; ++k) {
        if (tid + k * kJoinThreads >= parts) {
            m[k] = kNegInf;
            l[k] = 0.0f;
        }
        M = fmaxf(M, m[k]);
    }
    for (int x = 32; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    if ((tid & 63) == 0) red[0][wave] = M;
    __syncthreads();
    for (uint32_t w = 0; w < kJoinThreads / 64; ++w) M = fmaxf(M, red[0][w]);
    const float base = M == kNegInf ? 0.0f : M;
#pragma unroll
    for (uint32_t k = 0; k < kMostParts / kJoinThreads; ++k) {
        const float x = l[k] * __builtin_amdgcn_exp2f(m[k] - base);
        weight[tid + k * kJoinThreads] = x;
        L += x;
    }
    for (int x = 32; x; x >>= 1) L += __shfl_xor(L, x);
    if ((tid & 63) == 0) red[1][wave] = L;
    __syncthreads();
    L = 0.0f;
    for (uint32_t w = 0; w < kJoinThreads / 64; ++w) L += red[1][w];
    float o = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kFirst; ++k) {
        const uint32_t i = tid / width + k * every;
        o = fmaf(i < parts ? weight[i] : 0.0f, x[k], o);
    }
#pragma unroll 8
    for (uint32_t i = tid / width + kFirst * every; i < parts; i += every) o = fmaf(weight[i], at[i * step + d], o);
    sums[tid] = o;
    __syncthreads();
    if (tid < D) {
        o = 0.0f;
        for (uint32_t k = 0; k < every; ++k) o += sums[tid + k * width];
        out[tid] = L != 0.0f ? o / L : 0.0f;
    }
}

// A sequence's parts together.
__global__ __launch_bounds__(kJoinThreads) void kv_attention_merge(KvAttn p, Split sp, const float *ws, uint32_t ws_rows)
{
    const KvCall &c = p.call;
    const uint32_t h = blockIdx.y, row = blockIdx.z, D = c.c.head_dim, group = p.heads / c.c.kv_heads;
    Slot sl;
    sl.b = blockIdx.x;
    uint32_t slot = 0;
    if (!find_slot(p, sp, true, slot, sl) || sl.parts < 2) return;
    const kv::Seq seq = kv::sequence(c, sl.b);
    if (row >= seq.n * group) return;
    const uint64_t step = static_cast<uint64_t>(c.c.kv_heads) * ws_rows * (D + 2);
    const float *at = ws + ((static_cast<uint64_t>(slot) * c.c.kv_heads + h) * ws_rows + row) * (D + 2);
    join_parts(at, step, sl.parts, D,
               p.O + kv::rows_base(c, p.o, sl.b, seq) + row / group * p.o.token + (h * group + row % group) * p.o.head);
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of four waves takes 64 RT rows, each wave 16 RT of
// them, and its part of the keys 64 at a time.  The chunk's K codes are copied
// into LDS in operand order, its V codes pass through registers to be turned into
// f16 once for the four waves; both of the next chunk are on their way while
// this one is computed, and one barrier a chunk hands the buffers over.
// Bound by the vector instructions: 64 keys of 32 rows take a wave 112 matrix
// instructions (16 cycles each) and about 490 others (4 cycles, exponentials 16):
// three conversions and sums for a score's digits, ten for a weight and its two
// halves.  Two waves a SIMD fill 70 % of its vector issue and 47 % of its matrix
// cores.  A step has few branches, so that its products and exponentials
// mix: with the rows one after another and conditions inside, 306 us instead of 256.
// 4096 tokens on themselves, causal, 32 heads of 128: 243 us, 566 TFLOP/s (a
// large f16 product of the library, which needs 2 of these 5 matrix
// instructions, 1109); heads of 64 161 us, of 256 (half the heads and tokens) 100 us.
// Workgroups of 8 waves and 256 rows: 254 us and worse where tiles are few.
// ---------------------------------------------------------------------------

struct Tiles {
    uint32_t per_seq;      // tiles a sequence (without seq_start)
    uint32_t count;        // room for tiles a kv head
    uint32_t parts;        // key ranges of a tile at most
    uint32_t per;          // chunks of a range at most
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

// Keys that a row sees; chunks of a tile and the ranges that share them evenly.
__device__ __forceinline__ int keys_of(const KvAttn &p, uint32_t len, uint32_t n, uint32_t row, uint32_t group)
{
    return p.causal ? max(0, static_cast<int>(len) - static_cast<int>(n) + static_cast<int>(row / group) + 1) : static_cast<int>(len);
}
template <uint32_t M>
__device__ __forceinline__ uint32_t tile_chunks(const KvAttn &p, uint32_t len, uint32_t n, uint32_t tile, uint32_t group)
{
    return (static_cast<uint32_t>(keys_of(p, len, n, min(n * group, tile * M + M) - 1, group)) + kChunk - 1) / kChunk;
}
__device__ __forceinline__ uint32_t ranges_of(const Tiles &tl, uint32_t chunks)
{
    return tl.parts == 1 ? 1 : max(1u, (chunks + tl.per - 1) / tl.per);
}

template <int DP, int RT, bool FULL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP * RT <= 128 ? 3 : 2) void kv_attention_tile(KvAttn p, Tiles tl, float *ws)
{
    constexpr int DS = DP / 64, DT = DP / 16;
    constexpr uint32_t M = 16 * RT * WAVES;
    constexpr uint32_t kK = 4 * DS * 1024, kV = DT * 2048, kBuf = kK + kV;   // bytes of a chunk's operands
    extern __shared__ __align__(1024) int8_t lds[];
    const KvCall &c = p.call;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t G = c.c.kv_heads, h = blockIdx.x % G, D = FULL ? DP : c.c.head_dim, ps = c.c.page_size, group = p.heads / G;
    if (blockIdx.x == 0 && blockIdx.y == 0) kv::check_all(c, false, p.max_kv, p.max_tokens);
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
    const uint32_t chunks = tile_chunks<M>(p, len, n, tile, group), ranges = ranges_of(tl, chunks);
    if (blockIdx.y >= ranges) return;
    auto sees = [&](uint32_t row) { return keys_of(p, len, n, row, group); };
    // Keys of the wave; below `least` every row of the wave sees all.
    const int wave_keys = row0 < rows ? sees(min(rows, row0 + 16 * RT) - 1) : 0, least = row0 < rows ? sees(row0) : 0;
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * blockIdx.y / ranges);
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (blockIdx.y + 1) / ranges);

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
    constexpr int VW = (DT + WAVES - 1) / WAVES, KW = (4 * DS + WAVES - 1) / WAVES;   // tiles of V, pieces of K that a wave brings in
    v4i vf[VW];
    float ks = 0.0f, vs = 0.0f;
    // A page's codes, of all heads, are less than 2^32 bytes.
    const uint32_t page_bytes = G * ps * D;
    const int8_t *k_lane = c.c.k + static_cast<uint64_t>(h * ps + (col & 3)) * D, *v_lane = c.c.v + static_cast<uint64_t>(h * D + col) * ps;
    auto fetch = [&](uint32_t chunk, int8_t *buf) {
        const uint32_t in_k = (16 * min(4 * chunk + kb, last16)) & (ps - 1);
        const int8_t *kat = k_lane + (static_cast<uint64_t>(checked(k_id)) * page_bytes + in_k * D);
#pragma unroll
        for (int i = 0; i < KW; ++i) {   // operand (tile t, step s) is piece t * DS + s
            const uint32_t piece = wave + WAVES * i, t = piece / DS, s = piece % DS, d = 64 * s + 16 * g;
            if (4 * DS % WAVES == 0 || piece < 4 * DS) lds::dma16(kat + 4 * t * D + (d < D ? d : 0), buf + piece * 1024);
        }
        const uint32_t in_v = (16 * min(4 * chunk + g, last16)) & (ps - 1), id = checked(v_id);
        const uint64_t unit_v = static_cast<uint64_t>(id) * G + h;
        const int8_t *vat = v_lane + (static_cast<uint64_t>(id) * page_bytes + in_v);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const uint32_t t = wave + WAVES * i;
            vf[i] = *reinterpret_cast<const v4i *>(vat + static_cast<uint64_t>(FULL ? 16 * t : min(16 * t, D - 16)) * ps);
        }
        ks = c.c.ks[unit_v];
        vs = c.c.vs[unit_v];
    };
    auto turn_v = [&](int8_t *buf) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const uint32_t t = wave + WAVES * i;
            if (!FULL && 16 * t >= D) continue;
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
    auto step = [&](uint32_t chunk, auto works, auto masks) {
        constexpr bool WORK = decltype(works)::value, MASK = decltype(masks)::value;
        int8_t *now = lds + ((chunk - begin) & 1) * kBuf, *next = lds + ((chunk - begin + 1) & 1) * kBuf;
        const float k_scale = fmaf(ks, 0.0f, ks), v_scale = vs;   // infinite as NaN: scores of minus infinity are none
        const bool more = chunk + 1 < end;
        if (more) {
            fetch(chunk + 1, next);
            ids(min(chunk + 2, end - 1));
        }
        if constexpr (WORK) {
            // The lane's 16 keys are of one page.  What is multiplied with its scale stays finite
            // whatever U is: a row with a U so far below it has no weight there.
            const float power = __builtin_amdgcn_fmed3f(__builtin_amdgcn_logf(v_scale), -100.0f, 127.0f);
            const float most_shift = 126.0f - fmaxf(power, 0.0f);
            const int first = static_cast<int>(kChunk * chunk + 16 * g);
            v4f f[RT][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                v4i a[RT][3];
#pragma unroll
                for (int s = 0; s < DS; ++s) {
                    const v4i k = *reinterpret_cast<const v4i *>(now + (t * DS + s) * 1024 + lane * 16);
#pragma unroll
                    for (int d = 0; d < 3; ++d)
#pragma unroll
                        for (int r = 0; r < RT; ++r)
                            a[r][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q[r].digit[d][s], s ? a[r][d] : v4i{}, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        f[r][t][i] = fmaf(static_cast<float>(a[r][0][i] * 256 + a[r][1][i]), 256.0f, static_cast<float>(a[r][2][i]));
            }
            float ck[RT], base[RT], top[RT];
            bool move = false;
            uint32_t covered = 0xffffu;   // rows with a product of 2^-12 U or more, or none at all
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                ck[r] = q[r].factor * k_scale;
                top[r] = largest<MASK>(f[r], ck[r], limit[r] - first);   // of the lane's keys
                const float over = top[r] - st[r].m + (power - 14.0f + st[r].shift);   // log2 of the largest product / U
                move = move || top[r] > st[r].m + kAhead || over > 1.0f;
                const uint64_t rows_of = __ballot(over >= -12.0f || (MASK && limit[r] <= static_cast<int>(kChunk * chunk)));
                const uint32_t halves = static_cast<uint32_t>(rows_of | rows_of >> 32);
                covered &= halves | halves >> 16;
            }
            if (__any(move) || covered != 0xffffu) {   // else o is left alone
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float now = fmaxf(st[r].m, groups_max(top[r]));
                    const float alpha = now > st[r].m ? __builtin_amdgcn_exp2f(st[r].m - now) : 1.0f;
                    const float need = groups_max(top[r] + power) - now;
                    // A row without keys or numbers keeps its unit.
                    float to = st[r].shift;
                    // U up: 2^-4 U is the largest now, so that the next ones may be larger; 2 U where it
                    // is far above what came before and above others of its chunk: their last bits count.
                    const bool jump = need > 15.0f + kJump - to;
                    bool far = false;
                    if (__any(jump)) {
                        float least = f[r][0][0];
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) least = fminf(least, f[r][t][i]);
                        far = jump && -groups_max(-fmaf(least, ck[r], power)) - now < need - kFar;
                    }
                    if (need > 15.0f - to) to = (far ? 15.0f : 10.0f) - ceilf(need);
                    const bool low = need < 2.0f - to;
                    if (__any(low)) {
                        float held = 0.0f;
#pragma unroll
                        for (int t = 0; t < DT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) held = fmaxf(held, fabsf(st[r].o[t][i]));
                        const float room = 226.0f - static_cast<float>(__float_as_uint(groups_max(held)) >> 23);
                        if (low) to = fminf(fminf(8.0f - ceilf(fmaxf(need, -200.0f)), to + fmaxf(0.0f, room)), kMostShift);   // 2^-6 U
                    }
                    const float by = ldexpf(alpha, static_cast<int>(to - st[r].shift));
                    st[r].l *= alpha;
                    st[r].l_rest *= alpha;
#pragma unroll
                    for (int t = 0; t < DT; ++t) st[r].o[t] *= by;
                    st[r].m = now;
                    st[r].shift = to;
                }
            }
            float fv[RT], sum[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                sum[r] = 0.0f;
                base[r] = st[r].m == kNegInf ? 0.0f : st[r].m;
                fv[r] = ldexpf(v_scale, static_cast<int>(fminf(st[r].shift, most_shift)));
            }
            // The products of the first half's weights go beside the second half's exponentials.
            v8h hi[RT][2], lo[RT][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int r = 0; r < RT; ++r) weigh<MASK>(sum[r], f[r], k, ck[r], base[r], fv[r], limit[r] - first, hi[r][k], lo[r][k]);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) add_kept(st[r].l, st[r].l_rest, sum[r]);
            if (more) turn_v(next);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    if (!FULL && 16 * t >= static_cast<int>(D)) continue;
                    const v8h v = *reinterpret_cast<const v8h *>(now + kK + (2 * t + k) * 1024 + lane * 16);
#pragma unroll
                    for (int r = 0; r < RT; ++r) st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[r][k], st[r].o[t], 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < RT; ++r) st[r].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[r][k], st[r].o[t], 0, 0, 0);
                }
        } else if (more) {
            turn_v(next);
        }
        lds::wait_vmcnt<0>();
        __syncthreads();
    };
    // Chunks that every row of the wave sees, that some see, that are other waves'.
    const uint32_t all_end = min(max(static_cast<uint32_t>(least) / kChunk, begin), end);
    const uint32_t wave_end = min(max((static_cast<uint32_t>(wave_keys) + kChunk - 1) / kChunk, all_end), end);
    uint32_t chunk = begin;
    for (; chunk < all_end; ++chunk) step(chunk, std::true_type(), std::false_type());
    for (; chunk < wave_end; ++chunk) step(chunk, std::true_type(), std::true_type());
    for (; chunk < end; ++chunk) step(chunk, std::false_type(), std::false_type());

    const bool out_aligned = ((reinterpret_cast<uintptr_t>(p.O) & 15) | (p.o.batch & 3) | (p.o.token & 3) | (p.o.head & 3)) == 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t row = row0 + 16 * r + col;
        const float l = groups_sum(st[r].l + st[r].l_rest);
        const float by = l != 0.0f ? 1.0f / l : 0.0f;
        const int down = -static_cast<int>(st[r].shift);
        auto result = [&](int t) { return v4f{ldexpf(st[r].o[t][0] * by, down), ldexpf(st[r].o[t][1] * by, down), ldexpf(st[r].o[t][2] * by, down), ldexpf(st[r].o[t][3] * by, down)}; };
        if (row >= rows) continue;
        if (ranges == 1) {
            float *at = p.O + kv::rows_base(c, p.o, b, seq) + (row / group) * p.o.token + (h * group + row % group) * p.o.head + 4 * g;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (16 * t >= static_cast<int>(D)) continue;
                const v4f x = result(t);
                if (out_aligned) *reinterpret_cast<v4f *>(at + 16 * t) = x;
                else
                    for (int i = 0; i < 4; ++i) at[16 * t + i] = x[i];
            }
        } else {
            float *at = ws + (((static_cast<uint64_t>(unit) * G + h) * tl.parts + blockIdx.y) * M + (row - tile * M)) * (D + 4);
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t < static_cast<int>(D)) *reinterpret_cast<v4f *>(at + 4 * g + 16 * t) = result(t);
            if (g == 0) {
                at[D] = st[r].m;
                at[D + 1] = l;
            }
        }
    }
}

// A tile's key ranges, at most 64, together: kJoinRows rows a wave, a range's
// weight a lane.  Lanes behind head_dim load its last element: loads under a
// condition are waited for one by one (10.8 us instead of 7.9 for 220 tiles of 64 rows
// and up to 5 ranges).
constexpr int kJoinRows = 2;
template <uint32_t M, int DS>
__global__ __launch_bounds__(256) void kv_attention_join(KvAttn p, Tiles tl, const float *ws)
{
    const KvCall &c = p.call;
    const uint32_t G = c.c.kv_heads, h = blockIdx.x % G, unit = blockIdx.x / G, D = c.c.head_dim, group = p.heads / G;
    uint32_t b, tile, len;
    kv::Seq seq;
    if (!find_tile<M>(p, tl, group, unit, b, tile) || !tile_sequence(p, tl, group, b, seq, len)) return;
    const uint32_t lane = threadIdx.x & 63, in = (blockIdx.y * 4 + (threadIdx.x >> 6)) * kJoinRows, row = tile * M + in;
    if (static_cast<uint64_t>(tile) * M + in >= static_cast<uint64_t>(seq.n) * group) return;
    const uint32_t ranges = __builtin_amdgcn_readfirstlane(ranges_of(tl, tile_chunks<M>(p, len, seq.n, tile, group)));
    if (ranges == 1) return;   // written by the tile itself
    const uint64_t step = static_cast<uint64_t>(M) * (D + 4);
    const float *first = ws + (static_cast<uint64_t>(unit) * G + h) * tl.parts * step;
    const float *at[kJoinRows];
    float m[kJoinRows], l[kJoinRows], weight[kJoinRows], sum[kJoinRows], o[kJoinRows][DS] = {};
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {   // a row behind the last is the last again
        at[k] = first + static_cast<uint64_t>(min(row + k, seq.n * group - 1) - tile * M) * (D + 4);
        m[k] = at[k][min(lane, ranges - 1) * step + D];
        l[k] = at[k][min(lane, ranges - 1) * step + D + 1];
    }
    uint32_t d[DS];
#pragma unroll
    for (int r = 0; r < DS; ++r) d[r] = min(lane + 64 * r, D - 1);
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
        const float top = groups_max(row_max(m[k]));
        weight[k] = lane < ranges ? l[k] * __builtin_amdgcn_exp2f(m[k] - (top == kNegInf ? 0.0f : top)) : 0.0f;
        sum[k] = groups_sum(row_sum(weight[k]));
    }
#pragma unroll 4
    for (uint32_t i = 0; i < ranges; ++i)
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k) {
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight[k]), i));
#pragma unroll
            for (int r = 0; r < DS; ++r) o[k][r] = fmaf(w, at[k][i * step + d[r]], o[k][r]);
        }
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
        const uint32_t to = min(row + k, seq.n * group - 1);
        float *out = p.O + kv::rows_base(c, p.o, b, seq) + (to / group) * p.o.token + (h * group + to % group) * p.o.head;
#pragma unroll
        for (int r = 0; r < DS; ++r)
            if (lane + 64 * r < D) out[lane + 64 * r] = sum[k] != 0.0f ? o[k][r] / sum[k] : 0.0f;
    }
}

// Rows that the kernel of few rows takes: one workgroup's, or two's where all
// sequences' keys together are few.  (20 rows of 8 heads of 128, 3001 keys:
// 1 sequence 17.4 us and 16.7 in tiles, heads of 64 14.3 and 14.7, 12 rows of 256 22.9 and
// 24.0; 4 of 700 to 3001 keys 25.0 and 18.7, 4 of 3001 keys 42.1 and 20.3.)
uint32_t few_rows(const KvAttn &p)
{
    const uint32_t one = p.call.c.head_dim > 128 ? 8 : 16;
    const double keys = (p.call.seq_start ? 0.6 : 1.0) * p.call.batch * p.call.c.kv_heads * p.max_kv;
    return keys <= 32768 ? 2 * one : one;
}

struct Plan {
    bool few = false, tiled = false;   // kernels of the call: sequences of few rows, of many
    Split split{};
    uint32_t slots = 0, rows = 0;   // of the kernel of few rows: slots a kv head, rows a slot at most
    Tiles tiles{};
    uint32_t tile_rows = 0;
    size_t few_ws = 0, ws = 0;
};
Plan plan_of(const KvAttn &p)
{
    Plan r;
    const KvCall &c = p.call;
    const uint32_t G = c.c.kv_heads, group = p.heads / G, D = c.c.head_dim;
    const uint64_t most = static_cast<uint64_t>(p.max_tokens) * group;
    const uint32_t at_most = few_rows(p);
    r.tiled = most > at_most;
    // Without seq_start all sequences have max_tokens.  Beside sequences of many
    // rows the few-row ones have a launch of their own where they may be many;
    // some more tiles cost less than that (6 sequences of 4 heads: 22 us).
    r.few = !r.tiled || (c.seq_start && static_cast<uint64_t>(c.batch) * G >= p.cus / 2);
    if (r.few) {
        r.rows = static_cast<uint32_t>(std::min<uint64_t>(most, at_most));
        // Slots for as many workgroups as run at a time (16 rows take the LDS
        // of a CU), the ragged ends among them.
        const uint32_t tile = D > 128 ? (r.rows <= 4 ? 4 : 8) : r.rows <= 4 ? 4 : r.rows <= 8 ? 8 : 16;
        const uint32_t at_once = (tile == 16 ? 1 : 2) * p.cus / (G * ((r.rows + tile - 1) / tile));
        r.split.target = std::min(std::max(at_once > c.batch ? at_once - c.batch / 2 : at_once / 2, 1u), kMostParts);
        r.split.min_per = 4;
        // A sequence and kv head as one workgroup: 9 us and 1.05 us for each 256
        // keys of the longest, or the codes at 6.4 TB/s; split: 12 us with the join
        // and the codes (8 heads of 128, 4096 keys: 1 sequence 27.9 and 11.1 us, 16 sequences
        // 29.3 and 29.9; 32 heads, 8 sequences 43.0 and 54.8; 8 heads, 16 sequences of 100 to
        // 8000 keys 51.2 and 38.8; 1 sequence of 768 keys 9.6 and 10.9, of 1024 11.1 and 11.0).
        // Sequences are taken to be 0.8 of max_kv long, with seq_start 0.6.  It does not know
        // that more rows and larger heads take longer for a chunk (16 sequences of 4096 keys,
        // 16 rows on 8 heads of 128: 67 whole as it says, 56 split).
        const double mb = (c.seq_start ? 1.2e-6 : 1.6e-6) * c.batch * G * D * p.max_kv;
        r.split.whole = std::max(9.0 + 1.05 * ((p.max_kv + 255) / 256), mb / 6.4) <= 12.0 + mb / 6.4;
        r.split.low_rows = 0;
        r.split.high_rows = at_most;
        // No more slots than parts of the longest: a workgroup without work takes its turn too.
        r.slots = r.split.whole ? c.batch
                                : static_cast<uint32_t>(std::min<uint64_t>(
                                      r.split.target + c.batch,
                                      static_cast<uint64_t>(c.batch) * ((p.max_kv + r.split.min_per * kChunk - 1) / (r.split.min_per * kChunk))));
        if (!r.split.whole) r.few_ws = (static_cast<size_t>(r.slots) * G * r.rows * (D + 2) * sizeof(float) + 15) / 16 * 16;
    }
    r.ws = r.few_ws;
    if (r.tiled) {
        r.tiles.low_rows = r.few ? at_most : 0;
        auto tiles_of = [&](uint32_t rows) {   // of all kv heads
            r.tile_rows = rows;
            r.tiles.per_seq = static_cast<uint32_t>((most + rows - 1) / rows);
            r.tiles.count = c.seq_start ? static_cast<uint32_t>(static_cast<uint64_t>(c.tokens) * group / rows) + c.batch
                                        : r.tiles.per_seq * c.batch;
            return static_cast<uint64_t>(r.tiles.count) * G;
        };
        const uint32_t chunks = (p.max_kv + kChunk - 1) / kChunk;
        // 128 rows share K and V of a chunk where the card has more of such tiles
        // than run at a time (32 heads of 128, causal: 4096 tokens of 8 kv heads
        // 248 us against 254 with 64 rows, 2048 of 32 kv heads 84 and 81), or a few
        // even ones with keys for 16 chunks a range (512 tokens of 4096, 8 kv heads: 76 us
        // against 79; a ragged batch of 1 to 331 tokens, 4 kv heads of 80, 43 against 35).
        uint64_t grid = D <= 128 ? tiles_of(128) : 0;
        if (grid <= 2 * p.cus && (c.seq_start || grid >= p.cus || grid * (chunks / 16) < 2 * p.cus)) grid = tiles_of(64);
        // Key ranges of 4 chunks at least for a workgroup a CU, of 8 for as many as
        // run at a time (32 tiles, 47 chunks: 8 ranges 20.5 us, 5 24.2, 10 22.1; 64 chunks: 8
        // ranges 23.7 us, 5 28.8, 10 26.2).  Where sequences differ the shorter have fewer.
        const uint64_t at_once = (D > 128 ? 1 : r.tile_rows == 128 ? 2 : 3) * p.cus;
        const uint64_t parts = std::max(std::min<uint64_t>(p.cus / grid, chunks / 4),
                                        std::min<uint64_t>(at_once * (c.seq_start ? 5 : 3) / (3 * grid), chunks / (c.seq_start ? 5 : 8)));
        r.tiles.parts = static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(parts, 1), 64));
        r.tiles.per = (chunks + r.tiles.parts - 1) / r.tiles.parts;
        if (r.tiles.parts > 1) r.ws += static_cast<size_t>(grid) * r.tiles.parts * r.tile_rows * (D + 4) * sizeof(float);
    }
    return r;
}

template <int DP, int RT>
void launch_few(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    constexpr int W = DP > 128 ? 2 : 4;
    constexpr uint32_t bytes = few_lds<DP, RT, W>();
    const bool full = p.call.c.head_dim == DP;
    const auto kernel = full ? kv_attention_few<DP, RT, true, W> : kv_attention_few<DP, RT, false, W>;
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const uint32_t tiles = (pl.rows + 4 * RT - 1) / (4 * RT);
    kernel<<<dim3(pl.slots, p.call.c.kv_heads, tiles), 64 * W, bytes, s>>>(p, pl.split, ws, pl.rows);
}
template <int DP, int RT, int WAVES>
void launch_tile(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    constexpr uint32_t bytes = 2 * (4 * (DP / 64) * 1024 + (DP / 16) * 2048);
    const auto kernel = p.call.c.head_dim == DP ? kv_attention_tile<DP, RT, true, WAVES> : kv_attention_tile<DP, RT, false, WAVES>;
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const uint32_t grid = pl.tiles.count * p.call.c.kv_heads;
    kernel<<<dim3(grid, pl.tiles.parts), 64 * WAVES, bytes, s>>>(p, pl.tiles, ws);
    if (pl.tiles.parts > 1) kv_attention_join<16 * RT * WAVES, DP / 64><<<dim3(grid, 4 * RT * WAVES / kJoinRows), 256, 0, s>>>(p, pl.tiles, ws);
}
template <int DP>
void launch(hipStream_t s, const KvAttn &p, const Plan &pl, float *ws)
{
    if (pl.few) {
        if (pl.rows <= 4) launch_few<DP, 1>(s, p, pl, ws);
        else if (DP > 128 || pl.rows <= 8) launch_few<DP, 2>(s, p, pl, ws);
        else if constexpr (DP <= 128) launch_few<DP, 4>(s, p, pl, ws);
        if (pl.few_ws)
            kv_attention_merge<<<dim3(p.call.batch, p.call.c.kv_heads, pl.rows), kJoinThreads, 0, s>>>(p, pl.split, ws, pl.rows);
    }
    if (pl.tiled) {
        float *rest = ws + pl.few_ws / sizeof(float);
        if (DP > 128 || pl.tile_rows == 64) launch_tile<DP, 1, 4>(s, p, pl, rest);
        else if constexpr (DP <= 128) launch_tile<DP, 2, 4>(s, p, pl, rest);
    }
}

}  // namespace

std::string kv_attention_route(const KvAttn &p)
{
    const Plan pl = plan_of(p);
    char text[96];
    std::snprintf(text, sizeof(text), "few=%u rows=%u tile=%u parts=%u", pl.few ? pl.slots : 0, pl.rows,
                  pl.tile_rows, pl.tiles.parts);
    return text;
}

// A grid's work-items count in 32 bits.
bool kv_attention_fits(const KvAttn &p)
{
    const Plan pl = plan_of(p);
    return static_cast<uint64_t>(pl.slots) * 256 < (1ull << 32) &&
           static_cast<uint64_t>(p.call.batch) * kJoinThreads < (1ull << 32) &&
           static_cast<uint64_t>(pl.tiles.count) * p.call.c.kv_heads * 256 < (1ull << 32);
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
