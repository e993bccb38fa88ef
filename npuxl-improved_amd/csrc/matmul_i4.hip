// matmul_i4.hip - MATMUL_I4: f32 rows times 4-bit weights with group scales, on
// gfx950.
//
//   C[m][n] = epi(sum_g scale[g][n] * sum_{k in g} A[m][k] (code[k][n] - zero[g][n]) + bias[n])
//
// code - zero is a whole number from -15 to 15 and exact in int8 and f16; what has to be
// split is A.  Three kernels: whole numbers of 31 bits for up to 8 rows (bound by the
// codes' bytes: few instructions a code), two f16 halves of a row's 128 of K for tens of rows (bound by
// unpacking), two f16 halves split beforehand for more (bound by the matrix cores).  Sums are
// exact or f32, and each group's is scaled once.  estimate() chooses.
//
// Weights in device memory, strips of 16 columns and blocks of 128 of K:
//   codes  [Np/16][KB][64][16]: byte j of lane (kg, c) holds k = 128 kb + 32 (j / 8)
//          + 8 kg + j % 8 in its lower half and k + 64 in its upper, so that a lane's
//          16 bytes and two masks are its operands of two products; 1 KiB a block, a
//          strip's blocks in a row.
//   scales [Np/16][groups][16] f32, zeros the same in bytes; padding 0.
#include "device_math.hpp"
#include "kernels.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <type_traits>

namespace vnpu {
namespace k {
namespace {

using v4i = int __attribute__((ext_vector_type(4)));
using v4f = float __attribute__((ext_vector_type(4)));
using v2h = _Float16 __attribute__((ext_vector_type(2)));
using v8h = _Float16 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(256) void pack_codes(const uint8_t *B, uint32_t K, uint32_t N, uint32_t ldb, uint32_t trans_b,
                                                  uint8_t *codes, uint32_t KB, uint64_t pieces)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= pieces) return;
    const uint32_t lane = at & 63, c = lane & 15, kg = lane >> 4;
    const uint64_t block = at >> 6;
    const uint32_t kb = static_cast<uint32_t>(block % KB), n = static_cast<uint32_t>(block / KB) * 16 + c;
    auto code = [&](uint32_t k) -> uint32_t {
        if (k >= K || n >= N) return 0;
        const uint32_t row = trans_b ? n : k, col = trans_b ? k : n;
        return (B[static_cast<uint64_t>(row) * ldb + col / 2] >> (4 * (col & 1))) & 15;
    };
    uint32_t w[4] = {};
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) {
        const uint32_t k = 128 * kb + 32 * (j / 8) + 8 * kg + j % 8;
        w[j / 4] |= (code(k) | code(k + 64) << 4) << (8 * (j % 4));
    }
    reinterpret_cast<uint4 *>(codes)[at] = make_uint4(w[0], w[1], w[2], w[3]);
}

// groups of the caller's, slots of a strip in the packed arrays.
__global__ __launch_bounds__(256) void pack_scales(const float *scales, const uint8_t *zeros, uint32_t groups, uint32_t slots,
                                                   uint32_t N, float *to, uint8_t *to_zeros, uint64_t count, uint32_t *bad)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= count) return;
    const uint64_t row = at >> 4;
    const uint32_t g = static_cast<uint32_t>(row % slots), n = static_cast<uint32_t>(row / slots) * 16 + (at & 15);
    const bool in = g < groups && n < N;
    to[at] = in ? scales[static_cast<uint64_t>(g) * N + n] : 0.0f;
    if (!zeros) return;
    const uint8_t z = in ? zeros[static_cast<uint64_t>(g) * N + n] : 0;
    if (z > 15) *bad = 1;
    to_zeros[at] = z;
}

// ---------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------

// A function's relative error is its argument's absolute one: GELU's arguments, 88 and 10 in size where results are still
// normal numbers, are worked out in 64 bits and go in as f32 and what that leaves.  The tiles' kernels have this once
// for each of 64 elements, so it is kept short (with an exponential and a division more, 2048 x 4096 x 11008 took 358 us
// instead of 341 without any epilogue).
__device__ __forceinline__ float finished(float x, uint32_t epilogue)
{
    if (epilogue == 0) return x;
    if (epilogue == 1) return x > 0.0f ? x : x != x ? x : 0.0f;
    if (__builtin_expect(epilogue != 4, 1)) {
        // x / (1 + exp(-u)); u = x, or sqrt(8 / pi) (x + 0.044715 x^3): 1 + tanh(u / 2) = 2 / (1 + exp(-u)).  exp(-|u|) ends in
        // 0 and not in infinity.
        float top = -fabsf(x), rest = 0.0f;
        if (__builtin_expect(epilogue == 3, 0)) {
            const double y = x, u = fmax(-fabs(y) * fma(0.07135481627260025 * y, y, 1.5957691216057308), -200.0);
            top = static_cast<float>(u);
            rest = static_cast<float>(u - top);
        }
        const float e = expf(top), down = fmaf(e, rest, e);
        return (x < 0.0f ? x * down : x) / (1.0f + down);
    }
    // erfc' = -2 / sqrt(pi) exp(-y^2)
    const double u = -0.70710678118654752440 * x;
    const float y = static_cast<float>(u), rest = fabsf(y) < 16.0f ? static_cast<float>(u - y) : 0.0f;
    return 0.5f * x * fmaf(-1.12837917f * rest, __builtin_amdgcn_exp2f(-1.44269504f * y * y), erfcf(y));
}

// ---------------------------------------------------------------------------
// Few rows: bound by the codes.  128 of a row of A become whole numbers of up to 31 bits
// in a unit of their own (a power of two), four balanced base-256 digits each, and
// codes are 0 to 15 as they stand, so that a group's sums run on the int8 matrix cores without a
// rounding.  The 16 operand rows of v_mfma_i32_16x16x64_i8 are 4 rows of A times 4 digits: one
// product gives a lane the four digit sums of one result.  Zeros enter as the product's
// first summand, -zero * (sum of the digits), which a product with ones gives.
//
// 1 x 4096 x 4096 4.5 us (a launch; the codes are 1.7 us of a copy), 1 x 4096 x 32000, groups of
// 128, zeros 13.2 us with three sets of weights in turn, which the last cache holds, and 13.9 with twelve, which it does not:
// 5.1 TB/s; 8 x 11008 x 4096, groups of 64, 12.5 us with the join, vector instructions in 57% of the SIMD cycles
// (A's digits, made again in each of 64 workgroups) and 3 us of start.  Blocks asked for two ahead instead of one: no
// gain.
// ---------------------------------------------------------------------------

// Largest over the 4 groups of 16 lanes; NaN is above all.
__device__ __forceinline__ float groups_largest(float x)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// And over 4 lanes side by side: the lanes of a row of A.
__device__ __forceinline__ float row_largest(float x)
{
    auto dpp = [](float y, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    x = __builtin_elementwise_maximum(x, dpp(x, std::integral_constant<int, 0xB1>()));
    return groups_largest(__builtin_elementwise_maximum(x, dpp(x, std::integral_constant<int, 0x4E>())));
}
// Biased exponent e: x * 2^(157 - e) of an x no larger than these bits fits four balanced digits,
// 127 * (2^24 + 2^16 + 2^8 + 1) = 2139062143 = 2^30 (2 - 65793 / 2^23), 0x10400 is 66560.
// From 31 up, so that 2^(e - 157) is a normal number.
__device__ __forceinline__ uint32_t digits_exponent(uint32_t bits) { return max((bits + 0x10400u) >> 23, 31u); }

// Bytes i of four words in word i.
__device__ __forceinline__ void planes_of(const uint32_t u[4], uint32_t p[4])
{
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), d = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
    p[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    p[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    p[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    p[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}
// Sum of four digit sums, digit i counting 256^i.
__device__ __forceinline__ float digits_sum(const v4i &a)
{
    return fmaf(static_cast<float>(a[3] * 256 + a[2]), 65536.0f, static_cast<float>(a[1] * 256 + a[0]));
}

constexpr int kBufferWord3 = 0x00020000;   // raw buffer, 32-bit data format
constexpr uint32_t kOut = 0x80000000u;      // an offset past any buffer

// Buffers over a workgroup's T strips and blocks begin .. end: what is behind them is zero.  A load's whole offset is in the
// lanes' operand, which the range check covers; a scalar operand's part it would not.
template <int T, int GB>
struct Weights {
    v4i codes[T];
    float scale[T][GB];
    uint32_t zero[T][GB];
};
template <int T, int GB, bool ZEROS>
struct Strips {
    __amdgpu_buffer_rsrc_t codes[T], scales[T], zeros[T];
    uint32_t slot0, begin, factor, shift;
    __device__ __forceinline__ Strips(const I4Gemm &p, uint32_t strip0, uint32_t first, uint32_t end)
    {
        begin = first;
        factor = p.group_factor;
        shift = p.group_shift;
        slot0 = slot(begin);
        const uint32_t strips = p.Np / 16, slots = GB > 1 ? GB * (end - begin) : slot(end - 1) + 1 - slot0;
        uint8_t *c = const_cast<uint8_t *>(p.codes) + (static_cast<uint64_t>(strip0) * p.KB + begin) * 1024;
        const uint64_t at = (static_cast<uint64_t>(strip0) * p.slots + slot0) * 16;
        float *s = const_cast<float *>(p.scales) + at;
        uint8_t *z = const_cast<uint8_t *>(p.zeros) + at;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const bool in = strip0 + t < strips;
            codes[t] = __builtin_amdgcn_make_buffer_rsrc(c + static_cast<uint64_t>(t) * p.KB * 1024, 0, in ? (end - begin) * 1024 : 0, kBufferWord3);
            scales[t] = __builtin_amdgcn_make_buffer_rsrc(s + static_cast<uint64_t>(t) * p.slots * 16, 0, in ? slots * 64 : 0, kBufferWord3);
            if (ZEROS) zeros[t] = __builtin_amdgcn_make_buffer_rsrc(z + static_cast<uint64_t>(t) * p.slots * 16, 0, in ? slots * 16 : 0, kBufferWord3);
        }
    }
    // kb / blocks_of_group without the division's 15 scalar instructions, and without a condition for groups of one block: that
    // becomes a branch, and where one lies between a product and its first use the compiler has counted the longer of
    // the two ways alone for the wait that the result needs.
    __device__ __forceinline__ uint32_t slot(uint32_t kb) const { return GB > 1 ? GB * kb : __umulhi(kb << 9, factor) >> shift; }
    // Block begin + at.
    __device__ __forceinline__ void load(Weights<T, GB> &w, uint32_t at) const
    {
        const uint32_t lane = threadIdx.x & 63, from = (slot(begin + at) - slot0) * 16 + (lane & 15);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            w.codes[t] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(codes[t], at * 1024 + lane * 16, 0, 2));   // nontemporal
#pragma unroll
            for (int g = 0; g < GB; ++g) {
                w.scale[t][g] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(scales[t], (from + 16 * g) * 4, 0, 0));
                w.zero[t][g] = ZEROS ? __builtin_amdgcn_raw_buffer_load_b8(zeros[t], from + 16 * g, 0, 0) : 8;
            }
        }
    }
};

// A workgroup has T strips, 4 RQ rows and a range of the blocks of 128 of K, its waves every
// W-th block of that.  GB: groups of a block (4, 2, or 1 where a group is
// a block or more).  Every load is a buffer's, whose range check gives zeros behind
// the range, the last row and K without a branch.
template <int RQ, int T, int W, int GB, bool ZEROS>
__global__ __launch_bounds__(64 * W) void matmul_i4_few(I4Gemm p, uint32_t per, float *part)
{
    extern __shared__ __align__(16) int8_t lds[];
    const uint32_t lane = threadIdx.x & 63, m = (lane & 15) >> 2, d = lane & 3, kg = lane >> 4, c = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t strip0 = blockIdx.x * T, row0 = blockIdx.y * 4 * RQ, strips = p.Np / 16;
    const uint32_t begin = blockIdx.z * per, end = min(begin + per, p.KB);
    int8_t *mine = lds + wave * 2048;
    const Strips<T, GB, ZEROS> strip(p, strip0, begin, end);
    const uint32_t rows = min(p.M - row0, 4u * RQ), last = min(p.K, 128 * end);
    const auto a = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p.A) + static_cast<uint64_t>(row0) * p.lda, 0,
                                                     ((rows - 1) * p.lda + p.K) * 4, kBufferWord3);
    struct Block {
        Weights<T, GB> w;
        v4f x[RQ][2];
    };
    auto load_rows = [&](Block &b, uint32_t i, int q) {   // of the wave's i-th block
        const uint32_t k = 128 * (begin + wave + W * i) + 32 * d + 8 * kg;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bool in = 4 * q + m < rows && k + 4 * j < last;
            b.x[q][j] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(a, in ? ((4 * q + m) * p.lda + k + 4 * j) * 4 : kOut, 0, 0));
        }
    };

    float acc[RQ][T] = {};   // row 4 q + kg, column c
    auto of_row_kg = [&](float x) {   // as lane 4 kg has it
        return __int_as_float(__builtin_amdgcn_ds_bpermute(static_cast<int>(16 * kg), __float_as_int(x)));
    };
    auto work = [&](Block &b, uint32_t i) {
        v4i low[T], high[T];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                low[t][j] = b.w.codes[t][j] & 0x0f0f0f0f;
                high[t][j] = (b.w.codes[t][j] >> 4) & 0x0f0f0f0f;
            }
        const uint32_t kb = begin + wave + W * i;
#pragma unroll
        for (int q = 0; q < RQ; ++q) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = b.x[q][j / 4][j % 4];
            if (128 * kb + 128 > p.K) {   // four that begin before K may end behind it
                const uint32_t k = 128 * kb + 32 * d + 8 * kg;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = k + j < p.K ? x[j] : 0.0f;
            }
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = __builtin_elementwise_maximum(most, fabsf(x[j]));
            most = row_largest(most);
            // Below 2^-96 the unit would not be a normal number: 2^96 times as large, and back at the end.
            const bool tiny = __float_as_uint(most) - 1u < 0x0f800000u - 1u, rare = __any(tiny);
            float down = 1.0f;
            if (rare) {
                const float by = tiny ? 7.922816251426434e28f : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= by;
                most *= by;
                down = of_row_kg(tiny ? 1.262177448353619e-29f : 1.0f);
            }
            const uint32_t e = digits_exponent(__float_as_uint(most));
            const float up = __uint_as_float((284u - e) << 23);
            uint32_t u[8], plane[2][4];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                u[j] = (static_cast<uint32_t>(static_cast<int>(rintf(x[j] * up))) + 0x80808080u) ^ 0x80808080u;   // bytes: balanced digits
            planes_of(u, plane[0]);
            planes_of(u + 4, plane[1]);
            // Lane (m, d, kg) has 8 of K and all digits; as an operand it wants digit d of 32 of K.
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint2 *>(mine + ((m * 4 + j) * 4 + kg) * 32 + d * 8) = make_uint2(plane[0][j], plane[1][j]);
            __builtin_amdgcn_wave_barrier();
            load_rows(b, i + 1, q);   // before the products and the next weights: its digits are made while those come
            __builtin_amdgcn_sched_barrier(0x86);   // no product or load passes
            const v4i a0 = *reinterpret_cast<const v4i *>(mine + (c * 4 + kg) * 32), a1 = *reinterpret_cast<const v4i *>(mine + (c * 4 + kg) * 32 + 16);
            __builtin_amdgcn_wave_barrier();
            const float unit = of_row_kg(__float_as_uint(most) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((e - 30u) << 23));
            // Less the digits' sum, times the zero: 8 where there are none.
            const int less = ZEROS ? -1 : static_cast<int>(0xf8f8f8f8u);
            const v4i minus = {less, less, less, less}, none = {0, 0, 0, 0};
            auto product = [&](const v4i &x, const v4i &y, const v4i &s) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, s, 0, 0, 0); };
            auto half = [&](const v4i &x, const v4i &y, int j, const v4i &s) {
                const long xs = static_cast<long>(static_cast<uint32_t>(x[2 * j])) | static_cast<long>(x[2 * j + 1]) << 32;
                const long ys = static_cast<long>(static_cast<uint32_t>(y[2 * j])) | static_cast<long>(y[2 * j + 1]) << 32;
                return __builtin_amdgcn_mfma_i32_16x16x32_i8(xs, ys, s, 0, 0, 0);
            };
            auto first = [&](const v4i &sums, uint32_t zero) {
                v4i r = sums;
                if (ZEROS)
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[j] = __mul24(sums[j], static_cast<int>(zero));
                return r;
            };
            v4i sums[GB];
            if constexpr (GB == 1) {
                sums[0] = product(a1, minus, product(a0, minus, none));
            } else if constexpr (GB == 2) {
                sums[0] = product(a0, minus, none);
                sums[1] = product(a1, minus, none);
            } else {
                sums[0] = half(a0, minus, 0, none);
                sums[1] = half(a0, minus, 1, none);
                sums[2] = half(a1, minus, 0, none);
                sums[3] = half(a1, minus, 1, none);
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                v4i r[GB];
                if constexpr (GB == 1) {
                    r[0] = product(a1, high[t], product(a0, low[t], first(sums[0], b.w.zero[t][0])));
                } else if constexpr (GB == 2) {
                    r[0] = product(a0, low[t], first(sums[0], b.w.zero[t][0]));
                    r[1] = product(a1, high[t], first(sums[1], b.w.zero[t][1]));
                } else {
                    r[0] = half(a0, low[t], 0, first(sums[0], b.w.zero[t][0]));
                    r[1] = half(a0, low[t], 1, first(sums[1], b.w.zero[t][1]));
                    r[2] = half(a1, high[t], 0, first(sums[2], b.w.zero[t][2]));
                    r[3] = half(a1, high[t], 1, first(sums[3], b.w.zero[t][3]));
                }
#pragma unroll
                for (int g = 0; g < GB; ++g) {
                    float x = digits_sum(r[g]) * b.w.scale[t][g];   // the unit last: its product with a scale may be denormal
                    if (rare) x *= down;
                    acc[q][t] = fmaf(x, unit, acc[q][t]);
                }
            }
        }
    };
    Block block;
#pragma unroll
    for (int q = 0; q < RQ; ++q) load_rows(block, 0, q);
    __builtin_amdgcn_sched_barrier(0);
    strip.load(block.w, wave);
    for (uint32_t i = 0; wave + W * i < end - begin; ++i) {
        work(block, i);
        strip.load(block.w, wave + W * (i + 1));
    }
    // The waves' sums together, in the waves' order.
    __syncthreads();
    float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int q = 0; q < RQ; ++q)
#pragma unroll
        for (int t = 0; t < T; ++t) sums[(wave * RQ * T + q * T + t) * 64 + lane] = acc[q][t];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < RQ * T * 64; e += 64 * W) {
        const uint32_t q = e / (T * 64), row = row0 + 4 * q + (e >> 4 & 3), n = (strip0 + e / 64 % T) * 16 + (e & 15);
        if (row >= p.M || n >= p.N) continue;
        float x = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) x += sums[w * RQ * T * 64 + e];
        if (part) {
            part[(static_cast<uint64_t>(blockIdx.z) * p.M + row) * p.N + n] = x;
        } else {
            if (p.bias) x += p.bias[n];
            p.C[static_cast<uint64_t>(row) * p.ldc + n] = finished(x, p.epilogue);
        }
    }
}

// part: where the sums of ranges of K go, null if there is one range.
template <int RQ, int T, int W, int GB>
void launch_few(hipStream_t s, const I4Gemm &p, float *part)
{
    const dim3 grid((p.Np / 16 + T - 1) / T, (p.M + 4 * RQ - 1) / (4 * RQ), p.splits);
    constexpr uint32_t bytes = W * (RQ * T > 8 ? RQ * T * 256 : 2048);
    const auto kernel = p.zeros ? matmul_i4_few<RQ, T, W, GB, true> : matmul_i4_few<RQ, T, W, GB, false>;
    kernel<<<grid, 64 * W, bytes, s>>>(p, p.per, part);
}
template <int RQ, int T, int W>
void launch_few(hipStream_t s, const I4Gemm &p, float *part)
{
    if (p.groups_of_block == 4) launch_few<RQ, T, W, 4>(s, p, part);
    else if (p.groups_of_block == 2) launch_few<RQ, T, W, 2>(s, p, part);
    else launch_few<RQ, T, W, 1>(s, p, part);
}

// ---------------------------------------------------------------------------
// Tens of rows: a row's 128 of K times a power of two, so that their largest is below
// 2^15, are hi + lo, two f16 (22 bits, and 2^-25 where those end); code - zero is exact in
// f16, and v_mfma_f32_16x16x32_f16 sums the products with each part in f32.  A lane has
// the f32 values that it needs as operands, so nothing goes through LDS, and 16 rows take
// one product where whole numbers of 4 digits take four.  Vector instructions bound it, 38 a
// strip and block to unpack and 130 for 16 rows' halves, made again for each T strips: 16 x 4096 x 11008
// 13.4 us, 32 rows 24.0, 64 x 4096 x 4096 14.2.
// ---------------------------------------------------------------------------

// Place in 8 of K of a fragment's element e: the order in which codes come out of a word.
__device__ __forceinline__ constexpr uint32_t order(uint32_t e) { return (e & 4) | (e & 1) << 1 | (e >> 1 & 1); }

// Codes of 32 of K: words w of a strip's block, their lower or upper halves, less zero.  A code set under the exponent of
// 1024 is 1024 + code, a published way that f16's format gives.  The mask
// and the exponent bits are in registers: as literals they would take an instruction each.
struct Masks {
    uint32_t low, high, bits;
    __device__ __forceinline__ Masks()
    {
        asm("s_mov_b32 %0, 0x000f000f" : "=s"(low));
        asm("s_mov_b32 %0, 0x00f000f0" : "=s"(high));
        asm("v_mov_b32 %0, 0x64006400" : "=v"(bits));
    }
};
template <bool HIGH>
__device__ __forceinline__ v8h differences(const Masks &m, uint32_t w0, uint32_t w1, v2h zero)
{
    auto two = [&](uint32_t w) {
        if constexpr (HIGH) {   // 1024 + 16 code
            const v2h x = __builtin_bit_cast(v2h, (w & m.high) | m.bits), sixteenth = {0.0625f16, 0.0625f16};
            return __builtin_elementwise_fma(x, sixteenth, v2h{960.0f16, 960.0f16} - zero);
        } else {
            return __builtin_bit_cast(v2h, (w & m.low) | m.bits) - zero;
        }
    };
    const v2h a = two(w0), b = two(w0 >> 8), c = two(w1), d = two(w1 >> 8);
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

using v2f = float __attribute__((ext_vector_type(2)));

// A workgroup has T strips, 16 RT rows and a range of the blocks of K, its waves every W-th.
template <int RT, int T, int W, int GB, bool ZEROS>
__global__ __launch_bounds__(64 * W) void matmul_i4_mid(I4Gemm p, uint32_t per, float *part)
{
    extern __shared__ __align__(16) int8_t lds[];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t strip0 = blockIdx.x * T, row0 = blockIdx.y * 16 * RT;
    const uint32_t begin = blockIdx.z * per, end = min(begin + per, p.KB);
    const Strips<T, GB, ZEROS> strip(p, strip0, begin, end);
    const uint32_t rows = min(p.M - row0, 16u * RT), last = min(p.K, 128 * end);
    const auto a = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p.A) + static_cast<uint64_t>(row0) * p.lda, 0,
                                                     ((rows - 1) * p.lda + p.K) * 4, kBufferWord3);
    const Masks masks;
    struct Block {
        Weights<T, GB> w;
        v4f x[RT][4][2];
    };
    auto load = [&](Block &b, uint32_t i) {
        const uint32_t at = wave + W * i, k = 128 * (begin + at) + 8 * g;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool in = 16 * r + c < rows && k + 32 * h + 4 * j < last;
                    b.x[r][h][j] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(a, in ? ((16 * r + c) * p.lda + k + 32 * h + 4 * j) * 4 : kOut, 0, 0));
                }
        if (GB == 1) __builtin_amdgcn_sched_barrier(0);   // A's first: its halves are made while the weights come
        strip.load(b.w, at);
    };
    v4f total[RT][T];   // rows 16 r + 4 g + i, column c
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) total[r][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    auto work = [&](const Block &b, uint32_t i) {
        const uint32_t kb = begin + wave + W * i;
        v8h hi[RT][4], lo[RT][4];
        float unit[RT][4], down[RT][4];
        bool rare = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = b.x[r][j / 8][j / 4 % 2][j % 4];
            if (128 * kb + 128 > p.K) {   // four that begin before K may end behind it
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = 128 * kb + 32 * (j / 8) + 8 * g + j % 8 < p.K ? x[j] : 0.0f;
            }
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) most = __builtin_elementwise_maximum(most, fabsf(x[j]));
            most = groups_largest(most);
            // As for few rows.
            const bool tiny = __float_as_uint(most) - 1u < 0x0f800000u - 1u;
            if (__any(tiny)) {
                const float by = tiny ? 7.922816251426434e28f : 1.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] *= by;
                most *= by;
                rare = true;
            }
            const uint32_t e = max(__float_as_uint(most) >> 23, 31u);
            const float up = __uint_as_float((268u - min(e, 254u)) << 23);   // 2^(141 - e)
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const v2f y = {x[8 * h + order(j)] * up, x[8 * h + order(j + 1)] * up};
                    const v2h top = __builtin_convertvector(y, v2h), rest = __builtin_convertvector(y - __builtin_convertvector(top, v2f), v2h);
                    hi[r][h][j] = top[0];
                    hi[r][h][j + 1] = top[1];
                    lo[r][h][j] = rest[0];
                    lo[r][h][j + 1] = rest[1];
                }
            // Of rows 4 g + i: lane 4 g + i has row 4 g + i.
            const float own = __float_as_uint(most) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((e - 14u) << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int from = static_cast<int>(4 * (4 * g + j));
                unit[r][j] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(own)));
                down[r][j] = rare ? __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(tiny ? 1.262177448353619e-29f : 1.0f))) : 1.0f;
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            v4f acc[RT], sum[RT];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                constexpr int of = 4 / GB;   // of 32 of K in a group
                const _Float16 z = __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x6400 + b.w.zero[t][h / of]));   // 1024 + zero
                const uint32_t w0 = static_cast<uint32_t>(b.w.codes[t][2 * (h & 1)]), w1 = static_cast<uint32_t>(b.w.codes[t][2 * (h & 1) + 1]);
                const v8h w = h < 2 ? differences<false>(masks, w0, w1, v2h{z, z}) : differences<true>(masks, w0, w1, v2h{z, z});
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[r][h], w, h % of ? acc[r] : v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[r][h], w, acc[r], 0, 0, 0);
                if (h % of == of - 1)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[r][j] = h == of - 1 ? acc[r][j] * b.w.scale[t][0] : fmaf(acc[r][j], b.w.scale[t][h / of], sum[r][j]);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (rare) sum[r][j] *= down[r][j];
                    total[r][t][j] = fmaf(sum[r][j], unit[r][j], total[r][t][j]);
                }
        }
    };
    Block block;
    load(block, 0);
    for (uint32_t i = 0; wave + W * i < end - begin; ++i) {
        work(block, i);
        load(block, i + 1);
    }
    // The waves' sums together, in the waves' order.
    v4f *sums = reinterpret_cast<v4f *>(lds);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sums[((wave * RT + r) * T + t) * 64 + lane] = total[r][t];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < RT * T * 64; e += 64 * W) {
        const uint32_t n = (strip0 + e / 64 % T) * 16 + (e & 15), row = row0 + 16 * (e / (64 * T)) + 4 * (e >> 4 & 3);
        if (n >= p.N) continue;
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) x += sums[w * RT * T * 64 + e];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (row + j >= p.M) continue;
            if (part) {
                part[(static_cast<uint64_t>(blockIdx.z) * p.M + row + j) * p.N + n] = x[j];
            } else {
                float y = x[j];
                if (p.bias) y += p.bias[n];
                p.C[static_cast<uint64_t>(row + j) * p.ldc + n] = finished(y, p.epilogue);
            }
        }
    }
}

template <int RT, int T, int W, int GB>
void launch_mid(hipStream_t s, const I4Gemm &p, float *part)
{
    const dim3 grid((p.Np / 16 + T - 1) / T, (p.M + 16 * RT - 1) / (16 * RT), p.splits);
    constexpr uint32_t bytes = W * RT * T * 1024;
    const auto kernel = p.zeros ? matmul_i4_mid<RT, T, W, GB, true> : matmul_i4_mid<RT, T, W, GB, false>;
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    kernel<<<grid, 64 * W, bytes, s>>>(p, p.per, part);
}
template <int RT, int T, int W>
void launch_mid(hipStream_t s, const I4Gemm &p, float *part)
{
    if (p.groups_of_block == 4) launch_mid<RT, T, W, 4>(s, p, part);
    else if (p.groups_of_block == 2) launch_mid<RT, T, W, 2>(s, p, part);
    else launch_mid<RT, T, W, 1>(s, p, part);
}

// ---------------------------------------------------------------------------
// Many rows: bound by the matrix cores.  A row of A times a power of two, so that its
// largest is below 2^15, is hi + lo, two f16 (22 bits, and 2^-25 where those end);
// code - zero is exact in f16, a product with each part sums in f32, and a group's sum
// is scaled into the result's.  A kernel splits A into fragments, operands of
// v_mfma_f32_16x16x32_f16 as they are read: [row tile of 16][32 of K][hi, lo][64
// lanes][8], lane (kg, row), element e the K of place order(e) among its 8.
//
// 2048 x 4096 x 11008, groups of 128: 337 to 358 us as the card's clock goes, 530 TFLOP/s of the result's, 1.06 PFLOP/s of
// products (a large f16 product of the library 1.16), the split 19 of them; in groups of 32, which take four times as many
// scalings, 422.  A tile's wave has its strips' codes alone and shares the rows' fragments through LDS.  Its matrix cores are
// busy in 56% of the cycles, its vector issue in 43%; 2.7 tiles for each that runs at a time are 3 rounds.
// ---------------------------------------------------------------------------

// A workgroup has 16 rows and a part of their blocks; it looks for the rows' largest
// itself, in all of K.
constexpr uint32_t kSplitThreads = 1024;
template <bool ALIGNED>
__global__ __launch_bounds__(kSplitThreads) void matmul_i4_split(I4Gemm p, uint32_t row0, int8_t *frags, float *down)
{
    __shared__ uint32_t largest[16];
    const uint32_t tid = threadIdx.x, tile = blockIdx.x;
    if (tid < 16) largest[tid] = 0;
    __syncthreads();
    {
        const uint32_t r = tid / (kSplitThreads / 16), at = tid % (kSplitThreads / 16);
        const float *row = p.A + static_cast<uint64_t>(min(row0 + tile * 16 + r, p.M - 1)) * p.lda;
        uint32_t most = 0;
        if constexpr (ALIGNED) {
#pragma unroll 8
            for (uint32_t k = 4 * at; k < p.K; k += kSplitThreads / 4) {
                const v4f x = *reinterpret_cast<const v4f *>(row + k);
#pragma unroll
                for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
            }
        } else {
#pragma unroll 8
            for (uint32_t k = at; k < p.K; k += kSplitThreads / 16) most = max(most, __float_as_uint(row[k]) & 0x7fffffffu);
        }
        for (int o = kSplitThreads / 32; o; o >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o)));
        if (at == 0) largest[r] = most;
    }
    __syncthreads();
    const uint32_t lane = tid & 63, r = lane & 15, kg = lane >> 4, most = largest[r], e = max(most >> 23, 1u);
    // 2^(141 - e) in two factors; a row's results take it back.
    const uint32_t up = 141 - min(e, 141u), first = min(up, 100u);
    const float by = e <= 141 ? __uint_as_float((127 + first) << 23) : __uint_as_float((268 - min(e, 254u)) << 23);
    const float more = __uint_as_float((127 + up - first) << 23);
    if (blockIdx.y == 0 && tid < 16)
        down[tile * 16 + r] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, static_cast<int>(e) - 141);
    const float *row = p.A + static_cast<uint64_t>(min(row0 + tile * 16 + r, p.M - 1)) * p.lda;
    const uint32_t blocks = 4 * p.KB, begin = static_cast<uint32_t>(static_cast<uint64_t>(blocks) * blockIdx.y / gridDim.y);
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(blocks) * (blockIdx.y + 1) / gridDim.y);
    for (uint32_t b = begin + tid / 64; b < end; b += kSplitThreads / 64) {
        const uint32_t k = 32 * b + 8 * kg;
        float x[8];
        if constexpr (ALIGNED) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const v4f v = *reinterpret_cast<const v4f *>(row + (k + 4 * i < p.K ? k + 4 * i : 0));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = row[k + i < p.K ? k + i : 0];
        }
        v8h hi, lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t at = order(i);
            const float y = k + at < p.K ? x[at] * by * more : 0.0f;
            const _Float16 h = static_cast<_Float16>(y);
            hi[i] = h;
            lo[i] = static_cast<_Float16>(y - static_cast<float>(h));
        }
        v8h *to = reinterpret_cast<v8h *>(frags + (static_cast<uint64_t>(tile) * blocks + b) * 2048) + lane;
        to[0] = hi;
        to[64] = lo;
    }
}

// The work of a call of many rows.
struct I4Tiles {
    uint32_t row_tiles, col_tiles;   // workgroups' tiles
    uint32_t splits, per;            // ranges of K, blocks of a range
    uint32_t row0, rows;             // of this pass
};

constexpr uint32_t kBand = 8;
template <int RT, int CT, int GB, bool ZEROS>
__global__ __launch_bounds__(256, RT * CT <= 16 ? 2 : 1) void matmul_i4_tile(I4Gemm p, I4Tiles tl, const int8_t *frags, const float *down, float *part)
{
    extern __shared__ __align__(1024) int8_t lds[];
    constexpr uint32_t kStage = RT * 8192;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Neighbouring tiles on one XCD, in bands of 8 row tiles: the 64 that run there at a time share 8 tiles of rows and
    // 8 of columns (2048 x 4096 x 11008: 347 us; a column tile's row tiles one after the other 356, timed in turn).
    const uint32_t tiles = tl.row_tiles * tl.col_tiles, each = (tiles + 7) / 8, id = blockIdx.x % 8 * each + blockIdx.x / 8;
    if (blockIdx.x / 8 >= each || id >= tiles) return;
    const uint32_t band = id / (kBand * tl.col_tiles), in = id - band * kBand * tl.col_tiles;
    const uint32_t high = min(kBand, tl.row_tiles - band * kBand), row_tile = band * kBand + in % high, col_tile = in / high, strips = p.Np / 16;
    const uint32_t begin = blockIdx.y * tl.per, end = min(begin + tl.per, p.KB);

    const uint8_t *codes[CT];
    const float *scales[CT];
    const uint8_t *zeros[CT];
    const uint32_t strip0 = (col_tile * 4 + wave) * CT;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const uint64_t strip = min(strip0 + t, strips - 1);
        codes[t] = p.codes + strip * p.KB * 1024;
        scales[t] = p.scales + strip * p.slots * 16;
        zeros[t] = ZEROS ? p.zeros + strip * p.slots * 16 : nullptr;
    }
    const int8_t *from = frags + static_cast<uint64_t>(row_tile) * RT * p.KB * 8192;
    auto copy = [&](uint32_t kb, int8_t *buf) {
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) {
            const uint32_t piece = wave * 2 * RT + i;
            lds::dma16_s(from + (static_cast<uint64_t>(piece / 8) * p.KB + kb) * 8192 + piece % 8 * 1024, lane * 16, buf + piece * 1024);
        }
    };
    struct Block {
        v4i codes[CT];
        float scale[CT][GB];
        uint32_t zero[CT][GB];
    };
    auto load = [&](Block &b, uint32_t kb) {
        const uint32_t slot = GB > 1 ? GB * kb : kb / p.blocks_of_group;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            b.codes[t] = *reinterpret_cast<const v4i *>(codes[t] + static_cast<uint64_t>(kb) * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < GB; ++i) {
                b.scale[t][i] = scales[t][(slot + i) * 16 + c];
                b.zero[t][i] = ZEROS ? zeros[t][(slot + i) * 16 + c] : 8;
            }
        }
    };

    v4f total[RT][CT], acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) total[r][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    Block now, next;
    copy(begin, lds);
    load(now, begin);
    lds::wait_vmcnt<0>();
    __syncthreads();
    const Masks masks;
    constexpr int per = 4 / GB;   // of 32 of K in a group
    auto weights = [&](int h, int t) {
        const _Float16 z = __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x6400 + now.zero[t][h / per]));   // 1024 + zero
        const uint32_t w0 = static_cast<uint32_t>(now.codes[t][2 * (h & 1)]), w1 = static_cast<uint32_t>(now.codes[t][2 * (h & 1) + 1]);
        return h < 2 ? differences<false>(masks, w0, w1, v2h{z, z}) : differences<true>(masks, w0, w1, v2h{z, z});
    };
    for (uint32_t kb = begin; kb < end; ++kb) {
        const int8_t *buf = lds + ((kb - begin) & 1) * kStage;
        if (kb + 1 < end) {
            copy(kb + 1, lds + ((kb + 1 - begin) & 1) * kStage);
            load(next, kb + 1);
        }
        // Steps of 32 of K and a row tile.  A step's fragments are read a step ahead, the next 32 of K's weights are
        // made beside its products.
        auto fragment = [&](int step, int part) { return *reinterpret_cast<const v8h *>(buf + (step % RT * 8 + 2 * (step / RT) + part) * 1024 + lane * 16); };
        v8h hi = fragment(0, 0), lo = fragment(0, 1), b[CT], soon[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) b[t] = weights(0, t);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // the first step's
#pragma unroll
        for (int step = 0; step < 4 * RT; ++step) {
            const int h = step / RT, r = step % RT;
            const v8h next_hi = step + 1 < 4 * RT ? fragment(step + 1, 0) : hi, next_lo = step + 1 < 4 * RT ? fragment(step + 1, 1) : lo;
#pragma unroll
            for (int t = 0; t < CT; ++t)
                acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, b[t], h % per ? acc[r][t] : v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, b[t], acc[r][t], 0, 0, 0);
            if (h < 3)
#pragma unroll
                for (int t = r * CT / RT; t < (r + 1) * CT / RT; ++t) soon[t] = weights(h + 1, t);
            if (h % per == per - 1) {
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) total[r][t][i] = fmaf(acc[r][t][i], now.scale[t][h / per], total[r][t][i]);
            }
            hi = next_hi;
            lo = next_lo;
            if (r == RT - 1)
#pragma unroll
                for (int t = 0; t < CT; ++t) b[t] = soon[t];
            if (step + 1 < 4 * RT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // the next step's, then each product with what else there is
#pragma unroll
            for (int t = 0; t < 2 * CT; ++t) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
            }
        }
        lds::wait_vmcnt<0>();
        __syncthreads();
        now = next;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const uint32_t tile_row = (row_tile * RT + r) * 16 + 4 * g;
        const v4f by = *reinterpret_cast<const v4f *>(down + tile_row);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const uint32_t n = (strip0 + t) * 16 + c;
            if (n >= p.N) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (tile_row + i >= tl.rows) continue;
                float x = total[r][t][i] * by[i];
                if (tl.splits > 1) {
                    part[(static_cast<uint64_t>(blockIdx.y) * tl.rows + tile_row + i) * p.N + n] = x;
                } else {
                    if (p.bias) x += p.bias[n];
                    p.C[static_cast<uint64_t>(tl.row0 + tile_row + i) * p.ldc + n] = finished(x, p.epilogue);
                }
            }
        }
    }
}

// The ranges of K together, in their order.
__global__ __launch_bounds__(256) void matmul_i4_join(I4Gemm p, I4Tiles tl, const float *part)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<uint64_t>(tl.rows) * p.N;
    if (at >= all) return;
    float x = 0.0f;
    for (uint32_t z = 0; z < tl.splits; ++z) x += part[z * all + at];
    const uint32_t row = static_cast<uint32_t>(at / p.N), n = static_cast<uint32_t>(at % p.N);
    if (p.bias) x += p.bias[n];
    p.C[static_cast<uint64_t>(tl.row0 + row) * p.ldc + n] = finished(x, p.epilogue);
}

template <int RT, int CT, int GB>
void launch_tile(hipStream_t s, const I4Gemm &p, const I4Tiles &tl, const int8_t *frags, const float *down, float *part)
{
    constexpr uint32_t bytes = 2 * RT * 8192;
    const auto kernel = p.zeros ? matmul_i4_tile<RT, CT, GB, true> : matmul_i4_tile<RT, CT, GB, false>;
    if (bytes > 60 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    kernel<<<dim3((tl.row_tiles * tl.col_tiles + 7) / 8 * 8, tl.splits), 256, bytes, s>>>(p, tl, frags, down, part);
}
template <int RT, int CT>
void launch_tile(hipStream_t s, const I4Gemm &p, const I4Tiles &tl, const int8_t *frags, const float *down, float *part)
{
    if (p.groups_of_block == 4) launch_tile<RT, CT, 4>(s, p, tl, frags, down, part);
    else if (p.groups_of_block == 2) launch_tile<RT, CT, 2>(s, p, tl, frags, down, part);
    else launch_tile<RT, CT, 1>(s, p, tl, frags, down, part);
}
constexpr uint64_t kMostFragments = 256ull << 20, kMostParts = 256ull << 20;   // bytes
size_t frag_bytes(const I4Gemm &p) { return static_cast<size_t>(p.pass_rows) * p.KB * 512; }
size_t down_bytes(const I4Gemm &p) { return (static_cast<size_t>(p.pass_rows) * 4 + 255) / 256 * 256; }
size_t part_bytes(const I4Gemm &p)
{
    const uint64_t rows = p.kernel == I4Gemm::kTile ? std::min(p.pass_rows, p.M) : p.M;
    return p.splits > 1 ? static_cast<size_t>(p.splits) * rows * p.N * 4 : 0;
}

void launch_join(hipStream_t s, const I4Gemm &p, const I4Tiles &tl, const float *part)
{
    const uint64_t all = static_cast<uint64_t>(tl.rows) * p.N;
    matmul_i4_join<<<static_cast<uint32_t>((all + 255) / 256), 256, 0, s>>>(p, tl, part);
}
void launch_tiles(hipStream_t s, const I4Gemm &p, int8_t *ws)
{
    int8_t *frags = ws;
    float *down = reinterpret_cast<float *>(ws + frag_bytes(p)), *part = reinterpret_cast<float *>(ws + frag_bytes(p) + down_bytes(p));
    const bool aligned = !((reinterpret_cast<uintptr_t>(p.A) & 15) | (p.lda & 3) | (p.K & 3));
    for (uint32_t row0 = 0; row0 < p.M; row0 += p.pass_rows) {
        I4Tiles tl;
        tl.row0 = row0;
        tl.rows = std::min(p.pass_rows, p.M - row0);
        tl.row_tiles = (tl.rows + 16 * p.rows - 1) / (16 * p.rows);
        tl.col_tiles = (p.Np + 64 * p.strips - 1) / (64 * p.strips);
        tl.splits = p.splits;
        tl.per = p.per;
        const uint32_t tiles = tl.row_tiles * p.rows, parts = std::max(1u, std::min(p.cus / tiles, p.KB / 4));
        (aligned ? matmul_i4_split<true> : matmul_i4_split<false>)<<<dim3(tiles, parts), kSplitThreads, 0, s>>>(p, row0, frags, down);
        if (p.rows == 2 && p.strips == 1) launch_tile<2, 1>(s, p, tl, frags, down, part);
        else if (p.rows == 2) launch_tile<2, 2>(s, p, tl, frags, down, part);
        else if (p.strips == 2) launch_tile<4, 2>(s, p, tl, frags, down, part);
        else launch_tile<4, 4>(s, p, tl, frags, down, part);
        if (tl.splits > 1) launch_join(s, p, tl, part);
    }
}
template <int RQ>
void launch_few_of(hipStream_t s, const I4Gemm &p, float *part)
{
    if (p.waves == 16) p.strips == 1 ? launch_few<RQ, 1, 16>(s, p, part) : launch_few<RQ, 2, 16>(s, p, part);
    else if (p.strips == 2) launch_few<RQ, 2, 8>(s, p, part);
    else if (p.strips == 3) launch_few<RQ, 3, 8>(s, p, part);
    else launch_few<RQ, 4, 8>(s, p, part);
}
void launch_mid_of(hipStream_t s, const I4Gemm &p, float *part)
{
    if (p.rows == 2) p.strips == 3 ? launch_mid<2, 3, 8>(s, p, part) : launch_mid<2, 4, 8>(s, p, part);
    else if (p.strips == 1) launch_mid<1, 1, 8>(s, p, part);
    else if (p.strips == 2) launch_mid<1, 2, 8>(s, p, part);
    else if (p.strips == 3) launch_mid<1, 3, 8>(s, p, part);
    else launch_mid<1, 4, 8>(s, p, part);
}

uint32_t parts_of(uint64_t x, uint32_t y) { return static_cast<uint32_t>((x + y - 1) / y); }

// The time of a call as p says, us: a fit to 7000 measured ones (1 to 256 rows, K 512 to 16384,
// N 512 to 28672, groups of 32 and 128; within 15 to 18 %; what it chooses is 3 % slower in the
// mean than the fastest).  ops: vector instructions of a wave and block.
double estimate(const I4Gemm &p, uint32_t kernel, uint32_t rows, uint32_t strips, uint32_t waves, uint32_t per, uint32_t splits)
{
    const double GB = p.groups_of_block, joined = splits > 1 ? 4.0 * splits * p.M * p.N / 3e6 : 0.0;
    if (kernel == I4Gemm::kTile) {
        const double groups = static_cast<double>(parts_of(p.M, 16 * rows)) * parts_of(p.Np / 16, 4 * strips) * splits;
        const double load = std::ceil(groups / p.cus), tiles = rows * strips, at_once = tiles <= 2 ? 4 : tiles <= 4 ? 3 : 2;
        const double matrix = load * per * tiles * 128 / 2400, vector = load * per * (40 * strips + 4 * tiles * GB) * 4 / 2400;
        return 6.4 + 2.2 * std::max(matrix, vector) + 0.35 * std::ceil(groups / (p.cus * at_once)) * per +
               3.6e-6 * p.M * p.K + 1.9 * std::ceil(p.K / 2048.0) +
               (splits > 1 ? 2.25 : 0.0) + 1.5 * joined;
    }
    const uint32_t wg_rows = kernel == I4Gemm::kFew ? 4 * rows : 16 * rows;
    const double again = parts_of(p.M, wg_rows), groups = parts_of(p.Np / 16, strips) * again * splits, load = std::ceil(groups / p.cus);
    const double ops = kernel == I4Gemm::kFew ? 95.0 * rows + strips * (12 + rows * GB * 11) : 130.0 * rows + strips * (38 + rows * (4 * GB + 4));
    const double vector = load * per * ops / 2400, rounds = std::ceil(groups / (p.cus * (waves == 16 ? 1 : 2)));
    if (kernel == I4Gemm::kFew) return 3.0 + 1.7 * vector + 0.094 * rounds * parts_of(per, waves) + (splits > 1 ? 2.7 : 0.0) + 8.8 * joined;
    return 3.7 + 2.7 * vector + (splits > 1 ? 2.2 : 0.0) + 4.5 * joined;
}

}  // namespace

void pack_i4(hipStream_t s, const uint8_t *B, const float *scales, const uint8_t *zeros, uint32_t K, uint32_t N, uint32_t groups,
             uint32_t ldb, uint32_t trans_b, const I4Weights &w, uint32_t *bad)
{
    const uint64_t pieces = static_cast<uint64_t>(w.Np / 16) * w.KB * 64, count = static_cast<uint64_t>(w.Np) * w.slots;
    pack_codes<<<static_cast<uint32_t>((pieces + 255) / 256), 256, 0, s>>>(B, K, N, ldb, trans_b, w.codes, w.KB, pieces);
    pack_scales<<<static_cast<uint32_t>((count + 255) / 256), 256, 0, s>>>(scales, zeros, groups, w.slots, N, w.scales, w.zeros, count, bad);
}

bool matmul_i4_lay_out(I4Gemm &p)
{
    // kb / g = (kb 2^9 f / 2^32) / 2^s for kb below 2^23, s = log2 g rounded up, f = 2^(23 + s) / g rounded up: f g is less than g
    // above 2^(23 + s), so the quotient is less than 2^-s, at most 1 / g, too high.
    while ((1u << p.group_shift) < p.blocks_of_group) ++p.group_shift;
    p.group_factor = static_cast<uint32_t>(((1ull << (23 + p.group_shift)) + p.blocks_of_group - 1) / p.blocks_of_group);
    // Offsets into A and a strip's codes are 31 bits in the kernels of few and tens of rows.
    const uint64_t most_rows = std::min(p.M, 32u);
    const bool short_offsets = ((most_rows - 1) * p.lda + p.K) * 4 < (1ull << 31) && p.KB < (1u << 21);
    double best = 1e30;
    auto consider = [&](uint32_t kernel, uint32_t rows, uint32_t strips, uint32_t waves) {
        for (uint32_t splits = 1; splits <= 8; splits *= 2) {
            const uint32_t per = parts_of(p.KB, splits);
            if (splits > 1 && (per < 4 || 4ull * splits * std::min<uint64_t>(p.M, 1u << 20) * p.N > kMostParts)) break;
            if (parts_of(p.KB, per) != splits || (waves == 16 && per < 16)) continue;
            const double us = estimate(p, kernel, rows, strips, waves, per, splits);
            if (us >= best) continue;
            best = us;
            p.kernel = static_cast<decltype(p.kernel)>(kernel);
            p.rows = rows;
            p.strips = strips;
            p.waves = waves;
            p.per = per;
            p.splits = splits;
        }
    };
    if (p.M <= 8 && short_offsets) {
        const uint32_t quads = p.M <= 4 ? 1 : 2;
        consider(I4Gemm::kFew, quads, 1, 16);
        consider(I4Gemm::kFew, quads, 2, 16);
        for (uint32_t t = 2; t <= 4; ++t) consider(I4Gemm::kFew, quads, t, 8);
    }
    if (p.M > 4 && p.M <= 512 && short_offsets)
        for (uint32_t t = 1; t <= 4; ++t) {
            consider(I4Gemm::kMid, 1, t, 8);
            if (p.M > 16 && t >= 3) consider(I4Gemm::kMid, 2, t, 8);
        }
    if (p.M > 16 || !short_offsets) {
        consider(I4Gemm::kTile, 2, 1, 4);
        consider(I4Gemm::kTile, 2, 2, 4);
        consider(I4Gemm::kTile, 4, 2, 4);
        consider(I4Gemm::kTile, 4, 4, 4);
    }
    uint64_t groups = static_cast<uint64_t>(parts_of(p.Np / 16, p.strips)), pass = p.M;
    if (p.kernel == I4Gemm::kTile) {
        const uint32_t wg_rows = 16 * p.rows;
        p.pass_rows = static_cast<uint32_t>(std::max<uint64_t>(1, kMostFragments / (512ull * p.KB * wg_rows))) * wg_rows;
        p.pass_rows = std::min(p.pass_rows, parts_of(p.M, wg_rows) * wg_rows);
        pass = std::min(p.pass_rows, p.M);
        groups = static_cast<uint64_t>(p.pass_rows / wg_rows) * parts_of(p.Np / 16, 4 * p.strips) + 7;
    }
    // A grid's work-items count in 32 bits.
    return groups * 64 * p.waves < (1ull << 32) && (p.splits == 1 || pass * p.N < (1ull << 32) - 256);
}

size_t matmul_i4_ws_bytes(const I4Gemm &p)
{
    return p.kernel == I4Gemm::kTile ? frag_bytes(p) + down_bytes(p) + part_bytes(p) : part_bytes(p);
}

void matmul_i4(hipStream_t s, const I4Gemm &p, void *ws)
{
    if (p.kernel == I4Gemm::kTile) {
        launch_tiles(s, p, static_cast<int8_t *>(ws));
        return;
    }
    float *part = p.splits > 1 ? static_cast<float *>(ws) : nullptr;
    if (p.kernel == I4Gemm::kFew) p.rows == 1 ? launch_few_of<1>(s, p, part) : launch_few_of<2>(s, p, part);
    else launch_mid_of(s, p, part);
    if (part) {
        I4Tiles tl{};
        tl.splits = p.splits;
        tl.rows = p.M;
        launch_join(s, p, tl, part);
    }
}

std::string matmul_i4_route(const I4Gemm &p)
{
    static const char *names[] = {"few", "mid", "tile"};
    char text[96];
    std::snprintf(text, sizeof(text), "%s rows=%u strips=%u waves=%u splits=%u", names[p.kernel], p.rows, p.strips, p.waves, p.splits);
    return text;
}

}  // namespace k
}  // namespace vnpu
