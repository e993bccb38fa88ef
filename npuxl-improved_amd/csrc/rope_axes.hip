// rope_axes.hip - ROPE_AXES_F32: rotary positions with several axes, on gfx950.
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),
//   a = positions[axis(j)][t] * scaling * theta^-e(j) for pair j of token t.
// Which axis a pair has and its exponent are worked out on the host.
#include "device_math.hpp"
#include "kernels.hpp"

#include <algorithm>

namespace vnpu {
namespace k {
namespace {

using v4f = float __attribute__((ext_vector_type(4)));

// Elements of a thread: U pairs of a token that begin with pair U * i, or, behind the last
// pair, 2 U elements that are copied; in the heads h0, h0 + 1, .. of Q or K.
template <int U, bool HALF>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxes p, uint32_t units, uint32_t per, uint32_t q_parts)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t token = static_cast<uint32_t>(at / units), i = static_cast<uint32_t>(at % units);
    if (token >= p.tokens) return;
    const bool is_q = blockIdx.y < q_parts;
    const uint32_t part = is_q ? blockIdx.y : blockIdx.y - q_parts, h0 = part * per;
    const uint32_t h1 = min(is_q ? p.heads : p.kv_heads, h0 + per), n = p.tokens / p.batch, b = token / n, t = token - b * n;
    const KvRows &from = is_q ? p.q : p.k, &to = is_q ? p.qo : p.ko;
    const float *in = (is_q ? p.Q : p.K) + b * from.batch + t * from.token + h0 * from.head;
    float *out = (is_q ? p.Q_out : p.K_out) + b * to.batch + t * to.token + h0 * to.head;
    const bool turn = U * i < p.pairs;
    const uint32_t first = turn && HALF ? U * i : 2 * U * i, second = turn && HALF ? first + p.pairs : first + U;
    double c[U], s[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        c[j] = 1.0;
        s[j] = 0.0;
        if (!turn) continue;
        const uint32_t pair = U * i + j;
        dev::cos_sin_turns(static_cast<double>(p.positions[static_cast<uint64_t>(p.axis[pair]) * p.position_ld + token]) * p.turns[pair], c[j], s[j]);
    }
    for (uint32_t h = h0; h < h1; ++h, in += from.head, out += to.head) {
        float x[2 * U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            x[j] = in[first + j];
            x[U + j] = in[second + j];
        }
        if (turn) {
            float y[2 * U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int a = HALF ? j : 2 * j, o = HALF ? U + j : 2 * j + 1;
                const double u = x[a], v = x[o];
                y[a] = static_cast<float>(fma(u, c[j], -(v * s[j])));
                y[o] = static_cast<float>(fma(u, s[j], v * c[j]));
            }
#pragma unroll
            for (int j = 0; j < 2 * U; ++j) x[j] = y[j];
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            out[first + j] = x[j];
            out[second + j] = x[U + j];
        }
    }
}

}  // namespace

// A grid's work-items count in 32 bits.
bool rope_axes_fits(const RopeAxes &p) { return static_cast<uint64_t>(p.tokens) * (p.head_dim / 2) < (1ull << 32) - 256; }

void rope_axes(hipStream_t s, const RopeAxes &p)
{
    const uint32_t units = p.head_dim / 2, per = 8, q_parts = (p.heads + per - 1) / per, k_parts = (p.kv_heads + per - 1) / per;
    const dim3 grid(static_cast<uint32_t>((static_cast<uint64_t>(p.tokens) * units + 255) / 256), q_parts + k_parts);
    (p.half ? rope_axes_kernel<1, true> : rope_axes_kernel<1, false>)<<<grid, 256, 0, s>>>(p, units, per, q_parts);
}

}  // namespace k
}  // namespace vnpu
