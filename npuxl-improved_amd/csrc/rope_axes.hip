// rope_axes.hip - ROPE_AXES_F32: rotary positions with several axes, on gfx950.
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),
//   a = positions[axis(j)][t] * scaling * theta^-e(j) for pair j of token t.
// Which axis a pair has and its exponent are worked out on the host.  A thread has a pair of a
// token and turns it in some heads, whose values are asked for before the cosine is computed.
// Bound by the rows in and out: 4096 tokens of 32 and 8 heads of 128 in 35 us as rows of a fused
// projection, 32 us head-major, 4.8 and 5.2 TB/s (a large copy: 5.1); 1601 tokens of 16 and 16 heads
// of 80 in 7.5 us; 8 tokens in 3.1 us, a launch and its latency.
#include "device_math.hpp"
#include "kernels.hpp"

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

namespace vnpu {
namespace k {
namespace {

// Unit i of a token is pair i, or behind the last pair two elements that are copied; in PER heads of Q or K.
// (Four pairs a thread and 16 bytes a load: 4096 tokens 38 us whatever PER, 64 tokens 4.0 us instead of 3.3;
// a thread asks for the axis and rate of each of its pairs one after another.)
template <int PER, bool HALF>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxes p, uint32_t units, uint32_t q_parts)
{
    const uint32_t at = blockIdx.x * 256 + threadIdx.x, token = at / units, i = at - token * units;
    if (token >= p.tokens) return;
    const bool is_q = blockIdx.y < q_parts;
    const uint32_t h0 = (is_q ? blockIdx.y : blockIdx.y - q_parts) * PER, heads = is_q ? p.heads : p.kv_heads;
    const uint32_t b = token / (p.tokens / p.batch), t = token - b * (p.tokens / p.batch);
    const bool turn = i < p.pairs;
    const uint32_t first = turn && HALF ? i : 2 * i, second = turn && HALF ? i + p.pairs : 2 * i + 1;
    const KvRows &from = is_q ? p.q : p.k, &to = is_q ? p.qo : p.ko;
    const float *in = (is_q ? p.Q : p.K) + b * from.batch + t * from.token;
    float x[PER], y[PER];
#pragma unroll
    for (int h = 0; h < PER; ++h) {   // heads behind the last: the last again
        const float *row = in + min(h0 + h, heads - 1) * from.head;
        x[h] = row[first];
        y[h] = row[second];
    }
    if (turn) {
        double c, s;
        dev::cos_sin_turns(static_cast<double>(p.positions[static_cast<uint64_t>(p.of.axis[i]) * p.position_ld + token]) * p.of.turns[i], c, s);
#pragma unroll
        for (int h = 0; h < PER; ++h) {
            const double u = x[h], v = y[h];
            x[h] = static_cast<float>(fma(u, c, -(v * s)));
            y[h] = static_cast<float>(fma(u, s, v * c));
        }
    }
    float *out = (is_q ? p.Q_out : p.K_out) + b * to.batch + t * to.token;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
        if (h0 + h >= heads) break;
        float *row = out + (h0 + h) * to.head;
        row[first] = x[h];
        row[second] = y[h];
    }
}

template <int PER>
void launch(hipStream_t s, const RopeAxes &p)
{
    const uint32_t units = p.head_dim / 2, q_parts = (p.heads + PER - 1) / PER, k_parts = (p.kv_heads + PER - 1) / PER;
    const dim3 grid(static_cast<uint32_t>((static_cast<uint64_t>(p.tokens) * units + 255) / 256), q_parts + k_parts);
    (p.half ? rope_axes_kernel<PER, true> : rope_axes_kernel<PER, false>)<<<grid, 256, 0, s>>>(p, units, q_parts);
}

}  // namespace

// Kept by value for a call's parameters: the powers of 64 pairs are microseconds on the host.
void rope_axes_rates(RopeAxes &p, bool in_turn, bool own_ladders, uint32_t axes, const uint32_t *sections, float theta, float scaling)
{
    using Key = std::tuple<bool, bool, std::vector<uint32_t>, float, float>;
    static std::mutex mutex;
    static auto *known = new std::map<Key, RopeAxes::Pairs>();
    std::lock_guard<std::mutex> lock(mutex);
    const Key key(in_turn, own_ladders, std::vector<uint32_t>(sections, sections + axes), theta, scaling);
    const auto it = known->find(key);
    if (it != known->end()) {
        p.of = it->second;
        return;
    }
    p.of = {};
    uint32_t used[4] = {}, axis = 0;
    for (uint32_t j = 0; j < p.pairs; ++j) {
        while (used[axis] == sections[axis]) axis = (axis + 1) % axes;
        const double power = own_ladders ? static_cast<double>(used[axis]) / sections[axis] : static_cast<double>(j) / p.pairs;
        p.of.axis[j] = static_cast<uint8_t>(axis);
        p.of.turns[j] = static_cast<double>(scaling) * std::pow(static_cast<double>(theta), -power) / (2.0 * M_PI);
        ++used[axis];
        if (in_turn) axis = (axis + 1) % axes;
    }
    if (known->size() >= 64) known->clear();
    known->emplace(key, p.of);
}

// A grid's work-items count in 32 bits.
bool rope_axes_fits(const RopeAxes &p) { return static_cast<uint64_t>(p.tokens) * (p.head_dim / 2) < (1ull << 32) - 256; }

// More heads a thread share its cosine, fewer make more threads (us with 2, 4, 8 heads: 64 tokens of 40 heads of 128 3.2,
// 3.4, 3.3; 512 tokens 6.7, 5.7, 5.9; 4096 tokens 43, 39, 35).
void rope_axes(hipStream_t s, const RopeAxes &p)
{
    const uint64_t work = static_cast<uint64_t>(p.tokens) * (p.head_dim / 2) * (p.heads + p.kv_heads);
    const uint32_t heads = std::max(p.heads, p.kv_heads);
    if (work < 30000) launch<1>(s, p);
    else if (work < 400000 || heads <= 2) launch<2>(s, p);
    else if (work < 1600000 || heads <= 4) launch<4>(s, p);
    else launch<8>(s, p);
}

}  // namespace k
}  // namespace vnpu
