// kv_attention.hip - KV_ATTENTION_I8: attention over the paged int8 KV cache
// on gfx950.
//
//   o = sum_j softmax_j(scale * q . k_j) v_j,  k_j = code * k_scale(page, head)
// over the keys j that the query sees.  One pass over the keys with the
// running maximum m and sum l of the softmax.
#include "kv_common.hpp"

namespace vnpu {
namespace k {
namespace {

// One wave per token and query head; lane = key for the scores, lane = head
// dimension for the products with V.
__global__ __launch_bounds__(64) void kv_attention_simple(KvAttn p)
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
    if (!s.ok || i >= s.n || len < 0 || static_cast<uint32_t>(len) > p.max_kv) return;
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

std::string kv_attention_route(const KvAttn &) { return "rowwise"; }

size_t kv_attention_ws_bytes(const KvAttn &) { return 0; }

void kv_attention(hipStream_t s, const KvAttn &p, void *)
{
    kv_attention_simple<<<dim3(p.call.tokens, p.heads), 64, 0, s>>>(p);
}

}  // namespace k
}  // namespace vnpu
