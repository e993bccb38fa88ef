// kv_common.hpp - what the kernels of the paged int8 KV cache share: where a
// call's sequences, pages and rows are, and the checks that keep every access
// inside the caller's buffers whatever the arrays on the device hold.
#pragma once

#include "kernels.hpp"

namespace vnpu {
namespace k {
namespace kv {

// A length, seq_start or page was out of range: the stream fails at its sync.
__device__ __forceinline__ void fail(uint32_t *err)
{
    __hip_atomic_store(err, 2u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Sequence b's rows [row, row + n) of the call, and whether they are in range.
struct Seq {
    uint32_t row, n;
    bool ok;
};
__device__ __forceinline__ Seq sequence(const KvCall &c, uint32_t b)
{
    if (!c.seq_start) {
        const uint32_t n = c.tokens / c.batch;
        return {b * n, n, true};
    }
    const int32_t a = c.seq_start[b], e = c.seq_start[b + 1];
    return {static_cast<uint32_t>(a), static_cast<uint32_t>(e - a),
            a >= 0 && e >= a && static_cast<uint32_t>(e) <= c.tokens};
}
__device__ __forceinline__ uint32_t capacity(const KvCall &c) { return c.c.table_ld << c.c.log_page; }

// Element 0 of head 0 of sequence b's token 0.
__device__ __forceinline__ uint64_t rows_base(const KvCall &c, const KvRows &r, uint32_t b, const Seq &s)
{
    return c.seq_start ? s.row * r.token : b * r.batch;
}

// Append and read work page by page.  The pages that sequences touch are not
// known to the host: sequence b of n tokens touches at most n / page_size + 2,
// so its units are given room for that many.  unit -> (b, which of its pages);
// false: no sequence's.  Every thread of the workgroup calls it.
__device__ __forceinline__ uint32_t unit_room(const KvCall &c, uint32_t row, uint32_t b)
{
    return (row >> c.c.log_page) + 2 * b;
}
__device__ __forceinline__ bool find_unit(const KvCall &c, uint32_t unit, uint32_t &b, uint32_t &j)
{
    if (!c.seq_start) {
        const uint32_t room = ((c.tokens / c.batch) >> c.c.log_page) + 2;
        b = unit / room;
        j = unit % room;
        return b < c.batch;
    }
    // How many sequences begin at this unit or before it, counted by each wave.
    uint32_t before = 0;
    for (uint32_t i = 0; i < c.batch; i += 64) {
        const uint32_t at = i + (threadIdx.x & 63);
        const bool here = at < c.batch && unit_room(c, static_cast<uint32_t>(c.seq_start[at]), at) <= unit;
        before += __popcll(__ballot(here));
    }
    if (!before) return false;
    b = before - 1;
    j = unit - unit_room(c, static_cast<uint32_t>(c.seq_start[b]), b);
    return true;
}
inline uint32_t unit_count(const KvCall &c)
{
    return c.seq_start ? (c.tokens >> c.c.log_page) + 2 * c.batch
                       : c.batch * (((c.tokens / c.batch) >> c.c.log_page) + 2);
}

// Every sequence's rows and lengths, looked over by one workgroup of a call so
// that what no workgroup meets is an error too.  extra: the call's tokens count
// towards the length (append, read).  most: tokens of a sequence.
__device__ __forceinline__ void check_all(const KvCall &c, bool extra, uint32_t limit, uint32_t most)
{
    for (uint32_t b = threadIdx.x; b < c.batch; b += blockDim.x) {
        const Seq s = sequence(c, b);
        const int64_t len = c.lengths ? c.lengths[b] : 0;
        if (!s.ok || s.n > most || len < 0 || len + (extra ? static_cast<int64_t>(s.n) : 0) > static_cast<int64_t>(limit)) fail(c.err);
    }
}

// What a workgroup of append and read works on: m tokens at slots slot.. of a
// page, the sequence's tokens first.. of the call.
struct Piece {
    uint32_t page, slot, m, first;
    Seq seq;
};
__device__ __forceinline__ bool find_piece(const KvCall &c, uint32_t unit, uint32_t &b, Piece &p)
{
    uint32_t j;
    if (!find_unit(c, unit, b, j)) return false;
    p.seq = sequence(c, b);
    const int64_t past = c.lengths ? c.lengths[b] : 0;
    if (!p.seq.ok || past < 0 || past + p.seq.n > static_cast<int64_t>(capacity(c))) return false;   // check_all told
    const uint32_t ps = c.c.page_size, begin = static_cast<uint32_t>(past), end = begin + p.seq.n;
    const uint32_t pg = (begin >> c.c.log_page) + j;
    if (pg >= c.c.table_ld) return false;
    const uint32_t lo = max(begin, pg << c.c.log_page), hi = min(end, (pg << c.c.log_page) + ps);
    if (lo >= hi) return false;
    const int32_t id = c.c.table[static_cast<uint64_t>(b) * c.c.table_ld + pg];
    if (static_cast<uint32_t>(id) >= c.c.pages) {
        fail(c.err);
        return false;
    }
    p.page = static_cast<uint32_t>(id);
    p.slot = lo & (ps - 1);
    p.m = hi - lo;
    p.first = lo - begin;
    return true;
}

}  // namespace kv
}  // namespace k
}  // namespace vnpu
