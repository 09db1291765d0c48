// sgq_paged.h -- sequences of new tokens over a paged cache, as the kernels of
// sgq_rope.hip and sgq_attention.hip read them.  Device-only; include from .hip files.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sgq_internal.h"

namespace sgq {
namespace {

// A sequence's new rows [row0, row0 + n) and its keys.  ok: within the call's bounds, and
// so within its arrays; otherwise n rows from row0, which lie within `rows`, become NaN.
struct SeqRows {
    int row0, n, len;
    bool ok;
    __device__ __forceinline__ int position(int row) const { return len - n + (row - row0); }
};

__device__ __forceinline__ SeqRows seq_rows(const Sequences& s, int b) {
    SeqRows r;
    const int s0 = s.starts[b], s1 = s.starts[b + 1];
    r.len = s.lens[b];
    r.ok = s0 >= 0 && s1 >= s0 && s1 <= s.rows;
    r.row0 = min(max(s0, 0), s.rows);
    r.n = max(min(s1, s.rows) - r.row0, 0);
    r.ok = r.ok && r.n <= s.max_new && r.n <= r.len && r.len <= s.max_len && r.len <= s.capacity;
    return r;
}

// The sequence whose rows hold `row`: how many of starts[1 ..] are not past it (B: the row is of none).  By a whole
// wavefront, which narrows the sequences down to a 64th at a time: the loads wait for each other
// (appending for 4096 sequences of one token 20 us; counting 64 by 64 took 36).
__device__ __forceinline__ int seq_of_row(const Sequences& s, int row) {
    const int lane = threadIdx.x & 63;
    int b = 0, n = s.B;  // it is one of [b, b + n]
    while (n > 0) {
        const int step = (n + 63) / 64, at = (lane + 1) * step;  // a lane's: the last of a block of `step`
        const int whole = __popcll(__ballot(at <= n && s.starts[b + min(at, n)] <= row));
        b += whole * step;
        n = min(step - 1, n - whole * step);
    }
    return b;
}

// Element offset of key j's row (head 0) in the pool, -1 where the table names no page.
__device__ __forceinline__ int64_t key_offset(const PagedCache& c, const int32_t* table, int j) {
    const int page = table[j >> c.page_log];
    if ((unsigned)page >= (unsigned)c.pages) return -1;
    return (int64_t)page * c.page_stride + (int64_t)(j & ((1 << c.page_log) - 1)) * c.token_stride;
}

// Sixteen bytes of a type's elements.
template <typename T>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(N)));
};

}  // namespace
}  // namespace sgq
