// sgq_attention.hip -- attention of new tokens over a paged key/value cache.
//
// Mathematics.  Row i of a sequence (position p) sees the keys of one interval [lo, hi)
// (causal, window, document start, prefix); with s_j its scores
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j,
// in one pass over the keys with a running maximum: when it grows from m to m', what
// was summed is multiplied by exp(m - m').  All of it in fp32.
#include "sgq_paged.h"

namespace sgq {
namespace {

constexpr float kLog2e = 1.44269504f;

// The keys [lo, hi) that a row sees.
__device__ __forceinline__ void row_keys(const AttendArgs& a, const SeqRows& r, int b, int row, int& lo, int& hi) {
    const int p = r.position(row);
    lo = a.first_key ? max(a.first_key[row], 0) : 0;
    if (a.window > 0) lo = max(lo, p - a.window + 1);
    hi = p + 1;
    if (a.prefix) hi = max(hi, min(a.prefix[b], r.len));
}

// A wavefront per row and head, a key at a time.
template <typename T>
__global__ __launch_bounds__(256) void k_attend_rows(const AttendArgs a, const PagedCache c, const Sequences s) {
    const int row = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (h >= a.heads) return;
    const int b = seq_of_row(s, row);
    if (b >= s.B) return;
    const SeqRows r = seq_rows(s, b);
    const bool inside = row >= r.row0 && row < r.row0 + r.n;
    if (!inside && r.ok) return;
    const int d = c.head_dim, kvh = h / (a.heads / c.kv_heads);
    const T* q = (const T*)a.q.p + (int64_t)row * a.q.row + (int64_t)h * a.q.head;
    T* out = (T*)a.out.p + (int64_t)row * a.out.row + (int64_t)h * a.out.head;
    float x[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 4; ++i) x[i] = lane + 64 * i < d ? (float)q[lane + 64 * i] : 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool ok = r.ok;
    if (ok) {
        int lo, hi;
        row_keys(a, r, b, row, lo, hi);
        const float slope = a.slopes ? a.slopes[h] : 0.0f;
        for (int j = lo; j < hi; ++j) {
            const int64_t off = key_offset(c, s.table + b * s.table_ld, j);
            if (off < 0) {
                ok = false;
                break;
            }
            const T* k = (const T*)c.k + off + kvh * c.head_stride;
            const T* v = (const T*)c.v + off + kvh * c.head_stride;
            float sc = 0.0f;
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < d) sc = fmaf(x[i], (float)k[lane + 64 * i], sc);
            for (int t = 32; t > 0; t >>= 1) sc += __shfl_xor(sc, t, 64);
            sc *= a.scale;
            if (a.softcap > 0.0f) sc = a.softcap * tanhf(sc / a.softcap);
            sc -= slope * fabsf((float)(r.position(row) - j));
            const float mn = fmaxf(m, sc);
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float w = expf(m - base), e = sc != sc ? sc : expf(sc - base);
            l = l * w + e;
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < d) o[i] = o[i] * w + e * (float)v[lane + 64 * i];
            m = mn;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < d) out[lane + 64 * i] = ok ? (T)(o[i] * inv) : (T)NAN;
}

}  // namespace

hipError_t launch_attend(const AttendArgs& a, const PagedCache& c, const Sequences& s, void* ws, hipStream_t st) {
    if (s.rows <= 0 || s.B <= 0) return hipSuccess;
    const dim3 grid((unsigned)s.rows, (unsigned)ceil_div(a.heads, 4));
    switch (c.t) {
        case DType::f32: k_attend_rows<float><<<grid, 256, 0, st>>>(a, c, s); break;
        case DType::bf16: k_attend_rows<__bf16><<<grid, 256, 0, st>>>(a, c, s); break;
        case DType::f16: k_attend_rows<_Float16><<<grid, 256, 0, st>>>(a, c, s); break;
    }
    return hipGetLastError();
}

}  // namespace sgq
