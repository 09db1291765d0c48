// sgq_rope.hip -- norms of the heads of queries and keys, the position rotation, and the
// new tokens' keys and values into their pages, in one pass over q, k and v.
//
// Mathematics.  Per head x of q and k: u = x * g / sqrt(sum(x^2) / d + eps), then pairs
// (a, b) of u turned by angle = position * freqs[i]:
//   a' = a cos - b sin,  b' = b cos + a sin.
// fp32 throughout, one rounding to the type at the store.  The angle is a 64-bit
// product: at position 10^6 fp32 would be off by 0.06 rad.  In 64 bits it is taken to
// half turns t = 2 (r - rint(r)), r = angle / 2 pi, |t| <= 1; sin and cos of pi t come
// from fp32's sincospi of t rounded and the rounding's rest e (sin' = sin + pi e cos).
//
// Layout.  A thread takes two 16-byte chunks of a head that hold both sides of their
// pairs (i and i + rotary_dim / 2, or neighbours), so that nothing is exchanged but the
// sum of squares, over the lanes of a head.  Pairs that do not fall on whole chunks go
// through LDS.  A workgroup is one token and some or all of its heads: it finds the
// sequence, the page and the sines once; where tokens are few (a decode step) its heads go to several workgroups.
//
// HBM bounds it: 16384 tokens, 64 on 8 heads of 128 in bf16, 671 MB read and written in 124 us, 5.4 TB/s; 2048 tokens,
// 32 heads, 50 MB 12 us, 4.1.  A decode step of eight tokens takes 4.2 us, a launch and three latencies (the
// sequence, its page, the row).
#include "sgq_paged.h"

namespace sgq {
namespace {

constexpr int kBlock = 256;

enum class Pairs : int { chunks, lds, neighbours };

template <typename T, Pairs P>
__global__ __launch_bounds__(kBlock) void k_norm_rope_append(const RopeArgs a, const PagedCache c, const Sequences s,
                                                             int lanes_log, int heads_per_wg) {
    constexpr int N = Chunk<T>::N;
    typedef typename Chunk<T>::type Vec;
    __shared__ float2 turn[kMaxHeadDim / 2];
    __shared__ float part[P == Pairs::lds ? kBlock * 2 * N : 1];

    const int row = blockIdx.x;
    const int b = seq_of_row(s, row);
    if (b >= s.B) return;
    const SeqRows r = seq_rows(s, b);
    if (row < r.row0 || row >= r.row0 + r.n) return;  // before the first sequence, or starts that decrease
    const int at = r.position(row);
    const int64_t slot = r.ok ? key_offset(c, s.table + b * s.table_ld, at) : -1;
    const bool ok = slot >= 0;

    const double pos = a.positions ? a.positions[row] : at;
    for (int i = threadIdx.x; i < a.half; i += kBlock) {
        double t = pos * a.freqs[i] * 0.15915494309189533577;  // 1 / (2 pi)
        t = 2.0 * (t - rint(t));
        const float f = (float)t, e = 3.14159265f * (float)(t - f);
        float sn, cs;
        sincospif(f, &sn, &cs);
        turn[i] = make_float2(fmaf(-e, sn, cs), fmaf(e, cs, sn));
    }
    __syncthreads();

    // Two chunks (of a head's 2 * pairs chunks) per thread, 2^lanes_log lanes a head.
    const int d = c.head_dim, pairs = d / (2 * N);
    const int t = threadIdx.x & ((1 << lanes_log) - 1), slots = kBlock >> lanes_log;
    const bool mine = t < pairs;
    const int hc = a.half / N;  // chunks of one side of the pairs
    int e0, e1;                 // first elements of the two chunks
    if (P != Pairs::chunks) {
        e0 = 2 * t * N, e1 = e0 + N;
    } else if (t < hc) {
        e0 = t * N, e1 = e0 + a.half;
    } else {
        e0 = 2 * t * N, e1 = e0 + N;  // behind the turned ones, which are 2 hc chunks
    }
    const int nq = a.heads, nk = nq + c.kv_heads, all = nk + c.kv_heads;
    const int h0 = blockIdx.y * heads_per_wg, h1 = min(all, h0 + heads_per_wg);
    for (int hb = h0; hb < h1; hb += slots) {
        const int h = hb + (threadIdx.x >> lanes_log);
        const bool on = mine && h < h1;
        const bool is_q = h < nq, is_v = h >= nk;
        const HeadRows& in = is_q ? a.q : (is_v ? a.v : a.k);
        const int hh = is_q ? h : (is_v ? h - nk : h - nq);
        const T* x = (const T*)in.p + (int64_t)row * in.row + (int64_t)hh * in.head;
        Vec x0 = {}, x1 = {};
        if (on) x0 = *(const Vec*)(x + e0), x1 = *(const Vec*)(x + e1);
        float u0[N], u1[N];
#pragma unroll
        for (int i = 0; i < N; ++i) u0[i] = (float)x0[i], u1[i] = (float)x1[i];
        const float* g = is_q ? a.q_norm : a.k_norm;
        if (a.q_norm || a.k_norm) {  // the sum by all lanes
            auto squares = [&] {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) ss = fmaf(u0[i], u0[i], ss);
#pragma unroll
                for (int i = 0; i < N; ++i) ss = fmaf(u1[i], u1[i], ss);
                for (int o = 1 << lanes_log >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
                return ss;
            };
            float ss = squares(), eps = a.eps;
            // Heads whose squares fp32 does not hold are taken 2^-72 or (where eps does not outweigh them) 2^72 times, which the norm
            // takes out again; where one of a wavefront is, all of it comes along.
            if (__builtin_expect(__any(h < h1 && !(ss >= 0x1p-90f && ss < INFINITY)), 0)) {
                const bool large = ss == INFINITY, far = (large || (ss < 0x1p-90f && a.eps < 0x1p-100f)) && g && !is_v;
                const float unit = !far ? 1.0f : large ? 0x1p-72f : 0x1p72f;
#pragma unroll
                for (int i = 0; i < N; ++i) u0[i] *= unit, u1[i] *= unit;
                ss = squares(), eps = eps * unit * unit;  // (unit * unit by itself would pass fp32)
            }
            if (on && g && !is_v) {
                const float rstd = 1.0f / sqrtf(ss / (float)d + eps);
#pragma unroll
                for (int i = 0; i < N; ++i) u0[i] = u0[i] * rstd * g[e0 + i], u1[i] = u1[i] * rstd * g[e1 + i];
            }
        }
        Vec y0 = x0, y1 = x1;  // values as they are
        if constexpr (P == Pairs::lds) {
            float* p = part + (threadIdx.x >> lanes_log << lanes_log) * 2 * N;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) p[2 * t * N + i] = u0[i], p[(2 * t + 1) * N + i] = u1[i];
            __syncthreads();
            if (on && !is_v) {
                auto turned = [&](int e, float u) {
                    if (e >= 2 * a.half) return u;
                    const bool low = e < a.half;
                    const float2 w = turn[low ? e : e - a.half];
                    const float o = p[low ? e + a.half : e - a.half];
                    return low ? u * w.x - o * w.y : u * w.x + o * w.y;
                };
#pragma unroll
                for (int i = 0; i < N; ++i) y0[i] = (T)turned(e0 + i, u0[i]), y1[i] = (T)turned(e1 + i, u1[i]);
            }
        } else if (on && !is_v) {
            if constexpr (P == Pairs::neighbours) {
                auto two = [&](int e, float p, float q, T& yp, T& yq) {
                    float2 w = make_float2(1.0f, 0.0f);
                    if (e < 2 * a.half) w = turn[e / 2];
                    yp = (T)(p * w.x - q * w.y), yq = (T)(q * w.x + p * w.y);
                };
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    T p, q;
                    two(e0 + i, u0[i], u0[i + 1], p, q), y0[i] = p, y0[i + 1] = q;
                    two(e1 + i, u1[i], u1[i + 1], p, q), y1[i] = p, y1[i + 1] = q;
                }
                if (e1 + N > 2 * a.half)  // as below
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (e0 + i >= 2 * a.half) y0[i] = (T)u0[i];
                        if (e1 + i >= 2 * a.half) y1[i] = (T)u1[i];
                    }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float2 w = make_float2(1.0f, 0.0f);
                    if (t < hc) w = turn[e0 + i];
                    y0[i] = (T)(u0[i] * w.x - u1[i] * w.y), y1[i] = (T)(u1[i] * w.x + u0[i] * w.y);
                }
                // Not by an angle of 0: 0 times what is not finite is a NaN.  (A branch that wavefronts skip whose
                // heads are turned whole; with one around the products 16384 tokens took 125.4 us instead of 124.9.)
                if (t >= hc)
#pragma unroll
                    for (int i = 0; i < N; ++i) y0[i] = (T)u0[i], y1[i] = (T)u1[i];
            }
        }
        if (!on) continue;
        T* y;
        if (is_q) {
            y = (T*)a.out.p + (int64_t)row * a.out.row + (int64_t)hh * a.out.head;
            if (!ok)
#pragma unroll
                for (int i = 0; i < N; ++i) y0[i] = y1[i] = (T)NAN;
        } else {
            if (!ok) continue;
            y = (T*)(is_v ? c.v : c.k) + slot + (int64_t)hh * c.head_stride;
        }
        *(Vec*)(y + e0) = y0;
        *(Vec*)(y + e1) = y1;
    }
}

template <typename T>
void start(const RopeArgs& a, const PagedCache& c, const Sequences& s, hipStream_t st) {
    constexpr int N = Chunk<T>::N;
    const int pairs = c.head_dim / (2 * N);
    int lanes_log = 0;
    while (1 << lanes_log < pairs) ++lanes_log;
    const int slots = kBlock >> lanes_log, all = a.heads + 2 * c.kv_heads;
    const int rounds = (int)ceil_div(all, slots);
    const int wgs = (int)std::min<int64_t>(rounds, ceil_div(1024, s.rows));
    const int per = (int)ceil_div(rounds, wgs) * slots;
    const dim3 grid((unsigned)s.rows, (unsigned)ceil_div(all, per));
    if (a.interleaved)
        k_norm_rope_append<T, Pairs::neighbours><<<grid, kBlock, 0, st>>>(a, c, s, lanes_log, per);
    else if (a.half % N == 0)
        k_norm_rope_append<T, Pairs::chunks><<<grid, kBlock, 0, st>>>(a, c, s, lanes_log, per);
    else
        k_norm_rope_append<T, Pairs::lds><<<grid, kBlock, 0, st>>>(a, c, s, lanes_log, per);
}

}  // namespace

hipError_t launch_norm_rope_append(const RopeArgs& a, const PagedCache& c, const Sequences& s, hipStream_t st) {
    if (s.rows <= 0 || s.B <= 0) return hipSuccess;
    switch (c.t) {
        case DType::f32: start<float>(a, c, s, st); break;
        case DType::bf16: start<__bf16>(a, c, s, st); break;
        case DType::f16: start<_Float16>(a, c, s, st); break;
    }
    return hipGetLastError();
}

}  // namespace sgq
