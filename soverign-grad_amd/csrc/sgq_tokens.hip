// sgq_tokens.hip -- 8-bit tokens for gfx950: rows of activations as int8 codes
// with one fp32 scale per row, with or without the RMSNorm (and the residual's
// addition) in front, and their values read back.
//
// Mathematics.  The quantizer is the one of sgq_quant.hip over a row v[0..K):
//   m = max(1e-8, max|v|) where NaN never wins, scale = m / 127, inv = 127 / m,
//   code = clamp(round half away from zero(v * inv), -127, 127),
// single IEEE operations, so the codes are fixed bits.  Behind the norm the row is
// n = u * rstd with u = h * g, rstd = 1 / sqrt(sum(h^2) / K + eps).  rstd is one
// positive factor of the whole row: it cancels out of n / max|n|, so the codes are
// taken from u (m = max(max|u|, 1e-8 / rstd)) and do not depend on the order of
// the sum; rstd only enters the scale, m * rstd / 127.
// Rows that are not finite: behind the norm the sum of squares carries them into the
// scale.  Without it the rule is the weights' (NaN never wins the maximum), which would
// turn the hidden row of NaN of an MLP into small finite tokens; KEEP sums v * 0, zero
// or, of an infinity or a NaN, a NaN, beside the maximum and adds it to the scale (2048 x
// 11008 fp32 20.9 us against 20.8 without, bf16 14.7 against 14.5).
// Nothing in this file may be contracted into FMAs but the sum of squares.
#include "sgq_internal.h"

#pragma clang fp contract(off)

namespace sgq {
namespace {

constexpr int kBlock = 256;
constexpr int kV = 8;  // elements a thread takes at a time

// Eight elements at an address of their type's alignment.
template <typename T>
struct Eight {
    typedef T type __attribute__((ext_vector_type(kV), aligned(sizeof(T))));
};
typedef Eight<float>::type f32x8_u;

// round half away from zero(u * inv), at most 127 (as a NaN is).  |u * inv| stays
// below 127.5 but for a NaN, and adding the float below 0.5 with its sign before
// the truncation rounds every such value as roundf does.
__device__ __forceinline__ uint32_t code_of(float u, float inv) {
    const float v = fminf(u * inv, 127.0f);
    return (uint32_t)(int)(v + copysignf(0.49999997f, v)) & 0xFFu;
}

struct TokensArgs {
    const void* x;
    const void* r;  // residual, or null
    void* h;        // x + r
    const float* g; // the norm's weights
    float eps;
    int64_t ldx, ldr, ldh, ldc;
    int64_t M, K, Kpad;
    signed char* codes;
    float* scales;
};

// Sum of ss and maximum of m over NT threads of the workgroup (a wavefront, or all).
template <int NT>
__device__ __forceinline__ void row_reduce(float& ss, float& m, float (*red)[16]) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        ss += __shfl_xor(ss, o, 64);
        m = fmaxf(m, __shfl_xor(m, o, 64));
    }
    if constexpr (NT > 64) {
        __syncthreads();  // the last row's
        if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = ss, red[1][threadIdx.x >> 6] = m;
        __syncthreads();
        ss = red[0][0], m = red[1][0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) ss += red[0][w], m = fmaxf(m, red[1][w]);
    }
}

// Scale of a row, and m as the codes take it, from its sum of squares (KEEP: of v * 0)
// and its maximum.
template <bool NORM, bool KEEP>
__device__ __forceinline__ float row_scale(float ss, float& m, float K, float eps) {
    if constexpr (NORM) {
        const float rstd = 1.0f / sqrtf(ss / K + eps);
        m = fmaxf(m, 1e-8f / rstd);
        return m * rstd / 127.0f;
    } else {
        m = fmaxf(m, 1e-8f);
        return KEEP ? m / 127.0f + ss : m / 127.0f;
    }
}

// 127 / m, at most the largest float: without eps the norm of a row of zeros has m = 0, and
// an infinite factor would leave no zeros past K (nor the signs of values below 2^-126).
__device__ __forceinline__ float row_inv(float m) { return fminf(127.0f / m, 3.40282347e38f); }

// NT threads a row (a wavefront of several in a workgroup, or a workgroup), C
// chunks of eight elements a thread: the row stays in registers.
template <typename T, bool NORM, bool RES, bool KEEP, int NT, int C>
__global__ __launch_bounds__(NT < kBlock ? kBlock : NT) void k_tokens_row(const TokensArgs a) {
    __shared__ float red[2][16];
    constexpr int kRows = NT < kBlock ? kBlock / NT : 1;
    typedef typename Eight<T>::type T8;
    const int t = NT < kBlock ? threadIdx.x % NT : threadIdx.x;
    const int K = (int)a.K, nq = (int)(a.Kpad / kV);
    for (int64_t row = blockIdx.x * (int64_t)kRows + (NT < kBlock ? threadIdx.x / NT : 0); row < a.M;
         row += (int64_t)gridDim.x * kRows) {
        const T* x = (const T*)a.x + row * a.ldx;
        const T* r = RES ? (const T*)a.r + row * a.ldr : nullptr;
        T* h = RES ? (T*)a.h + row * a.ldh : nullptr;
        T8 xv[C], rv[C];
        f32x8_u gv[C];
        auto load_g = [&](f32x8_u& v, int k) {
            if (k + kV <= K) {
                v = *(const f32x8_u*)(a.g + k);
            } else {
#pragma unroll
                for (int e = 0; e < kV; ++e) v[e] = k + e < K ? a.g[k + e] : 0.0f;
            }
        };
        // Every load is issued before the first is used.
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int k = (t + i * NT) * kV;
            if (k + kV <= K) {
                xv[i] = *(const T8*)(x + k);
                if constexpr (RES) rv[i] = *(const T8*)(r + k);
            } else {
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    xv[i][e] = k + e < K ? x[k + e] : (T)0.0f;
                    if constexpr (RES) rv[i][e] = k + e < K ? r[k + e] : (T)0.0f;
                }
            }
            if constexpr (NORM) load_g(gv[i], k);
        }
        float u[C][kV], ss = 0.0f, m = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int k = (t + i * NT) * kV;
            if constexpr (RES) {
#pragma unroll
                for (int e = 0; e < kV; ++e) xv[i][e] = (T)((float)xv[i][e] + (float)rv[i][e]);
                if (k + kV <= K) {
                    *(T8*)(h + k) = xv[i];
                } else {
#pragma unroll
                    for (int e = 0; e < kV; ++e)
                        if (k + e < K) h[k + e] = xv[i][e];
                }
            }
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                float v = (float)xv[i][e];
                if constexpr (KEEP) ss = fmaf(v, 0.0f, ss);
                if constexpr (NORM) {
                    ss = fmaf(v, v, ss);
                    v = v * gv[i][e];
                }
                u[i][e] = v;
                m = fmaxf(m, fabsf(v));
            }
        }
        row_reduce<NT>(ss, m, red);
        const float scale = row_scale<NORM, KEEP>(ss, m, (float)K, a.eps), inv = row_inv(m);
        if (t == 0) a.scales[row] = scale;
        signed char* c = a.codes + row * a.ldc;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int q = t + i * NT;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < kV; ++e) w[e / 4] |= code_of(u[i][e], inv) << (8 * (e % 4));
            if (q < nq) *(uint2*)(c + q * kV) = make_uint2(w[0], w[1]);
        }
    }
}

// Longer rows, read again (from the caches) for the codes.  With the norm that is
// from 16384 on: x, the residual, g and u of four chunks do not fit the 128 registers
// that sixteen wavefronts leave a thread.
constexpr int kLoopBlock = 1024;
template <typename T, bool NORM, bool RES, bool KEEP>
__global__ __launch_bounds__(kLoopBlock) void k_tokens_loop(const TokensArgs a) {
    __shared__ float red[2][16];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.ldx;
        const T* r = RES ? (const T*)a.r + row * a.ldr : nullptr;
        T* h = RES ? (T*)a.h + row * a.ldh : nullptr;
        float ss = 0.0f, m = 0.0f;
#pragma unroll 4
        for (int64_t k = threadIdx.x; k < a.K; k += kLoopBlock) {
            float v = (float)x[k];
            if constexpr (RES) {
                const T t = (T)(v + (float)r[k]);
                h[k] = t;
                v = (float)t;
            }
            if constexpr (KEEP) ss = fmaf(v, 0.0f, ss);
            if constexpr (NORM) {
                ss = fmaf(v, v, ss);
                v = v * a.g[k];
            }
            m = fmaxf(m, fabsf(v));
        }
        row_reduce<kLoopBlock>(ss, m, red);
        const float scale = row_scale<NORM, KEEP>(ss, m, (float)a.K, a.eps), inv = row_inv(m);
        if (threadIdx.x == 0) a.scales[row] = scale;
        const T* src = RES ? h : x;  // each thread reads what it wrote
#pragma unroll 4
        for (int64_t k = threadIdx.x; k < a.Kpad; k += kLoopBlock) {
            float v = k < a.K ? (float)src[k] : 0.0f;
            if constexpr (NORM) v = k < a.K ? v * a.g[k] : 0.0f;
            a.codes[row * a.ldc + k] = (signed char)code_of(v, inv);
        }
    }
}

// Values of eight codes a thread.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_tokens_values(const signed char* __restrict__ codes, int64_t ldc,
                                                          const float* __restrict__ scales, int64_t M, int K,
                                                          T* __restrict__ out, int64_t ldo) {
    const int k = (blockIdx.x * kBlock + threadIdx.x) * kV;
    if (k >= K) return;
    for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
        const float s = scales[row];
        const uint2 w = *(const uint2*)(codes + row * ldc + k);  // within the row: it holds K rounded up to 128
        typename Eight<T>::type v;
#pragma unroll
        for (int e = 0; e < kV; ++e) v[e] = (T)((float)(signed char)((e < 4 ? w.x : w.y) >> (8 * (e % 4))) * s);
        T* o = out + row * ldo + k;
        if (k + kV <= K) {
            *(typename Eight<T>::type*)o = v;
        } else {
#pragma unroll
            for (int e = 0; e < kV - 1; ++e)
                if (k + e < K) o[e] = v[e];
        }
    }
}

constexpr int64_t kMaxRowGroups = (int64_t)1 << 20;  // workgroups of a launch (fewer than 2^32 threads)

// Threads of a row by its chunks q.  Measured (us, graphs; bf16 with a residual unless
// said): a wavefront against 256 threads, 4096 x 1024 7.5 / 10.0, but 2048 x 2048 8.3 / 7.6 and
// 8 x 2048 fp32 4.0 / 2.9; 256 threads of three chunks against four, 1023 x 5003 fp16 without
// 7.0 / 7.9; 512 of two against 256 of four, 8192 x 8192 84 / 87, 16 x 8192 3.9 / 4.3.  HBM bounds
// them from there: 2048 x 4096 11.3 us, 5.2 TB/s, 2048 x 11008 fp32 tokens 20.7, 5.4 TB/s (a large
// copy reaches 5.1); a few rows are one row's latency.
template <typename T, bool NORM, bool RES, bool KEEP>
hipError_t launch_rows(const TokensArgs& a, hipStream_t s) {
    const auto grid = [&](int rows) { return (unsigned)(ceil_div(a.M, rows) < kMaxRowGroups ? ceil_div(a.M, rows) : kMaxRowGroups); };
    const int64_t q = a.Kpad / kV;
    if (q <= 64)
        k_tokens_row<T, NORM, RES, KEEP, 64, 1><<<grid(4), kBlock, 0, s>>>(a);
    else if (q <= 128)
        k_tokens_row<T, NORM, RES, KEEP, 64, 2><<<grid(4), kBlock, 0, s>>>(a);
    else if (q <= 256)
        k_tokens_row<T, NORM, RES, KEEP, 256, 1><<<grid(1), 256, 0, s>>>(a);
    else if (q <= 512)
        k_tokens_row<T, NORM, RES, KEEP, 256, 2><<<grid(1), 256, 0, s>>>(a);
    else if (q <= 768)
        k_tokens_row<T, NORM, RES, KEEP, 256, 3><<<grid(1), 256, 0, s>>>(a);
    else if (q <= 1024)
        k_tokens_row<T, NORM, RES, KEEP, 512, 2><<<grid(1), 512, 0, s>>>(a);
    else if (q <= 2048)
        k_tokens_row<T, NORM, RES, KEEP, 512, 4><<<grid(1), 512, 0, s>>>(a);
    else if constexpr (!NORM) {
        if (q <= 4096)
            k_tokens_row<T, NORM, RES, KEEP, 1024, 4><<<grid(1), 1024, 0, s>>>(a);
        else
            k_tokens_loop<T, NORM, RES, KEEP><<<grid(1), kLoopBlock, 0, s>>>(a);
    } else {
        k_tokens_loop<T, NORM, RES, KEEP><<<grid(1), kLoopBlock, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const TokensArgs& a, bool keep, hipStream_t s) {
    if (!a.g) return keep ? launch_rows<T, false, false, true>(a, s) : launch_rows<T, false, false, false>(a, s);
    return a.r ? launch_rows<T, true, true, false>(a, s) : launch_rows<T, true, false, false>(a, s);
}

}  // namespace

hipError_t launch_tokens(const void* x, DType t, int64_t ldx, const void* r, int64_t ldr, void* h, int64_t ldh,
                         const float* g, float eps, bool keep_nan, int64_t M, int64_t K, void* codes, int64_t ldc,
                         float* scales, hipStream_t s) {
    TokensArgs a{};
    a.x = x, a.r = r, a.h = h, a.g = g, a.eps = eps;
    a.ldx = ldx, a.ldr = ldr, a.ldh = ldh, a.ldc = ldc;
    a.M = M, a.K = K, a.Kpad = K > 0 ? round_up(K, kTokenPadK) : kTokenPadK;
    a.codes = (signed char*)codes, a.scales = scales;
    return t == DType::f32 ? launch_t<float>(a, keep_nan, s)
                           : (t == DType::bf16 ? launch_t<__bf16>(a, keep_nan, s) : launch_t<_Float16>(a, keep_nan, s));
}

hipError_t launch_tokens_values(const void* codes, int64_t ldc, const float* scales, int64_t M, int64_t K, void* out,
                                DType t, int64_t ldo, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(K, kBlock * kV), (unsigned)(M < 32768 ? M : 32768));
    const signed char* c = (const signed char*)codes;
    if (t == DType::f32)
        k_tokens_values<float><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, (int)K, (float*)out, ldo);
    else if (t == DType::bf16)
        k_tokens_values<__bf16><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, (int)K, (__bf16*)out, ldo);
    else
        k_tokens_values<_Float16><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, (int)K, (_Float16*)out, ldo);
    return hipGetLastError();
}

}  // namespace sgq
