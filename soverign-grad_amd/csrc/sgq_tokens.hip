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
// Nothing in this file may be contracted into FMAs but the sum of squares.
#include "sgq_internal.h"

#pragma clang fp contract(off)

namespace sgq {
namespace {

constexpr int kBlock = 256;
__device__ __forceinline__ float ref_max(float m, float a) { return (a > m) ? a : m; }

__device__ __forceinline__ int code_of(float u, float inv) {
    const float v = roundf(u * inv);
    const float m = (v < 127.0f) ? v : 127.0f;  // NaN gives 127, as the weights' quantizer does
    return (int)((-127.0f < m) ? m : -127.0f);
}

struct TokensArgs {
    const void* x;
    const void* r;  // residual, or null
    void* h;        // x + r
    const float* g; // the norm's weights
    float eps;
    int64_t ldx, ldr, ldh, ldc;
    int64_t K, Kpad;
    signed char* codes;
    float* scales;
};

// One workgroup per row, the row read again for the codes.
template <typename T, bool NORM, bool RES>
__global__ __launch_bounds__(kBlock) void k_tokens(const TokensArgs a) {
    __shared__ float red[2][kBlock / 64];
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ldx;
    const T* r = RES ? (const T*)a.r + row * a.ldr : nullptr;
    T* h = RES ? (T*)a.h + row * a.ldh : nullptr;
    float ss = 0.0f, m = NORM ? 0.0f : 1e-8f;
    for (int64_t k = threadIdx.x; k < a.K; k += kBlock) {
        float v = (float)x[k];
        if constexpr (RES) {
            const T t = (T)(v + (float)r[k]);
            h[k] = t;
            v = (float)t;
        }
        if constexpr (NORM) {
            ss = fmaf(v, v, ss);
            v = v * a.g[k];
        }
        m = ref_max(m, fabsf(v));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        ss += __shfl_xor(ss, o, 64);
        m = ref_max(m, __shfl_xor(m, o, 64));
    }
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = ss, red[1][threadIdx.x >> 6] = m;
    __syncthreads();
    ss = red[0][0], m = red[1][0];
#pragma unroll
    for (int w = 1; w < kBlock / 64; ++w) ss += red[0][w], m = ref_max(m, red[1][w]);
    float scale;
    if constexpr (NORM) {
        const float rstd = 1.0f / sqrtf(ss / (float)a.K + a.eps);
        m = ref_max(m, 1e-8f / rstd);
        scale = m * rstd / 127.0f;
    } else {
        scale = m / 127.0f;
    }
    const float inv = 127.0f / m;
    if (threadIdx.x == 0) a.scales[row] = scale;
    const T* src = RES ? h : x;
    for (int64_t k = threadIdx.x; k < a.Kpad; k += kBlock) {
        int c = 0;
        if (k < a.K) {
            float v = (float)src[k];
            if constexpr (NORM) v = v * a.g[k];
            c = code_of(v, inv);
        }
        a.codes[row * a.ldc + k] = (signed char)c;
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_tokens_values(const signed char* __restrict__ codes, int64_t ldc,
                                                          const float* __restrict__ scales, int64_t M, int64_t K,
                                                          T* __restrict__ out, int64_t ldo) {
    for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
        const float s = scales[row];
        for (int64_t k = blockIdx.x * (int64_t)kBlock + threadIdx.x; k < K; k += (int64_t)gridDim.x * kBlock)
            out[row * ldo + k] = (T)((float)codes[row * ldc + k] * s);
    }
}

template <typename T>
hipError_t launch_t(const TokensArgs& a, int64_t M, hipStream_t s) {
    const unsigned grid = (unsigned)M;
    if (!a.g)
        k_tokens<T, false, false><<<grid, kBlock, 0, s>>>(a);
    else if (!a.r)
        k_tokens<T, true, false><<<grid, kBlock, 0, s>>>(a);
    else
        k_tokens<T, true, true><<<grid, kBlock, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tokens(const void* x, DType t, int64_t ldx, const void* r, int64_t ldr, void* h, int64_t ldh,
                         const float* g, float eps, int64_t M, int64_t K, void* codes, int64_t ldc, float* scales,
                         hipStream_t s) {
    TokensArgs a{};
    a.x = x, a.r = r, a.h = h, a.g = g, a.eps = eps;
    a.ldx = ldx, a.ldr = ldr, a.ldh = ldh, a.ldc = ldc;
    a.K = K, a.Kpad = round_up(K, kTokenPadK);
    a.codes = (signed char*)codes, a.scales = scales;
    return t == DType::f32 ? launch_t<float>(a, M, s)
                           : (t == DType::bf16 ? launch_t<__bf16>(a, M, s) : launch_t<_Float16>(a, M, s));
}

hipError_t launch_tokens_values(const void* codes, int64_t ldc, const float* scales, int64_t M, int64_t K, void* out,
                                DType t, int64_t ldo, hipStream_t s) {
    const dim3 grid((unsigned)(ceil_div(K, kBlock) < 1024 ? ceil_div(K, kBlock) : 1024), (unsigned)(M < 32768 ? M : 32768));
    const signed char* c = (const signed char*)codes;
    if (t == DType::f32)
        k_tokens_values<float><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, K, (float*)out, ldo);
    else if (t == DType::bf16)
        k_tokens_values<__bf16><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, K, (__bf16*)out, ldo);
    else
        k_tokens_values<_Float16><<<grid, kBlock, 0, s>>>(c, ldc, scales, M, K, (_Float16*)out, ldo);
    return hipGetLastError();
}

}  // namespace sgq
