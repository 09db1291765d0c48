// sgq_w8a8.hip -- int8 tokens times int8 weights on the matrix cores (gfx950),
// and the layout of such weights.
//
// Mathematics.  acc[m,n] = sum_k cx[m,k] * cw[k,n] in int32, exact while K * 128^2
// < 2^31, so neither the order of the sum nor a split of K changes a bit;
// y = (acc * sx[m]) * sw[n] + bias[n] in fp32, rounded once more to the output's
// type.  The gated form takes two such products and h = silu(gate) * up.
#include "sgq_device.h"
#include "sgq_internal.h"

namespace sgq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kWG = 256;

__device__ __forceinline__ float ref_max(float m, float a) { return (a > m) ? a : m; }

// ---- weights ------------------------------------------------------------

constexpr int kTileK = 128, kTileN = 64;  // of the pack kernels: one workgroup

// top[n] (bits of a float, starting at 1e-8) = max |w[k][n]|, NaN never winning.
// A maximum does not depend on the order the workgroups come in, and floats of
// one sign compare as their bits do.
__global__ void k_channels_start(uint32_t* __restrict__ top, int64_t N) {
    const int64_t n = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (n < N) top[n] = __float_as_uint(1e-8f);
}

__global__ __launch_bounds__(kWG) void k_channels_top(const float* __restrict__ w, int64_t K, int64_t N, int64_t rows,
                                                      uint32_t* __restrict__ top) {
    __shared__ float red[kWG / 64][64];
    const int64_t n = blockIdx.x * (int64_t)64 + (threadIdx.x & 63);
    const int64_t k0 = blockIdx.y * rows, k1 = min(K, k0 + rows);
    float m = 0.0f;
    if (n < N)
#pragma unroll 8
        for (int64_t k = k0 + (threadIdx.x >> 6); k < k1; k += kWG / 64) m = ref_max(m, fabsf(w[k * N + n]));
    red[threadIdx.x >> 6][threadIdx.x & 63] = m;
    __syncthreads();
    if (threadIdx.x < 64 && n < N) {
#pragma unroll
        for (int q = 1; q < kWG / 64; ++q) m = ref_max(m, red[q][threadIdx.x]);
        atomicMax(top + n, __float_as_uint(m));
    }
}

// Codes of a kTileK x kTileN tile: FROM_CODES reads fp32 codes (validated into
// *bad), else w with the columns' maxima in top; through LDS into the layout.
template <bool FROM_CODES>
__global__ __launch_bounds__(kWG) void k_channels_pack(const float* __restrict__ src, int64_t K, int64_t N, int64_t nkt,
                                                       const uint32_t* __restrict__ top, float* __restrict__ scales,
                                                       float* __restrict__ qdata, signed char* __restrict__ packed,
                                                       int* __restrict__ bad) {
#pragma clang fp contract(off)
    __shared__ __attribute__((aligned(16))) signed char col[kTileN][kTileK + 16];
    const int64_t kt = blockIdx.x % nkt, nt = blockIdx.x / nkt;
    const int c = threadIdx.x & 63;
    const int64_t n = nt * kTileN + c;
    float inv = 0.0f;
    if (!FROM_CODES && n < N) {
        const float m = __uint_as_float(top[n]);
        inv = 127.0f / m;
        if (kt == 0 && threadIdx.x < 64) scales[n] = m / 127.0f;
    }
    bool wrong = false;
    for (int r = threadIdx.x >> 6; r < kTileK; r += kWG / 64) {
        const int64_t k = kt * kTileK + r;
        float v = 0.0f;
        if (k < K && n < N) {
            v = src[k * N + n];
            if constexpr (FROM_CODES) {
                if (!(v == truncf(v) && v >= -128.0f && v <= 127.0f)) wrong = true, v = 0.0f;
            } else {
                v = roundf(v * inv);
                v = (v < 127.0f) ? v : 127.0f;
                v = (-127.0f < v) ? v : -127.0f;
                if (qdata) qdata[k * N + n] = v;
            }
        }
        col[c][r] = (signed char)(int)v;
    }
    if (wrong) atomicOr(bad, 1);
    if (!packed) return;
    __syncthreads();
    // Chunk t: column t % 16 of column block t / 128, k chunk (t / 16) % 8.
    const ChannelsGeom g(K, N);
    for (int t = threadIdx.x; t < kTileN * kTileK / 16; t += kWG) {
        const int cb = t >> 7, kc = (t >> 4) & 7, cc = t & 15;
        const int64_t gcb = nt * (kTileN / 16) + cb;
        if (gcb < g.NB)
            *(uint4*)(packed + ((gcb * g.KC + kt * (kTileK / 16) + kc) * 16 + cc) * 16) =
                *(const uint4*)&col[16 * cb + cc][16 * kc];
    }
}

// out[k][n] = code (* scales[n]).
__global__ __launch_bounds__(kWG) void k_channels_unpack(const signed char* __restrict__ packed, int64_t K, int64_t N,
                                                         int64_t nkt, const float* __restrict__ scales,
                                                         float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) signed char col[kTileN][kTileK + 16];
    const int64_t kt = blockIdx.x % nkt, nt = blockIdx.x / nkt;
    const ChannelsGeom g(K, N);
    for (int t = threadIdx.x; t < kTileN * kTileK / 16; t += kWG) {
        const int cb = t >> 7, kc = (t >> 4) & 7, cc = t & 15;
        const int64_t gcb = nt * (kTileN / 16) + cb;
        if (gcb < g.NB)
            *(uint4*)&col[16 * cb + cc][16 * kc] =
                *(const uint4*)(packed + ((gcb * g.KC + kt * (kTileK / 16) + kc) * 16 + cc) * 16);
    }
    __syncthreads();
    const int c = threadIdx.x & 63;
    const int64_t n = nt * kTileN + c;
    if (n >= N) return;
    const float s = scales ? scales[n] : 1.0f;
    for (int r = threadIdx.x >> 6; r < kTileK; r += kWG / 64) {
        const int64_t k = kt * kTileK + r;
        if (k < K) out[k * N + n] = scales ? (float)col[c][r] * s : (float)col[c][r];
    }
}

// ---- products -----------------------------------------------------------

// Four neighbouring values of type T at an address of T's alignment.
template <typename T>
struct Four {
    typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
typedef Four<float>::type f32x4_u;

// (acc * sx) * sw + bias of four neighbouring columns.
__device__ __forceinline__ floatx4 product4(i32x4 acc, float sx, floatx4 sw, floatx4 b) {
#pragma clang fp contract(off)
    floatx4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = ((float)acc[r] * sx) * sw[r] + b[r];
    return v;
}

// v rounded to T into columns n .. n + 3 of a row, those below N.
template <typename T>
__device__ __forceinline__ void store4(T* row, int64_t n, int64_t N, floatx4 v) {
    typename Four<T>::type o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (T)v[r];
    if (n + 4 <= N) {
        *(typename Four<T>::type*)(row + n) = o;
    } else {
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (n + r < N) row[n + r] = o[r];
    }
}

__device__ __forceinline__ floatx4 silu_mul4(floatx4 g, floatx4 u) {
    floatx4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = silu_f32(g[r]) * u[r];
    return v;
}

// v[n .. n + 3], zeros from N on or without v.
__device__ __forceinline__ floatx4 load4(const float* v, int64_t n, int64_t N) {
    if (v && n + 4 <= N) return *(const f32x4_u*)(v + n);
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    if (v)
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (n + r < N) o[r] = v[n + r];
    return o;
}

// A wavefront per 16 tokens by 16 columns, operands straight from memory.  A
// lane's A operand is a chunk of the packed weight (column lane & 15, k chunk lane
// >> 4), its B operand 16 codes of token lane & 15, so that it ends up with four
// neighbouring columns of one token.
template <int NG, typename T>
__global__ __launch_bounds__(kWG) void k_w8a8_simple(const W8A8Args a) {
    const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    const int64_t wave = (int64_t)blockIdx.x * (kWG / 64) + (threadIdx.x >> 6);
    const ChannelsGeom geo(a.K, a.N);
    if (wave >= geo.NB * ceil_div(a.M, 16)) return;
    const int64_t cb = wave % geo.NB, mb = wave / geo.NB;
    const int64_t m = mb * 16 + lr;
    const signed char* x = a.x + (m < a.M ? m : a.M - 1) * a.ldx + 16 * g;
    i32x4 acc[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) acc[q] = i32x4{0, 0, 0, 0};
    for (int64_t kc = 0; kc < geo.KC; kc += 4) {
        const i32x4 b = *(const i32x4*)(x + 16 * kc);
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            const i32x4 w = *(const i32x4*)(a.w[q] + ((cb * geo.KC + kc) * 16 + lane) * 16);
            acc[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, b, acc[q], 0, 0, 0);
        }
    }
    if (m >= a.M) return;
    const bool sums = a.K > 0;  // else the biases
    const float sx = sums ? a.sx[m] : 0.0f;
    const int64_t n = cb * 16 + 4 * g;
    floatx4 v = product4(acc[0], sx, load4(sums ? a.sw[0] : nullptr, n, a.N), load4(a.bias[0], n, a.N));
    if constexpr (NG == 2)
        v = silu_mul4(v, product4(acc[1], sx, load4(sums ? a.sw[1] : nullptr, n, a.N), load4(a.bias[1], n, a.N)));
    store4((T*)a.y + m * a.ldy, n, a.N, v);
}

// ---- the tile kernel ------------------------------------------------------

typedef __attribute__((address_space(3))) void lds_void;

constexpr int kStage = 128;  // k per stage

template <int NG, int BM, int BN, int WM, int WN>
struct TileCfg {
    static constexpr int kThreads = 64 * WM * WN;
    static constexpr int TM = BM / WM / 16;       // token blocks of a wavefront
    static constexpr int TN = BN / WN / 16;       // column blocks of a wavefront, NG > 1: of all weights
    static constexpr int kXLoads = BM * kStage / 16 / kThreads;  // 16-byte loads a thread and stage
    static constexpr int kWLoads = BN * kStage / 16 / kThreads;
};

template <int NG, typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_w8a8_tile(const W8A8Args a, int tiles_m, int tiles_n, int xlog) {
    using C = TileCfg<NG, BM, BN, WM, WN>;
    constexpr int TM = C::TM, TN = C::TN;
    __shared__ __attribute__((aligned(128))) signed char xs0[BM * kStage], xs1[BM * kStage];
    __shared__ __attribute__((aligned(128))) signed char ws0[BN * kStage], ws1[BN * kStage];
    __shared__ float esx[BM];
    __shared__ __attribute__((aligned(16))) float esw[BN], eb[BN];  // scales and biases, as the weights' blocks lie
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;

    // Tiles in groups of eight rows of tiles, column by column.
    const int b = xcd_swizzle(blockIdx.x, gridDim.x, xlog);
    constexpr int kGroup = 8;
    const int group = b / (kGroup * tiles_n), in = b - group * (kGroup * tiles_n);
    const int gm = min(kGroup, tiles_m - group * kGroup);
    const int tm = group * kGroup + in % gm, tn = in / gm;

    const int64_t m0 = (int64_t)tm * BM;
    const ChannelsGeom geo(a.K, a.N);
    const int64_t cb0 = (int64_t)tn * (BN / 16 / NG);  // first column block of each weight
    const int rows = (int)min((int64_t)BM, a.M - m0), ncb = (int)min((int64_t)(BN / 16 / NG), geo.NB - cb0);
    const int ldx = (int)a.ldx, cbytes = (int)geo.KC * 256;
    const signed char* const xp = a.x + m0 * a.ldx;
    const uint32_t xbytes = (uint32_t)((rows - 1) * ldx) + (uint32_t)geo.Kpad, wbytes = (uint32_t)ncb * (uint32_t)cbytes;
    const int n = (int)(geo.Kpad / kStage);

    // A stage's loads.  Tokens: eight rows of 128 bytes a wavefront and load, the 16-byte
    // chunk at place p of row r being chunk p ^ (r & 7) (no bank twice when sixteen rows
    // are read at one k).  Weights: the layout as it is, half a column block a load.
    const int xrow = lane >> 3, xoff = ((lane & 7) ^ xrow) * 16;
    // Past the last stage the buffers have no bytes: the loads are issued (the compiler
    // counts them to know which ones a read has to wait for) and fetch nothing.
    auto load = [&](signed char* xs, signed char* ws, int s) {
        const __amdgpu_buffer_rsrc_t rx = make_rsrc(xp, s < n ? xbytes : 0);
#pragma unroll
        for (int i = 0; i < C::kXLoads; ++i) {
            const int r = (i * (C::kThreads / 64) + wave) * 8;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_void*)(xs + r * kStage), 16, (r + xrow) * ldx + xoff, s * kStage, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < C::kWLoads; ++i) {
            const int u = i * (C::kThreads / 64) + wave;  // of 1024 bytes
            const int q = NG == 1 ? 0 : i / (C::kWLoads / NG);
            const int v = NG == 1 ? u : u - q * (BN / NG / 8);
            const __amdgpu_buffer_rsrc_t rw = make_rsrc(a.w[q] + cb0 * cbytes, s < n ? wbytes : 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_void*)(ws + u * 1024), 16, (v >> 1) * cbytes + (v & 1) * 1024 + lane * 16, s * 2048, 0, 0);
        }
    };
    // Operands of half a stage: 64 k.
    auto read = [&](i32x4 (&x)[TM], i32x4 (&w)[TN], const signed char* xs, const signed char* ws, int h) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            x[i] = *(const i32x4*)(xs + (wm * (BM / WM) + i * 16 + lr) * kStage + (((4 * h + g) ^ (lr & 7)) * 16));
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            // NG weights: each wavefront has the same columns of all.
            const int cb = NG == 1 ? wn * TN + j : (j / (TN / NG)) * (BN / 16 / NG) + wn * (TN / NG) + j % (TN / NG);
            w[j] = *(const i32x4*)(ws + cb * 2048 + h * 1024 + lane * 16);
        }
    };
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    auto mfma = [&](const i32x4 (&x)[TM], const i32x4 (&w)[TN]) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
    };

    i32x4 x0[TM], w0[TN], x1[TM], w1[TN];
    load(xs0, ws0, 0);
    for (int t = threadIdx.x; t < BM; t += C::kThreads) esx[t] = t < rows ? a.sx[m0 + t] : 0.0f;
    for (int t = threadIdx.x; t < BN; t += C::kThreads) {
        const int q = t / (BN / NG);
        const int64_t nn = cb0 * 16 + t - q * (BN / NG);
        esw[t] = nn < a.N ? a.sw[q][nn] : 0.0f;
        eb[t] = nn < a.N && a.bias[q] ? a.bias[q][nn] : 0.0f;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load(xs1, ws1, 1);
    read(x0, w0, xs0, ws0, 0);
    auto step = [&](signed char* xs, signed char* ws, const signed char* xn, const signed char* wsn, int s) {
        read(x1, w1, xs, ws, 1);
        __builtin_amdgcn_sched_barrier(0);
        mfma(x0, w0);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        load(xs, ws, s + 2);
        read(x0, w0, xn, wsn, 0);
        __builtin_amdgcn_sched_barrier(0);
        mfma(x1, w1);
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int s = 0; s < n - 1; s += 2) {
        step(xs0, ws0, xs1, ws1, s);
        step(xs1, ws1, xs0, ws0, s + 1);
    }
    if (n & 1) step(xs0, ws0, xs1, ws1, n - 1);
    // No load may still be writing to LDS when the workgroup's share of it is given away.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    // A lane has columns 4 g .. 4 g + 3 of a block, of token lr.
    const int col0 = wn * (TN / NG) * 16 + 4 * g;  // of the first block, in its weight
    const int64_t nb = cb0 * 16 + col0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int r = wm * (BM / WM) + i * 16 + lr;
        if (r >= rows) continue;
        const float sx = esx[r];
        T* row = (T*)a.y + (m0 + r) * a.ldy;
#pragma unroll
        for (int j = 0; j < TN / NG; ++j) {
            const int c = col0 + 16 * j;
            floatx4 v = product4(acc[i][j], sx, *(const floatx4*)&esw[c], *(const floatx4*)&eb[c]);
            if constexpr (NG == 2)
                v = silu_mul4(v, product4(acc[i][j + TN / 2], sx, *(const floatx4*)&esw[c + BN / 2],
                                          *(const floatx4*)&eb[c + BN / 2]));
            store4(row, nb + 16 * j, a.N, v);
        }
    }
}

template <int NG, typename T, int BM, int BN, int WM, int WN>
void launch_tile(const W8A8Args& a, hipStream_t s) {
    const int64_t tm = ceil_div(a.M, BM), tn = ceil_div(ChannelsGeom(a.K, a.N).NB, BN / 16 / NG);
    k_w8a8_tile<NG, T, BM, BN, WM, WN>
        <<<(unsigned)(tm * tn), 64 * WM * WN, 0, s>>>(a, (int)tm, (int)tn, xcd_log2(device_xcds(s)));
}

template <int NG, typename T>
hipError_t launch_as(const W8A8Args& a, hipStream_t s) {
    if (a.K > 0 && a.M > 128) {
        launch_tile<NG, T, 256, 256, 4, 2>(a, s);
    } else {
        const int64_t waves = ChannelsGeom(a.K, a.N).NB * ceil_div(a.M, 16);
        k_w8a8_simple<NG, T><<<(unsigned)ceil_div(waves, kWG / 64), kWG, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <int NG>
hipError_t launch_ng(const W8A8Args& a, hipStream_t s) {
    return a.t == DType::f32 ? launch_as<NG, float>(a, s)
                             : (a.t == DType::bf16 ? launch_as<NG, __bf16>(a, s) : launch_as<NG, _Float16>(a, s));
}

}  // namespace

hipError_t launch_channels_quantize(const float* w, int64_t K, int64_t N, float* qdata, float* scales, void* packed,
                                    void* top, hipStream_t s) {
    k_channels_start<<<(unsigned)ceil_div(N, kWG), kWG, 0, s>>>((uint32_t*)top, N);
    const int64_t rows = 256;
    if (K > 0) {
        const dim3 grid((unsigned)ceil_div(N, 64), (unsigned)ceil_div(K, rows));
        k_channels_top<<<grid, kWG, 0, s>>>(w, K, N, rows, (uint32_t*)top);
    }
    const int64_t nkt = K > 0 ? ceil_div(K, kTileK) : 1;
    k_channels_pack<false><<<(unsigned)(nkt * ceil_div(N, kTileN)), kWG, 0, s>>>(
        w, K, N, nkt, (const uint32_t*)top, scales, qdata, K > 0 ? (signed char*)packed : nullptr, nullptr);
    return hipGetLastError();
}

hipError_t launch_channels_pack(const float* codes, int64_t K, int64_t N, void* packed, int* bad, hipStream_t s) {
    const int64_t nkt = ceil_div(K, kTileK);
    k_channels_pack<true><<<(unsigned)(nkt * ceil_div(N, kTileN)), kWG, 0, s>>>(codes, K, N, nkt, nullptr, nullptr,
                                                                               nullptr, (signed char*)packed, bad);
    return hipGetLastError();
}

hipError_t launch_channels_unpack(const void* packed, int64_t K, int64_t N, const float* scales, float* out,
                                  hipStream_t s) {
    const int64_t nkt = ceil_div(K, kTileK);
    k_channels_unpack<<<(unsigned)(nkt * ceil_div(N, kTileN)), kWG, 0, s>>>((const signed char*)packed, K, N, nkt,
                                                                           scales, out);
    return hipGetLastError();
}

int64_t w8a8_workspace_bytes(int, int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_w8a8(const W8A8Args& a, int ng, void*, hipStream_t s) {
    return ng == 2 ? launch_ng<2>(a, s) : launch_ng<1>(a, s);
}

}  // namespace sgq
