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

__global__ __launch_bounds__(kWG) void k_channels_top(const float* __restrict__ w, int64_t K, int64_t N, int64_t n0,
                                                      int64_t rows, uint32_t* __restrict__ top) {
    __shared__ float red[kWG / 64][64];
    const int64_t n = n0 + blockIdx.x * (int64_t)64 + (threadIdx.x & 63);
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

// Their bytes bound them: quantizing 4096 x 11008 takes 76 us (w read twice, the second
// time partly from the caches: 5.3 TB/s, a large copy reaches 5.1), 8192 x 28672 500 us
// (4.2 TB/s), unpacking 34 and 215 us (6.6 and 5.5 TB/s).  Packing fp32 codes of 8192 x
// 28672 takes 358 us with the wait for the flag (3.3 TB/s) and was left there: a weight is
// packed once.
//
// Codes of a kTileK x kTileN tile: FROM_CODES reads fp32 codes (validated into
// *bad), else w with the columns' maxima in top; through LDS into the layout.
template <bool FROM_CODES>
__global__ __launch_bounds__(kWG) void k_channels_pack(const float* __restrict__ src, int64_t K, int64_t N, int64_t nkt, int64_t t0,
                                                       const uint32_t* __restrict__ top, float* __restrict__ scales,
                                                       float* __restrict__ qdata, signed char* __restrict__ packed,
                                                       int* __restrict__ bad) {
#pragma clang fp contract(off)
    __shared__ __attribute__((aligned(16))) signed char col[kTileN][kTileK + 16];
    const int64_t kt = (t0 + blockIdx.x) % nkt, nt = (t0 + blockIdx.x) / nkt;
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
                                                         int64_t nkt, int64_t t0, const float* __restrict__ scales,
                                                         float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) signed char col[kTileN][kTileK + 16];
    const int64_t kt = (t0 + blockIdx.x) % nkt, nt = (t0 + blockIdx.x) / nkt;
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

// silu(g) * u.  With the whole number n nearest to g log2 e, within limits, and the rest
// f = n - g log2 e, which two fused operations give to 2^-25,
//   silu(g) = g / (1 + e^-g) = 2^n * g / (2^n + 2^f):
// the exponential's argument keeps its bits however large g is, and nothing overflows
// or is subnormal before the last step, down to the gates (-104) where silu leaves fp32.
// n's limits: from 43 on 2^f counts for nothing, and 2^-149 is the smallest number (f,
// which takes g itself, has what is left, and by it 2^f carries infinities and a NaN).
// The exponential and the reciprocal are the hardware's, each within a step.  Error over
// a million gates in each of eleven ranges of [-92, 100], in units of 2^-24: 0.9 rms, 3.3
// at most (expf and a division: 0.7 and 2.5, but zero from -88.7 on; g * -log2 e rounded
// into the exponential: 8 rms at -20, 32 at -85, zero from -87.3 on).  A 256 x 256 tile
// takes 64 of these a lane: 4096 x 4096 -> 11008 gated 319 us, 512 x 2048 -> 5632 17.7 (the
// rounded product 312 and 17.3; expf and a division 332 and 18.9).
__device__ __forceinline__ floatx4 silu_mul4(floatx4 g, floatx4 u) {
    constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f;  // their sum is log2 e to 48 bits
    floatx4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float n = rintf(__builtin_amdgcn_fmed3f(g[r] * kLog2e, -149.0f, 43.0f));
        const float f = fmaf(g[r], -kLog2eRest, fmaf(g[r], -kLog2e, n));
        const float s = __builtin_ldexpf(1.0f, (int)n);
        v[r] = g[r] * __builtin_amdgcn_rcpf(s + __builtin_amdgcn_exp2f(f)) * s * u[r];
    }
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

// ---- few tokens -----------------------------------------------------------

// A workgroup takes 16 MB tokens by 16 C columns (of NG weights); its NW wavefronts
// share K, a step of 64 k at a time in turn, with operands straight from memory: a
// lane's A operand is a chunk of the packed weight (column lane & 15, k chunk lane >>
// 4: a wavefront reads 1024 contiguous bytes), its B operand 16 codes of token lane &
// 15, so that it ends up with four neighbouring columns of one token.  The sums of
// the wavefronts are added through LDS; integers, so in any order.  The weight's bytes
// bound it (graphs of calls over weights that together pass the caches): 1 x 4096 -> 4096
// 5.0 us, 3.3 TB/s, 16 x 4096 -> 11008 gated 18.5 us, 4.9 TB/s, 8 x 8192 -> 28672 38.5 us, 6.1
// TB/s; below some 30 MB the launch and one latency.  With one row block a weight is read
// once and its loads are marked as streamed: from HBM 1 x 4096 -> 4096 5.0 us against 5.6
// without, 16 x 4096 -> 11008 gated 18.5 against 20.0 (a weight that the caches hold from
// the call before loses by it, 16 x 11008 -> 4096 11.9 against 10.2; the layers of a model
// come from HBM).
template <int NG, typename T, int MB, int C, int NW>
__global__ __launch_bounds__(64 * NW) void k_w8a8_few(const W8A8Args a, int mblocks, int xlog) {
    constexpr int B = MB * C * NG;  // 16 x 16 blocks of sums
    // Steps whose loads are in flight together.  Measured with 1 / 2 / 3 / 4 (us, bf16,
    // weights from HBM), one weight and the gated two:
    //   16 x 16, 16 x 4096 -> 11008   13.0 / 13.8 / 14.0 / 12.3   21.0 / 19.4 / 20.0 / 19.2
    //   32 x 16, 32 x 4096 -> 4096     8.2 /  8.1 /  8.8 /  7.9   10.8 / 11.1 / 11.8 / 10.9
    //   32 x 32, 48 x 4096 -> 4096     8.2 /  8.4 /  9.0 /  8.2   13.0 / 13.4 / 15.0 / 14.6
    //   64 x 32, 128 x 4096 -> 4096   12.9 / 13.4 / 14.2 / 13.4   18.1 / 17.4 / 21.3 / 22.3
    // One block of sums gains; from four on more of them gain little or lose, so it is not
    // single latencies that those forms wait for: their workgroups read tokens and weights
    // of 100 MB in all through the L2s in the last line, at 8 TB/s.
    constexpr int U = B >= 8 ? 1 : (B >= 4 ? 2 : 4);
    __shared__ i32x4 red[NW][B][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const ChannelsGeom geo(a.K, a.N);
    const int bs = xcd_swizzle(blockIdx.x, gridDim.x, xlog);  // row blocks of the same columns on one XCD
    const int64_t mb = bs % mblocks, cb0 = (int64_t)(bs / mblocks) * C;
    const int64_t m0 = mb * 16 * MB;
    const int rows = (int)min((int64_t)(16 * MB), a.M - m0), ncb = (int)min((int64_t)C, geo.NB - cb0);
    const int ldx = (int)a.ldx, cbytes = (int)geo.KC * 256, steps = (int)(geo.Kpad / 64);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(a.x + m0 * a.ldx, (uint32_t)((rows - 1) * ldx) + (uint32_t)geo.Kpad);
    __amdgpu_buffer_rsrc_t rw[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) rw[q] = make_rsrc(a.w[q] + cb0 * cbytes, (uint32_t)ncb * (uint32_t)cbytes);
    int xo[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) xo[i] = i * 16 + lr < rows ? (i * 16 + lr) * ldx + 16 * g : kOobOff;

    i32x4 acc[MB][NG * C];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int c = 0; c < NG * C; ++c) acc[i][c] = i32x4{0, 0, 0, 0};
    for (int st = wave; st < steps; st += NW * U) {
        i32x4 x[U][MB], w[U][NG * C];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Past the last step and the last column block: zeros.  The column block is in the
            // lane's offset, which a buffer's check is sure to count (on this card it counts the
            // scalar offset too).
            const int k = st + u * NW;
            const int wo = k < steps ? lane * 16 : kOobOff;
#pragma unroll
            for (int q = 0; q < NG; ++q)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    w[u][q * C + c] = __builtin_bit_cast(
                        i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw[q], wo + c * cbytes, k * 1024, MB == 1 ? kStreamPolicy : 0));
#pragma unroll
            for (int i = 0; i < MB; ++i)
                x[u][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, k < steps ? xo[i] : kOobOff, k * 64, 0));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < NG * C; ++c)
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    acc[i][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][c], x[u][i], acc[i][c], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int c = 0; c < NG * C; ++c) red[wave][i * NG * C + c][lane] = acc[i][c];
    __syncthreads();
    // A thread per four columns of a token.
    for (int t = threadIdx.x; t < MB * C * 64; t += 64 * NW) {
        const int b = t >> 6, i = b / C, c = b - i * C;
        const int64_t m = m0 + i * 16 + (t & 15), n = (cb0 + c) * 16 + 4 * ((t >> 4) & 3);
        i32x4 v[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            v[q] = red[0][i * NG * C + q * C + c][t & 63];
#pragma unroll 5
            for (int w = 1; w < NW; ++w) v[q] += red[w][i * NG * C + q * C + c][t & 63];
        }
        if (m >= a.M || n >= a.N) continue;
        const float sx = a.sx[m];
        floatx4 o = product4(v[0], sx, load4(a.sw[0], n, a.N), load4(a.bias[0], n, a.N));
        if constexpr (NG == 2) o = silu_mul4(o, product4(v[1], sx, load4(a.sw[1], n, a.N), load4(a.bias[1], n, a.N)));
        store4((T*)a.y + m * a.ldy, n, a.N, o);
    }
}

// Wavefronts of a workgroup with `blocks` 16 x 16 blocks a weight.  Up to two blocks:
// eight where K gives sixteen less than four steps each (us, sixteen -> eight: 1 x
// 2048 -> 2048 3.1 -> 2.5, 1 x 2048 -> 11008 7.5 -> 5.2; 1 x 4096 -> 4096 4.5 against
// 4.9, 16 x 11008 -> 4096 11.9 against 11.7).  More blocks: what LDS holds of their sums.
int few_waves(int blocks, int ng, int64_t K) {
    if (blocks <= 2) return K < 4096 ? 8 : 16;
    return (blocks <= 4 ? 16 : 8) / ng;
}

// K == 0: the biases.
template <int NG, typename T>
__global__ void k_w8a8_bias(const W8A8Args a) {
    for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y)
        for (int64_t n = 4 * (blockIdx.x * (int64_t)blockDim.x + threadIdx.x); n < a.N; n += 4 * (int64_t)gridDim.x * blockDim.x) {
            floatx4 o = load4(a.bias[0], n, a.N);
            if constexpr (NG == 2) o = silu_mul4(o, load4(a.bias[1], n, a.N));
            store4((T*)a.y + m * a.ldy, n, a.N, o);
        }
}

// ---- the tile kernel ------------------------------------------------------

typedef __attribute__((address_space(3))) void lds_void;

constexpr int kStage = 128;  // k per stage

// A workgroup of WM x WN wavefronts computes BM tokens by BN columns (of the NG weights
// together, so that the gated MLP's two products of an output are in one lane).  Both
// operands go to LDS by direct loads, 128 k a stage, in NB buffers; a wavefront reads
// each operand once for all of its products, and the weight's layout is its operands',
// so nothing is rearranged.
//
// What bounds it: at 8192 x 8192 -> 28672 (256 x 256 tiles, 1.35 to 1.40 ms, 2.8 POP/s; a library
// int8 product of the shape 1.66 ms) the matrix cores are busy 73 to 75% of the time with
// the clock at 1.65 GHz, the power limit: the same instructions alone, on operands of
// random bits, run at 3.3 to 3.4 POP/s (4.6 on zeros), and the 32 x 32 x 32 form is
// slower (1710 us against 1530 in the first tiles).  2048 x 4096 -> 4096 (128 x 256, one
// tile a CU, 29 to 31 us, the library 41): 22 us of stages, the rest the launch, the first
// loads and the stores.  Calls of it back to back gain 32 stages in 24.6 us, 2.8 POP/s again,
// and as much with all loads taken from one tile, so that memory is not what they wait
// for; on half of the CUs, with power to spare, a stage takes .55 us in place of .77.
// Smaller products wait for their stages' loads: a third and a fourth buffer take a 64 x
// 128 stage from .51 to .23 us and a 128 x 128 one from .61 to .48; where CUs hold several
// tiles, two buffers of 128 x 128 leave room for a second workgroup and do better (2048 x
// 4096 -> 4096 36 us against 39).
// Measured and not kept: a workgroup that takes its tiles one after another, the next
// one's first loads under the last products (4096 x 4096 -> 11008 176 us against 163: the
// loop over tiles left no registers); four wavefronts of 128 x 128 (1614 against 1440) or of
// 64 x 128 and 128 x 64 (128 x 256 tiles, 2048 x 4096 -> 4096 39 against 36): fewer LDS reads,
// but a SIMD's only wavefront waits for them.
template <int NG, int BM, int BN, int WM, int WN>
struct TileCfg {
    static constexpr int kThreads = 64 * WM * WN;
    static constexpr int TM = BM / WM / 16;       // token blocks of a wavefront
    static constexpr int TN = BN / WN / 16;       // column blocks of a wavefront, NG > 1: of all weights
    static constexpr int kXLoads = BM * kStage / 16 / kThreads;  // 16-byte loads a thread and stage
    static constexpr int kWLoads = BN * kStage / 16 / kThreads;
};

template <int NG, typename T, int BM, int BN, int WM, int WN, int NB>
__global__ __launch_bounds__(64 * WM * WN) void k_w8a8_tile(const W8A8Args a, int tiles_m, int tiles_n, int xlog,
                                                                   int KS, int* part) {
    using C = TileCfg<NG, BM, BN, WM, WN>;
    constexpr int TM = C::TM, TN = C::TN, kQuads = TM * TN / 4, kLoads = C::kXLoads + C::kWLoads, kReads = TM + TN;
    // Of n things issued between kQuads quads of products, those before quad q.
    constexpr auto part_of = [](int q, int n) { return q * n / kQuads; };
    // NB buffers of a stage, objects of their own: by them the compiler tells the loads a
    // read has to wait for from those it has not.
    constexpr int kX = BM * kStage, kW = BN * kStage;
    static_assert(NB >= 2 && NB <= 4, "buffers");
    __shared__ __attribute__((aligned(128))) signed char xs0[kX], xs1[kX], xs2[NB > 2 ? kX : 16], xs3[NB > 3 ? kX : 16];
    __shared__ __attribute__((aligned(128))) signed char ws0[kW], ws1[kW], ws2[NB > 2 ? kW : 16], ws3[NB > 3 ? kW : 16];
    __shared__ float esx[BM];
    __shared__ __attribute__((aligned(16))) float esw[BN], eb[BN];  // scales and biases, as the weights' blocks lie
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;

    // Tiles in groups of eight rows of tiles, column by column.
    // The K splits of a tile are neighbours.
    const int bs = xcd_swizzle(blockIdx.x, gridDim.x, xlog), b = bs / KS, split = bs - b * KS;
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
    const int stages = (int)(geo.Kpad / kStage), per = (stages + KS - 1) / KS;
    const int s0 = split * per, n = min(stages, s0 + per);  // stages s0 .. n - 1, at least one

    // A stage's loads, a 16-byte one of each thread at a time.  Tokens: eight rows of 128
    // bytes a wavefront, the chunk at place p of row r being chunk p ^ (r & 7) (no bank
    // twice when sixteen rows are read at one k).  Weights: the layout as it is, half a
    // column block a wavefront.  Past the last stage the buffers have no bytes: the loads
    // are issued (the compiler counts them to know which ones a read has to wait for)
    // and fetch nothing.
    const int xrow = lane >> 3, xoff = ((lane & 7) ^ xrow) * 16;
    auto load1 = [&](signed char* xs, signed char* ws, int s, int l) {
        if (l < C::kXLoads) {
            const __amdgpu_buffer_rsrc_t rx = make_rsrc(xp, s < n ? xbytes : 0);
            const int r = (l * (C::kThreads / 64) + wave) * 8;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_void*)(xs + r * kStage), 16, (r + xrow) * ldx + xoff,
                                                     s * kStage, 0, 0);
        } else {
            const int i = l - C::kXLoads, u = i * (C::kThreads / 64) + wave;  // of 1024 bytes
            const int q = NG == 1 ? 0 : i / (C::kWLoads / NG), v = NG == 1 ? u : u - q * (BN / NG / 8);
            const __amdgpu_buffer_rsrc_t rw = make_rsrc(a.w[q] + cb0 * cbytes, s < n ? wbytes : 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_void*)(ws + u * 1024), 16,
                                                     (v >> 1) * cbytes + (v & 1) * 1024 + lane * 16, s * 2048, 0, 0);
        }
    };
    // An operand of half a stage, 64 k: the first columns', the tokens', then the other
    // columns', as the products take them.
    auto read1 = [&](i32x4 (&x)[TM], i32x4 (&w)[TN], const signed char* xs, const signed char* ws, int h, int l) {
        if (l >= 1 && l <= TM) {
            const int i = l - 1;
            x[i] = *(const i32x4*)(xs + (wm * (BM / WM) + i * 16 + lr) * kStage + (((4 * h + g) ^ (lr & 7)) * 16));
        } else {
            // NG weights: each wavefront has the same columns of all.
            const int j = l == 0 ? 0 : l - TM;
            const int cb = NG == 1 ? wn * TN + j : (j / (TN / NG)) * (BN / 16 / NG) + wn * (TN / NG) + j % (TN / NG);
            w[j] = *(const i32x4*)(ws + cb * 2048 + h * 1024 + lane * 16);
        }
    };
    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    // Four products of half a stage.
    auto mfma4 = [&](const i32x4 (&x)[TM], const i32x4 (&w)[TN], int q) {
#pragma unroll
        for (int p = 4 * q; p < 4 * q + 4; ++p) {
            const int j = p / TM, i = p % TM;
            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x[i], acc[i][j], 0, 0, 0);
        }
    };

    i32x4 x0[TM], w0[TN], x1[TM], w1[TN];
    // The first stages and the scales and biases on their way together.
    auto load = [&](signed char* xs, signed char* ws, int s) {
#pragma unroll
        for (int l = 0; l < kLoads; ++l) load1(xs, ws, s, l);
    };
    load(xs0, ws0, s0);
    constexpr int kEX = (BM + C::kThreads - 1) / C::kThreads, kEW = (BN + C::kThreads - 1) / C::kThreads;
    float vx[kEX], vw[kEW], vb[kEW];
#pragma unroll
    for (int e = 0; e < kEX; ++e) {
        const int t = threadIdx.x + e * C::kThreads;
        vx[e] = t < rows ? a.sx[m0 + t] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < kEW; ++e) {
        const int t = threadIdx.x + e * C::kThreads, q = NG == 1 ? 0 : t / (BN / NG);
        const int64_t c = cb0 * 16 + t - q * (BN / NG);
        const float* sw = q == 0 ? a.sw[0] : a.sw[NG - 1];
        const float* b = q == 0 ? a.bias[0] : a.bias[NG - 1];
        const bool in = t < BN && c < a.N;
        vw[e] = in ? sw[c] : 0.0f;
        vb[e] = in && b ? b[c] : 0.0f;
    }
    load(xs1, ws1, s0 + 1);
    if constexpr (NB > 2) load(xs2, ws2, s0 + 2);
    if constexpr (NB > 3) load(xs3, ws3, s0 + 3);
#pragma unroll
    for (int e = 0; e < kEX; ++e)
        if (threadIdx.x + e * C::kThreads < BM) esx[threadIdx.x + e * C::kThreads] = vx[e];
#pragma unroll
    for (int e = 0; e < kEW; ++e)
        if (threadIdx.x + e * C::kThreads < BN) {
            esw[threadIdx.x + e * C::kThreads] = vw[e];
            eb[threadIdx.x + e * C::kThreads] = vb[e];
        }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((NB - 1) * kLoads) : "memory");
#pragma unroll
    for (int l = 0; l < kReads; ++l) read1(x0, w0, xs0, ws0, 0, l);
    // A stage: the products of its first half while the operands of the second are
    // read; all wavefronts are then done with its buffers, which the stage after the
    // next is loaded into while the products of the second half run and the first
    // operands of the next stage are read.  A load or read is issued every few products:
    // all of them at once held the products back until the queues had taken them (4096
    // x 8192 -> 4096 117 -> 104 us).
    auto step = [&](signed char* xs, signed char* ws, const signed char* xn, const signed char* wsn, int s) {
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
#pragma unroll
            for (int l = part_of(q, kReads); l < part_of(q + 1, kReads); ++l) read1(x1, w1, xs, ws, 1, l);
            __builtin_amdgcn_sched_barrier(0);
            mfma4(x0, w0, q);
            __builtin_amdgcn_sched_barrier(0);
        }
        // The next stage has come when all but the loads of the NB - 2 after it have.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((NB - 2) * kLoads) : "memory");
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
#pragma unroll
            for (int l = part_of(q, kReads); l < part_of(q + 1, kReads); ++l) read1(x0, w0, xn, wsn, 0, l);
#pragma unroll
            for (int l = part_of(q, kLoads); l < part_of(q + 1, kLoads); ++l) load1(xs, ws, s + NB, l);
            __builtin_amdgcn_sched_barrier(0);
            mfma4(x1, w1, q);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The buffers in turn; what is left past the last whole turn.
    int s = s0;
    for (; s + NB <= n; s += NB) {
        step(xs0, ws0, xs1, ws1, s);
        if constexpr (NB == 2) {
            step(xs1, ws1, xs0, ws0, s + 1);
        } else {
            step(xs1, ws1, xs2, ws2, s + 1);
            if constexpr (NB == 3) {
                step(xs2, ws2, xs0, ws0, s + 2);
            } else {
                step(xs2, ws2, xs3, ws3, s + 2);
                step(xs3, ws3, xs0, ws0, s + 3);
            }
        }
    }
    if (s < n) step(xs0, ws0, xs1, ws1, s);
    if constexpr (NB > 2)
        if (s + 1 < n) step(xs1, ws1, xs2, ws2, s + 1);
    if constexpr (NB > 3)
        if (s + 2 < n) step(xs2, ws2, xs3, ws3, s + 2);
    // No load may still be writing to LDS, which the results go through and which is
    // given away at the end.
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");

    // A lane has columns 4 g .. 4 g + 3 of a block, of token lr.
    const int col0 = wn * (TN / NG) * 16 + 4 * g;  // of the first block, in its weight
    const int64_t nb = cb0 * 16 + col0;
    if (KS > 1) {  // partial sums, [split][weight][M][16 NB]
        const int64_t np = geo.NB * 16;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int r = wm * (BM / WM) + i * 16 + lr;
            if (r >= rows) continue;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int q = j / (TN / NG);
                const int64_t nn = nb + 16 * (j - q * (TN / NG));
                if (nn < np) *(i32x4*)(part + ((split * NG + q) * a.M + m0 + r) * np + nn) = acc[i][j];
            }
        }
        return;
    }
    // Sixteen tokens at a time through a share of LDS of the wavefront's own, so that
    // neighbouring lanes store a row's 16-byte chunks: chunk c of row r lies at place
    // c ^ r (mod the chunks of a row).  Rows that begin with a 128-byte line are written
    // past the L2, which would else hold them until the kernel's end and write them back
    // at once; rows that share lines are left to the L2 to put together.  Measured (us,
    // bf16: stores from the registers, through LDS, past the L2): 4096 x 4096 -> 4096 58.6 /
    // 57.2 / 54.0, 2048 x 4096 -> 4096 35.2 / 34.7 / 33.0, 8192 x 8192 -> 28672 1447 / 1411 /
    // 1402; on 256 x 256 tiles 4096 x 4096 -> 5003 101 / 91 / 96.
    const bool whole = (((uintptr_t)a.y | (uintptr_t)(a.ldy * (int)sizeof(T))) & 127) == 0;
    constexpr int kCols = TN / NG * 16, kRowBytes = kCols * (int)sizeof(T), kChunks = kRowBytes / 16;
    constexpr int kRowsAt = 64 / kChunks, kPer = 16 / (int)sizeof(T);
    static_assert(WM * WN * 16 * kRowBytes <= BN * kStage, "the wavefronts' shares are in ws0");
    signed char* const share = ws0 + wave * 16 * kRowBytes;
    const int at_row = lane / kChunks, at_chunk = lane % kChunks;
    const int64_t col = cb0 * 16 + wn * kCols + at_chunk * kPer;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int r0 = wm * (BM / WM) + i * 16;
        const float sx = esx[r0 + lr];
#pragma unroll
        for (int j = 0; j < TN / NG; ++j) {
            const int c = col0 + 16 * j;
            floatx4 v = product4(acc[i][j], sx, *(const floatx4*)&esw[c], *(const floatx4*)&eb[c]);
            if constexpr (NG == 2)
                v = silu_mul4(v, product4(acc[i][j + TN / 2], sx, *(const floatx4*)&esw[c + BN / 2],
                                          *(const floatx4*)&eb[c + BN / 2]));
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
            const int byte = (16 * j + 4 * g) * (int)sizeof(T);
            *(T4*)(share + lr * kRowBytes + ((byte / 16) ^ (lr % kChunks)) * 16 + byte % 16) = o;
        }
        asm volatile("" ::: "memory");  // a wavefront's LDS accesses are in order
#pragma unroll
        for (int q = 0; q < (15 + kRowsAt) / kRowsAt; ++q) {
            const int row = q * kRowsAt + at_row;
            if (kRowsAt > 16 && row >= 16) continue;
            typedef T TP __attribute__((ext_vector_type(kPer)));
            typedef T TPu __attribute__((ext_vector_type(kPer), aligned(sizeof(T))));
            const TP o = *(const TP*)(share + row * kRowBytes + (at_chunk ^ (row % kChunks)) * 16);
            if (r0 + row < rows) {
                T* to = (T*)a.y + (m0 + r0 + row) * a.ldy + col;
                if (col + kPer <= a.N) {
                    if (whole)
                        __builtin_nontemporal_store(o, (TPu*)to);
                    else
                        *(TPu*)to = o;
                } else {
#pragma unroll
                    for (int e = 0; e < kPer - 1; ++e)
                        if (col + e < a.N) to[e] = o[e];
                }
            }
        }
        asm volatile("" ::: "memory");
    }
}

// y of the partial sums of KS splits.
template <int NG, typename T>
__global__ __launch_bounds__(kWG) void k_w8a8_reduce(const W8A8Args a, int KS, const int* __restrict__ part, int64_t np) {
    const int64_t n = 4 * (blockIdx.x * (int64_t)kWG + threadIdx.x);
    if (n >= a.N) return;
    for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y) {
        i32x4 v[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            const int* p = part + (q * a.M + m) * np + n;
            v[q] = *(const i32x4*)p;
            for (int s = 1; s < KS; ++s) v[q] += *(const i32x4*)(p + s * NG * a.M * np);
        }
        const float sx = a.sx[m];
        floatx4 o = product4(v[0], sx, load4(a.sw[0], n, a.N), load4(a.bias[0], n, a.N));
        if constexpr (NG == 2) o = silu_mul4(o, product4(v[1], sx, load4(a.sw[1], n, a.N), load4(a.bias[1], n, a.N)));
        store4((T*)a.y + m * a.ldy, n, a.N, o);
    }
}

template <int NG, typename T, int BM, int BN, int WM, int WN, int NB>
void launch_tile(const W8A8Args& a, int KS, int* part, hipStream_t s) {
    const int64_t tm = ceil_div(a.M, BM), tn = ceil_div(ChannelsGeom(a.K, a.N).NB, BN / 16 / NG);
    k_w8a8_tile<NG, T, BM, BN, WM, WN, NB>
        <<<(unsigned)(tm * tn * KS), 64 * WM * WN, 0, s>>>(a, (int)tm, (int)tn, xcd_log2(device_xcds(s)), KS, part);
    if (KS > 1) {
        const dim3 grid((unsigned)ceil_div(a.N, 4 * kWG), (unsigned)(a.M < 32768 ? a.M : 32768));
        k_w8a8_reduce<NG, T><<<grid, kWG, 0, s>>>(a, KS, part, ChannelsGeom(a.K, a.N).NB * 16);
    }
}

template <int NG, typename T, int MB, int C, int NW>
void launch_few(const W8A8Args& a, hipStream_t s) {
    const int64_t mbs = ceil_div(a.M, 16 * MB), cgs = ceil_div(ChannelsGeom(a.K, a.N).NB, C);
    const int xlog = xcd_log2(device_xcds(s));
    if constexpr (MB * C <= 2) {
        if (few_waves(MB * C, NG, a.K) == 8) {
            k_w8a8_few<NG, T, MB, C, 8><<<(unsigned)(mbs * cgs), 64 * 8, 0, s>>>(a, (int)mbs, xlog);
            return;
        }
    }
    k_w8a8_few<NG, T, MB, C, NW><<<(unsigned)(mbs * cgs), 64 * NW, 0, s>>>(a, (int)mbs, xlog);
}

template <int NG, typename T>
hipError_t launch_as(const W8A8Args& a, const W8A8Plan& p, int* part, hipStream_t s) {
    switch (p.form) {
        case W8A8Form::bias: {
            const dim3 grid((unsigned)min(ceil_div(a.N, 4 * kWG), (int64_t)4096), (unsigned)(a.M < 32768 ? a.M : 32768));
            k_w8a8_bias<NG, T><<<grid, kWG, 0, s>>>(a);
            break;
        }
        case W8A8Form::few1x1: launch_few<NG, T, 1, 1, 16>(a, s); break;
        case W8A8Form::few2x1: launch_few<NG, T, 2, 1, 16>(a, s); break;
        case W8A8Form::few2x2: launch_few<NG, T, 2, 2, 16 / NG>(a, s); break;
        case W8A8Form::few4x2: launch_few<NG, T, 4, 2, 8 / NG>(a, s); break;
        case W8A8Form::tile64x128: launch_tile<NG, T, 64, 128, 1, 4, 3>(a, p.KS, part, s); break;
        case W8A8Form::tile128: launch_tile<NG, T, 128, 128, 2, 2, 2>(a, p.KS, part, s); break;
        case W8A8Form::tile128deep: launch_tile<NG, T, 128, 128, 2, 2, 4>(a, p.KS, part, s); break;
        case W8A8Form::tile128x256: launch_tile<NG, T, 128, 256, 2, 4, 3>(a, p.KS, part, s); break;
        case W8A8Form::tile256: launch_tile<NG, T, 256, 256, 2, 4, 2>(a, p.KS, part, s); break;
    }
    return hipGetLastError();
}

template <int NG>
hipError_t launch_ng(const W8A8Args& a, const W8A8Plan& p, int* part, hipStream_t s) {
    return a.t == DType::f32 ? launch_as<NG, float>(a, p, part, s)
                             : (a.t == DType::bf16 ? launch_as<NG, __bf16>(a, p, part, s)
                                                   : launch_as<NG, _Float16>(a, p, part, s));
}

}  // namespace

// A launch holds fewer than 2^32 threads: f(first tile, tiles) over nkt times the
// column tiles.
constexpr int64_t kPackTiles = (int64_t)1 << 23;
template <typename F>
static void each_tiles(int64_t nkt, int64_t N, F f) {
    const int64_t tiles = nkt * ceil_div(N, kTileN);
    for (int64_t t = 0; t < tiles; t += kPackTiles) f(t, (unsigned)min(kPackTiles, tiles - t));
}

hipError_t launch_channels_quantize(const float* w, int64_t K, int64_t N, float* qdata, float* scales, void* packed,
                                    void* top, hipStream_t s) {
    k_channels_start<<<(unsigned)ceil_div(N, kWG), kWG, 0, s>>>((uint32_t*)top, N);
    if (K > 0) {
        constexpr int64_t rows = 256, cols = 64 * kPackTiles;
        for (int64_t n = 0; n < N; n += cols) {
            const dim3 grid((unsigned)ceil_div(min(cols, N - n), 64), (unsigned)ceil_div(K, rows));
            k_channels_top<<<grid, kWG, 0, s>>>(w, K, N, n, rows, (uint32_t*)top);
        }
    }
    const int64_t nkt = K > 0 ? ceil_div(K, kTileK) : 1;
    each_tiles(nkt, N, [&](int64_t t0, unsigned n) {
        k_channels_pack<false><<<n, kWG, 0, s>>>(w, K, N, nkt, t0, (const uint32_t*)top, scales, qdata,
                                                 K > 0 ? (signed char*)packed : nullptr, nullptr);
    });
    return hipGetLastError();
}

hipError_t launch_channels_pack(const float* codes, int64_t K, int64_t N, void* packed, int* bad, hipStream_t s) {
    const int64_t nkt = ceil_div(K, kTileK);
    each_tiles(nkt, N, [&](int64_t t0, unsigned n) {
        k_channels_pack<true><<<n, kWG, 0, s>>>(codes, K, N, nkt, t0, nullptr, nullptr, nullptr, (signed char*)packed, bad);
    });
    return hipGetLastError();
}

hipError_t launch_channels_unpack(const void* packed, int64_t K, int64_t N, const float* scales, float* out,
                                  hipStream_t s) {
    const int64_t nkt = ceil_div(K, kTileK);
    each_tiles(nkt, N, [&](int64_t t0, unsigned n) {
        k_channels_unpack<<<n, kWG, 0, s>>>((const signed char*)packed, K, N, nkt, t0, scales, out);
    });
    return hipGetLastError();
}

int64_t w8a8_plan_bytes(const W8A8Plan& p, int ng, int64_t M, int64_t K, int64_t N) {
    return p.KS > 1 ? (int64_t)p.KS * ng * M * ChannelsGeom(K, N).NB * 64 : 0;
}

// The form and the K splits with the least time by a model of a launch, in us: a form
// that puts w workgroups on a CU, each with st steps of K (stages of 128 k; a
// wavefront's steps of 64 k in the forms for few tokens), takes
//   fixed + max(alone * st, w * (step * st + end)), and at least 2 + the weights at 5 TB/s
// or at 36 GB/s a workgroup; a split of K 2.5 us and its partial sums at 3 TB/s more.
// The constants are fitted to 326 shapes (1 to 8192 tokens, K and N of 512 to 28672, one
// weight and two) with every form timed on each; the form this picks takes 1.03 times
// the fastest one's time on average, 1.11 times in one of ten.  For instance (us, 64 x
// 128 / 128 x 128 with two buffers / with four / 128 x 256 / 256 x 256): 333 x 2043 -> 5001 9.6 /
// 13.8 / 12.7 / 15.6 / 24.6, 1024 x 4096 -> 4096 23.4 / 24.4 / 20.2 / 23.7 / 38, 2048 x 4096 -> 4096
// 44 / 36 / 39 / 31 / 40, 4096 x 4096 -> 4096 86 / 69 / 75 / 61 / 54; 128 x 11008 -> 4096 on 64 x
// 128 (from HBM) without a split 40, with two 27, with four, its plan, 21, with eight 24.
// The forms for few tokens read a weight once for each of their row blocks: 48 x 4096 ->
// 4096 9.8 on 64 x 32 against 11.2, but 48 x 14336 -> 28672 132 against 73.
W8A8Plan w8a8_plan(int ng, int64_t M, int64_t K, int64_t N, int64_t cus) {
    W8A8Plan best;
    if (K == 0) return best;
    if (M <= 16) {  // one row block: a read of the weight, whatever the sizes
        best.form = W8A8Form::few1x1;
        return best;
    }
    static constexpr struct {
        W8A8Form form;
        int few, rows, cols;                  // rows and columns (of all weights) of a workgroup, in 16s for few
        struct { double fixed, alone, step, end; } t[2];  // one weight, two
    } forms[] = {
        {W8A8Form::few2x1, 1, 2, 1, {{1.0, .48, 1.0, 0.}, {1.0, 1.09, .88, 0.}}},
        {W8A8Form::few2x2, 1, 2, 2, {{1.75, .5, 1.07, 1.1}, {1.5, .85, .9, 1.3}}},
        {W8A8Form::few4x2, 1, 4, 2, {{1.4, .67, .74, 1.5}, {2.7, .7, .65, 1.2}}},
        {W8A8Form::tile64x128, 0, 64, 128, {{2.6, .226, .29, 1.25}, {2.6, .226, .29, 1.25}}},
        {W8A8Form::tile128, 0, 128, 128, {{3.4, .6, .46, 1.75}, {3.4, .6, .46, 1.75}}},
        {W8A8Form::tile128deep, 0, 128, 128, {{.2, .48, .45, 4.6}, {.2, .48, .45, 4.6}}},
        {W8A8Form::tile128x256, 0, 128, 256, {{0., .73, .74, 5.6}, {0., .73, .74, 5.6}}},
        {W8A8Form::tile256, 0, 256, 256, {{0., 1.33, 1.33, 7.2}, {0., 1.33, 1.33, 7.2}}},
    };
    constexpr int64_t kFewRows = 256, kFewBytes = 100 * 1000 * 1000, kMinSplitStages = 4;
    const ChannelsGeom g(K, N);
    const double cu = cus < 1 ? 1.0 : (double)cus;
    double least = 0.0;
    for (const auto& f : forms) {
        if (f.few && (M > kFewRows || ng * K * N > kFewBytes)) continue;
        const auto& t = f.t[ng - 1];
        for (int ks = 1; ks <= (f.few ? 1 : 8); ks *= 2) {
            const int64_t stages = g.Kpad / 128, per = ceil_div(stages, ks);
            if (ks > 1 && (per < kMinSplitStages || ceil_div(stages, per) != ks)) continue;
            double wgs, w, st;
            if (f.few) {
                wgs = (double)(ceil_div(M, 16 * f.rows) * ceil_div(g.NB, f.cols));
                w = wgs < cu ? 1.0 : wgs / cu;
                st = (double)ceil_div(2 * stages, few_waves(f.rows * f.cols, ng, K));
            } else {
                const int64_t n = ceil_div(M, f.rows) * ceil_div(g.NB, f.cols / 16 / ng) * ks;
                wgs = (double)n;
                w = (double)ceil_div(n, (int64_t)cu);
                st = (double)per;
            }
            const double busy = w * (t.step * st + t.end), alone = t.alone * st;
            double us = t.fixed + (busy > alone ? busy : alone);
            const double rate = wgs * 3.6e4 < 5.1e6 ? wgs * 3.6e4 : 5.1e6;  // bytes a us
            const double read = 2.0 + (double)(ng * K) * (double)N / rate;
            us = us > read ? us : read;
            if (ks > 1) us += 2.5 + (double)(ks * ng * 4) * (double)M * (double)N / 3.0e6;
            if (least == 0.0 || us < least) least = us, best.form = f.form, best.KS = ks;
        }
    }
    return best;
}

hipError_t launch_w8a8(const W8A8Args& a, int ng, const W8A8Plan& p, void* ws, hipStream_t s) {
    // A launch holds fewer than 2^32 threads: very wide or very many rows go in slices.
    constexpr int64_t kRows = (int64_t)1 << 26, kCols = (int64_t)1 << 24;
    if (a.M > kRows || a.N > kCols) {
        for (int64_t m = 0; m < a.M; m += kRows)
            for (int64_t n = 0; n < a.N; n += kCols) {
                W8A8Args b = a;
                b.M = min(kRows, a.M - m), b.N = min(kCols, a.N - n);
                b.x += m * a.ldx, b.sx += m;
                b.y = (char*)a.y + (m * a.ldy + n) * dtype_bytes(a.t);
                for (int q = 0; q < ng; ++q) {
                    b.w[q] += n / 16 * ChannelsGeom(a.K, a.N).KC * 256, b.sw[q] += n;
                    if (b.bias[q]) b.bias[q] += n;
                }
                const hipError_t e = launch_w8a8(b, ng, p, ws, s);
                if (e != hipSuccess) return e;
            }
        return hipSuccess;
    }
    return ng == 2 ? launch_ng<2>(a, p, (int*)ws, s) : launch_ng<1>(a, p, (int*)ws, s);
}

}  // namespace sgq
