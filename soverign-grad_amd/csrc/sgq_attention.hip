// sgq_attention.hip -- attention of new tokens over a paged key/value cache, for gfx950.
//
// Mathematics.  Row i of a sequence (position p) sees the keys of one interval [lo, hi)
// (causal, window, document start, prefix); with s_j its scores
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j,
// in one pass over the keys with a running maximum: when it grows from m to m', what
// was summed is multiplied by exp(m - m').  Ranges of keys that different workgroups (or
// wavefronts) took are joined the same way.  Scores, softmax and sums are fp32; in
// 16-bit types a weight is rounded to the type before its product with v, for the matrix
// instruction takes it so (half a step of each weight, while the sum of weights keeps them
// unrounded); fp32 stays fp32 throughout.
//
// Matrix layout.  A wavefront owns 32 rows (a row: a new token and one of the heads that
// share a kv head, heads next to each other) and computes transposed: S^T = K Q^T and O^T =
// V^T P^T with 32 x 32 products.  Column = row of the batch = lane & 31, so a row's
// maximum, sum and factor are one register of a lane, and the only exchange is with lane ^ 32,
// which has the other half of the keys.  The result registers of S^T are, in order, the
// B operand of the second product, if the k slots of that product are the keys in the order
// that the registers hold them: lane half h has keys 8 a + 4 h + 0..3 of each 32, and the A
// operand V^T is read in the same order.
//   16 bits: 32x32x16; K rows as 16-byte LDS reads, V^T by transposing 8-byte LDS reads
//   (four keys of a column a lane).
//   fp32: 32x32x2; a 16-byte read of K serves four products; V^T a float a lane.
// Keys and values go from their pages to LDS directly, the 16-byte chunks of a row permuted so
// that all reads are free of conflicts (counted: none).
//
// Forms.  Up to 32 rows of a sequence and kv head (single tokens, and a few): k_attend_few, or
// k_attend_lanes for up to four in fp32; more: k_attend_tiles.  Where their workgroups are too
// few for the device the keys are split, and k_attend_join joins the splits.
#include "sgq_lanes.h"
#include "sgq_paged.h"

#include <algorithm>
#include <type_traits>

namespace sgq {
namespace {

constexpr float kLog2e = 1.44269504f;
constexpr float kGrowth = 8.0f;  // a running maximum is raised where a score's weight passes 2^kGrowth
// How much lower (in powers of two) the weights of a row are held where a sum came out not finite: those of 2^30 keys sum to a
// quarter then, so that no sum of values passes what the largest of them is.
constexpr float kLower = 32.0f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Sixteen bytes that a lane without a row of its own reads: zeros.
__device__ const uint32_t g_zeros[4] = {0, 0, 0, 0};

template <typename T>
struct Mat;
template <>
struct Mat<__bf16> {
    typedef b16x8 Frag;
    static constexpr int kStep = 16;  // head elements of a fragment, both lane halves together
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mat<_Float16> {
    typedef h16x8 Frag;
    static constexpr int kStep = 16;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mat<float> {
    typedef f32x4 Frag;
    static constexpr int kStep = 8;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

constexpr int pow2_from(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// A tile of keys (or values) in LDS: rows of kRow bytes, chunk c of row r at position c ^ mix(r).
template <typename T, int DP>
struct TileRows {
    static constexpr int kRow = pow2_from(DP * (int)sizeof(T));
    static constexpr int kChunks = kRow / 16;
    // 16 bits: sixteen neighbouring rows have their chunk c in sixteen places of 256 bytes (K),
    // four neighbouring rows their 64 bytes in four places (V).  fp32: sixteen rows likewise,
    // rows four apart their 128 bytes in two places.
    static __device__ __forceinline__ int mix(int r) {
        if constexpr (sizeof(T) == 4) return ((r & 4) << 1) | ((r & 3) << 1) | ((r >> 3) & 1);
        if constexpr (kChunks == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
        return ((r & 3) << 2) | ((r >> 2) & 3);
    }
};

// The keys [lo, hi) that a row at position p sees.
__device__ __forceinline__ void row_keys(const AttendArgs& a, const SeqRows& r, int b, int row, int p, int& lo, int& hi) {
    lo = a.first_key ? max(a.first_key[row], 0) : 0;
    if (a.window > 0) lo = max(lo, p - a.window + 1);
    hi = p + 1;
    if (a.prefix) hi = max(hi, min(a.prefix[b], r.len));
}

// A row's column as T: its sum over that of the weights (inv: one over it).  A mean is no larger than the largest of the values,
// but rounded weights, and sums, may take it past the type's range by their last steps.
template <typename T>
__device__ __forceinline__ T mean(float sum, float inv) {
    constexpr float top = std::is_same_v<T, _Float16> ? 65504.0f : std::is_same_v<T, __bf16> ? 0x1.FEp127f : 0x1.FFFFFEp127f;
    const float x = sum * inv;
    return (T)(isfinite(sum) && inv == inv ? __builtin_amdgcn_fmed3f(x, -top, top) : x);
}

__device__ __forceinline__ float other_half(float v, bool take_max) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
    return take_max ? fmaxf(x, y) : x + y;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ int wave_max(int v) { return -wave_min(-v); }

// How scores become weights, the same for all of a launch.
struct Score {
    float c;         // exponent of 2 per raw score (without a cap)
    float in, out;   // cap: 2^ of out * tanh(in * raw)
    bool negate;     // scale < 0: the queries are negated instead
    bool capped, sloped;
    __device__ __forceinline__ explicit Score(const AttendArgs& a) {
        negate = a.scale < 0.0f;
        capped = a.softcap > 0.0f;
        sloped = a.slopes != nullptr;
        in = capped ? fminf(fabsf(a.scale) / a.softcap, 1.0e30f) : 0.0f;  // times 0 has to be 0
        out = a.softcap * kLog2e;
        // Never zero: a hidden score is -inf, and has to stay that.
        c = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);
    }
};

// A wavefront's 32 rows on tiles of 32 NK keys.
template <typename T, int DP, int NK>
struct Rows {
    typedef Mat<T> M;
    typedef typename M::Frag Frag;
    typedef TileRows<T, DP> Tile;
    static constexpr int kFrags = DP / M::kStep, kCols = DP / 32;
    // Weights and their sum are 2^kLift times what they are, which without it is 2^8 at most (softmax() says why).  With 2^-8
    // they are 1 at most, so that a sum of large values passes fp32's range no sooner than with a maximum that is raised at once.
    // In fp16, which has steps of 2^-24 only below 2^-14, those of many keys beside a large one would be off
    // together (4095 of e^-14.5: 5%); its values are 2^16 at most, and the weights go up to 2^15.
    static constexpr float kLift = std::is_same_v<T, _Float16> ? 7.0f : -kGrowth;

    Frag q[kFrags];
    f32x16 o[kCols];
    f32x16 s[NK];  // scores of a tile
    std::conditional_t<sizeof(T) == 4, f32x16, Frag> p[sizeof(T) == 4 ? NK : 2 * NK];  // weights of a tile
    float m, l;            // maximum of the scores (as c multiplies them), this half's sum of weights
    int lo, hi, pos;       // the row's keys and position
    float slope;           // times log2 e
    float lower = 0.0f;    // weights are 2^-lower times what kLift makes them: 0 or kLower
    int max_lo, min_hi, min_lo, max_hi;  // over the wavefront's rows

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kCols; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
        m = -INFINITY, l = 0.0f;
    }
    // Elements kStep i + (kStep / 2) half + 0 .. of the row's query, zeros from d on.
    __device__ __forceinline__ void load(const T* p, int d, bool negate) {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int i = 0; i < kFrags; ++i) {
            const int e = i * M::kStep + h * (M::kStep / 2);
            const Frag f = *(const Frag*)(p + min(e, d - M::kStep / 2)), none = {};
            q[i] = e < d ? (negate ? -f : f) : none;
        }
    }
    __device__ __forceinline__ void bounds() {
        max_lo = __builtin_amdgcn_readfirstlane(wave_max(lo)), min_hi = __builtin_amdgcn_readfirstlane(wave_min(hi));
        min_lo = __builtin_amdgcn_readfirstlane(wave_min(lo)), max_hi = __builtin_amdgcn_readfirstlane(wave_max(hi));
    }

    // Whether some row does not see some key of the tile at k0.
    __device__ __forceinline__ bool part(int k0) const { return k0 < max_lo || k0 + 32 * NK > min_hi; }

    // Scores of the keys from k0 on to weights, the sum and, where the maximum grows, the factor of what was summed.
    // LOWER: lower may be other than 0.
    template <bool LOWER>
    __device__ __forceinline__ void softmax(int k0, const Score& sc) {
        const int h = (threadIdx.x & 63) >> 5;
        // Key of register e of tile t: k0 + 32 t + 8 (e / 4) + 4 h + e % 4.
        const int kb = k0 + 4 * h;
        float c = sc.c;
        if (sc.capped || sc.sloped) c = 1.0f;
        if (sc.capped) {
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (sizeof(T) == 4) {
                        s[t][e] = sc.out * tanhf(s[t][e] * sc.in);
                    } else {
                        // tanh x = 1 - 2 / (1 + e^2x): off by some 2^-23 of the cap, which is 1024 at most here, and a
                        // 16-bit weight does not see it.  (With a series for the small x of
                        // wider caps 4 prompts of 8192 tokens, without a cap, took 4.49 ms instead of 4.22.)
                        const float u = __builtin_amdgcn_exp2f(s[t][e] * (2.0f * kLog2e * sc.in));
                        s[t][e] = fmaf(sc.out * -2.0f, __builtin_amdgcn_rcpf(1.0f + u), sc.out);
                    }
                }
        } else if (sc.sloped) {
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[t][e] *= sc.c;
        }
        if (sc.sloped)
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[t][e] = fmaf(-slope, (float)abs(pos - (kb + 32 * t + 8 * (e / 4) + e % 4)), s[t][e]);
        if (part(k0)) {
            const unsigned width = (unsigned)max(hi - lo, 0);
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if ((unsigned)(kb + 32 * t + 8 * (e / 4) + e % 4 - lo) >= width) s[t][e] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
        top = other_half(top, true);
        // The factor of what was summed is due only where a maximum grew by more than 2^8: until
        // then weights are up to 2^8 (times 2^kLift) and sums as exact as before.
        if (__any((top - m) * c > kGrowth)) {
            const float now = fmaxf(m, top);
            const float w = __builtin_amdgcn_exp2f((m - (now == -INFINITY ? 0.0f : now)) * c);
            m = now;
            l *= w;
#pragma unroll
            for (int i = 0; i < kCols; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= w;
        }
        // exp2(s c - m c) with m c rounded has one instruction for the exponent.  What is lost of m c, 2^-24 of it, is the same
        // for all keys under one maximum, but from 2^28 on it takes weights past the type's range: scores past 2^12 have
        // the maximum taken off first.
        const float lift = LOWER ? kLift - lower : kLift;
        float base = m == -INFINITY ? 0.0f : fmaf(-m, c, lift);
        if (__builtin_expect(__any(fabsf(base) > 4096.0f), 0)) {
            const float off = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[t][e] -= off;
            base = lift;
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, base));
                sum[e & 3] += w;
                if constexpr (sizeof(T) == 4)
                    p[t][e] = w;
                else
                    p[2 * t + e / 8][e % 8] = (T)w;
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // S^T of the keys in the tile at ks.  The LDS reads of four products are issued ahead of the four before
    // them; left alone, the compiler reads for each product as it comes and waits.  beside(g): what is issued
    // beside the g-th four.
    // (One ahead of one for the widest heads in 16 bits, which leave few registers: 1024 rows of 16 heads of 256, a window of
    // 4096 keys 123 us, with two 127, with four 160.)
    static constexpr int kAhead = DP == 256 && sizeof(T) == 2 ? 1 : 4, kScoreGroups = (kFrags * NK + kAhead - 1) / kAhead;
    template <typename F>
    __device__ __forceinline__ void scores(const char* ks, F beside) {
        const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
        const int x = (h ^ Tile::mix(n)) << 4;  // chunk 2 i + h of row n (mix has the period of 16 rows)
        const char* const row = ks + n * Tile::kRow;
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = 0.0f;
        constexpr int N = kFrags * NK, G = kAhead;
        auto read = [&](int j) { return *(const Frag*)(row + j % NK * 32 * Tile::kRow + ((j / NK * 32) ^ x)); };
        Frag f[2][G];
#pragma unroll
        for (int j = 0; j < G; ++j) f[0][j] = read(j);
#pragma unroll
        for (int g = 0; g < (N + G - 1) / G; ++g) {
#pragma unroll
            for (int j = 0; j < G; ++j)
                if ((g + 1) * G + j < N) f[(g + 1) & 1][j] = read((g + 1) * G + j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const int i = g * G + j;
                if (i < N) s[i % NK] = M::mma(f[g & 1][j], q[i / NK], s[i % NK]);
            }
            beside(g);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // O^T += V^T P^T with the values in the tile at vs.
    __device__ __forceinline__ void values(const char* vs) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // A 16-lane group reads four keys of sixteen columns, a lane eight bytes of them.
            const int i = lane & 15, r0 = 4 * h + (i >> 2);
            const int x = ((2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ Tile::mix(r0)) << 4;
            const char* const row = vs + r0 * Tile::kRow + 8 * (i & 1);
            constexpr int kNext = 2 << 4;  // how mix moves a chunk in a row eight further
#pragma unroll
            for (int u = 0; u < 2 * NK; ++u)
#pragma unroll
                for (int cidx = 0; cidx < kCols; ++cidx) {
                    const char* const at = row + u * 16 * Tile::kRow;
                    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + ((cidx * 64) ^ x)));
                    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(at + 8 * Tile::kRow + ((cidx * 64) ^ x ^ kNext)));
                    const Frag v = __builtin_bit_cast(Frag, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[cidx] = M::mma(v, p[u], o[cidx]);
                }
        } else {
            const int n = lane & 31;
#pragma unroll
            for (int t = 0; t < NK; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = t * 32 + 8 * (e / 4) + 4 * h + e % 4;
                    const char* row = vs + r * Tile::kRow + 4 * (n & 3);
                    const int x = ((n >> 2) ^ Tile::mix(r)) << 4;
#pragma unroll
                    for (int cidx = 0; cidx < kCols; ++cidx)
                        o[cidx] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(const float*)(row + ((cidx * 128) ^ x)), p[t][e],
                                                                       o[cidx], 0, 0, 0);
                }
        }
    }
    // Whether a column of the row is not finite (those from d on are zeros), though its sum of weights is: then a sum of zeros
    // times the columns is a NaN.  (An instruction a column; asking each whether it is finite took 2 us of 106.)
    __device__ __forceinline__ bool not_finite(float sum) const {
        float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kCols; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) z[e & 3] = fmaf(o[i][e], 0.0f, z[e & 3]);
        return (z[0] + z[1]) + (z[2] + z[3]) != 0.0f && sum == sum;
    }
    // For another pass: rows that were not finite have their weights lower (fp16's values cannot pass fp32).
    __device__ __forceinline__ void set_lower(bool bad) {
        // A row's columns are in two lanes.
        if (!std::is_same_v<T, _Float16>) lower = other_half(bad ? 1.0f : 0.0f, true) != 0.0f ? kLower : 0.0f;
    }
    // Which of the row's columns see an infinity of either sign or a NaN among the values, a bit each; of a lane in
    // LDS, words `step` apart (in registers they would cost every launch some).
    static constexpr int kWords = (16 * kCols + 31) / 32;
    struct Marks {
        uint32_t* at;
        int step;
        __device__ __forceinline__ uint32_t& operator()(int kind, int word) const { return at[(kind * kWords + word) * step]; }
    };
    static constexpr int kMarks = 3 * kWords;  // of a lane
    // Those of the tile of codes (code_values) at vs, whose keys are from k0 on, among the others.  The columns and the
    // weights are lost.
    __device__ __forceinline__ void mark(const char* vs, int k0, const Marks& marks) {
        const int kb = k0 + 4 * ((threadIdx.x & 63) >> 5);
        const unsigned width = (unsigned)max(hi - lo, 0);
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float sees = (unsigned)(kb + 32 * t + 8 * (e / 4) + e % 4 - lo) < width ? 1.0f : 0.0f;
                if constexpr (sizeof(T) == 4)
                    p[t][e] = sees;
                else
                    p[2 * t + e / 8][e % 8] = (T)sees;
            }
        clear();
        values(vs);
#pragma unroll
        for (int word = 0; word < kWords; ++word) {
            uint32_t plus = 0, minus = 0, nan = 0;
#pragma unroll
            for (int b = 0; b < 32 && 32 * word + b < 16 * kCols; ++b) {
                const int sum = (int)o[2 * word + b / 16][b % 16];  // how many of each, 64 at most, as digits
                plus |= (sum & 0x7f ? 1u : 0u) << b, minus |= (sum & 0x3f80 ? 1u : 0u) << b, nan |= (sum >> 14 ? 1u : 0u) << b;
            }
            marks(0, word) |= plus, marks(1, word) |= minus, marks(2, word) |= nan;
        }
    }
    __device__ __forceinline__ void add(const Marks& marks) {
#pragma unroll
        for (int word = 0; word < kWords; ++word) {
            const uint32_t plus = marks(0, word), minus = marks(1, word), nan = marks(2, word);
#pragma unroll
            for (int b = 0; b < 32 && 32 * word + b < 16 * kCols; ++b)
                o[2 * word + b / 16][b % 16] += ((plus >> b & 1 ? INFINITY : 0.0f) + (minus >> b & 1 ? -INFINITY : 0.0f)) +
                                                (nan >> b & 1 ? NAN : 0.0f);
        }
    }
    // The row's columns times w, as T, 16 bytes a store.
    __device__ __forceinline__ void store(T* out, int d, float w) const {
        const int h = (threadIdx.x & 63) >> 5;
        if constexpr (sizeof(T) == 4) {
            store_f32(out, d, [&](float x) { return mean<float>(x, w); });
        } else {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
                    T4 a, b;
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = mean<T>(o[i][e + j], w), b[j] = mean<T>(o[i][e + 4 + j], w);
                    const u32x2 ua = __builtin_bit_cast(u32x2, a), ub = __builtin_bit_cast(u32x2, b);
                    // Columns 0-3 | 4-7 and 8-11 | 12-15 of the halves: the lower lane takes 0-7, the upper 8-15.
                    const auto x = __builtin_amdgcn_permlane32_swap(ua[0], ub[0], false, false);
                    const auto y = __builtin_amdgcn_permlane32_swap(ua[1], ub[1], false, false);
                    const int col = 32 * i + 2 * e + 8 * h;
                    if (out && col < d) *(u32x4*)(out + col) = u32x4{x[0], y[0], x[1], y[1]};
                }
        }
    }
    // As fp32, by what(column) (out null: no store, but all lanes come along).
    template <typename F>
    __device__ __forceinline__ void store_f32(float* out, int d, F what) const {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int i = 0; i < kCols; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int col = 32 * i + 2 * e + 4 * h;
                if (out && col < d)
                    *(f32x4*)(out + col) = f32x4{what(o[i][e]), what(o[i][e + 1]), what(o[i][e + 2]), what(o[i][e + 3])};
            }
    }
};

// 16 bytes a lane to LDS, a wavefront's next to each other from `lds` on: from p, or from base + off.  Written
// out, because the compiler waits for such a load of its own before the next LDS read, whatever either is
// of; here the waits are the kernels'.  The load has no register of its own to be overwritten, and the
// compiler's count of loads in flight, which misses it, only makes its waits longer.
// (m0 is not among the clobbers: it is reserved, so the compiler would not heed that, and warned of it 4352 times a build.
// Nothing else in these kernels uses m0.)
__device__ __forceinline__ void load_lds(uint64_t p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}
__device__ __forceinline__ void load_lds(uint64_t base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Loads tiles of KEYS keys or their values: 16 bytes a lane, straight to LDS.  THREADS threads (whole
// wavefronts) share a tile.  A wavefront's load is kGroup neighbouring rows, at most eight, which are all of one
// page (pages have eight at least, tiles begin at multiples of kGroup): the page, looked up ahead by one lane a
// load, and the address are scalar, and a lane's offset is the same for every tile.  With a page and an address
// of each lane's own, a tile of 64 keys of 128 in bf16 took 80 vector instructions more.
template <typename T, int DP, int KEYS, int THREADS>
struct Loader {
    typedef TileRows<T, DP> Tile;
    static constexpr int kLoads = KEYS * Tile::kChunks / THREADS;  // of a lane
    static constexpr int kRowsApart = THREADS / Tile::kChunks;     // rows between a lane's loads
    static constexpr int kGroup = 64 / Tile::kChunks;
    static constexpr int kBytes = KEYS * Tile::kRow;
    static_assert(THREADS % 64 == 0 && 64 % Tile::kChunks == 0 && KEYS * Tile::kChunks % THREADS == 0 && kLoads <= 64, "");

    const PagedCache* c;
    const int32_t* table;
    uint64_t k_base, v_base;
    int first, row, chunk[kRowsApart % 16 ? kLoads : 1];  // first row of the wavefront's first load; the lane's in it
    uint32_t lds;                                         // of the wavefront's first load, from a tile's begin
    unsigned top_page = 0;

    // Pages of a tile's loads, lane i that of load i.
    struct Pages {
        unsigned of;
    };

    __device__ __forceinline__ Loader(const PagedCache& cache, const int32_t* t, int kvh, int thread) {
        c = &cache, table = t;
        const uint64_t head = (uint64_t)kvh * cache.head_stride * sizeof(T);
        k_base = (uint64_t)cache.k + head, v_base = (uint64_t)cache.v + head;
        const int wave = __builtin_amdgcn_readfirstlane(thread >> 6), lane = thread & 63;
        first = wave * kGroup, row = lane / Tile::kChunks;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(chunk) / 4); ++i)
            chunk[i] = (lane & (Tile::kChunks - 1)) ^ Tile::mix(first + row + i * kRowsApart);
        lds = wave * 1024;
    }
    // Where tiles of keys from lo on may begin.
    static __device__ __forceinline__ int begin(int lo) { return lo & ~(kGroup - 1); }
    // A page that is not in the pool was named (by any lane so far; its last page was read instead).
    __device__ __forceinline__ bool bad() const { return top_page >= (unsigned)c->pages; }
    // Pages of the keys from k0 on; from `end` on they are those of the key before it.
    __device__ __forceinline__ Pages pages(int k0, int end) const {
        Pages p;
        const int key = min(k0 + first + min((int)(threadIdx.x & 63), kLoads - 1) * kRowsApart, end - 1);
        p.of = *(const unsigned*)((const char*)table + 4u * (unsigned)(key >> c->page_log));
        return p;
    }
    // Load i of the keys and of the values from k0 on (from `end` on those of the one before it), to the tiles at LDS
    // addresses ks and vs.
    __device__ __forceinline__ void load(uint32_t ks, uint32_t vs, int k0, int end, const Pages& p, int i) {
        const int key = min(k0 + first + i * kRowsApart, (end - 1) & ~(kGroup - 1));
        const unsigned page = __builtin_amdgcn_readlane(p.of, i);
        top_page = max(top_page, page);
        const uint64_t at = (uint64_t)min(page, (unsigned)c->pages - 1) * c->page_bytes +
                            (unsigned)(key & ((1 << c->page_log) - 1)) * c->token_bytes;
        const uint32_t to = lds + i * THREADS * 16;
        const int ch = chunk[kRowsApart % 16 ? i : 0];
        const uint32_t off = (uint32_t)min(row, end - 1 - key) * c->token_bytes + ch * 16;
        if (Tile::kChunks * Chunk<T>::N != c->head_dim) {
            const bool on = ch * Chunk<T>::N < c->head_dim;
            load_lds(on ? k_base + at + off : (uint64_t)g_zeros, ks + to);
            load_lds(on ? v_base + at + off : (uint64_t)g_zeros, vs + to);
        } else {
            load_lds(k_base + at, off, ks + to);
            load_lds(v_base + at, off, vs + to);
        }
    }
    // All of them.  Where the pages have come is said first: the compiler does not count the loads here.
    __device__ __forceinline__ void load(uint32_t ks, uint32_t vs, int k0, int end, Pages& p) {
        arrived(p);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(ks, vs, k0, end, p, i);
    }
    static __device__ __forceinline__ void arrived(Pages& p) { asm volatile("" : "+v"(p.of)); }
};

// Ends a phase: nothing is scheduled across it.
__device__ __forceinline__ void phase_end() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A weight of 0 times an infinity or a NaN is a NaN: values that are not finite touch rows that do not see them, and an
// infinity that a row sees with a weight below fp32's range (exactly, it is positive) becomes a NaN.  A sum of finite values may
// also pass fp32 where their mean does not.  Where a row's result is not finite, the wavefront (workgroup) goes over its
// keys twice more: which columns see what that is not finite (mark_pass: codes of the values times who sees whom, on the matrix
// cores), then everything with such values taken out of the tiles (clean_values); what was marked is added at the end.  (Where all
// values are NaN, 4 prompts of 8192 tokens take 18.6 ms, one token on 131072 keys 0.42; 305 and 3.7 where the marks were
// found key by key.)  THREADS threads, all of which come along.
template <typename T, int BYTES, int THREADS>
__device__ __forceinline__ void clean_values(char* tile, int thread) {
    typedef typename Chunk<T>::type Vec;
    for (int i = thread * 16; i < BYTES; i += THREADS * 16) {
        Vec v = *(const Vec*)(tile + i);
#pragma unroll
        for (int e = 0; e < Chunk<T>::N; ++e) v[e] = isfinite((float)v[e]) ? v[e] : (T)0.0f;
        *(Vec*)(tile + i) = v;
    }
}
// Values as codes: infinities 1 and 2^7, NaN 2^14, others 0, so that sums of 64 of them say how many there are of each.  Whether
// there were any.
template <typename T, int BYTES, int THREADS>
__device__ __forceinline__ bool code_values(char* tile, int thread) {
    typedef typename Chunk<T>::type Vec;
    bool found = false;
    for (int i = thread * 16; i < BYTES; i += THREADS * 16) {
        Vec v = *(const Vec*)(tile + i);
#pragma unroll
        for (int e = 0; e < Chunk<T>::N; ++e) {
            const float x = (float)v[e];
            found = found || !isfinite(x);
            v[e] = (T)(x == INFINITY ? 1.0f : x == -INFINITY ? 128.0f : x == x ? 0.0f : 16384.0f);
        }
        *(Vec*)(tile + i) = v;
    }
    return found;
}
template <typename T, int DP, int NK, int THREADS>
__device__ __forceinline__ void mark_pass(Rows<T, DP, NK>& w, Loader<T, DP, 32 * NK, THREADS>& ld, char* lds, int k0, int k1,
                                          int step, const typename Rows<T, DP, NK>::Marks& marks) {
    static_assert(32 * NK <= 64, "a code's digits");
    constexpr int B = Loader<T, DP, 32 * NK, THREADS>::kBytes;
    constexpr bool kShared = THREADS > 64;  // the tile by a workgroup
#pragma unroll
    for (int i = 0; i < Rows<T, DP, NK>::kMarks; ++i) marks(0, i) = 0;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address(lds));
    int odd = 0;  // two buffers: a wavefront may still read the one
#pragma unroll 1
    for (int k = k0; k < k1; k += step, odd ^= 1) {
        auto p = ld.pages(k, k1);
        ld.load(at + odd * 2 * B, at + odd * 2 * B + B, k, k1, p);
        loads_done();
        if (kShared) phase_end();
        char* const codes = lds + odd * 2 * B + B;
        const bool found = code_values<T, B, THREADS>(codes, threadIdx.x & (THREADS - 1));
        bool any;
        if constexpr (kShared) {
            any = __syncthreads_or(found);
            phase_end();
        } else {
            any = __any(found);
        }
        if (any) w.mark(codes, k, marks);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// What a part with a factor below fp32's range adds to a join, with a factor of 1: what is not finite, as it is.
__device__ __forceinline__ f32x4 rest_of(f32x4 x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = isfinite(x[e]) ? 0.0f : x[e];
    return x;
}

// Where a launch's partial results lie: for (row, head) r and split s, fp32 columns at
// o[(r * splits + s) * d ..] and (maximum, sum) at ml[r * splits + s].  The maximum is of exponents of 2.
struct Parts {
    float* o;
    float2* ml;
    int splits;
    int fold;  // tiles of a sequence in falling order, before the others in rising order
};

// A split's share of the keys [lo, hi): whole steps of `step` keys.
__device__ __forceinline__ void split_range(int lo, int hi, int split, int splits, int step, int& k0, int& k1) {
    const int steps = (max(hi - lo, 0) + step - 1) / step;
    const int per = (steps + splits - 1) / splits;
    k0 = min(lo + split * per * step, hi);
    k1 = min(k0 + per * step, hi);
}

// The end of a wavefront's rows: out (one split) or a partial result.  on: the lane's row exists.
template <typename T, int DP, int NK>
__device__ __forceinline__ void finish(const Rows<T, DP, NK>& w, const AttendArgs& a, const Parts& parts, float c, int split,
                                       int d, int row, int head, bool on, bool bad) {
    float l = other_half(w.l, false);
    if (bad) l = NAN;
    if (parts.splits == 1) {
        T* out = on ? (T*)a.out.p + (int64_t)row * a.out.row + (int64_t)head * a.out.head : nullptr;
        w.store(out, d, l == 0.0f ? 0.0f : 1.0f / l);
    } else {
        const int64_t r = ((int64_t)row * a.heads + head) * parts.splits + split;
        if (on && (threadIdx.x & 63) < 32) parts.ml[r] = make_float2(w.m * c + w.lower, l);
        w.store_f32(on && l != 0.0f ? parts.o + r * d : nullptr, d, [](float x) { return x; });
    }
}

// What a workgroup of a sequence that breaks a bound does: NaN for rows [first, end).
template <typename T>
__device__ __forceinline__ void poison(const AttendArgs& a, const Parts& parts, int d, int first, int end, int h0, int heads,
                                       int split) {
    const int per = heads * d;
    for (int64_t i = threadIdx.x; i < (int64_t)(end - first) * per; i += blockDim.x) {
        const int row = first + (int)(i / per), e = (int)(i % per), h = h0 + e / d;
        if (parts.splits == 1)
            ((T*)a.out.p)[(int64_t)row * a.out.row + (int64_t)h * a.out.head + e % d] = (T)NAN;
        else if (e % d == 0)
            parts.ml[((int64_t)row * a.heads + h) * parts.splits + split] = make_float2(-INFINITY, NAN);
    }
}

// Joined parts have 2^-kRoom times their factors, for 2^kRoom parts at most: their sum passes what one holds no sooner.
constexpr float kRoom = 2.0f, kSplitRoom = 8.0f;

// Four columns (the i-th such) of the rows that the wavefronts of a workgroup have parts of: their maxima (exponents of
// 2), sums and columns, joined and left as finish() does.
template <typename T, int NW, typename M, typename L, typename C>
__device__ __forceinline__ void join_waves(const AttendArgs& a, const Parts& parts, const SeqRows& r, int kvh, int g, int split,
                                           int d, int i, bool bad, M max_of, L sum_of, C cols_of) {
    const int quads = d / 4, q = i / quads, col = 4 * (i % quads);
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NW; ++v) top = fmaxf(top, max_of(v, q) + kRoom);
    static_assert(NW <= 1 << (int)kRoom, "");
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        const float l = sum_of(v, q);
        if (l == 0.0f) continue;  // nothing seen, its maximum -inf
        float f = __builtin_amdgcn_exp2f(max_of(v, q) - (top == -INFINITY ? 0.0f : top));
        sum = fmaf(l, f, sum);
        f32x4 x = *(const f32x4*)(cols_of(v, q) + col);
        if (f == 0.0f) x = rest_of(x), f = 1.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    }
    if (bad) sum = NAN;
    const int row = r.row0 + q / g, head = kvh * g + q % g;
    if (parts.splits == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = mean<T>(o[e], inv);
        *(T4*)((T*)a.out.p + (int64_t)row * a.out.row + (int64_t)head * a.out.head + col) = y;
    } else {
        const int64_t at = ((int64_t)row * a.heads + head) * parts.splits + split;
        if (sum != 0.0f) *(f32x4*)(parts.o + at * d + col) = o;
        if (col == 0) parts.ml[at] = make_float2(top, sum);
    }
}

constexpr int kTileRows = 32;  // of a wavefront
constexpr int kJoinSplits = 256, kWaveSplits = 16;

// ---- tiles of rows ----------------------------------------------------------

// A workgroup of NW wavefronts takes 32 NW rows of one sequence and kv head, which share tiles of
// 32 NK keys in two buffers: while one is worked on, the next loads.  Two workgroups share a compute unit (64 KiB of LDS
// each, up to 256 registers a lane), and while the one has the matrix cores the other has the vector unit: a wavefront's 64
// keys of 128 in bf16 are 32 products of 32 cycles, 32 exponentials of 16 and some 180 vector instructions of 4, so that neither
// unit can be busy all the time.  4 prompts of 8192 tokens, 64 on 8 heads of 128 in bf16: 4.17 to 4.46 ms, 986 to 1055 TFLOP/s, matrix
// cores 54% and vector unit 57% busy at 1.9 GHz (a large library product: 1094 TFLOP/s); without the loads 3.8.  A prompt of 2048, 32 heads: 52 us,
// the longest tile's 32 steps one after another.  Measured and not kept: eight wavefronts, half of them a phase behind the other
// half and barriers between products and softmax (4.8 ms against 4.4: barriers cost more than the units' overlap gave).
// Heads of 256 leave too few registers: 28 to 30 spilled in 16 bits (72 bytes of scratch a lane), 22 (80) in fp32, some in the loop; two wavefronts
// a row's columns, or queries in LDS, would mend that.
template <typename T, int DP, int NW, int NK, bool CLEAN>
__device__ __forceinline__ void tile_pass(Rows<T, DP, NK>& w, Loader<T, DP, 32 * NK, 64 * NW>& ld, const Score& sc, char* lds,
                                          int k0, int k1) {
    typedef Loader<T, DP, 32 * NK, 64 * NW> L;
    constexpr int kKeys = 32 * NK, B = L::kBytes;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address(lds));  // keys, values; keys, values
    typename L::Pages p = ld.pages(k0, k1);
    ld.load(at, at + B, k0, k1, p);
    p = ld.pages(k0 + kKeys, k1);
    loads_done();
    phase_end();
    int odd = 0;
#pragma unroll 1
    for (int k = k0; k < k1; k += kKeys, odd ^= 1) {
        char* const cur = lds + odd * 2 * B;
        if constexpr (CLEAN) {
            clean_values<T, B, 64 * NW>(cur + B, threadIdx.x);
            phase_end();
        }
        const uint32_t next = at + (odd ^ 1) * 2 * B;
        L::arrived(p);
        // The next tile's loads beside the products of the scores, which leave the scalar unit idle (after the last
        // tile too, then of its last rows: a branch here would part the products).
        constexpr int NG = Rows<T, DP, NK>::kScoreGroups;
        w.scores(cur, [&](int g) {
#pragma unroll
            for (int i = 0; i < L::kLoads; ++i)
                if (i * NG / L::kLoads == g) ld.load(next, next + B, k + kKeys, k1, p, i);
        });
        p = ld.pages(k + 2 * kKeys, k1);
        w.template softmax<CLEAN>(k, sc);
        w.values(cur + B);
        loads_done();
        phase_end();
    }
}

template <typename T, int DP, int NW, int NK>
__global__ __launch_bounds__(64 * NW, DP * sizeof(T) <= 512 ? 2 : 1) void k_attend_tiles(const AttendArgs a, const PagedCache c, const Sequences s,
                                                          const Parts parts) {
    typedef Loader<T, DP, 32 * NK, 64 * NW> L;
    constexpr int kRows = kTileRows * NW;
    __shared__ __align__(16) char lds[4 * L::kBytes];
    __shared__ uint32_t lds_marks[Rows<T, DP, NK>::kMarks * 64 * NW];
    __shared__ int range[2][NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = a.heads / c.kv_heads;
    const int kvh = blockIdx.x % c.kv_heads, split = blockIdx.x / c.kv_heads % parts.splits;

    // The sequence and the tile of it that this workgroup is: tiles in order of the sequences.
    int want = blockIdx.x / (c.kv_heads * parts.splits), b = -1, tile = 0, tiles = 0;
    for (int i0 = 0; i0 < s.B; i0 += 64) {
        int n = 0;
        if (i0 + lane < s.B) {
            const SeqRows r = seq_rows(s, i0 + lane);
            n = (int)(((int64_t)min(r.n, s.max_new) * g + kRows - 1) / kRows);
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(upto, o, 64);
            if (lane >= o) upto += v;
        }
        const unsigned long long past = __ballot(upto > want);
        if (past) {
            const int at = __ffsll(past) - 1;
            b = i0 + at;
            tiles = __shfl(n, at, 64);
            tile = want - (__shfl(upto, at, 64) - tiles);
            break;
        }
        want -= __shfl(upto, 63, 64);
    }
    if (b < 0) return;
    const SeqRows r = seq_rows(s, b);
    if (!r.ok) {
        const int per = (r.n + tiles - 1) / tiles;
        poison<T>(a, parts, c.head_dim, r.row0 + min(r.n, tile * per), r.row0 + min(r.n, (tile + 1) * per), kvh * g, g, split);
        return;
    }
    // The longest rows first.  Where all workgroups are resident, two a compute unit: the ones that come second to a unit
    // the other way round, so that the shortest share with the longest (a prompt of 2048 tokens, 32 on 8 heads of 128).
    tile = tile < parts.fold ? tiles - 1 - tile : tile - parts.fold;

    const Score sc(a);
    Rows<T, DP, NK> w;
    const int64_t first = (int64_t)tile * kRows + wave * kTileRows + (lane & 31), last = (int64_t)r.n * g - 1;
    const bool on = first <= last;
    const int item = (int)min(first, last);
    const int row = r.row0 + item / g, head = kvh * g + item % g;
    w.pos = r.position(row);
    row_keys(a, r, b, row, w.pos, w.lo, w.hi);
    w.slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    w.load((const T*)a.q.p + (int64_t)row * a.q.row + (int64_t)head * a.q.head, c.head_dim, sc.negate);
    w.bounds();
    if (lane == 0) range[0][wave] = w.min_lo, range[1][wave] = w.max_hi;
    __syncthreads();
    int lo = range[0][0], hi = range[1][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) lo = min(lo, range[0][i]), hi = max(hi, range[1][i]);
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    int k0, k1;
    L ld(c, s.table + b * s.table_ld, kvh, threadIdx.x);
    split_range(ld.begin(lo), hi, split, parts.splits, 32 * NK, k0, k1);
    w.clear();
    if (k0 < k1) tile_pass<T, DP, NW, NK, false>(w, ld, sc, lds, k0, k1);
    const bool bad = __syncthreads_or(ld.bad());
    if (!bad && __builtin_expect(__syncthreads_or(k0 < k1 && on && w.not_finite(other_half(w.l, false))), 0)) {
        w.set_lower(w.not_finite(other_half(w.l, false)));
        const typename Rows<T, DP, NK>::Marks marks = {lds_marks + threadIdx.x, 64 * NW};
        mark_pass(w, ld, lds, k0, k1, 32 * NK, marks);
        phase_end();
        w.clear();
        tile_pass<T, DP, NW, NK, true>(w, ld, sc, lds, k0, k1);
        w.add(marks);
    }
    const float unit = sc.capped || sc.sloped ? 1.0f : sc.c;
    finish(w, a, parts, unit, split, c.head_dim, row, head, on, bad);
}

// ---- few rows ----------------------------------------------------------------

// Up to 32 rows of a sequence and kv head (single tokens and a few more): the NW wavefronts of a workgroup
// have tiles of 32 keys of their own, in two buffers each, and are joined at the end.  The cache's bytes bound it: 64 sequences of up
// to 8192 keys, 32 on 8 heads of 128 in bf16, 1.05 GB in 218 us, 4.8 TB/s; one of 131072 537 MB in 109 us with its join, 4.9.
// In fp32 the products are made for 32 rows and take longer than the bytes (64 on 8 heads over 8192 keys 38 us, 1.8 TB/s), most at a head size
// of 256, where one wavefront fits a compute unit and 35 registers are spilled (114 us, 1.2 TB/s).
template <typename T, int DP, int NW, bool CLEAN>
__device__ __forceinline__ void few_pass(Rows<T, DP, 1>& w, Loader<T, DP, 32, 64>& ld, const Score& sc, char* lds, int k0,
                                         int k1) {
    typedef Loader<T, DP, 32, 64> L;
    constexpr int B = L::kBytes, kStep = 32 * NW;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address(lds));  // keys, values; keys, values
    if (k0 >= k1) return;
    typename L::Pages p = ld.pages(k0, k1);
    ld.load(at, at + B, k0, k1, p);
    p = ld.pages(k0 + kStep, k1);
    int odd = 0;
#pragma unroll 1
    for (int k = k0; k < k1; k += kStep, odd ^= 1) {
        loads_done();
        if (k + kStep < k1) {
            const uint32_t next = at + (odd ^ 1) * 2 * B;
            ld.load(next, next + B, k + kStep, k1, p);
        }
        p = ld.pages(k + 2 * kStep, k1);
        char* const cur = lds + odd * 2 * B;
        if constexpr (CLEAN) clean_values<T, B, 64>(cur + B, threadIdx.x & 63);
        w.scores(cur, [](int) {});
        w.template softmax<CLEAN>(k, sc);
        w.values(cur + B);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void k_attend_few(const AttendArgs a, const PagedCache c, const Sequences s,
                                                        const Parts parts) {
    typedef Loader<T, DP, 32, 64> L;
    static_assert(L::kBytes * 4 >= 32 * DP * 4, "a wavefront's buffers hold its result");
    __shared__ __align__(16) char lds[NW][4 * L::kBytes];
    __shared__ uint32_t lds_marks[Rows<T, DP, 1>::kMarks * 64 * NW];
    __shared__ float ml[2][NW][32];
    __shared__ int wrong[NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = a.heads / c.kv_heads, d = c.head_dim;
    const int kvh = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int split = rest % parts.splits, b = rest / parts.splits;
    const SeqRows r = seq_rows(s, b);
    if (r.n == 0) return;
    if (!r.ok) {
        poison<T>(a, parts, d, r.row0, r.row0 + r.n, kvh * g, g, split);
        return;
    }
    const Score sc(a);
    Rows<T, DP, 1> w;
    const int rows = r.n * g, item = min(lane & 31, rows - 1);
    const int row = r.row0 + item / g, head = kvh * g + item % g;
    const bool on = (lane & 31) < rows;
    w.pos = r.position(row);
    row_keys(a, r, b, row, w.pos, w.lo, w.hi);
    w.slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    w.load((const T*)a.q.p + (int64_t)row * a.q.row + (int64_t)head * a.q.head, d, sc.negate);
    w.bounds();
    int k0, k1;
    L ld(c, s.table + b * s.table_ld, kvh, lane);
    split_range(ld.begin(w.min_lo), w.max_hi, split, parts.splits, 32 * NW, k0, k1);
    w.clear();
    few_pass<T, DP, NW, false>(w, ld, sc, lds[wave], k0 + 32 * wave, k1);
    float l = other_half(w.l, false);
    if (__builtin_expect(__any(on && w.not_finite(l)), 0)) {
        w.set_lower(w.not_finite(l));
        const typename Rows<T, DP, 1>::Marks marks = {lds_marks + threadIdx.x, 64 * NW};
        mark_pass(w, ld, lds[wave], k0 + 32 * wave, k1, 32 * NW, marks);
        w.clear();
        few_pass<T, DP, NW, true>(w, ld, sc, lds[wave], k0 + 32 * wave, k1);
        l = other_half(w.l, false);
        w.add(marks);
    }
    const float unit = sc.capped || sc.sloped ? 1.0f : sc.c;
    const bool bad = __any(ld.bad());
    if constexpr (NW == 1) {
        finish(w, a, parts, unit, split, d, row, head, on, bad);
    } else {
        if (lane < 32) ml[0][wave][lane] = w.m * unit + w.lower, ml[1][wave][lane] = l;
        if (lane == 0) wrong[wave] = bad;
        float* mine = (float*)lds[wave];
        w.store_f32(on ? mine + (lane & 31) * DP : nullptr, d, [](float x) { return x; });
        __syncthreads();
        bool any_bad = false;
#pragma unroll
        for (int i = 0; i < NW; ++i) any_bad = any_bad || wrong[i];
        for (int i = threadIdx.x; i < rows * (d / 4); i += 64 * NW)
            join_waves<T, NW>(a, parts, r, kvh, g, split, d, i, any_bad, [&](int v, int q) { return ml[0][v][q]; },
                              [&](int v, int q) { return ml[1][v][q]; },
                              [&](int v, int q) { return (const float*)lds[v] + q * DP; });
    }
}

// ---- few rows in fp32 -----------------------------------------------------------

// Up to four rows in fp32, of whose 32-row products on the matrix cores little would be used: a wavefront has the columns
// across its lanes (NV each) and takes eight keys at a time, keys and values straight from their page (pages have eight
// rows at least) and the next eight's loads in flight.  Scores of eight keys are summed over the lanes together,
// each lane ending with one key's, so that eight keys take one exponential; a weight goes to all lanes as a scalar.
// HBM bounds it (us, k_attend_few in brackets: 32 sequences of 1024 keys, 16 heads of 128, 537 MB 85 [222]; 8 of 512
// 18.3 [37]; four rows, 8 of 2048, 32 on 8 heads 41 [67]; with eight rows it would lose, 51 [39] at a head size of 64).
template <int NV, int R, int NW>
__global__ __launch_bounds__(64 * NW) void k_attend_lanes(const AttendArgs a, const PagedCache c, const Sequences s,
                                                          const Parts parts) {
    constexpr int U = kMinPage;
    typedef float Vec __attribute__((ext_vector_type(NV), aligned(NV == 4 ? 16 : 4 * NV)));
    __shared__ __align__(16) float cols[NW][R][64 * NV];
    __shared__ float ml[2][NW][R];
    __shared__ int wrong[NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = a.heads / c.kv_heads, d = c.head_dim;
    const int kvh = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int split = rest % parts.splits, b = rest / parts.splits;
    const SeqRows r = seq_rows(s, b);
    if (r.n == 0) return;
    if (!r.ok) {
        poison<float>(a, parts, d, r.row0, r.row0 + r.n, kvh * g, g, split);
        return;
    }
    const int rows = r.n * g, col = lane * NV;
    const bool on = col < d;
    float q[R][NV], o[R][NV], m[R], l[R], slope[R];
    int lo[R], hi[R], pos[R], first = 0x7fffffff, end = 0, max_lo = 0, min_hi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int item = min(i, rows - 1), row = r.row0 + item / g, head = kvh * g + item % g;
        pos[i] = r.position(row);
        row_keys(a, r, b, row, pos[i], lo[i], hi[i]);
        lo[i] = __builtin_amdgcn_readfirstlane(lo[i]), hi[i] = __builtin_amdgcn_readfirstlane(hi[i]);
        slope[i] = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
        const Vec x = *(const Vec*)((const float*)a.q.p + (int64_t)row * a.q.row + (int64_t)head * a.q.head + min(col, d - NV));
#pragma unroll
        for (int e = 0; e < NV; ++e) q[i][e] = on ? x[e] : 0.0f, o[i][e] = 0.0f;
        m[i] = -INFINITY, l[i] = 0.0f;
        first = min(first, lo[i]), end = max(end, hi[i]);
        max_lo = max(max_lo, lo[i]), min_hi = min(min_hi, hi[i]);
    }
    int k0, k1;
    split_range(first & ~(U - 1), end, split, parts.splits, U * NW, k0, k1);
    const int32_t* const table = s.table + b * s.table_ld;
    const float* const kp = (const float*)c.k + (int64_t)kvh * c.head_stride + min(col, d - NV);
    const float* const vp = (const float*)c.v + (int64_t)kvh * c.head_stride + min(col, d - NV);
    const int last = k1 - 1, mask = (1 << c.page_log) - 1;
    const bool narrow = d < 64 * NV, sloped = a.slopes != nullptr, capped = a.softcap > 0.0f;
    const float unit = a.scale * kLog2e, in = capped ? __builtin_amdgcn_fmed3f(a.scale / a.softcap, -1.0e30f, 1.0e30f) : 0.0f, out_cap = a.softcap * kLog2e;
    unsigned top_page = 0;

    auto row_top = [&](float v) {  // over the lanes of the eight keys
        v = fmaxf(v, __shfl_xor(v, 32, 64));
        v = fmaxf(v, __shfl_xor(v, 16, 64));
        return fmaxf(v, __shfl_xor(v, 1, 64));
    };
    auto page_of = [&](int k) { return (unsigned)table[min(k, last) >> c.page_log]; };
    auto load = [&](int k, unsigned page, Vec (&kx)[U], Vec (&vx)[U]) {
        top_page = max(top_page, page);
        const int64_t at = (int64_t)min(page, (unsigned)c.pages - 1) * c.page_stride;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t off = at + (int64_t)(min(k + u, last) & mask) * c.token_stride;
            kx[u] = __builtin_nontemporal_load((const Vec*)(kp + off));
            vx[u] = __builtin_nontemporal_load((const Vec*)(vp + off));
        }
    };
    float extra[R][NV], lower[R];  // of a second pass: what is not finite among the values seen, how much lower the weights are
#pragma unroll
    for (int i = 0; i < R; ++i) lower[i] = 0.0f;
    auto take = [&](auto clean, int k, Vec (&kx)[U], Vec (&vx)[U]) {
        if (narrow && !on)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < NV; ++e) kx[u][e] = 0.0f;
        const bool part = k < max_lo || k + U > min_hi;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                x[u] = q[i][0] * kx[u][0];
#pragma unroll
                for (int e = 1; e < NV; ++e) x[u] = fmaf(q[i][e], kx[u][e], x[u]);
            }
            int mine = 0;
            lane_reduce<U, 0>(x, lane, mine);
            const int key = k + mine;
            float v = x[0];
            v = capped ? out_cap * tanhf(v * in) : v * unit;
            if (sloped) v = fmaf(-slope[i], (float)abs(pos[i] - key), v);
            if (part && (key < lo[i] || key >= hi[i])) v = -INFINITY;
            if (__any(v - m[i] > kGrowth)) {
                const float now = fmaxf(m[i], row_top(v));
                const float w = __builtin_amdgcn_exp2f(m[i] - (now == -INFINITY ? 0.0f : now));
                m[i] = now, l[i] *= w;
#pragma unroll
                for (int e = 0; e < NV; ++e) o[i][e] *= w;
            }
            const float less = clean() ? kGrowth + lower[i] : kGrowth;  // so that a weight is 1 at most
            const float p = __builtin_amdgcn_exp2f(v - (m[i] == -INFINITY ? 0.0f : m[i]) - less);
            l[i] += p;  // each key's in the lanes that have it
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), (u & 4) * 8 + (u & 2) * 8 + (u & 1)));
                const bool seen = !part || (k + u >= lo[i] && k + u < hi[i]);
#pragma unroll
                for (int e = 0; e < NV; ++e) {
                    const bool in_sum = seen && (!clean() || isfinite(vx[u][e]));
                    if (clean() && seen && !in_sum) extra[i][e] += vx[u][e];
                    o[i][e] = in_sum ? fmaf(w, vx[u][e], o[i][e]) : o[i][e];  // what is not seen may be anything
                }
            }
        }
    };
    int k = k0 + U * wave;
    constexpr int step = U * NW;
    if (k < k1) {
        Vec ka[U], va[U], kb[U], vb[U];
        unsigned page = page_of(k), next = page_of(k + step);
        load(k, page, ka, va);
#pragma unroll 1
        for (;;) {
            page = page_of(k + 2 * step);
            load(k + step, next, kb, vb);
            take(std::false_type{}, k, ka, va);
            if ((k += step) >= k1) break;
            next = page_of(k + 2 * step);
            load(k + step, page, ka, va);
            take(std::false_type{}, k, kb, vb);
            if ((k += step) >= k1) break;
        }
    }
    // A weight below fp32's range is 0 and makes a NaN of an infinity: again without them, and they as they are at the end.
    bool wrong_row[R], not_finite = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        bool bad = false;
#pragma unroll
        for (int e = 0; e < NV; ++e) bad = bad || !isfinite(o[i][e]);
        wrong_row[i] = __any(bad), not_finite = not_finite || wrong_row[i];
    }
    if (__builtin_expect(not_finite, 0)) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            lower[i] = wrong_row[i] ? kLower : 0.0f;
            m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < NV; ++e) o[i][e] = extra[i][e] = 0.0f;
        }
#pragma unroll 1
        for (k = k0 + U * wave; k < k1; k += step) {
            Vec kx[U], vx[U];
            load(k, page_of(k), kx, vx);
            take(std::true_type{}, k, kx, vx);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < NV; ++e) o[i][e] += extra[i][e];
    }
    // A key's weight is in eight lanes of a wavefront's sum.
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int t = 32; t > 0; t >>= 1) l[i] += __shfl_xor(l[i], t, 64);
        l[i] *= 0.125f;
        if (lane == 0) ml[0][wave][i] = m[i] + lower[i], ml[1][wave][i] = l[i];
        Vec x;
#pragma unroll
        for (int e = 0; e < NV; ++e) x[e] = o[i][e];
        *(Vec*)&cols[wave][i][col] = x;
    }
    if (lane == 0) wrong[wave] = top_page >= (unsigned)c.pages;
    __syncthreads();
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NW; ++i) bad = bad || wrong[i];
    for (int i = threadIdx.x; i < rows * (d / 4); i += 64 * NW)
        join_waves<float, NW>(a, parts, r, kvh, g, split, d, i, bad, [&](int w, int q) { return ml[0][w][q]; },
                              [&](int w, int q) { return ml[1][w][q]; }, [&](int w, int q) { return (const float*)cols[w][q]; });
}

// ---- the splits of a row joined ------------------------------------------------

// W wavefronts per row and head (a workgroup has four): the factors of the splits first, to LDS, then four columns and a
// share of the splits a thread, whose loads are independent (64 splits of 32 heads 4 us; one thread's loads one after
// another took 30 for 256 splits).  About 3.5 TB/s where there are many rows.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_attend_join(const AttendArgs a, int d, const Sequences s, const Parts parts) {
    constexpr int kThreads = 64 * W, kItems = 4 / W, kSplits = W == 4 ? kJoinSplits : kWaveSplits;
    __shared__ float factor[kItems][kSplits];
    __shared__ f32x4 red[256];
    __shared__ float part[2][4];
    const int own = threadIdx.x / kThreads, t = threadIdx.x % kThreads;
    const int item = min((int)blockIdx.x * kItems + own, s.rows * a.heads - 1);  // the last again: the same result
    const int row = item / a.heads, head = item % a.heads;
    const int b = seq_of_row(s, row);
    bool on = b < s.B;
    if (on) {
        const SeqRows r = seq_rows(s, b);
        on = row >= r.row0 && row < r.row0 + r.n;
    }
    const int64_t at = (int64_t)item * parts.splits;
    const float2 v = on && t < parts.splits ? parts.ml[at + t] : make_float2(-INFINITY, 0.0f);
    float top = v.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if constexpr (W == 4) {
        if ((t & 63) == 0) part[0][t >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
    }
    static_assert(kSplits <= 1 << (int)kSplitRoom, "");
    const float f = v.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(v.x - (top == -INFINITY ? 0.0f : top) - kSplitRoom);
    float sum = v.y == 0.0f ? 0.0f : v.y * f;
    // Columns have been written where something was seen; beside a sum of NaN they may not have been, and need not.
    if (t < kSplits) factor[own][t] = v.y != 0.0f && v.y == v.y ? f : -1.0f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if constexpr (W == 4)
        if ((t & 63) == 0) part[1][t >> 6] = sum;
    __syncthreads();
    if constexpr (W == 4) sum = (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]);
    const int quads = d / 4, groups = kThreads / quads, grp = t / quads, col = 4 * (t % quads);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (on && grp < groups) {
        constexpr int U = 8;
        for (int i0 = grp; i0 < parts.splits; i0 += U * groups) {
            f32x4 x[U];
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * groups;
                w[u] = i < parts.splits ? factor[own][i] : -1.0f;
                x[u] = w[u] >= 0.0f ? *(const f32x4*)(parts.o + (at + i) * d + col) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (w[u] == 0.0f) x[u] = rest_of(x[u]), w[u] = 1.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(x[u][e], w[u], o[e]);
        }
    }
    red[threadIdx.x] = o;
    __syncthreads();
    if (!on || t >= quads) return;
    for (int i = 1; i < groups; ++i) o += red[threadIdx.x + i * quads];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = mean<T>(o[e], inv);
    *(T4*)((T*)a.out.p + (int64_t)row * a.out.row + (int64_t)head * a.out.head + col) = y;
}

constexpr int kTileWaves = 4;

// Wavefronts of k_attend_few whose buffers (two of 32 keys and values each) fit 128 KiB.
constexpr int few_waves(int row_bytes) { return row_bytes <= 256 ? 4 : 1024 / row_bytes; }

constexpr int kLaneRows = 4, kLaneWaves = 4;

template <int NV>
void start_lanes(const AttendArgs& a, const PagedCache& c, const Sequences& s, const AttendPlan& p, const Parts& parts,
                 hipStream_t st) {
    const unsigned wgs = (unsigned)((int64_t)s.B * c.kv_heads * p.splits);
    const int rows = s.max_new * (a.heads / c.kv_heads);
    if (rows <= 1) k_attend_lanes<NV, 1, kLaneWaves><<<wgs, 64 * kLaneWaves, 0, st>>>(a, c, s, parts);
    else if (rows <= 2) k_attend_lanes<NV, 2, kLaneWaves><<<wgs, 64 * kLaneWaves, 0, st>>>(a, c, s, parts);
    else k_attend_lanes<NV, 4, kLaneWaves><<<wgs, 64 * kLaneWaves, 0, st>>>(a, c, s, parts);
}

template <typename T, int DP>
void start(const AttendArgs& a, const PagedCache& c, const Sequences& s, const AttendPlan& p, const Parts& parts,
           hipStream_t st) {
    constexpr int kRow = TileRows<T, DP>::kRow;
    if (p.lanes) {
        start_lanes<(DP <= 64 ? 1 : DP <= 128 ? 2 : 4)>(a, c, s, p, parts, st);
    } else if (p.few) {
        constexpr int NW = few_waves(kRow);
        k_attend_few<T, DP, NW><<<(unsigned)((int64_t)s.B * c.kv_heads * p.splits), 64 * NW, 0, st>>>(a, c, s, parts);
    } else {
        constexpr int NK = kRow <= 256 ? 2 : 1;
        k_attend_tiles<T, DP, kTileWaves, NK>
            <<<(unsigned)(p.tiles * c.kv_heads * p.splits), 64 * kTileWaves, 0, st>>>(a, c, s, parts);
    }
    const int64_t items = (int64_t)s.rows * a.heads;
    if (p.splits > kWaveSplits)
        k_attend_join<T, 4><<<(unsigned)items, 256, 0, st>>>(a, c.head_dim, s, parts);
    else if (p.splits > 1)
        k_attend_join<T, 1><<<(unsigned)ceil_div(items, 4), 256, 0, st>>>(a, c.head_dim, s, parts);
}

template <typename T>
void start(const AttendArgs& a, const PagedCache& c, const Sequences& s, const AttendPlan& p, const Parts& parts,
           hipStream_t st) {
    const int d = c.head_dim;
    if (d <= 64) start<T, 64>(a, c, s, p, parts, st);
    else if (d <= 96) start<T, 96>(a, c, s, p, parts, st);
    else if (d <= 128) start<T, 128>(a, c, s, p, parts, st);
    else if (d <= 192) start<T, 192>(a, c, s, p, parts, st);
    else start<T, 256>(a, c, s, p, parts, st);
}

}  // namespace

static int64_t attend_split_bytes(const AttendShape& q) { return q.rows * q.heads * (q.head_dim * 4 + 8); }

// Splits share the keys of too few workgroups for the device.  Few rows: four workgroups a compute unit, of at least 128
// keys (fp32: 256), so that sequences of different lengths come out even; a sequence by itself two, for its splits are
// alike and each costs its beginning (us, two / four / eight a unit: 131072 keys of one sequence 115 / 122 / 140, 64
// sequences of up to 8192 240 / 221 / 221).  Tiles: the number, a power of two, of the least time by a model of the launch.
AttendPlan attend_plan(const AttendShape& q, int64_t cus) {
    AttendPlan p;
    const int64_t g = q.heads / q.kv_heads, len = std::max<int64_t>(q.max_len, 1);
    const bool f32 = q.t == DType::f32;
    p.few = q.max_new * g <= kTileRows;
    p.lanes = f32 && q.max_new * g <= kLaneRows;
    p.splits = 1;
    // Rows behind the last sequence have their places among the partial results too: 1 GiB of those at most, which only a
    // call padded to many times its tokens would need.
    const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 30) / attend_split_bytes(q));
    int64_t wgs;
    if (p.few) {
        p.tiles = 0;
        wgs = q.B * q.kv_heads;
        p.splits = (int)std::max<int64_t>(1, std::min({ceil_div((q.B == 1 ? 2 : 4) * cus, wgs), ceil_div(len, f32 && !p.lanes ? 256 : 128),
                                                       (int64_t)kJoinSplits, most}));
    } else {
        const int64_t rows = kTileRows * kTileWaves;
        p.tiles = std::min(q.rows * g / rows + q.B, q.B * ceil_div(q.max_new * g, rows));
        wgs = p.tiles * q.kv_heads;
        // us that a workgroup takes for 64 keys where it shares a compute unit with others (their number times this
        // each), and by itself, as measured at head sizes of 64, 128 and 256; joining: the partial sums there and back.
        const double width = (double)round_up(q.head_dim, 32) / 128;
        const double step = f32 ? 7.3 * width : (width <= 1 ? 0.35 + 0.7 * width : 1.05 + 2.4 * (width - 1));
        const double alone = (f32 ? 1.5 : 1.4) * step;
        const int64_t seen = q.window > 0 ? std::min(len, q.window + rows / g) : len;
        const double longest = ceil_div(seen, 64);
        const double mean = q.window > 0 ? longest : std::max(1.0, longest - (double)q.max_new / 128);
        double best = 0;
        for (int S = 1; S <= std::min<int64_t>(kWaveSplits, most) && (S == 1 || S * 128 <= seen); S *= 2) {
            const double rounds = (double)ceil_div(wgs * S, cus);
            const double work = rounds <= 1 ? alone * longest / S : std::max(step * rounds * mean / S, 2 * step * longest / S);
            const double join = S == 1 ? 0 : 4 + (double)(q.rows * q.heads) * (S * q.head_dim * 8 + 256) / 3.5e6;
            const double t = work + 1.5 * std::max(rounds, 2.0) + join;
            if (S == 1 || t < best) best = t, p.splits = S;
        }
    }
    p.workgroups = wgs * p.splits;
    p.fold = q.B == 1 && p.workgroups <= 2 * cus ? (int)std::max<int64_t>(1, cus / (q.kv_heads * p.splits)) : 1 << 30;
    return p;
}

int64_t attend_plan_bytes(const AttendPlan& p, const AttendShape& q) {
    if (p.splits == 1) return 0;
    return attend_split_bytes(q) * p.splits;
}

hipError_t launch_attend(const AttendArgs& a, const PagedCache& c, const Sequences& s, const AttendPlan& p, void* ws,
                         hipStream_t st) {
    if (s.rows <= 0 || s.B <= 0) return hipSuccess;
    const int64_t n = (int64_t)s.rows * a.heads * p.splits;
    const Parts parts = {(float*)ws, (float2*)((float*)ws + n * c.head_dim), p.splits, p.fold};
    switch (c.t) {
        case DType::f32: start<float>(a, c, s, p, parts, st); break;
        case DType::bf16: start<__bf16>(a, c, s, p, parts, st); break;
        case DType::f16: start<_Float16>(a, c, s, p, parts, st); break;
    }
    return hipGetLastError();
}

}  // namespace sgq
