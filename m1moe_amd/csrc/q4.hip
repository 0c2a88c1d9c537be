// q4.hip — products of rows with weights in 4 bits: y[t][n] = sum_k x[t][k] (q s + b)[n][k] (+ r).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "device.hpp"
#include "drafts.hpp"

namespace m1moe {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

// Of a workgroup of many tokens: tiles of 16 of them, tiles of 16 rows of a wave.
constexpr int kManyTiles = 2, kManyRows = 2;
// Most tokens that every workgroup stages for itself (with 16, 17 to 32 tokens as many: 6144 x 4096
// f32, 17 tokens 16.1 us as few, 21.9 as many, 32 tokens 19.3 and 23.5; 50304 x 2048, whose rows fill the
// card either way, 25.6 and 25.6, 32.0 and 27.2), the LDS that it does so in, so that two fit a CU,
// and the rows of LDS that it takes for r.
constexpr int kFewTokens = 32, kFewLds = 76 * 1024;
__host__ __device__ constexpr int few_rows(int r) { return r | 1; }

// With the columns' groups G, y = sum_G (s_G sum_{k in G} x_k (q_k - 8) + (b_G + 8 s_G) X_G),
// X_G = sum_{k in G} x_k: the inner sum is an MFMA of f16 operands, exact products in f32
// sums, which the 8 keeps small.
//
// A nibble q, masked where it stands in the low (or second) four bits of a 16-bit half, under the
// exponent of 1024 is 1024 + q (or 1024 + 16 q): nine instructions make the MFMA operand q - 8 of
// a word's eight columns, in the order 0 4 1 5 2 6 3 7.  (q 2^-24 as a subnormal would take
// five, but an MFMA aligns its products by their operands' exponents, and of subnormals
// drops the last 7 bits.)  x meets them in that order, times a power of two 2^e that
// brings the row's largest value (up to 32 tokens: of a unit of columns) to 2^14 .. 2^15: an f32 x as
// two f16 parts, a bf16 x as one.  An f16 ends at steps of 2^-24, half of which are 2^-39 of the largest
// value (of 2^-112 where that is less): two parts are 22 bits of what is at least 2^-16 of it, below
// which the second one is a subnormal, one part is all of a bf16 of at least 2^-31 of it, and smaller values
// are kept to that half step.

// ---- few tokens ------------------------------------------------------------------------
//
// Bound by reading the weights once.  A wave has a tile of 16 rows n of W, its lane (c, g) the
// row n = c: 16 bytes, 32 columns, of each 128 at a time straight from memory into registers,
// a unit of columns ahead; v_permlane swaps bring the words of one group together.  x is staged
// in LDS as the other operand, a chunk of columns at a time; its rows are the tokens, or
// of f32 tokens the two parts of each, which fill the rows of one MFMA for up to 8 tokens.
// KS waves of a workgroup share a tile's columns, or KW workgroups.
//
// Group 64, us (at the rate of a large copy): 2048 x 2048, 1 token 5.1 (0.5), the launch, x, a row's
// words and the join in turn; 6144 x 4096 8.0 (2.7); 50304 x 2048, 1 token 15.4 (11.4), 16 f32 20.6, 26
// bf16 24.4 (12.2), where a tile's nibbles, MFMAs and LDS reads of x follow each other in a wave,
// 16 waves fill a CU and 197 such workgroups leave 59 CUs without one.
template <int G>
struct Unit {
    static constexpr int NQ = G == 32 ? 2 : 4;          // 128-column blocks
    static constexpr int kCols = 128 * NQ, kGroups = kCols / G;
    uint4 w[NQ];
    uint32_t s[kGroups / 2], b[kGroups / 2];            // bf16 pairs
};

// A lane's row of W.
struct Weights {
    const uint8_t* w;                  // at the lane's 32 columns of the first block
    const uint16_t *s, *b;             // all rows' scales and biases,
    int64_t at, total;                 // where the row's begin and how many there are
    int cols, groups, g;

    Weights() = default;
    __device__ __forceinline__ Weights(const Q4Args& a, int row, int lane_g) {
        cols = a.cols;
        groups = a.cols / a.group;
        g = lane_g;
        w = reinterpret_cast<const uint8_t*>(a.w) + (int64_t)row * (a.cols / 2) + 16 * g;
        s = a.scales;
        b = a.biases;
        at = (int64_t)row * groups;
        total = (int64_t)a.rows * groups;
    }
    // A unit's N values (N <= total), the first `left` of which belong to it, `late` of them before
    // the place that was read from.
    template <int N>
    struct __attribute__((packed, aligned(2))) Halves {
        uint32_t x[N / 2];
    };
    template <int N>
    __device__ __forceinline__ static void shift(uint32_t (&x)[N / 2], int late, int left) {
        uint64_t v[2] = {x[0] | (uint64_t)x[1] << 32, 0};
        if (N == 8) v[1] = x[N / 2 - 2] | (uint64_t)x[N / 2 - 1] << 32;
        if (late >= 4) v[0] = v[1], v[1] = 0;
        const int bits = 16 * (late & 3);
        v[0] = v[0] >> bits | (bits ? v[1] << (64 - bits) : 0);
        v[1] >>= bits;
        v[0] &= left >= 4 ? ~0ull : (1ull << 16 * left) - 1;
        v[1] &= left >= 8 ? ~0ull : left <= 4 ? 0ull : (1ull << 16 * (left - 4)) - 1;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[i] = (uint32_t)(v[i >> 1] >> 32 * (i & 1));
    }
    // A unit that ends in the row (all without a test: what a load may need would be kept in
    // registers beside the units).
    template <int G>
    __device__ __forceinline__ void load_whole(int u, Unit<G>& x) const {
        typedef Unit<G> U;
        constexpr int N = U::kGroups;
#pragma unroll
        for (int i = 0; i < U::NQ; ++i) x.w[i] = *reinterpret_cast<const uint4*>(w + (u * U::kCols / 2 + 64 * i));
        const int64_t from = at + u * N;
        const Halves<N> p = *reinterpret_cast<const Halves<N>*>(s + from), q = *reinterpret_cast<const Halves<N>*>(b + from);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x.s[i] = p.x[i], x.b[i] = q.x[i];
    }
    // The words of any 128-column block (past the row its last columns again, which meet x = 0 and
    // scales of 0).
    __device__ __forceinline__ uint4 words(int block) const {
        return *reinterpret_cast<const uint4*>(w + (min(128 * block, cols - 32 * (g + 1)) >> 1));
    }
    // N of the row's scales or biases from group q on, past its last one 0.
    template <int N>
    __device__ __forceinline__ void halves(const uint16_t* from_all, int q, uint32_t (&x)[N / 2]) const {
        raw_halves<N>(from_all, q, x);
        settle<N>(q, x);
    }
    // Their load, and what puts them in place where it could not begin at group q: apart, as a test
    // behind each load would wait for it.
    template <int N>
    __device__ __forceinline__ void raw_halves(const uint16_t* from_all, int q, uint32_t (&x)[N / 2]) const {
        const Halves<N> p = *reinterpret_cast<const Halves<N>*>(from_all + min(at + q, total - N));
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[i] = p.x[i];
    }
    template <int N>
    __device__ __forceinline__ void settle(int q, uint32_t (&x)[N / 2]) const {
        const int left = max(groups - q, 0);
        if (left < N) shift<N>(x, (int)(at + q - min(at + q, total - N)), left);
    }
    // A last unit that the row has only some groups of.
    template <int G>
    __device__ __forceinline__ void load_part(int u, Unit<G>& x) const {
        typedef Unit<G> U;
        constexpr int N = U::kGroups;
#pragma unroll
        for (int i = 0; i < U::NQ; ++i) x.w[i] = words(u * U::NQ + i);
        halves<N>(s, u * N, x.s);
        halves<N>(b, u * N, x.b);
    }
};

// The same number, but addresses made of it are made where they are used (or the compiler keeps
// 90 registers of them over a loop's rounds).
__device__ __forceinline__ int opaque(int u) {
    asm volatile("" : "+s"(u));
    return u;
}

__device__ __forceinline__ float bf16_pair(const uint32_t* p, int i) {
    return __uint_as_float(i & 1 ? p[i >> 1] & 0xFFFF0000u : p[i >> 1] << 16);
}

// Eight nibbles as an operand.
__device__ __forceinline__ f16x8 nibbles(uint32_t v, const NibK& k) {
    const uint32_t w = v >> 8;
    const half2_t off = {(_Float16)-1032.f, (_Float16)-1032.f}, off16 = {(_Float16)-72.f, (_Float16)-72.f},
                  by16 = {(_Float16)0.0625f, (_Float16)0.0625f};
    const auto low = [&](uint32_t x) { return __builtin_bit_cast(half2_t, (x & k.lo) | k.mg) + off; };
    const auto high = [&](uint32_t x) {
        return __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (x & k.hi) | k.mg), by16, off16);
    };
    const half2_t a = low(v), b = high(v), c = low(w), d = high(w);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A 128-column block's words, lane (c, g) holding columns 32 g .. 32 g + 31, as four steps of 32
// columns, each of one group: step i, lane g has the columns col(i, g) .. + 7.
template <int G>
__device__ __forceinline__ void steps(const uint4& x, uint32_t (&v)[4]) {
    if constexpr (G == 128) {
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else if constexpr (G == 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(x.x, x.y, false, false);
        const auto q = __builtin_amdgcn_permlane32_swap(x.z, x.w, false, false);
        v[0] = p[0], v[1] = q[0], v[2] = p[1], v[3] = q[1];
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(x.x, x.z, false, false);
        const auto q = __builtin_amdgcn_permlane32_swap(x.y, x.w, false, false);
        const auto r = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
        const auto s = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
        v[0] = r[0], v[1] = r[1], v[2] = s[0], v[3] = s[1];
    }
}
// The step i and lane g that have octet o (of 16) of a block.
template <int G>
__device__ __forceinline__ void place(int o, int& i, int& g) {
    if (G == 128) {
        i = o & 3, g = o >> 2;
    } else if (G == 64) {     // columns 64 h + 32 (g & 1) + 8 (2 s + (g >> 1)), i = 2 h + s
        i = (o >> 3) * 2 + ((o >> 1) & 1), g = ((o >> 2) & 1) | (o & 1) << 1;
    } else {
        i = o >> 2, g = o & 3;
    }
}

__device__ __forceinline__ float largest(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    return m;
}
// e such that 2^e brings the largest value of the wave to 2^14 .. 2^15 (zeros: as 2^-112).
__device__ __forceinline__ int scale_of(float m) {
    return 14 - max((int)(__float_as_uint(wave_max(m)) >> 23) - 127, -112);
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight columns of x from p on.
template <bool XB>
__device__ __forceinline__ void read8(const Q4Args& a, int64_t at, float (&v)[8]) {
    if constexpr (XB) {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + at);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = bf16x8_at(x, j);
    } else {
        const float4* x = reinterpret_cast<const float4*>(static_cast<const float*>(a.x) + at);
        const float4 p = x[0], q = x[1];
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
        v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
    }
}
// They, times 2^e (before they are summed, or large ones would pass the largest float).
__device__ __forceinline__ void scale(float (&v)[8], float up) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= up;
}
// As f16 parts, in the order of a word's nibbles.
__device__ __forceinline__ void parts(const float (&v)[8], f16x8& hi, f16x8& lo) {
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = v[order[j]];
        hi[j] = (_Float16)x;
        lo[j] = (_Float16)(x - (float)hi[j]);
    }
}
// The sum of a group's columns, eight a lane, in all its lanes.
template <int G>
__device__ __forceinline__ float group_sum(const float (&v)[8]) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
#pragma unroll
    for (int l = 1; l < G / 8; l <<= 1) sum += __shfl_xor(sum, l);
    return sum;
}

// NT operand tiles of 16 rows, P operands of a tile (an f32 x with one: its parts are rows 2 t
// and 2 t + 1 of the tile).
template <int G, int NT, int P, bool XB>
struct Few {
    typedef Unit<G> U;
    static constexpr int RT = !XB && P == 1 ? 2 : 1;     // rows of a token
    static constexpr int kSteps = 4 * U::NQ;             // of a unit

    const Q4Args& a;
    int R, rows;                 // rows staged, and those apart of a step's lanes in LDS: an odd number
    uint8_t* s_x;                // [units][P][steps][4][R] 16 bytes
    float* s_sum;                // [units][groups][16 NT]: X_G 2^e, rows as above (their second: 0)
    float* s_down;               // [units][16 NT]: 2^-e

    __host__ __device__ static constexpr int unit_bytes(int r) {
        return P * kSteps * 64 * r + (U::kGroups + 1) * 64 * NT;
    }
    __device__ __forceinline__ Few(const Q4Args& a, uint8_t* s) : a(a) {
        rows = RT * a.tokens;
        R = few_rows(rows);
        s_x = s;
        s_sum = reinterpret_cast<float*>(s + a.chunk * P * kSteps * 64 * R);
        s_down = s_sum + a.chunk * U::kGroups * 16 * NT;
    }

    // n units from column k0 on, by all waves, four of a token's units each at a time.
    __device__ __forceinline__ void stage(int k0, int n) {
        const int lane = (int)threadIdx.x & 63, waves = (int)blockDim.x >> 6;
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), at0 = 8 * lane, tn = a.tokens;
        for (int i0 = wave; i0 < tn * n; i0 += 4 * waves) {
            float v[4][8] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * waves, t = i / n, col = k0 + (i - t * n) * U::kCols + at0;
                if (i < tn * n && at0 < U::kCols && col < a.cols)
                    read8<XB>(a, (int64_t)t * a.x_stride + col, v[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * waves, t = i / n, u = i - t * n, row = RT * t;
                if (i >= tn * n) break;
                const int e = scale_of(largest(v[k]));
                scale(v[k], power(e));
                const float sum = group_sum<G>(v[k]);
                if (lane < RT) s_down[16 * NT * u + row + lane] = power(-e);
                if (at0 >= U::kCols) continue;
                if (at0 % G == 0) {
                    float* to = s_sum + (u * U::kGroups + at0 / G) * 16 * NT + row;
                    to[0] = sum;
                    if (RT == 2) to[1] = 0.f;
                }
                f16x8 hi, lo;
                parts(v[k], hi, lo);
                int step, g;
                place<G>(lane & 15, step, g);
                step += 4 * (lane >> 4);
                uint8_t* to = s_x + 16 * (((u * P * kSteps + step) * 4 + g) * R + row);
                *reinterpret_cast<f16x8*>(to) = hi;
                if (RT == 2) *reinterpret_cast<f16x8*>(to + 16) = lo;
                if (P == 2) *reinterpret_cast<f16x8*>(to + 64 * kSteps * R) = lo;
            }
        }
    }

    // Unit x, unit u of the chunk.
    __device__ __forceinline__ void add(const U& x, int u, int c, int g, f32x4v (&acc)[NT]) const {
        const uint8_t* y[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
            y[t] = s_x + 16 * ((u * P * kSteps * 4 + g) * R + min(16 * t + c, rows - 1));
        const NibK k = nib_consts();
        f32x4v unit[NT], part[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) unit[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < U::NQ; ++i) {
            __builtin_amdgcn_sched_barrier(0);   // (a block's operands at a time: registers)
            uint32_t v[4];
            steps<G>(x.w[i], v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x8 w = nibbles(v[j], k);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (j % (G / 32) == 0) part[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = P - 1; p >= 0; --p)
                        part[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            *reinterpret_cast<const f16x8*>(y[t] + p * 64 * kSteps * R), w, part[t], 0, 0, 0);
                    y[t] += 64 * R;
                }
                if (j % (G / 32) == G / 32 - 1) {
                    const int q = (4 * i + j) / (G / 32);     // group of the unit
                    const float s = bf16_pair(x.s, q), b = fmaf(8.f, s, bf16_pair(x.b, q));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const f32x4v sum =
                            *reinterpret_cast<const f32x4v*>(s_sum + (u * U::kGroups + q) * 16 * NT + 16 * t + 4 * g);
#pragma unroll
                        for (int e = 0; e < 4; ++e) unit[t][e] = fmaf(b, sum[e], fmaf(s, part[t][e], unit[t][e]));
                        asm volatile("" : "+v"(unit[t]));   // (here and now: or all parts are kept for later)
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const f32x4v down = *reinterpret_cast<const f32x4v*>(s_down + 16 * NT * u + 16 * t + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(unit[t][e], down[e], acc[t][e]);
        }
    }
};

__device__ __forceinline__ void put(const Q4Args& a, int t, int n, float y) {
    const int64_t at = (int64_t)t * a.y_stride + n;
    if (a.y_bf16) {
        if (a.residual) y += bf16_to_f32(static_cast<const uint16_t*>(a.residual)[at]);
        static_cast<__bf16*>(a.y)[at] = (__bf16)y;
    } else {
        if (a.residual) y += static_cast<const float*>(a.residual)[at];
        static_cast<float*>(a.y)[at] = y;
    }
}

// Weights of fewer groups in all than a unit of one row has (a unit's scales are one load): a
// wave per token and row.
template <bool XB>
__global__ __launch_bounds__(64) void q4_tiny_kernel(Q4Args a) {
    const int lane = (int)threadIdx.x, t = (int)blockIdx.x, n = (int)blockIdx.y, groups = a.cols / a.group;
    float sum = 0.f;
    for (int k = lane; k < a.cols; k += 64) {
        const int64_t at = (int64_t)t * a.x_stride + k, g = (int64_t)n * groups + k / a.group;
        const float x = XB ? bf16_to_f32(static_cast<const uint16_t*>(a.x)[at]) : static_cast<const float*>(a.x)[at];
        const float q = (float)(a.w[((int64_t)n * a.cols + k) / 8] >> 4 * (k & 7) & 15);
        sum = fmaf(x, fmaf(q, bf16_to_f32(a.scales[g]), bf16_to_f32(a.biases[g])), sum);
    }
    sum = wave_sum(sum);
    if (lane == 0) put(a, t, n, sum);
}

// KW workgroups share a block's columns, this one kw: the last of them to end joins their sums,
// N tiles of a wave, and goes on alone (true).  id: of the block.
template <int N>
__device__ __forceinline__ bool join_split(const Q4Args& a, int id, int KW, int kw, int waves, int wave, bool mine,
                                           f32x4v (&acc)[N], int* s_flag) {
    const int lane = (int)threadIdx.x & 63;
    const int64_t wg = (int64_t)waves * N * 256;
    float* part = a.part + (int64_t)id * KW * wg + (int64_t)wave * N * 256 + 4 * lane;   // [KW][waves][N][64][4]
    if (mine)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float y[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
            store4_coh(part + kw * wg + i * 256, y);
        }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        *s_flag = __hip_atomic_fetch_add(a.counters + id, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                  (uint32_t)(KW - 1);
        if (*s_flag) __hip_atomic_store(a.counters + id, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*s_flag) return false;
    // (in the order of the columns, whoever is last; as many loads at once as pay)
    constexpr int L = N > 1 ? 16 : 8, K = L / N;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < KW; k0 += K) {
        const float* at[L];
        f32x4v y[L];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) at[k * N + i] = part + min(k0 + k, KW - 1) * wg + i * 256;
        if constexpr (L == 16) load16_coh(at, y);
        else load8_coh(at, y);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k0 + k < KW)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += y[k * N + i];
    }
    return true;
}

template <int G, int NT, int P, bool XB>
__global__ __launch_bounds__(1024) void q4_few_kernel(Q4Args a) {
    typedef Few<G, NT, P, XB> F;
    typedef Unit<G> U;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_buf[];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int waves = (int)blockDim.x >> 6, c = lane & 15, g = lane >> 4, KS = a.wave_split, ks = wave % KS;
    const int KW = a.split, kw = (int)blockIdx.x % KW, block = (int)blockIdx.x / KW;
    const int tile = block * (waves / KS) + wave / KS;
    F f(a, s_buf);
    const int units = (a.cols + U::kCols - 1) / U::kCols;
    const int u0 = (int)((int64_t)units * kw / KW), u1 = (int)((int64_t)units * (kw + 1) / KW);
    const bool on = 16 * tile < a.rows;
    const int n = 16 * tile + c;
    const Weights w(a, min(n, a.rows - 1), g);
    f32x4v acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
    for (int k = u0; k < u1; k += a.chunk) {
        const int nu = min(a.chunk, u1 - k), lo = nu * ks / KS, end = nu * (ks + 1) / KS;
        const int hi = min(end, a.cols / U::kCols - k);    // (a last unit in part: behind the others)
        U x[2];
        if (on && lo < hi) w.load_whole<G>(k + lo, x[0]);
        if (k != u0) __syncthreads();
        f.stage(k * U::kCols, nu);
        __syncthreads();
        if (!on) continue;
        if (lo < hi) {
            int u = lo;
            for (; u + 2 < hi; u += 2) {   // (no load under a condition: its unit would be held twice)
                w.load_whole<G>(k + opaque(u) + 1, x[1]);
                f.add(x[0], opaque(u), c, g, acc);
                w.load_whole<G>(k + opaque(u) + 2, x[0]);
                f.add(x[1], opaque(u) + 1, c, g, acc);
            }
            if (u + 1 < hi) {
                w.load_whole<G>(k + u + 1, x[1]);
                f.add(x[0], u, c, g, acc);
                x[0] = x[1];
                ++u;
            }
            f.add(x[0], u, c, g, acc);
        }
        if (max(lo, hi) < end) {
            w.load_part<G>(k + end - 1, x[0]);
            f.add(x[0], end - 1, c, g, acc);
        }
    }
    // the waves of a tile, in their order
    if (KS > 1) {
        f32x4v* s = reinterpret_cast<f32x4v*>(s_buf);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t) s[(wave * NT + t) * 64 + lane] = acc[t];
        __syncthreads();
        if (ks == 0) {
            for (int i = 1; i < KS; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t] += s[((wave + i) * NT + t) * 64 + lane];
        }
    }
    if (KW > 1) {
        __syncthreads();
        if (!join_split<NT>(a, block, KW, kw, waves, wave, ks == 0, acc, reinterpret_cast<int*>(s_buf))) return;
    }
    if (ks || !on || n >= a.rows) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if constexpr (F::RT == 2) {
            if (2 * g < a.tokens) put(a, 2 * g, n, acc[t][0] + acc[t][1]);
            if (2 * g + 1 < a.tokens) put(a, 2 * g + 1, n, acc[t][2] + acc[t][3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (16 * t + 4 * g + i < a.tokens) put(a, 16 * t + 4 * g + i, n, acc[t][i]);
        }
    }
}

// ---- many tokens -----------------------------------------------------------------------
//
// x is made into operands once, by a kernel of its own: f16 parts in records of 16 tokens' 128
// columns, [P parts][4 steps][64 lanes] 16 bytes, as the MFMAs take them; the groups' sums
// X_G 2^e as three bf16 parts, 32 groups together, [3][64 lanes] 16 bytes; and the tokens' 2^-e
// (e: of a token's whole row).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr int record_bytes(int p) { return 4096 * p; }
constexpr int kSumBytes = 3 * 1024;

// x as three bf16 parts.
__device__ __forceinline__ void bf16_parts(float x, __bf16 (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i] = (__bf16)x;
        x -= (float)p[i];
    }
}

// Workgroup = (four tokens, a share of the columns, 4096 at most), a wave per token, which holds
// its share in registers and reads the rest of its row for the largest value only.  (800 x 4096
// f32: 9.3 us.)
template <int G, bool XB>
__global__ __launch_bounds__(256) void q4_parts_kernel(Q4Args a) {
    constexpr int P = XB ? 1 : 2, kRecord = record_bytes(P), N = 8;
    const int lane = (int)threadIdx.x & 63, t = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int quads = (a.cols + 511) / 512, tile = t >> 4, row = t & 15, sums = (a.cols / G + 31) / 32;
    const int64_t from = (int64_t)min(t, a.tokens - 1) * a.x_stride;
    const int q0 = (int)((int64_t)quads * blockIdx.x / gridDim.x), q1 = (int)((int64_t)quads * (blockIdx.x + 1) / gridDim.x);
    float v[N][8] = {}, m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int col = 512 * (q0 + i) + 8 * lane;
        if (q0 + i < q1 && col < a.cols && t < a.tokens) read8<XB>(a, from + col, v[i]);
    }
    if (gridDim.x > 1) {
#pragma unroll 4
        for (int col = 8 * lane; col < a.cols; col += 512) {
            float x[8];
            read8<XB>(a, from + col, x);
            m = fmaxf(m, largest(x));
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, largest(v[i]));
    const int e = scale_of(m);
    const float up = power(e);
    if (blockIdx.x == 0 && lane == 0) a.down[t] = power(-e);
    const auto put_sum = [&](int q, float x) {      // group q's
        __bf16 p[3];
        bf16_parts(x, p);
        uint8_t* to = a.xsums + ((int64_t)tile * sums + (q >> 5)) * kSumBytes + 16 * (16 * (q >> 3 & 3) + row) + 2 * (q & 7);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<__bf16*>(to + 1024 * k) = p[k];
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int b = 4 * (q0 + i) + (lane >> 4), col = 128 * b + 8 * (lane & 15);
        if (q0 + i >= q1) break;
        scale(v[i], up);
        const float sum = group_sum<G>(v[i]);
        uint8_t* rec = a.xparts + ((int64_t)tile * 4 * quads + b) * kRecord;
        if (col % G == 0) put_sum(col / G, sum);
        f16x8 hi, lo;
        parts(v[i], hi, lo);
        int step, g;
        place<G>(lane & 15, step, g);
        *reinterpret_cast<f16x8*>(rec + 16 * (64 * step + 16 * g + row)) = hi;
        if (P == 2) *reinterpret_cast<f16x8*>(rec + 4096 + 16 * (64 * step + 16 * g + row)) = lo;
    }
    if (blockIdx.x == 0)
        for (int q = 512 * quads / G + lane; q < 32 * sums; q += 64) put_sum(q, 0.f);
}

// Workgroup = 16 NT tokens, 16 MW rows of W a wave.  A wave's words come straight from memory,
// two blocks of 128 columns ahead, its scales four; the records through LDS, copied by the
// loads themselves, a block ahead.  The biases' part, sum_G b'_G X_G with b' = b + 8 s, is a
// product of its own before the others, of bf16 parts, six MFMAs for 32 groups: per value and
// group, with the sums read from LDS, it took as many instructions as the nibbles.
//
// Bound by a SIMD's two waves, whose MFMAs (35% of the time), vector work (37%: nibbles, scales) and LDS
// reads (34%, no bank conflicts) overlap only in part; setting them one beside the other by hand,
// operands a group ahead, changed nothing (122 us and 124).  800 x 6144 x 4096 f32, group 64: 107 us, 376
// TFLOP/s and, with both parts of x, 753 of the 1174 that a large f16 product reaches; 800 x 50304 x 2048
// 380 to 400 us (on different cards), of bf16 rows 294 to 311.
template <int G, int NT, int MW, bool XB>
__global__ __launch_bounds__(512, 4) void q4_many_kernel(Q4Args a) {
    constexpr int P = XB ? 1 : 2, kRecord = record_bytes(P), kStage = NT * kRecord, kSteps = G / 32, kWaves = 8;
    constexpr int kGroups = 512 / G, N = kGroups < 8 ? kGroups : 8;    // of a unit of four blocks, of one load
    __shared__ __attribute__((aligned(16))) uint8_t s_x[2 * kStage];
    __shared__ int s_last;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    // this workgroup's tile: one of the `whole` ones, or a share of one of the others
    const int id = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if (id >= a.grid) return;
    const int rest = id - a.whole, KW = rest < 0 ? 1 : a.split, kw = rest < 0 ? 0 : rest % KW;
    const int tile = rest < 0 ? id : a.whole + rest / KW;
    // all tokens of 32 blocks of rows, then of the next: an XCD's L2 keeps four blocks' words (800 x
    // 50304 x 2048 400 us, row by row of tiles 422; 800 x 50304 x 4096 786 and 851; of 16 blocks 405, 797)
    const int tall = (a.tokens + 16 * NT - 1) / (16 * NT), group = tile / (32 * tall), in = tile - group * 32 * tall;
    const int wide = min(32, a.grid_x - 32 * group), ty = in / wide, block = 32 * group + in - ty * wide;
    const int t0 = ty * 16 * NT, tile0 = (block * kWaves + wave) * MW;
    const int units = (a.cols + 511) / 512, sums = (a.cols / G + 31) / 32;
    const int u0 = (int)((int64_t)units * kw / KW), u1 = (int)((int64_t)units * (kw + 1) / KW), last = 4 * u1 - 1;
    const int tiles = min(NT, (a.tokens - t0 + 15) / 16);   // of tokens that there are
    int n[MW];
    Weights w[MW];
#pragma unroll
    for (int m = 0; m < MW; ++m) {
        n[m] = 16 * (tile0 + m) + c;
        w[m] = Weights(a, min(n[m], a.rows - 1), g);
    }
    const uint8_t* rec = a.xparts + (int64_t)ty * NT * 4 * units * kRecord;
    // block k's records to buffer s
    const auto copy = [&](int k, int s) {
#pragma unroll
        for (int i = 0; i < NT * 4 * P; i += kWaves) {
            if (NT * 4 * P % kWaves && i + wave >= NT * 4 * P) break;
            const int t = (i + wave) / (4 * P), j = (i + wave) % (4 * P);
            const uint8_t* from = rec + ((int64_t)min(t, tiles - 1) * 4 * units + k) * kRecord + 1024 * j;
            lds_copy16(16 * lane, from, lds_addr(s_x) + s * kStage + t * kRecord + 1024 * j);
        }
    };
    const auto scales = [&](int u, uint32_t (&x)[MW][kGroups / 2]) {
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < kGroups / N; ++i)
                w[m].template raw_halves<N>(w[m].s, u * kGroups + N * i, reinterpret_cast<uint32_t(&)[N / 2]>(x[m][i * N / 2]));
    };
    const auto settle = [&](int u, uint32_t (&x)[MW][kGroups / 2]) {
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < kGroups / N; ++i)
                w[m].template settle<N>(u * kGroups + N * i, reinterpret_cast<uint32_t(&)[N / 2]>(x[m][i * N / 2]));
    };
    f32x4v acc[MW * NT];
#pragma unroll
    for (int i = 0; i < MW * NT; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    for (int k = (sums * kw + KW - 1) / KW; k < (sums * (kw + 1) + KW - 1) / KW; ++k) {   // (the first shares have fewer units)
        constexpr int H = G == 128 ? 4 : 8;     // (a row has as many groups at least, or all rows together)
        bf16x8 y[NT][3], b[MW][3];
        uint32_t sv[MW][8 / H][H / 2], bv[MW][8 / H][H / 2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                y[t][p] = *reinterpret_cast<const bf16x8*>(
                    a.xsums + (((int64_t)ty * NT + min(t, tiles - 1)) * sums + k) * kSumBytes + 1024 * p + 16 * lane);
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < 8 / H; ++i) {
                w[m].template raw_halves<H>(w[m].s, 32 * k + 8 * g + H * i, sv[m][i]);
                w[m].template raw_halves<H>(w[m].b, 32 * k + 8 * g + H * i, bv[m][i]);
            }
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i % H == 0) {
                    w[m].template settle<H>(32 * k + 8 * g + i, sv[m][i / H]);
                    w[m].template settle<H>(32 * k + 8 * g + i, bv[m][i / H]);
                }
                __bf16 p[3];
                bf16_parts(fmaf(8.f, bf16_pair(sv[m][i / H], i % H), bf16_pair(bv[m][i / H], i % H)), p);
                b[m][0][i] = p[0], b[m][1][i] = p[1], b[m][2][i] = p[2];
            }
#pragma unroll
        for (int o = 2; o >= 0; --o)      // (small products first)
#pragma unroll
            for (int p = 0; p <= o; ++p)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int m = 0; m < MW; ++m)
                        acc[m * NT + t] =
                            __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[t][p], b[m][o - p], acc[m * NT + t], 0, 0, 0);
    }
    uint4 x[4][MW];
    uint32_t s_now[MW][kGroups / 2], s_next[MW][kGroups / 2];
    const auto words = [&](int k, uint4 (&y)[MW]) {
#pragma unroll
        for (int m = 0; m < MW; ++m) y[m] = w[m].words(k);
    };
    words(4 * u0, x[0]);
    scales(u0, s_now);
    copy(4 * u0, 0);
    words(4 * u0 + 1, x[1]);
    settle(u0, s_now);
    const NibK nk = nib_consts();
    for (int u = u0; u < u1; ++u) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int k = 4 * opaque(u) + b;
            wait_vm<MW>();        // (but for the next block's words)
            __syncthreads();      // (the block's records are there, and the other buffer read)
            uint32_t v[MW][4];
#pragma unroll
            for (int m = 0; m < MW; ++m) steps<G>(x[b][m], v[m]);
            // (past the last block: that one again, into a buffer that is not read)
            if (b == 2) scales(min(u + 1, u1 - 1), s_next), settle(min(u + 1, u1 - 1), s_next);
            copy(min(k + 1, last), ~b & 1);
            words(min(k + 2, last), x[(b + 2) & 3]);
            const uint8_t* s = s_x + (b & 1) * kStage;
            // (a tile's sums are added while the next one's MFMAs run; here and now: or the
            // compiler keeps all tiles' sums of a block for later)
            f32x4v part[2][MW];
            float sc[2][MW];
            const auto flush = [&](int i) {
#pragma unroll
                for (int m = 0; m < MW; ++m) {
                    f32x4v& y = acc[m * NT + i % NT];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = fmaf(sc[i / NT & 1][m], part[i & 1][m][e], y[e]);
                    asm volatile("" : "+v"(y));
                }
            };
#pragma unroll
            for (int qb = 0; qb < 4 / kSteps; ++qb) {     // the block's groups
                f16x8 q[MW][kSteps];
#pragma unroll
                for (int m = 0; m < MW; ++m) {
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) q[m][j] = nibbles(v[m][kSteps * qb + j], nk);
                    sc[qb & 1][m] = bf16_pair(s_now[m], 4 / kSteps * b + qb);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int i = qb * NT + t;
#pragma unroll
                    for (int m = 0; m < MW; ++m) part[i & 1][m] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int p = P - 1; p >= 0; --p)
#pragma unroll
                        for (int j = 0; j < kSteps; ++j) {
                            const f16x8 y = *reinterpret_cast<const f16x8*>(s + t * kRecord + 4096 * p +
                                                                            1024 * (kSteps * qb + j) + 16 * lane);
#pragma unroll
                            for (int m = 0; m < MW; ++m)
                                part[i & 1][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, q[m][j], part[i & 1][m], 0, 0, 0);
                        }
                    if (i > 0) flush(i - 1);
                }
            }
            flush(4 / kSteps * NT - 1);
        }
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < kGroups / 2; ++i) s_now[m][i] = s_next[m][i];
    }
    wait_vm<0>();     // (the last copy into LDS, before the LDS may be another workgroup's)
    if (KW > 1 && !join_split<MW * NT>(a, tile - a.whole, KW, kw, kWaves, wave, true, acc, &s_last)) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t >= tiles) break;
        const f32x4v down = *reinterpret_cast<const f32x4v*>(a.down + t0 + 16 * t + 4 * g);
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = t0 + 16 * t + 4 * g + i;
                if (n[m] < a.rows && tok < a.tokens) put(a, tok, n[m], acc[m * NT + t][i] * down[i]);
            }
    }
}

template <int G, int NT, int P, bool XB>
void launch_few(const Q4Args& a, hipStream_t st) {
    hipLaunchKernelGGL((q4_few_kernel<G, NT, P, XB>), dim3((unsigned)a.grid), dim3((unsigned)(64 * a.waves)),
                       (size_t)a.lds, st, a);
}

template <int G, int NT, int MW, bool XB>
void launch_many(const Q4Args& a, hipStream_t st) {
    hipLaunchKernelGGL((q4_parts_kernel<G, XB>), dim3((unsigned)a.part_split, (unsigned)((a.tokens + 15) / 16 * 4)), dim3(256),
                       0, st, a);
    // (a dimension of a grid holds less than 2^32 threads)
    const int x = std::min(a.grid, 1 << 14);
    hipLaunchKernelGGL((q4_many_kernel<G, NT, MW, XB>), dim3((unsigned)x, (unsigned)((a.grid + x - 1) / x)),
                       dim3((unsigned)(64 * a.waves)), 0, st, a);
}

template <int G, bool XB>
void launch_group(const Q4Args& a, hipStream_t st) {
    if (a.tiny)
        hipLaunchKernelGGL((q4_tiny_kernel<XB>), dim3((unsigned)a.tokens, (unsigned)a.rows), dim3(64), 0, st, a);
    else if (a.tokens > kFewTokens)
        launch_many<G, kManyTiles, kManyRows, XB>(a, st);
    else if (a.tokens <= (XB ? 16 : 8))
        launch_few<G, 1, 1, XB>(a, st);
    else if (!XB && a.tokens <= 16)
        launch_few<G, 1, XB ? 1 : 2, XB>(a, st);
    else
        launch_few<G, 2, XB ? 1 : 2, XB>(a, st);
}

}  // namespace

// Floats of the most partials that a call has: workgroups that share columns are at most two a CU, of 8
// waves with kManyRows by kManyTiles tiles, or one of 16 waves with two.  (This call's own would be
// fewer, but more than those of some calls of more tokens: a program that has run its largest step
// captures any other.)
static int64_t most_partials(int cus) { return (int64_t)2 * cus * 8 * kManyRows * kManyTiles * 256; }

int64_t matmul_q4_plan(Q4Args& a, int cus) {
    const int unit = a.group == 32 ? 256 : 512, units = (a.cols + unit - 1) / unit, groups = unit / a.group;
    const int tiles = (a.rows + 15) / 16;
    a.waves = 8;
    a.split = a.wave_split = 1;
    a.tiny = (int64_t)a.rows * (a.cols / a.group) < groups;
    if (a.tiny) return 0;
    if (a.tokens <= kFewTokens) {
        const bool flat = !a.x_bf16 && a.tokens <= 8;
        const int nt = a.tokens <= 16 ? 1 : 2, p = a.x_bf16 || flat ? 1 : 2;
        const int bytes = p * (unit / 32) * 64 * few_rows(flat ? 2 * a.tokens : a.tokens) + (groups + 1) * 64 * nt;
        // A tile's columns are shared by the waves of a workgroup, which need no second pass, as long as
        // staging x costs little: 4 tokens, all of whose columns fit the LDS at once; behind that by
        // workgroups, each of which stages its share only (2048 x 2048: 1 token 5.3 us so, 7.5 by
        // workgroups, 8 tokens 8.2 and 8.0; 6144 x 4096: 1 token 8.0 and 9.9, 4 bf16 ones 10.6 and
        // 11.0, 4 f32 ones, whose columns do not fit, 12.4 and 10.5, 8 15.3 and 11.3).
        // Tiles for every wave that the CUs hold: waves of workgroups that share them evenly, one a CU,
        // where that is a wave of a SIMD less than the 16 that fit (2048 columns, f32: 33000 rows, 9 waves,
        // 1 token 11.8 us, of 8 waves 14.8, 8 tokens 14.3, of 16 16.5; 50304 rows, 13 waves, 26 tokens 31.9,
        // of 16 30.5; 100000, twice 13, 1 token 28.6, of 8 26.4).
        const int rounds = (tiles + 16 * cus - 1) / (16 * cus), even = (tiles + rounds * cus - 1) / (rounds * cus);
        const bool apart = tiles > 8 * cus && even <= 12;
        if (a.tokens <= 4 && units * bytes <= kFewLds) {
            while (a.wave_split < 8 && 2 * a.wave_split <= units && tiles * a.wave_split * 2 <= 16 * cus) a.wave_split *= 2;
            // (workgroups of 4 while there are few: 2048 x 2048, 1 token 5.3 us, of 8 waves 5.6)
            if (a.wave_split <= 4 && tiles * a.wave_split < 8 * cus) a.waves = 4;
            if (apart) a.waves = std::max(8, even);
        } else {
            // (x is staged once for 16 waves where these still fill the card: 50304 x 2048, 16 f32 tokens
            // 20.6 us, of 8 waves 23.9; 2048 x 2048 8.9, of 16 waves 10.9)
            a.waves = apart ? std::max(8, even) : tiles >= 8 * cus ? 16 : 8;
            a.split = std::max(1, std::min(units, cus / ((tiles + a.waves - 1) / a.waves)));
        }
        const int per = a.waves / a.wave_split;
        // all of a workgroup's columns at once, of 16 waves in the LDS of two workgroups of 8
        a.chunk = std::max(1, std::min((a.waves > 8 ? 2 : 1) * kFewLds / bytes, (units + a.split - 1) / a.split));
        a.grid = (tiles + per - 1) / per * a.split;
        a.lds = std::max(a.chunk * bytes, a.wave_split > 1 ? a.waves * nt * 1024 : 16);
        return a.split > 1 ? most_partials(cus) : 0;
    }
    constexpr int nt = kManyTiles, mw = kManyRows;
    const int tt = (a.tokens + 15) / 16, quads = (a.cols + 511) / 512, sums = (a.cols / a.group + 31) / 32;
    // Whole tiles as long as there is one for every CU (two workgroups fit one); the columns of the
    // rest are shared by as many workgroups as there are CUs.  A join costs as much as two units of
    // columns, a second workgroup on a CU 0.6 of its time: f32, 4096 columns, n tiles, whole
    // and shared, 16 45.6 and 23.6 us, 64 47.1 and 28.9 (by twice as many 36.9), 112 48.4 and 37.9,
    // 208 50.3 and 53.7, 312 (256 of them whole) 78.3 and 61.4.  By twice as many where these are three
    // a tile and have units enough (168, 8 units: 48.4 and 43.4, 4 units: 28.1 and 28.9).
    a.grid_x = (tiles + mw * a.waves - 1) / (mw * a.waves);
    const int all = a.grid_x * ((tt + nt - 1) / nt);
    a.whole = all / cus * cus;
    const int rest = all - a.whole;
    if (rest) a.split = std::min(quads, cus / rest > 1 ? cus / rest : 2 * cus / rest == 3 && quads >= 8 ? 3 : 1);
    if (a.split == 1) a.whole = all;
    a.grid = a.whole + (all - a.whole) * a.split;
    // (as many workgroups as CUs where there are few tokens, though each reads whole rows for their
    // largest: 64 x 6144 x 4096 bf16 23.2 us, by the fewest 25.7)
    a.part_split = std::max((quads + 7) / 8, std::min(quads, cus / (4 * tt)));
    a.sums_at = (int64_t)tt * quads * record_bytes(a.x_bf16 ? 1 : 2);
    a.down_at = a.sums_at + (int64_t)tt * sums * kSumBytes / 4;
    a.part_at = a.down_at + 16 * tt;
    return a.part_at + most_partials(cus);
}

int launch_matmul_q4(const Q4Args& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (a.group) {
        case 32: a.x_bf16 ? launch_group<32, true>(a, st) : launch_group<32, false>(a, st); break;
        case 64: a.x_bf16 ? launch_group<64, true>(a, st) : launch_group<64, false>(a, st); break;
        case 128: a.x_bf16 ? launch_group<128, true>(a, st) : launch_group<128, false>(a, st); break;
        default: return (int)hipErrorInvalidValue;
    }
    return (int)hipGetLastError();
}

}  // namespace m1moe
