// q4.hip — products of rows with weights in 4 bits: y[t][n] = sum_k x[t][k] (q s + b)[n][k] (+ r).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "drafts.hpp"

namespace m1moe {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

constexpr int kFewTokens = 8;

// With the columns' groups G, y = sum_G (s_G sum_{k in G} x_k (q_k - 8) + (b_G + 8 s_G) X_G),
// X_G = sum_{k in G} x_k: the inner sum is an MFMA of f16 operands, exact products in f32
// sums, which the 8 keeps small.
//
// A nibble q, masked where it stands in the low (or second) four bits of a 16-bit half, under the
// exponent of 1024 is 1024 + q (or 1024 + 16 q): nine instructions make the MFMA operand q - 8 of
// a word's eight columns, in the order 0 4 1 5 2 6 3 7.  (q 2^-24 as a subnormal would take
// five, but an MFMA aligns its products by their operands' exponents, and of subnormals
// drops the last 7 bits.)  x meets them in that order, times a power of two 2^e that
// brings the row's largest value (of a chunk of columns) to 2^14 .. 2^15: an f32 x as two f16
// parts (22 bits; what is below 2^-28 of the row's largest is kept to 2^-39 of that one), a
// bf16 x as one.

// ---- few tokens ------------------------------------------------------------------------
//
// Bound by reading the weights once.  A wave has a tile of 16 rows n of W, its lane (c, g) the
// row n = c: 16 bytes, 32 columns, of each 128 at a time straight from memory into registers,
// a unit of columns ahead; v_permlane swaps bring the words of one group together.  x is staged
// in LDS as the other operand, a chunk of columns at a time; its rows are the tokens, or
// of f32 tokens the two parts of each, which fill the rows of one MFMA for up to 8 tokens.
// KS waves of a workgroup share a tile's columns.
template <int G>
struct Unit {
    static constexpr int NQ = G == 32 ? 2 : 4;          // 128-column blocks
    static constexpr int kCols = 128 * NQ, kGroups = kCols / G;
    uint4 w[NQ];
    uint32_t s[kGroups / 2], b[kGroups / 2];            // bf16 pairs
};

struct Weights {
    const uint8_t* w;                  // the lane's row, at its 32 columns of the first block
    const uint16_t *s, *b;             // its scales and biases
    int cols, groups, g;
    bool whole;                        // units' scales are whole aligned vectors

    Weights() = default;
    __device__ __forceinline__ Weights(const Q4Args& a, int row, int lane_g, int unit_groups) {
        cols = a.cols;
        groups = a.cols / a.group;
        g = lane_g;
        w = reinterpret_cast<const uint8_t*>(a.w) + (int64_t)row * (a.cols / 2) + 16 * g;
        s = a.scales + (int64_t)row * groups;
        b = a.biases + (int64_t)row * groups;
        whole = groups % unit_groups == 0;
    }

    template <int G>
    __device__ __forceinline__ void load(int u, Unit<G>& x) const {
        typedef Unit<G> U;
#pragma unroll
        for (int i = 0; i < U::NQ; ++i) {
            // (past the row: its last columns again, which meet x = 0 and scales of 0)
            const int col = min(u * U::kCols + 128 * i, cols - 32 * (g + 1));
            x.w[i] = *reinterpret_cast<const uint4*>(w + (col >> 1));
        }
        const int q0 = u * U::kGroups;
        if (whole) {
            if constexpr (U::kGroups == 8) {
                const uint4 p = *reinterpret_cast<const uint4*>(s + q0), q = *reinterpret_cast<const uint4*>(b + q0);
                x.s[0] = p.x, x.s[1] = p.y, x.s[2] = p.z, x.s[3] = p.w;
                x.b[0] = q.x, x.b[1] = q.y, x.b[2] = q.z, x.b[3] = q.w;
            } else {
                const uint2 p = *reinterpret_cast<const uint2*>(s + q0), q = *reinterpret_cast<const uint2*>(b + q0);
                x.s[0] = p.x, x.s[1] = p.y;
                x.b[0] = q.x, x.b[1] = q.y;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < U::kGroups; i += 2) {
            const int i0 = min(q0 + i, groups - 1), i1 = min(q0 + i + 1, groups - 1);
            const uint32_t s0 = s[i0], s1 = s[i1], b0 = b[i0], b1 = b[i1];
            x.s[i / 2] = (q0 + i < groups ? s0 : 0u) | (q0 + i + 1 < groups ? s1 << 16 : 0u);
            x.b[i / 2] = (q0 + i < groups ? b0 : 0u) | (q0 + i + 1 < groups ? b1 << 16 : 0u);
        }
    }
};

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

// The largest of eight values over the wave: 2^e brings it to 2^14 .. 2^15 (zeros: as 2^-112).
__device__ __forceinline__ int scale_of(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
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
// They times 2^e as f16 parts, in the order of a word's nibbles.
__device__ __forceinline__ void parts(const float (&v)[8], float up, f16x8& hi, f16x8& lo) {
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = v[order[j]] * up;
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

// A unit's sums into the whole: acc += unit 2^-e, row by row.
__device__ __forceinline__ void flush(f32x4v& acc, f32x4v unit, f32x4v down) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(unit[e], down[e], acc[e]);
}

// RT: operand rows of a token.
template <int G, bool XB>
struct Few {
    typedef Unit<G> U;
    static constexpr int kTokens = 8, RT = XB ? 1 : 2;

    const Q4Args& a;
    int t0, tn, R;               // tokens, rows staged
    uint8_t* s_x;                // [units][4 NQ steps][4][R] 16 bytes
    float* s_sum;                // [units][groups][16]: X_G 2^e, row 2 t (or t)
    float* s_down;               // [units][16]: 2^-e

    __device__ __forceinline__ uint8_t* at(int u, int step, int g, int row) const {
        return s_x + 16 * (((u * 4 * U::NQ + step) * 4 + g) * R + row);
    }

    // n units from column k0 on, by all waves, a token's unit each.
    __device__ __forceinline__ void stage(int k0, int n) {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
        for (int i = wave; i < tn * n; i += waves) {
            const int t = i / n, u = i - t * n, row = RT * t, at0 = 8 * lane, col = k0 + u * U::kCols + at0;
            float v[8] = {};
            if (at0 < U::kCols && col < a.cols) read8<XB>(a, (int64_t)(t0 + t) * a.x_stride + col, v);
            const int e = scale_of(v);
            const float up = power(e), sum = group_sum<G>(v);
            if (lane < RT) s_down[16 * u + row + lane] = power(-e);
            if (at0 >= U::kCols) continue;
            if (at0 % G == 0) {
                float* to = s_sum + (u * U::kGroups + at0 / G) * 16 + row;
                to[0] = sum * up;
                if (RT == 2) to[1] = 0.f;
            }
            f16x8 hi, lo;
            parts(v, up, hi, lo);
            int step, g;
            place<G>(lane & 15, step, g);
            step += 4 * (lane >> 4);
            *reinterpret_cast<f16x8*>(at(u, step, g, row)) = hi;
            if (RT == 2) *reinterpret_cast<f16x8*>(at(u, step, g, row + 1)) = lo;
        }
    }

    // Unit x, unit u of the chunk.
    __device__ __forceinline__ void add(const U& x, int u, int c, int g, f32x4v& acc) const {
        constexpr int kSteps = G / 32;                 // of a group
        const int row = min(c, R - 1);
        const NibK k = nib_consts();
        f32x4v unit = {0.f, 0.f, 0.f, 0.f}, part;
#pragma unroll
        for (int i = 0; i < U::NQ; ++i) {
            uint32_t v[4];
            steps<G>(x.w[i], v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j % kSteps == 0) part = f32x4v{0.f, 0.f, 0.f, 0.f};
                part = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    *reinterpret_cast<const f16x8*>(at(u, 4 * i + j, g, row)), nibbles(v[j], k), part, 0, 0, 0);
                if (j % kSteps == kSteps - 1) {
                    const int q = (4 * i + j) / kSteps;     // group of the unit
                    const float s = bf16_pair(x.s, q), b = fmaf(8.f, s, bf16_pair(x.b, q));
                    const f32x4v sum = *reinterpret_cast<const f32x4v*>(s_sum + (u * U::kGroups + q) * 16 + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) unit[e] = fmaf(b, sum[e], fmaf(s, part[e], unit[e]));
                }
            }
        }
        flush(acc, unit, *reinterpret_cast<const f32x4v*>(s_down + 16 * u + 4 * g));
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

template <int G, bool XB>
__global__ __launch_bounds__(512) void q4_few_kernel(Q4Args a) {
    typedef Few<G, XB> F;
    typedef Unit<G> U;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_buf[];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = (int)blockDim.x >> 6;
    const int c = lane & 15, g = lane >> 4, KS = a.wave_split, ks = wave % KS;
    const int tile = (int)blockIdx.x * (waves / KS) + wave / KS;
    F f{a};
    f.t0 = 0;
    f.tn = a.tokens;
    f.R = F::RT * f.tn;
    f.s_x = s_buf;
    f.s_sum = reinterpret_cast<float*>(s_buf + a.chunk * (4 * U::NQ) * 64 * f.R);
    f.s_down = f.s_sum + a.chunk * U::kGroups * 16;
    const int units = (a.cols + U::kCols - 1) / U::kCols;
    const bool on = 16 * tile < a.rows;
    const int n = 16 * tile + c;
    const Weights w(a, min(n, a.rows - 1), g, U::kGroups);
    f32x4v acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < units; k += a.chunk) {
        const int nu = min(a.chunk, units - k), lo = nu * ks / KS, hi = nu * (ks + 1) / KS;
        U x[2];
        if (on && lo < hi) w.load<G>(k + lo, x[0]);
        if (k) __syncthreads();
        f.stage(k * U::kCols, nu);
        __syncthreads();
        if (!on) continue;
        for (int u = lo; u < hi; u += 2) {
            if (u + 1 < hi) w.load<G>(k + u + 1, x[1]);
            f.add(x[0], u, c, g, acc);
            if (u + 1 >= hi) break;
            if (u + 2 < hi) w.load<G>(k + u + 2, x[0]);
            f.add(x[1], u + 1, c, g, acc);
        }
    }
    // the waves of a tile, in their order
    if (KS > 1) {
        f32x4v* s = reinterpret_cast<f32x4v*>(s_buf);
        __syncthreads();
        s[tid] = acc;
        __syncthreads();
        if (ks) return;
        for (int i = 1; i < KS; ++i) acc += s[tid + 64 * i];
    }
    if (!on || n >= a.rows) return;
    if constexpr (F::RT == 2) {
        if (2 * g < f.tn) put(a, 2 * g, n, acc[0] + acc[1]);
        if (2 * g + 1 < f.tn) put(a, 2 * g + 1, n, acc[2] + acc[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * g + i < f.tn) put(a, 4 * g + i, n, acc[i]);
    }
}

// ---- many tokens -----------------------------------------------------------------------
//
// x is made into f16 parts once, by a kernel of its own: records of 16 tokens' 128 columns, [P
// parts][4 steps][64 lanes] 16 bytes, as the MFMAs take them, then the groups' sums [4][16]
// and 2^-e [16] (e: of a token's unit of columns).
constexpr int record_bytes(int p) { return 4096 * p + 512; }

// Workgroup = (16 tokens, unit of columns), a wave per token.
template <int G, bool XB>
__global__ __launch_bounds__(1024) void q4_parts_kernel(Q4Args a) {
    typedef Unit<G> U;
    constexpr int P = XB ? 1 : 2, kRecord = record_bytes(P);
    __shared__ __attribute__((aligned(16))) uint8_t s_rec[U::NQ * kRecord];
    const int tid = (int)threadIdx.x, lane = tid & 63, row = tid >> 6;
    const int tile = (int)blockIdx.y, u = (int)blockIdx.x, blocks = (int)gridDim.x * U::NQ;
    const int t = 16 * tile + row, at0 = 8 * lane, col = u * U::kCols + at0;
    float v[8] = {};
    if (t < a.tokens && at0 < U::kCols && col < a.cols) read8<XB>(a, (int64_t)t * a.x_stride + col, v);
    const int e = scale_of(v);
    const float up = power(e), sum = group_sum<G>(v);
    if (at0 < U::kCols) {
        uint8_t* rec = s_rec + (lane >> 4) * kRecord;
        float* tail = reinterpret_cast<float*>(rec + 4096 * P);
        if (at0 % G == 0) tail[(at0 & 127) / G * 16 + row] = sum * up;
        if ((lane & 15) == 0) tail[64 + row] = power(-e);
        f16x8 hi, lo;
        parts(v, up, hi, lo);
        int step, g;
        place<G>(lane & 15, step, g);
        *reinterpret_cast<f16x8*>(rec + 16 * (64 * step + 16 * g + row)) = hi;
        if (P == 2) *reinterpret_cast<f16x8*>(rec + 4096 + 16 * (64 * step + 16 * g + row)) = lo;
    }
    __syncthreads();
    uint4* to = reinterpret_cast<uint4*>(a.xparts + ((int64_t)tile * blocks + u * U::NQ) * kRecord);
    for (int i = tid; i < U::NQ * kRecord / 16; i += 1024) to[i] = reinterpret_cast<const uint4*>(s_rec)[i];
}

// Workgroup = 16 NT tokens, 16 MW rows of W a wave; a wave's words come straight from memory as
// above, the records through LDS, copied by the loads themselves, SB blocks of 128 columns
// at a time, the next ones on their way while some are computed.
template <int G, int NT, int MW, bool XB>
struct Many {
    typedef Unit<G> U;
    static constexpr int P = XB ? 1 : 2, kRecord = record_bytes(P);
    static constexpr int SB = std::min(U::NQ, std::max(1, 8 / (NT * P)));
    static constexpr int kStage = SB * NT * kRecord;
};

template <int G, int NT, int MW, bool XB>
__global__ __launch_bounds__(512, 2) void q4_many_kernel(Q4Args a) {
    typedef Many<G, NT, MW, XB> M;
    typedef Unit<G> U;
    constexpr int P = M::P, SB = M::SB, kRecord = M::kRecord, kSteps = G / 32;
    __shared__ __attribute__((aligned(16))) uint8_t s_x[2 * M::kStage];
    __shared__ int s_last;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int waves = (int)blockDim.x >> 6, c = lane & 15, g = lane >> 4, KW = a.split;
    const int kw = (int)blockIdx.x % KW, block = (int)blockIdx.x / KW;
    const int t0 = (int)blockIdx.y * 16 * NT, tile0 = (block * waves + wave) * MW;
    const int units = (a.cols + U::kCols - 1) / U::kCols, blocks = units * U::NQ;
    const int u0 = (int)((int64_t)units * kw / KW), u1 = (int)((int64_t)units * (kw + 1) / KW);
    const bool on = 16 * tile0 < a.rows;
    const int tiles = min(NT, (a.tokens - t0 + 15) / 16);   // of tokens that there are
    int n[MW];
    Weights w[MW];
#pragma unroll
    for (int m = 0; m < MW; ++m) {
        n[m] = 16 * (tile0 + m) + c;
        w[m] = Weights(a, min(n[m], a.rows - 1), g, U::kGroups);
    }
    const uint8_t* rec = a.xparts + (int64_t)blockIdx.y * NT * blocks * kRecord;
    // SB blocks from block k on to buffer s
    const auto copy = [&](int k, int s) {
        constexpr int kUnits = kRecord / 512;      // half-kilobytes of a record
#pragma unroll 1
        for (int i = wave; i < NT * SB; i += waves) {
            const int t = i / SB, b = i - t * SB;
            const uint8_t* from = rec + ((int64_t)min(t, tiles - 1) * blocks + k + b) * kRecord;
            const uint32_t to = lds_addr(s_x) + s * M::kStage + (t * SB + b) * kRecord;
#pragma unroll
            for (int j = 0; j + 1 < kUnits; j += 2) lds_copy16(16 * lane + 512 * j, from, to + 512 * j);
            if (lane < 32) lds_copy16(16 * lane + 512 * (kUnits - 1), from, to + 512 * (kUnits - 1));
        }
    };
    f32x4v acc[MW][NT], unit[MW][NT];
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = unit[m][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
    U x[2][MW];
    const NibK nk = nib_consts();
    int turn = 0;
    // Unit u, x; the next one's words, y, are asked for behind the second stage's records.
    const auto compute = [&](const U (&x)[MW], U (&y)[MW], int u, bool more) {
#pragma unroll
        for (int b0 = 0; b0 < U::NQ; b0 += SB) {
            if (b0 == SB && on && more)
                wait_vm<MW * (U::NQ + 2)>();
            else
                wait_vm<0>();
            __syncthreads();      // (the stage is there, and the other one read)
            if (b0 + SB < U::NQ || more) copy(u * U::NQ + b0 + SB, turn ^ 1);
            if (b0 == 0 && on && more) {
#pragma unroll
                for (int m = 0; m < MW; ++m) w[m].template load<G>(u + 1, y[m]);
            }
            const uint8_t* s = s_x + turn * M::kStage;
            turn ^= 1;
            if (!on) continue;
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                uint32_t v[MW][4];
#pragma unroll
                for (int m = 0; m < MW; ++m) steps<G>(x[m].w[b0 + b], v[m]);
                f32x4v part[MW][NT];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f16x8 q[MW];
#pragma unroll
                    for (int m = 0; m < MW; ++m) q[m] = nibbles(v[m][j], nk);
#pragma unroll
                    for (int p = P - 1; p >= 0; --p)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const f16x8 y = *reinterpret_cast<const f16x8*>(s + (t * SB + b) * kRecord + 4096 * p +
                                                                            1024 * j + 16 * lane);
#pragma unroll
                            for (int m = 0; m < MW; ++m) {
                                if (j % kSteps == 0 && p == P - 1) part[m][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
                                part[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, q[m], part[m][t], 0, 0, 0);
                            }
                        }
                    if (j % kSteps == kSteps - 1) {
                        const int qb = j / kSteps, qu = (4 * (b0 + b) + j) / kSteps;   // group of the block, the unit
                        float sc[MW], bi[MW];
#pragma unroll
                        for (int m = 0; m < MW; ++m) {
                            sc[m] = bf16_pair(x[m].s, qu);
                            bi[m] = fmaf(8.f, sc[m], bf16_pair(x[m].b, qu));
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const f32x4v sum = *reinterpret_cast<const f32x4v*>(s + (t * SB + b) * kRecord + 4096 * P +
                                                                                64 * qb + 16 * g);
#pragma unroll
                            for (int m = 0; m < MW; ++m)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    unit[m][t][e] = fmaf(bi[m], sum[e], fmaf(sc[m], part[m][t][e], unit[m][t][e]));
                        }
                    }
                }
            }
            if (b0 + SB == U::NQ) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f32x4v down = *reinterpret_cast<const f32x4v*>(s + t * SB * kRecord + 4096 * P + 256 + 16 * g);
#pragma unroll
                    for (int m = 0; m < MW; ++m) {
                        flush(acc[m][t], unit[m][t], down);
                        unit[m][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
                    }
                }
            }
        }
    };
    copy(u0 * U::NQ, 0);
    if (on) {
#pragma unroll
        for (int m = 0; m < MW; ++m) w[m].template load<G>(u0, x[0][m]);
    }
    for (int u = u0; u < u1; u += 2) {
        compute(x[0], x[1], u, u + 1 < u1);
        if (u + 1 < u1) compute(x[1], x[0], u + 1, u + 2 < u1);
    }
    if (KW > 1) {
        // the last of the workgroups that share a block's columns to end joins them
        const int id = (int)blockIdx.y * ((int)gridDim.x / KW) + block;
        const int64_t wg = (int64_t)waves * MW * NT * 256;
        float* part = a.part + (int64_t)id * KW * wg + (int64_t)wave * MW * NT * 256 + 4 * lane;   // [KW][waves][MW][NT][64][4]
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float y[4] = {acc[m][t][0], acc[m][t][1], acc[m][t][2], acc[m][t][3]};
                store4_coh(part + kw * wg + (m * NT + t) * 256, y);
            }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0) {
            s_last = __hip_atomic_fetch_add(a.counters + id, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                     (uint32_t)(KW - 1);
            if (s_last) __hip_atomic_store(a.counters + id, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!s_last) return;
        // (in the order of the columns, whoever is last)
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4v sum = {0.f, 0.f, 0.f, 0.f};
                for (int i0 = 0; i0 < KW; i0 += 8) {
                    const float* at[8];
                    f32x4v y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) at[i] = part + min(i0 + i, KW - 1) * wg + (m * NT + t) * 256;
                    load8_coh(at, y);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i0 + i < KW) sum += y[i];
                }
                acc[m][t] = sum;
            }
    }
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = t0 + 16 * t + 4 * g + i;
                if (n[m] < a.rows && tok < a.tokens) put(a, tok, n[m], acc[m][t][i]);
            }
}

template <int G, int NT, int MW, bool XB>
void launch_many(const Q4Args& a, hipStream_t st) {
    hipLaunchKernelGGL((q4_many_kernel<G, NT, MW, XB>), dim3((unsigned)a.grid, (unsigned)a.grid_y),
                       dim3((unsigned)(64 * a.waves)), 0, st, a);
}

template <int G, bool XB>
void launch_group(const Q4Args& a, hipStream_t st) {
    if (a.tokens <= kFewTokens) {
        hipLaunchKernelGGL((q4_few_kernel<G, XB>), dim3((unsigned)a.grid), dim3((unsigned)(64 * a.waves)), (size_t)a.lds, st, a);
        return;
    }
    const int units = (a.cols + Unit<G>::kCols - 1) / Unit<G>::kCols;
    hipLaunchKernelGGL((q4_parts_kernel<G, XB>), dim3((unsigned)units, (unsigned)((a.tokens + 15) / 16)), dim3(1024), 0, st, a);
    switch (a.tiles) {
        case 1: launch_many<G, 1, 2, XB>(a, st); break;
        case 2: launch_many<G, 2, 2, XB>(a, st); break;
        default: launch_many<G, 4, 2, XB>(a, st); break;
    }
}

}  // namespace

int64_t matmul_q4_plan(Q4Args& a, int cus) {
    const int unit = a.group == 32 ? 256 : 512, units = (a.cols + unit - 1) / unit;
    const int tiles = (a.rows + 15) / 16;
    a.waves = 8;
    a.split = a.wave_split = 1;
    if (a.tokens <= kFewTokens) {
        const int rows = (a.x_bf16 ? 1 : 2) * a.tokens, bytes = rows * unit * 2 + unit / a.group * 64 + 64;
        // chunks of at most 48 KB, so that three workgroups fit a CU
        a.chunk = std::max(1, std::min(49152 / bytes, units));
        while (a.wave_split < 8 && 2 * a.wave_split <= units && tiles * a.wave_split * 2 <= 16 * cus) a.wave_split *= 2;
        if (a.wave_split <= 4 && tiles * a.wave_split < 8 * cus) a.waves = 4;
        const int per = a.waves / a.wave_split;
        a.grid = (tiles + per - 1) / per;
        a.lds = std::max(a.chunk * bytes, a.waves * 1024);
        return 0;
    }
    const int tt = (a.tokens + 15) / 16;
    a.tiles = tt == 1 ? 1 : tt == 2 ? 2 : 4;
    a.grid_y = (tt + a.tiles - 1) / a.tiles;
    const int blocks = (tiles + 2 * a.waves - 1) / (2 * a.waves);
    a.split = std::max(1, std::min(units, cus / (blocks * a.grid_y)));
    a.grid = blocks * a.split;
    const int64_t record = record_bytes(a.x_bf16 ? 1 : 2), records = (int64_t)tt * units * (unit / 128) * record / 4;
    a.part_at = records;
    return records + (a.split > 1 ? (int64_t)a.grid * a.grid_y * a.waves * 2 * a.tiles * 256 : 0);
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
