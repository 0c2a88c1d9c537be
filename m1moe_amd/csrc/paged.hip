// paged.hip — a KV cache in pages for a batch of sequences: append (per-head
// q/k RMSNorm, RoPE and the store in one pass) and attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged.hpp"

namespace m1moe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

// Sequence s of the batch as m1moe_paged_batch requires it.
__device__ __forceinline__ bool seq_ok(const PagedView& p, int lo, int hi, int len) {
    if (lo < 0 || hi < lo || hi > p.num_rows || len < hi - lo) return false;
    if ((int64_t)len > (int64_t)p.table_stride << p.page_shift) return false;
    return hi == lo || len - (hi - lo) >= p.prefix_len;
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{x, y}, bf16x2));
}

// ---- append --------------------------------------------------------------------------

template <int VEC>
__device__ __forceinline__ void store_vec(void* base, int64_t at, const float (&x)[VEC], bool bf16) {
    if (bf16) {
        uint32_t* d = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(base) + at);
        uint32_t w[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
        if (VEC == 8)
            *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[VEC / 2 - 2], w[VEC / 2 - 1]);
        else
            *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    } else {
        float* d = static_cast<float*>(base) + at;
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<float4*>(d + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
}

// Workgroup = (row, a share of its q, k and v heads).  A lane holds VEC
// neighbouring dims (16 bytes) of a head; the head's sum of squares and, in
// the half layout, a pair's other dim come from the head's other lanes.  The
// row's cos and sin are made once per workgroup: the angle is an exact product
// of an int and an f32 in f64, reduced there by multiples of 2 pi (in two
// parts, so that a position of 2^24 loses nothing), the rest in f32.
template <int HD, bool XB>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    constexpr int VEC = XB ? 8 : 4, LPH = HD / VEC, HPB = 256 / LPH;
    __shared__ unsigned long long s_place;
    __shared__ float2 s_cs[HD / 2];
    const PagedView& p = a.p;
    const int tid = threadIdx.x, row = (int)blockIdx.x, slot = tid / LPH, l = tid % LPH;
    if (tid == 0) s_place = ~0ull;
    __syncthreads();
    // the row's sequence and position (the lowest sequence, should the starts be wrong)
    for (int s = tid; s < p.num_seqs; s += 256) {
        const int lo = p.row_start[s], hi = p.row_start[s + 1], len = p.kv_len[s];
        if (!seq_ok(p, lo, hi, len)) {
            if (row == 0 && blockIdx.y == 0) flag_error(p.err, kErrPagedBatch);
        } else if (row >= lo && row < hi) {
            atomicMin(&s_place, (unsigned long long)s << 32 | (uint32_t)(len - (hi - row)));
        }
    }
    __syncthreads();
    const unsigned long long place = s_place;
    if (place == ~0ull) return;
    const int seq = (int)(place >> 32), pos = (int)(uint32_t)place;
    const int page = p.pages[(int64_t)seq * p.table_stride + (pos >> p.page_shift)];
    if (tid < a.rotary / 2) {
        const double ang = (double)pos * (double)a.inv_freq[tid];
        const double k = rint(ang * 0.15915494309189533577);
        const float r = (float)fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586232, ang));
        s_cs[tid] = make_float2(cosf(r) * a.amp, sinf(r) * a.amp);
    }
    __syncthreads();
    const bool page_ok = page >= 0 && page < p.num_pages;
    if (!page_ok && tid == 0) flag_error(p.err, kErrPagedPage);
    const int64_t cell =
        (((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) * p.kv_heads * HD;
    const int total = a.heads + 2 * p.kv_heads, h2 = a.rotary / 2, c = VEC * l;
    for (int b = (int)blockIdx.y * HPB; b < total; b += (int)gridDim.y * HPB) {
        const int head = b + slot;
        const bool on = head < total, is_q = head < a.heads, is_v = head >= a.heads + p.kv_heads;
        const int kh = head - a.heads - (is_v ? p.kv_heads : 0);
        float x[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = 0.f;
        if (on) {
            const void* src = is_q ? a.q : is_v ? a.v : a.k;
            const int64_t at = (int64_t)row * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) +
                               (int64_t)(is_q ? head : kh) * HD + c;
            if constexpr (XB) {
                const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = bf16x8_at(w, i);
            } else {
                const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(src) + at);
                x[0] = w.x;
                x[1] = w.y;
                x[2] = w.z;
                x[3] = w.w;
            }
        }
        const uint16_t* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
        // (lanes of other heads of the wave take part in the exchanges)
        if (a.q_norm || a.k_norm) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) s = fmaf(x[i], x[i], s);
#pragma unroll
            for (int m = 1; m < LPH; m <<= 1) s += __shfl_xor(s, m, LPH);
            if (w) {
                const float f = 1.0f / sqrtf(s * (1.0f / HD) + a.eps);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = x[i] * f * bf16_to_f32(w[c + i]);
            }
        }
        if (a.rotary && a.interleaved) {
            if (!is_v && c < a.rotary) {
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    const float2 cs = s_cs[(c + i) / 2];
                    const float x0 = x[i], x1 = x[i + 1];
                    x[i] = x0 * cs.x - x1 * cs.y;
                    x[i + 1] = x0 * cs.y + x1 * cs.x;
                }
            }
        } else if (a.rotary) {
            const bool lower = c < h2;
            const int other = lower ? l + h2 / VEC : l - h2 / VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float y = __shfl(x[i], other & (LPH - 1), LPH);
                if (!is_v && c < a.rotary) {
                    const float2 cs = s_cs[lower ? c + i : c - h2 + i];
                    x[i] = lower ? x[i] * cs.x - y * cs.y : y * cs.y + x[i] * cs.x;
                }
            }
        }
        if (!on) continue;
        if (is_q)
            store_vec(a.q_out, (int64_t)row * a.q_out_stride + (int64_t)head * HD + c, x, XB);
        else if (page_ok)
            store_vec(is_v ? p.v : p.k, cell + (int64_t)kh * HD + c, x, a.cache_bf16 != 0);
    }
}

// ---- attention -----------------------------------------------------------------------

// Eight f32 values as three bf16 parts that add up to them exactly.
struct Parts8 {
    bf16x8 h, m, l;
};
__device__ __forceinline__ Parts8 parts8(const float (&v)[8]) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x0 = v[2 * i], x1 = v[2 * i + 1];
        h[i] = pack_bf16(x0, x1);
        const float r0 = x0 - __uint_as_float(h[i] << 16), r1 = x1 - __uint_as_float(h[i] & 0xFFFF0000u);
        m[i] = pack_bf16(r0, r1);
        l[i] = pack_bf16(r0 - __uint_as_float(m[i] << 16), r1 - __uint_as_float(m[i] & 0xFFFF0000u));
    }
    Parts8 s;
    s.h = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
    s.m = __builtin_bit_cast(bf16x8, make_uint4(m[0], m[1], m[2], m[3]));
    s.l = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
    return s;
}

__device__ __forceinline__ f32x4v mfma(bf16x8 a, bf16x8 b, f32x4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quads_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float w = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(w), __float_as_uint(w), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float quads_add(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float w = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(w), __float_as_uint(w), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// e^(x scale) of a difference of raw scores, as the hardware exp2.
__device__ __forceinline__ float weight(float x, float unit) { return __builtin_amdgcn_exp2f(x * unit); }

constexpr int kCut = 256;        // keys: where a tile's keys may be cut between workgroups
constexpr int kFewKeys = 128;    // least keys per workgroup

// How the rows and keys are shared.  A tile is up to R = 64 NT rows (token,
// head) of one sequence and kv head, whole tokens: TT = R / share tokens.  Its
// keys are the positions from `org` (the prefix' end rounded down to 32) to its
// last token's; all tiles' keys, sequence by sequence, head by head, tile by
// tile, form one line that is cut into equal shares, one per workgroup, the
// cuts moved down to a multiple of kCut inside their tile.
struct Tile {
    int seq, head, r;            // sequence, kv head, tile of its rows
    int row0, n, base;           // the sequence's first row, rows, positions before them
    int64_t start, end;          // on the line
};

struct Line {
    int64_t* cum;                // LDS [num_seqs + 1]: the sequences' starts on the line
    int64_t total;
    int wgs;                     // workgroups that have a share
    int org, TT, kv_heads;

    // keys of the first r tiles of a head (r below the number of tiles)
    __device__ int64_t before(int base, int r) const {
        return (int64_t)r * (base - org) + (int64_t)TT * r * (r + 1) / 2;
    }
    __device__ int64_t head_keys(int base, int n, int tiles) const {
        return before(base, tiles - 1) + (base - org) + n;
    }
    __device__ int64_t cut(int w) const {
        return w >= wgs ? total : (int64_t)((double)total * w / wgs);
    }
    // The tile that holds place x (0 <= x < total) of sequence s.
    __device__ Tile tile(const PagedView& p, int s, int64_t x) const {
        Tile t;
        t.seq = s;
        t.row0 = p.row_start[s];
        t.n = p.row_start[s + 1] - t.row0;
        t.base = p.kv_len[s] - t.n;
        const int tiles = (t.n + TT - 1) / TT;
        const int64_t hk = head_keys(t.base, t.n, tiles);
        int64_t off = x - cum[s];
        t.head = (int)(off / hk);
        off -= (int64_t)t.head * hk;
        int lo = 0, hi = tiles - 1;       // the last tile that starts at or before off
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before(t.base, mid) <= off)
                lo = mid;
            else
                hi = mid - 1;
        }
        t.r = lo;
        t.start = cum[s] + (int64_t)t.head * hk + before(t.base, lo);
        t.end = t.start + (t.base - org) + min(t.n, (lo + 1) * TT);
        return t;
    }
    __device__ int64_t rounded(const Tile& t, int64_t x) const {
        return t.start + (x - t.start) / kCut * kCut;
    }
};

// Fills cum (and line): the whole workgroup of 256.  tmp: LDS, 4 values.
__device__ __forceinline__ void make_line(const PagedView& p, Line& ln, int64_t* tmp, int grid, bool flag) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int64_t carry = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += 256) {
        const int s = b0 + tid;
        int64_t keys = 0;
        if (s < p.num_seqs) {
            const int lo = p.row_start[s], hi = p.row_start[s + 1], len = p.kv_len[s], n = hi - lo;
            if (!seq_ok(p, lo, hi, len)) {
                if (flag) flag_error(p.err, kErrPagedBatch);
            } else if (n > 0) {
                keys = ln.kv_heads * ln.head_keys(len - n, n, (n + ln.TT - 1) / ln.TT);
            }
        }
        int64_t sum = keys;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int64_t o = __shfl_up(sum, m);
            if (lane >= m) sum += o;
        }
        if (lane == 63) tmp[wave] = sum;
        __syncthreads();
        int64_t at = carry;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += tmp[w];
            carry += tmp[w];
        }
        if (s < p.num_seqs) ln.cum[s] = at + sum - keys;
        __syncthreads();
    }
    if (tid == 0) ln.cum[p.num_seqs] = carry;
    ln.total = carry;
    ln.wgs = (int)min((int64_t)grid, max((int64_t)1, carry / kFewKeys));
    __syncthreads();
}

// The sequence that holds place x < total.
__device__ __forceinline__ int find_seq(const PagedView& p, const Line& ln, int64_t x) {
    int lo = 0, hi = p.num_seqs - 1;      // the last start at or before x: of equal ones
    while (lo < hi) {                     // (empty sequences) the last
        const int mid = (lo + hi + 1) / 2;
        if (ln.cum[mid] <= x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// What a workgroup computes at once: rows of one kv head over a range of keys.
struct Work {
    int token0, tokens;       // rows of q and out
    int pos0;                 // position of token0
    int row_pos;              // positions per token: 1, or 0 where all see every key (the prefix)
    int head0;                // first query head
    int lo, hi;               // keys [lo, hi), lo a multiple of 32
    int first, last;          // positions that may be read and seen (others are not)
    int head;                 // kv head
    const int32_t* table;
};

// One wave's 16 NT rows: running softmax and transposed output.  Lane l holds
// query column l % 16 of each group of 16 and, in row group g = l / 16, of a
// 32-key block the scores of keys 8 g .. 8 g + 7 (S^T = K Q^T with the K rows
// of two 16-key MFMAs chosen so: row 4 g + v of MFMA t is key 8 g + 4 t + v):
// the lane's P is then the operand of O^T = V^T P^T as it stands.  Its V
// operand is eight keys of one dim: the lane loads the VD = HD / 16 dims VD (l %
// 16) .. of its eight keys and picks dim j of them for MFMA j, whose output
// row 4 g + v is dim VD (4 g + v) + j.
template <int HD, int QP, int KP, int NT>
struct Wave {
    static constexpr int NS = HD / 32, VD = HD / 16;
    bf16x8 q[NT][QP][NS];
    f32x4v acc[NT][VD];
    float m[NT], l[NT];
    int qpos[NT];
    int g, c;
    const uint8_t *kc, *vc;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int j = 0; j < VD; ++j) acc[t][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ bool row_at(const PagedAttnArgs& a, const Work& w, int rho, int& token,
                                           int& head) const {
        const int t = rho / a.share;
        token = w.token0 + min(t, w.tokens - 1);
        head = w.head0 + rho - t * a.share;
        return t < w.tokens;
    }
    // rows rho0 ..
    __device__ __forceinline__ void load_q(const PagedAttnArgs& a, const Work& w, int rho0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            int token, head;
            const bool on = row_at(a, w, rho0 + 16 * t + c, token, head);
            qpos[t] = w.pos0 + (token - w.token0) * w.row_pos;
            const int64_t at = (int64_t)token * a.q_stride + (int64_t)head * HD + 8 * g;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if constexpr (QP == 1) {
                    uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at + 32 * s);
                    if (!on) x = make_uint4(0, 0, 0, 0);
                    q[t][0][s] = __builtin_bit_cast(bf16x8, x);
                } else {
                    const float4* x = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + 32 * s);
                    float4 y = x[0], z = x[1];
                    if (!on) y = z = make_float4(0.f, 0.f, 0.f, 0.f);
                    const Parts8 r = parts8({y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w});
                    q[t][0][s] = r.h;
                    q[t][QP - 2][s] = r.m;
                    q[t][QP - 1][s] = r.l;
                }
            }
        }
    }

    // The page of position pos (clamped to the readable ones).
    __device__ __forceinline__ int page_of(const PagedView& p, const Work& w, int pos, bool& bad) const {
        const int at = min(max(pos, w.first), w.last) >> p.page_shift;
        int page = w.table[at];
        if ((unsigned)page >= (unsigned)p.num_pages) {
            bad = true;
            page = 0;
        }
        return page;
    }
    // Element offset of position pos of page `page`.
    __device__ __forceinline__ int64_t cell(const PagedView& p, const Work& w, int page, int pos) const {
        const int in = min(max(pos, w.first), w.last) & ((1 << p.page_shift) - 1);
        return ((((int64_t)page << p.page_shift) + in) * p.kv_heads + w.head) * HD;
    }

    // Keys lo, lo + step, ... of the work in blocks of 32.
    __device__ __forceinline__ void run(const PagedAttnArgs& a, const Work& w, int lo, int step, float unit,
                                        bool& bad) {
        const PagedView& p = a.p;
        // a block with a key that some row does not see, or that is not readable
        int see = w.last;
#pragma unroll
        for (int t = 0; t < NT; ++t) see = min(see, qpos[t]);
        int most = -1;
#pragma unroll
        for (int t = 0; t < NT; ++t) most = max(most, qpos[t]);
        for (int x = 1; x < 16; x <<= 1) {
            see = min(see, __shfl_xor(see, x));
            most = max(most, __shfl_xor(most, x));
        }
        const int hi = min(w.hi, min(most, w.last) + 1);
        for (int kb = lo; kb < hi; kb += step) {
            const int pk = page_of(p, w, kb + 8 * (c >> 2), bad), pv = page_of(p, w, kb + 8 * g, bad);
            f32x4v s[NT][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t at = cell(p, w, pk, kb + 8 * (c >> 2) + 4 * u + (c & 3)) + 8 * g;
#pragma unroll
                for (int t = 0; t < NT; ++t) s[t][u] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if constexpr (KP == 1) {
                        const bf16x8 k = *reinterpret_cast<const bf16x8*>(kc + 2 * (at + 32 * i));
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int b = QP - 1; b >= 0; --b) s[t][u] = mfma(k, q[t][b][i], s[t][u]);
                    } else {
                        const float4* x = reinterpret_cast<const float4*>(kc + 4 * (at + 32 * i));
                        const float4 y = x[0], z = x[1];
                        const Parts8 k = parts8({y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w});
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            s[t][u] = mfma(k.l, q[t][0][i], s[t][u]);
                            s[t][u] = mfma(k.h, q[t][QP - 1][i], s[t][u]);
                            s[t][u] = mfma(k.m, q[t][QP / 2][i], s[t][u]);
                            s[t][u] = mfma(k.m, q[t][0][i], s[t][u]);
                            s[t][u] = mfma(k.h, q[t][QP / 2][i], s[t][u]);
                            s[t][u] = mfma(k.h, q[t][0][i], s[t][u]);
                        }
                    }
                }
            }
            // V of the lane's eight keys
            float vf[KP == 3 ? 8 : 1][KP == 3 ? VD : 1];
            uint32_t vw[KP == 1 ? 8 : 1][KP == 1 ? VD / 2 : 1];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t at = cell(p, w, pv, kb + 8 * g + e) + VD * c;
                if constexpr (KP == 1) {
                    typedef uint32_t words __attribute__((ext_vector_type(VD / 2)));
                    const words x = *reinterpret_cast<const words*>(vc + 2 * at);
#pragma unroll
                    for (int i = 0; i < VD / 2; ++i) vw[e][i] = x[i];
                } else {
#pragma unroll
                    for (int i = 0; i < VD; i += 4) {
                        const f32x4v x = *reinterpret_cast<const f32x4v*>(vc + 4 * (at + i));
#pragma unroll
                        for (int y = 0; y < 4; ++y) vf[e][i + y] = x[y];
                    }
                }
            }
            bf16x8 pp[NT][QP];
            const bool whole = kb >= w.first && kb + 31 <= see && kb + 32 <= w.hi;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[t][e >> 2][e & 3];
                if (!whole) {
                    const int top = min(min(qpos[t], w.last), w.hi - 1);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int pos = kb + 8 * g + e;
                        x[e] = pos >= w.first && pos <= top ? x[e] : -INFINITY;
                    }
                }
                float bm = x[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) bm = fmaxf(bm, x[e]);
                const float mn = fmaxf(m[t], quads_max(bm));
                const float mc = mn == -INFINITY ? 0.f : mn;   // (no key seen yet: all weights 0)
                if (__any(mn > m[t])) {
                    const float f = weight(m[t] - mc, unit);
                    l[t] *= f;
#pragma unroll
                    for (int j = 0; j < VD; ++j) acc[t][j] *= f;
                    m[t] = mn;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = weight(x[e] - mc, unit);
                    l[t] += x[e];
                }
                if constexpr (QP == 1) {
                    pp[t][0] = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                                                     pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])));
                } else {
                    const Parts8 r = parts8(x);
                    pp[t][0] = r.h;
                    pp[t][QP - 2] = r.m;
                    pp[t][QP - 1] = r.l;
                }
            }
#pragma unroll
            for (int j = 0; j < VD; ++j) {
                if constexpr (KP == 1) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[i] = __builtin_amdgcn_perm(vw[2 * i + 1][j >> 1], vw[2 * i][j >> 1],
                                                     j & 1 ? 0x07060302u : 0x05040100u);
                    const bf16x8 v = __builtin_bit_cast(bf16x8, make_uint4(o[0], o[1], o[2], o[3]));
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int b = QP - 1; b >= 0; --b) acc[t][j] = mfma(v, pp[t][b], acc[t][j]);
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = vf[e][j];
                    const Parts8 v = parts8(x);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        acc[t][j] = mfma(v.l, pp[t][0], acc[t][j]);
                        acc[t][j] = mfma(v.h, pp[t][QP - 1], acc[t][j]);
                        acc[t][j] = mfma(v.m, pp[t][QP / 2], acc[t][j]);
                        acc[t][j] = mfma(v.m, pp[t][0], acc[t][j]);
                        acc[t][j] = mfma(v.h, pp[t][QP / 2], acc[t][j]);
                        acc[t][j] = mfma(v.h, pp[t][0], acc[t][j]);
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) l[t] = quads_add(l[t]);
    }

    // Whether an infinity or a NaN came up in some row: one in q, k or v, also at a
    // position that a row does not see (0 times it is not 0), or an f32 value
    // whose bf16 part rounds to infinity.
    __device__ __forceinline__ bool odd() const {
        float z = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            z = fmaf(l[t], 0.f, z);
#pragma unroll
            for (int j = 0; j < VD; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) z = fmaf(acc[t][j][v], 0.f, z);
        }
        return __any(z != 0.f);
    }
    // The same keys for such a wave, row by row and key by key in f32: positions
    // that a row does not see are passed over.  tmp: HD floats of LDS of the wave.
    __device__ __forceinline__ void run_plain(const PagedAttnArgs& a, const Work& w, int rho0, int lo, int step,
                                              float unit, float* tmp) {
        constexpr int PL = HD / 64;
        const PagedView& p = a.p;
        const int lane = threadIdx.x & 63;
        clear();
        for (int rr = 0; rr < 16 * NT; ++rr) {
            int token, head;
            if (!row_at(a, w, rho0 + rr, token, head)) continue;   // (uniform)
            const int pos = w.pos0 + (token - w.token0) * w.row_pos, top = min(min(pos, w.last), w.hi - 1);
            float qr[PL], o[PL], rm = -INFINITY, rl = 0.f;
#pragma unroll
            for (int i = 0; i < PL; ++i) {
                const int64_t at = (int64_t)token * a.q_stride + (int64_t)head * HD + PL * lane + i;
                qr[i] = QP == 1 ? bf16_to_f32(static_cast<const uint16_t*>(a.q)[at]) : static_cast<const float*>(a.q)[at];
                o[i] = 0.f;
            }
            for (int kb = lo; kb <= top; kb += step)
                for (int k = max(kb, w.first); k <= min(kb + 31, top); ++k) {
                    int page = w.table[k >> p.page_shift];
                    if ((unsigned)page >= (unsigned)p.num_pages) page = 0;
                    const int64_t at = cell(p, w, page, k) + PL * lane;
                    float s = 0.f, v[PL];
#pragma unroll
                    for (int i = 0; i < PL; ++i) {
                        const float kx = KP == 1 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(kc)[at + i])
                                                 : reinterpret_cast<const float*>(kc)[at + i];
                        v[i] = KP == 1 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(vc)[at + i])
                                       : reinterpret_cast<const float*>(vc)[at + i];
                        s = fmaf(qr[i], kx, s);
                    }
                    s = wave_sum(s);
                    const float mn = fmaxf(rm, s), mc = mn == -INFINITY ? 0.f : mn;
                    const float f = weight(rm - mc, unit), x = weight(s - mc, unit);
                    rl = fmaf(rl, f, x);
#pragma unroll
                    for (int i = 0; i < PL; ++i) o[i] = fmaf(x, v[i], o[i] * f);
                    rm = mn;
                }
#pragma unroll
            for (int i = 0; i < PL; ++i) tmp[PL * lane + i] = o[i];
            __threadfence_block();
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (16 * t + c == rr) {
                    m[t] = rm;
                    l[t] = rl;
#pragma unroll
                    for (int j = 0; j < VD; ++j)
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[t][j][v] = tmp[VD * (4 * g + v) + j];
                }
            __threadfence_block();
        }
    }
};

// Sizes of a workgroup's LDS and partials.
template <int HD, int NT>
struct Sizes {
    static constexpr int R = 64 * NT;                      // rows of a tile
    static constexpr int kTile = 16 * NT * HD;             // floats of a wave's output
    static constexpr int64_t kSlot = (int64_t)R * (HD + 2);  // a partial: o [R][HD], m [R], l [R]
};

// joins (m1, l1) with (m0, l0): the factors of both
__device__ __forceinline__ void join(float& m0, float& l0, float m1, float l1, float unit, float& f0, float& f1) {
    const float mn = fmaxf(m0, m1), mc = mn == -INFINITY ? 0.f : mn;
    f0 = weight(m0 - mc, unit);
    f1 = weight(m1 - mc, unit);
    l0 = l0 * f0 + l1 * f1;
    m0 = mn;
}

template <int HD, bool OB, int N>
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int token, int head, int d, const float (&x)[N]) {
    const int64_t at = (int64_t)token * a.out_stride + (int64_t)head * HD + d;
    if constexpr (OB) {
        uint16_t* o = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<uint2*>(o + i) = make_uint2(pack_bf16(x[i], x[i + 1]), pack_bf16(x[i + 2], x[i + 3]));
    } else {
        float* o = static_cast<float*>(a.out) + at;
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<float4*>(o + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
}

// Adds the prefix' pieces of (token, head), dims d .., to x with m and l.
template <int HD, int N>
__device__ __forceinline__ void add_prefix(const PagedAttnArgs& a, int token, int head, int d, float unit, float& m,
                                           float& l, float (&x)[N]) {
    const int64_t rows = (int64_t)a.p.num_rows * a.heads, row = (int64_t)token * a.heads + head;
    for (int s = 0; s < a.splits; ++s) {
        const float* o = a.pre + ((int64_t)s * rows + row) * (HD + 2);
        float f0, f1;
        join(m, l, o[HD], o[HD + 1], unit, f0, f1);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = x[i] * f0 + o[d + i] * f1;
    }
}

// The work's rows over its keys by the four waves: as many waves side by side
// over the rows as they fill (1, 2 or 4), the others taking every second or
// fourth block of 32 keys; those are joined into the first waves' registers.
// Returns whether this wave holds rows, from rho0 on.
template <int HD, int QP, int KP, int NT>
__device__ __forceinline__ bool work_rows(const PagedAttnArgs& a, const Work& w, Wave<HD, QP, KP, NT>& wv, float unit,
                                          float* s_buf, int& rho0) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int groups = (w.tokens * a.share + 16 * NT - 1) / (16 * NT);
    const int side = groups <= 1 ? 1 : groups <= 2 ? 2 : 4, deep = 4 / side;
    const int ks = wave / side;
    rho0 = (wave % side) * 16 * NT;
    wv.kc = static_cast<const uint8_t*>(a.p.k);
    wv.vc = static_cast<const uint8_t*>(a.p.v);
    wv.g = lane >> 4;
    wv.c = lane & 15;
    wv.clear();
    const bool rows = rho0 < w.tokens * a.share;
    if (rows) {
        bool bad = false;
        wv.load_q(a, w, rho0);
        wv.run(a, w, w.lo + 32 * ks, 32 * deep, unit, bad);
        if (bad) flag_error(a.p.err, kErrPagedPage);
        if (wv.odd()) wv.run_plain(a, w, rho0, w.lo + 32 * ks, 32 * deep, unit, s_buf + wave * HD);
    }
    if (deep == 1) return rows;
    // halves the waves over the keys: those from `half` on hand theirs to the others
    constexpr int kWave = Sizes<HD, NT>::kTile + 128 * NT;
    for (int half = deep / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (rows && ks >= half && ks < 2 * half) {
            float* o = s_buf + ((ks - half) * side + wave % side) * kWave;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                o[(2 * t) * 64 + lane] = wv.m[t];
                o[(2 * t + 1) * 64 + lane] = wv.l[t];
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        o[128 * NT + ((t * HD / 16 + j) * 4 + v) * 64 + lane] = wv.acc[t][j][v];
            }
        }
        __syncthreads();
        if (rows && ks < half) {
            const float* o = s_buf + (ks * side + wave % side) * kWave;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float f0, f1;
                join(wv.m[t], wv.l[t], o[(2 * t) * 64 + lane], o[(2 * t + 1) * 64 + lane], unit, f0, f1);
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        wv.acc[t][j][v] =
                            wv.acc[t][j][v] * f0 + o[128 * NT + ((t * HD / 16 + j) * 4 + v) * 64 + lane] * f1;
            }
        }
    }
    return rows && ks == 0;
}

template <int HD, int NT>
constexpr int work_lds() {   // floats: two waves' results; the plain path's rows
    return 2 * (Sizes<HD, NT>::kTile + 128 * NT) > 4 * HD ? 2 * (Sizes<HD, NT>::kTile + 128 * NT) : 4 * HD;
}

// The sequences' own positions: one workgroup per share of the line.
template <int HD, int QP, int KP, int NT>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a) {
    constexpr int R = Sizes<HD, NT>::R, VD = HD / 16;
    __shared__ int64_t s_cum[kPagedMaxSeqs + 1];
    __shared__ int64_t s_tmp[4];
    __shared__ __attribute__((aligned(16))) float s_buf[work_lds<HD, NT>()];
    const PagedView& p = a.p;
    const float unit = a.scale * 1.44269504f;
    Line ln;
    ln.cum = s_cum;
    ln.org = p.prefix_len & ~31;
    ln.TT = R / a.share;
    ln.kv_heads = p.kv_heads;
    make_line(p, ln, s_tmp, a.grid, blockIdx.x == 0);
    if (ln.total == 0) return;
    // neighbouring shares on one XCD (workgroup id mod 8)
    const int per = (ln.wgs + 7) / 8, id = (int)blockIdx.x;
    const int wg = (id & 7) * per + (id >> 3);
    if ((id >> 3) >= per || wg >= ln.wgs) return;
    int64_t x = ln.cut(wg), x1 = ln.cut(wg + 1);
    Tile t = ln.tile(p, find_seq(p, ln, x), x);
    x = ln.rounded(t, x);
    if (x1 < ln.total) x1 = ln.rounded(ln.tile(p, find_seq(p, ln, x1), x1), x1);
    while (x < x1) {
        const int64_t end = min(t.end, x1);
        Work w;
        w.token0 = t.row0 + t.r * ln.TT;
        w.tokens = min(ln.TT, t.n - t.r * ln.TT);
        w.pos0 = t.base + t.r * ln.TT;
        w.row_pos = 1;
        w.head = t.head;
        w.head0 = t.head * a.share;
        w.lo = ln.org + (int)(x - t.start);
        w.hi = ln.org + (int)(end - t.start);
        w.first = p.prefix_len;
        w.last = w.pos0 + w.tokens - 1;
        w.table = p.pages + (int64_t)t.seq * p.table_stride;
        Wave<HD, QP, KP, NT> wv;
        int rho0;
        const bool holds = work_rows(a, w, wv, unit, s_buf, rho0);
        const bool all = x == t.start && end == t.end;
        float* slot = a.part + (int64_t)(2 * wg + (x > t.start ? 0 : 1)) * Sizes<HD, NT>::kSlot;
        if (holds) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int rho = rho0 + 16 * i + wv.c;
                int token, head;
                if (!wv.row_at(a, w, rho, token, head)) continue;
                if (!all && wv.g == 0) {
                    slot[(int64_t)R * HD + rho] = wv.m[i];
                    slot[(int64_t)R * HD + R + rho] = wv.l[i];
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    float o[VD];
#pragma unroll
                    for (int j = 0; j < VD; ++j) o[j] = wv.acc[i][j][v];
                    const int d = VD * (4 * wv.g + v);
                    if (all) {
                        float m = wv.m[i], l = wv.l[i];
                        add_prefix<HD>(a, token, head, d, unit, m, l, o);
                        const float f = 1.0f / l;
#pragma unroll
                        for (int j = 0; j < VD; ++j) o[j] *= f;
                        store_out<HD, QP == 1>(a, token, head, d, o);
                    } else {
#pragma unroll
                        for (int j = 0; j < VD; j += 4)
                            *reinterpret_cast<float4*>(slot + (int64_t)rho * HD + d + j) =
                                make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
            }
        }
        __syncthreads();   // (s_buf is the next tile's)
        x = end;
        if (x < x1) t = ln.tile(p, find_seq(p, ln, x), x);
    }
}

// The tiles that several workgroups shared: workgroup w joins the tile that cut w is
// the first inside of.
template <int HD, int QP, int NT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int R = Sizes<HD, NT>::R;
    __shared__ int64_t s_cum[kPagedMaxSeqs + 1];
    __shared__ int64_t s_tmp[4];
    const PagedView& p = a.p;
    const float unit = a.scale * 1.44269504f;
    Line ln;
    ln.cum = s_cum;
    ln.org = p.prefix_len & ~31;
    ln.TT = R / a.share;
    ln.kv_heads = p.kv_heads;
    make_line(p, ln, s_tmp, a.grid, false);
    const int wg = (int)blockIdx.x + 1;
    if (wg >= ln.wgs) return;
    const int64_t x = ln.cut(wg);
    const Tile t = ln.tile(p, find_seq(p, ln, x), x);
    if (ln.rounded(t, x) == t.start) return;                            // not cut here
    const int64_t prev = ln.cut(wg - 1);
    if (prev >= t.start && ln.rounded(t, prev) > t.start) return;       // nor first here
    const int tokens = min(ln.TT, t.n - t.r * ln.TT);
    for (int i = threadIdx.x; i < tokens * a.share * (HD / 4); i += 256) {
        const int rho = i / (HD / 4), d = 4 * (i % (HD / 4));
        const float* slot = a.part + (int64_t)(2 * (wg - 1) + 1) * Sizes<HD, NT>::kSlot;
        float4 y = *reinterpret_cast<const float4*>(slot + (int64_t)rho * HD + d);
        float m = slot[(int64_t)R * HD + rho], l = slot[(int64_t)R * HD + R + rho];
        float o[4] = {y.x, y.y, y.z, y.w};
        int64_t at = ln.rounded(t, x);
        for (int w = wg; at < t.end; ++w) {
            int64_t next = ln.cut(w + 1);
            next = next >= t.end ? t.end : ln.rounded(t, next);
            if (next > at) {
                slot = a.part + (int64_t)(2 * w) * Sizes<HD, NT>::kSlot;
                y = *reinterpret_cast<const float4*>(slot + (int64_t)rho * HD + d);
                float f0, f1;
                join(m, l, slot[(int64_t)R * HD + rho], slot[(int64_t)R * HD + R + rho], unit, f0, f1);
                o[0] = o[0] * f0 + y.x * f1;
                o[1] = o[1] * f0 + y.y * f1;
                o[2] = o[2] * f0 + y.z * f1;
                o[3] = o[3] * f0 + y.w * f1;
            }
            at = next;
        }
        const int token = t.row0 + t.r * ln.TT + rho / a.share, head = t.head * a.share + rho % a.share;
        add_prefix<HD>(a, token, head, d, unit, m, l, o);
        const float f = 1.0f / l;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] *= f;
        store_out<HD, QP == 1>(a, token, head, d, o);
    }
}

// The prefix, for all rows of the batch: workgroup = (tile of rows, kv head, piece of
// the prefix).
template <int HD, int QP, int KP, int NT>
__global__ __launch_bounds__(256) void paged_prefix_kernel(PagedAttnArgs a) {
    constexpr int R = Sizes<HD, NT>::R, VD = HD / 16;
    __shared__ __attribute__((aligned(16))) float s_buf[work_lds<HD, NT>()];
    const PagedView& p = a.p;
    const float unit = a.scale * 1.44269504f;
    const int TT = R / a.share, head = (int)blockIdx.y % p.kv_heads, piece = (int)blockIdx.y / p.kv_heads;
    const int rows = min(p.row_start[p.num_seqs], p.num_rows), blocks = (p.prefix_len + 31) / 32;
    Work w;
    w.token0 = (int)blockIdx.x * TT;
    w.tokens = min(TT, rows - w.token0);
    if (w.tokens <= 0) return;
    w.pos0 = p.prefix_len - 1;
    w.row_pos = 0;
    w.head = head;
    w.head0 = head * a.share;
    w.lo = 32 * (int)((int64_t)blocks * piece / a.splits);
    w.hi = min(p.prefix_len, 32 * (int)((int64_t)blocks * (piece + 1) / a.splits));
    w.first = 0;
    w.last = p.prefix_len - 1;
    w.table = p.prefix_pages;
    Wave<HD, QP, KP, NT> wv;
    int rho0;
    if (!work_rows(a, w, wv, unit, s_buf, rho0)) return;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        int token, qh;
        if (!wv.row_at(a, w, rho0 + 16 * i + wv.c, token, qh)) continue;
        float* o = a.pre + (((int64_t)piece * p.num_rows + token) * a.heads + qh) * (HD + 2);
        if (wv.g == 0) *reinterpret_cast<float2*>(o + HD) = make_float2(wv.m[i], wv.l[i]);
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int j = 0; j < VD; j += 2)
                *reinterpret_cast<float2*>(o + VD * (4 * wv.g + v) + j) =
                    make_float2(wv.acc[i][j][v], wv.acc[i][j + 1][v]);
    }
}

template <int HD, int QP, int KP, int NT>
void launch_attn(const PagedAttnArgs& a, hipStream_t st) {
    if (a.splits) {
        const int TT = 64 * NT / a.share;
        hipLaunchKernelGGL((paged_prefix_kernel<HD, QP, KP, NT>),
                           dim3((unsigned)((a.p.num_rows + TT - 1) / TT), (unsigned)(a.p.kv_heads * a.splits)),
                           dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL((paged_attn_kernel<HD, QP, KP, NT>), dim3((unsigned)a.grid), dim3(256), 0, st, a);
    hipLaunchKernelGGL((paged_join_kernel<HD, QP, NT>), dim3((unsigned)a.grid), dim3(256), 0, st, a);
}

int tile_groups(const PagedAttnArgs&) { return 1; }

template <int HD>
void launch_attn_hd(const PagedAttnArgs& a, hipStream_t st) {
    if (a.x_bf16)
        launch_attn<HD, 1, 1, 1>(a, st);
    else if (a.cache_bf16)
        launch_attn<HD, 3, 1, 1>(a, st);
    else
        launch_attn<HD, 3, 3, 1>(a, st);
}

template <int HD>
void launch_append_hd(const AppendArgs& a, dim3 grid, hipStream_t st) {
    if (a.x_bf16)
        hipLaunchKernelGGL((kv_append_kernel<HD, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((kv_append_kernel<HD, false>), grid, dim3(256), 0, st, a);
}

}  // namespace

int64_t paged_attention_plan(PagedAttnArgs& a, int cus, int64_t* own_floats) {
    const int nt = tile_groups(a), R = 64 * nt;
    a.grid = (2 * cus + 7) / 8 * 8;
    a.splits = 0;
    *own_floats = (int64_t)a.grid * 2 * R * (a.head_dim + 2);
    if (a.p.prefix_len == 0) return *own_floats;
    const int TT = R / a.share, tiles = (a.p.num_rows + TT - 1) / TT;
    const int64_t wgs = (int64_t)tiles * a.p.kv_heads;
    const int64_t most = std::max(1, a.p.prefix_len / 256);
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({most, (2 * cus + wgs - 1) / wgs, 32}));
    return *own_floats + (int64_t)a.splits * a.p.num_rows * a.heads * (a.head_dim + 2);
}

int launch_paged_attention(const PagedAttnArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (a.head_dim) {
        case 64: launch_attn_hd<64>(a, st); break;
        case 128: launch_attn_hd<128>(a, st); break;
        case 256: launch_attn_hd<256>(a, st); break;
        default: return (int)hipErrorInvalidValue;
    }
    return (int)hipGetLastError();
}

int launch_kv_append(const AppendArgs& a, int cus, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int per = 256 * (a.x_bf16 ? 8 : 4) / a.head_dim;   // heads a workgroup has at once
    const int passes = (a.heads + 2 * a.p.kv_heads + per - 1) / per;
    const int ny = std::max(1, std::min(passes, 4 * cus / a.p.num_rows));
    const dim3 grid((unsigned)a.p.num_rows, (unsigned)ny);
    switch (a.head_dim) {
        case 64: launch_append_hd<64>(a, grid, st); break;
        case 128: launch_append_hd<128>(a, grid, st); break;
        case 256: launch_append_hd<256>(a, grid, st); break;
        default: return (int)hipErrorInvalidValue;
    }
    return (int)hipGetLastError();
}

}  // namespace m1moe
