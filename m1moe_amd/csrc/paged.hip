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

// q and k of a head are divided by their root mean square (and multiplied by a
// weight), pairs of their dims are turned by the position's angles, then k and v go
// to the row's place in the cache, q to its output: every element is read and
// written once.  Prompts are bound by memory (five of 37 to 1900 tokens, 32 + 2 x 8 heads
// of 128, bf16: 28.8 us, of which 26.4 at the rate of a large copy; 20.8 where the same rows
// come again and the device's last-level cache still has them), steps by the launch and the
// chain sequence - page - store (64 tokens 4.4 us; one workgroup for all heads of a row 5.9).
//
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
        const double rest = fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586232, ang));
        // (what its rounding to f32 leaves, up to 2^-23, turns the pair once more)
        const float r = (float)rest, e = (float)(rest - (double)r), c = cosf(r), s = sinf(r);
        s_cs[tid] = make_float2(fmaf(-e, s, c) * a.amp, fmaf(e, c, s) * a.amp);
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
//
// out = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m), s_p = q . k_p / sqrt(head_dim), over the
// positions p up to the row's own, in one pass over them with a running m.  Scores and
// weighted sums are MFMAs of bf16 operands with f32 sums.  bf16 queries and
// cache: the weights are rounded to two bf16 parts and summed as rounded.  f32 ones are taken
// apart into three bf16 parts, whose products down to 2^-16 of the largest are formed, so
// that the result is as good as f32 arithmetic's.
//
// Steps are bound by reading the cache once (32 heads over 8, f32 queries, bf16 cache:
// 32 tokens behind 60 to 8100 positions 80.6 us, 4.5 TB/s; 16 heads, all bf16: 48 behind
// 100 to 4000 117 us, 4.8 TB/s), prompts and turns by a SIMD's two waves, whose MFMAs,
// softmax and LDS reads overlap only in part (2500 positions, all bf16: 95 us, 535 TFLOP/s;
// six turns of 9 to 400 tokens behind up to 4000, f32 queries: 73 us, of which 42.5 are
// the three products at a large matrix product's rate), one token behind few positions by
// the chain launch - lengths - page - rows - join (14.8 us).

// f32 values as three bf16 parts, each rounded to nearest, that add up to them
// exactly (24 bits), a pair at a time.  The rest of a pair is two v_dot2, (hi0, hi1) .
// (-1, 0) + x0 and (hi0, hi1) . (0, -1) + x1, exact: seven instructions a pair against
// eleven with the parts unpacked and subtracted.  The constants live in scalar registers:
// as literals the instruction would read them as f32.
struct Parts8 {
    bf16x8 h, m, l;
};
__device__ __forceinline__ void parts2(float x0, float x1, uint32_t& h, uint32_t& m, uint32_t& l) {
    uint32_t c0, c1;
    asm("s_mov_b32 %0, 0xbf80" : "=s"(c0));
    asm("s_mov_b32 %0, 0xbf800000" : "=s"(c1));
    const bf16x2 n0 = __builtin_bit_cast(bf16x2, c0), n1 = __builtin_bit_cast(bf16x2, c1);
    const bf16x2 hi = __builtin_convertvector(f32x2v{x0, x1}, bf16x2);
    const float r0 = __builtin_amdgcn_fdot2_f32_bf16(hi, n0, x0, false);
    const float r1 = __builtin_amdgcn_fdot2_f32_bf16(hi, n1, x1, false);
    const bf16x2 mid = __builtin_convertvector(f32x2v{r0, r1}, bf16x2);
    const float t0 = __builtin_amdgcn_fdot2_f32_bf16(mid, n0, r0, false);
    const float t1 = __builtin_amdgcn_fdot2_f32_bf16(mid, n1, r1, false);
    h = __builtin_bit_cast(uint32_t, hi);
    m = __builtin_bit_cast(uint32_t, mid);
    l = pack_bf16(t0, t1);
}
__device__ __forceinline__ Parts8 parts8(const float (&v)[8]) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) parts2(v[2 * i], v[2 * i + 1], h[i], m[i], l[i]);
    Parts8 s;
    s.h = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
    s.m = __builtin_bit_cast(bf16x8, make_uint4(m[0], m[1], m[2], m[3]));
    s.l = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
    return s;
}
__device__ __forceinline__ void parts4(f32x4v v, uint2& h, uint2& m, uint2& l) {
    parts2(v[0], v[1], h.x, m.x, l.x);
    parts2(v[2], v[3], h.y, m.y, l.y);
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

constexpr int kCut = 64;         // keys: where a tile's keys may be cut between workgroups
constexpr int kWhole = 512;      // keys of a tile that is not cut
constexpr int kFewKeys = 128;    // least places on the line per workgroup
constexpr int kTileKeys = 128;   // what a tile costs besides its keys, in keys

// How the rows and keys are shared.  A tile is up to R rows (token, head) of one
// sequence and kv head, whole tokens: TT = R / share tokens.  Its keys are the
// positions from `org` (the prefix' end rounded down to 32) to its last token's.
// All tiles, sequence by sequence, head by head, tile by tile, form one line, each
// with kTileKeys places for what it costs to begin and end it (about 5 us: the
// queries, the first page and rows one after the other, the waves' join) and one
// place per key; the line is cut into equal shares, one per workgroup, the cuts
// moved down to a multiple of kCut keys inside their tile, or to its start where it has
// at most kWhole keys: to join two pieces of one takes longer than to read it (a prompt of
// 2500 (one part per weight) and turns behind up to 4000: 104 and 88 us with every tile cut,
// 98 and 79 with 512 whole; later 84.2 and 73.2, with 768 whole 87.2 and 83.5).  (Without the places
// per tile the workgroups with the shortest sequences ended last: 32 steps of 60 to
// 8100 positions, 8 kv heads, median 61 us, last 116.)
struct Tile {
    int seq, head, r;            // sequence, kv head, tile of its rows
    int row0, n, base;           // the sequence's first row, rows, positions before them
    int64_t cum, start, end;     // on the line: the sequence's start, the tile's, its end

    // Lane `lane`'s in every lane, in scalar registers.
    __device__ __forceinline__ static int64_t lane64(int64_t x, int lane) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)x, lane));
    }
    __device__ __forceinline__ void of_lane(int lane) {
        for (int* x : {&seq, &head, &r, &row0, &n, &base}) *x = __builtin_amdgcn_readlane(*x, lane);
        for (int64_t* x : {&cum, &start, &end}) *x = lane64(*x, lane);
    }
};

struct Line {
    int64_t* cum;                // LDS [num_seqs + 1]: the sequences' starts on the line
    int64_t total, share;
    int rest;                    // the first shares have a place more
    int wgs;                     // workgroups that have a share
    int org, TT, kv_heads;

    // places of the first r tiles of a head (r below the number of tiles)
    __device__ int64_t before(int base, int r) const {
        return (int64_t)r * (base - org + kTileKeys) + (int64_t)TT * r * (r + 1) / 2;
    }
    __device__ int64_t head_places(int base, int n, int tiles) const {
        return before(base, tiles - 1) + (base - org + kTileKeys) + n;
    }
    // Equal shares but for one place, at least kFewKeys >= kCut places, so that every cut
    // inside a cut tile's keys begins a piece of its own.
    __device__ int64_t cut(int w) const { return w * share + min(w, rest); }
    // The last cut below place x > 0.
    __device__ int below(int64_t x) const {
        int w = min((int)((double)x / (double)share), wgs - 1);
        while (w + 1 < wgs && cut(w + 1) < x) ++w;
        while (w > 0 && cut(w) >= x) --w;
        return w;
    }
    // Sequence s of the batch, and its tile that holds place x of the line (all of a lane's
    // own: two places take no longer than one).
    __device__ void sequence(const PagedView& p, int s, Tile& t) const {
        t.seq = s;
        t.row0 = p.row_start[s];
        t.n = p.row_start[s + 1] - t.row0;
        t.base = p.kv_len[s] - t.n;
        t.cum = cum[s];
    }
    __device__ void find(int64_t x, Tile& t) const {
        const int tiles = (t.n + TT - 1) / TT;
        const int64_t hk = head_places(t.base, t.n, tiles);
        int64_t off = x - t.cum;
        // (the quotient in f64, within one of the whole one)
        int head = (int)((double)off / (double)hk);
        if ((int64_t)head * hk > off) --head;
        if ((int64_t)(head + 1) * hk <= off) ++head;
        off -= (int64_t)head * hk;
        int lo = 0, hi = tiles - 1;       // the last tile that starts at or before off
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before(t.base, mid) <= off)
                lo = mid;
            else
                hi = mid - 1;
        }
        t.head = head;
        t.r = lo;
        t.start = t.cum + (int64_t)head * hk + before(t.base, lo);
        t.end = t.start + kTileKeys + (t.base - org) + min(t.n, (lo + 1) * TT);
    }
    // Cut x inside tile t, moved down: to the tile's start or to a place of a key.
    __device__ int64_t rounded(const Tile& t, int64_t x) const {
        const int64_t keys = x - t.start - kTileKeys;
        return keys < kCut || t.end - t.start <= kTileKeys + kWhole ? t.start
                                                                    : t.start + kTileKeys + keys / kCut * kCut;
    }
    // The key (from org on) at place x of tile t.
    __device__ static int key(const Tile& t, int64_t x) { return (int)max((int64_t)0, x - t.start - kTileKeys); }
};

// Fills cum and the line: the whole workgroup of 256.  tmp: LDS, 4 values.
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
                keys = ln.kv_heads * ln.head_places(len - n, n, (n + ln.TT - 1) / ln.TT);
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
    static_assert(kFewKeys >= kCut, "a cut per piece");
    ln.share = (int64_t)((double)carry / ln.wgs);       // (within one)
    ln.share += ((ln.share + 1) * ln.wgs <= carry) - (ln.share * ln.wgs > carry);
    ln.rest = (int)(carry - ln.share * ln.wgs);
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

// The thread's number, opaque to the compiler: what depends on it is computed where
// it is used and not kept in registers over a workgroup's tiles (50 of them).
__device__ __forceinline__ int thread_id() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
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

    // (the same in every lane: into scalar registers)
    __device__ __forceinline__ void uniform() {
        for (int* x : {&token0, &tokens, &pos0, &head0, &lo, &hi, &last, &head}) *x = __builtin_amdgcn_readfirstlane(*x);
        const uint64_t t = reinterpret_cast<uint64_t>(table);
        table = reinterpret_cast<const int32_t*>(
            (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 32)) << 32 |
            (uint32_t)__builtin_amdgcn_readfirstlane((int)t));
    }
};

// The cache as a wave reads it: one kv head's rows.
template <int HD, int KP>
struct Cache {
    static constexpr int ES = KP == 1 ? 2 : 4;    // bytes of an element
    const uint8_t *k, *v;                         // at the kv head
    uint32_t row, page, mask;                     // bytes of a position and of a page; slots - 1
    int shift, pages, first, last;
    const int32_t* table;

    __device__ __forceinline__ Cache(const PagedView& p, const Work& w) {
        k = static_cast<const uint8_t*>(p.k) + (int64_t)w.head * HD * ES;
        v = static_cast<const uint8_t*>(p.v) + (int64_t)w.head * HD * ES;
        row = (uint32_t)p.kv_heads * HD * ES;
        shift = p.page_shift;
        page = row << shift;
        mask = (1u << shift) - 1;
        pages = p.num_pages;
        first = w.first;
        last = w.last;
        table = w.table;
    }
    __device__ __forceinline__ int clamp(int pos) const { return min(max(pos, first), last); }
    // Whether some of the n positions from kb on are not readable.  Their rows are read
    // all the same, from the slots they would have in a page that is looked up for them:
    // K's scores are passed over, V's rows are taken as 0.
    __device__ __forceinline__ bool edge(int kb, int n) const { return kb < first || kb + n - 1 > last; }
    __device__ __forceinline__ bool readable(int pos) const { return pos >= first && pos <= last; }
    // The page number of the aligned eight positions from pos on: of the readable one
    // among them, or of the nearest.  As the table has it: it is checked (known) where
    // it is used, as a test here would wait for it and for every load before it.
    // (a global load: a generic one would hold up the LDS reads that follow it)
    __device__ __forceinline__ int page_of(int pos) const {
        return ((const __attribute__((address_space(1))) int32_t*)table)[clamp(pos) >> shift];
    }
    // Page 0 for one outside the cache.
    __device__ __forceinline__ int known(int x, bool& bad) const {
        const bool out = (unsigned)x >= (unsigned)pages;
        bad |= out;
        return out ? 0 : x;
    }
    // Byte offset of position pos in page x.
    __device__ __forceinline__ int64_t at(int x, int pos) const {
        return (int64_t)((uint64_t)(uint32_t)x * page + ((uint32_t)pos & mask) * row);
    }
};

// The (token, query head) of row rho of the work; false past its rows.
__device__ __forceinline__ bool row_at(const PagedAttnArgs& a, const Work& w, int rho, int& token, int& head) {
    const int t = rho / a.share;
    token = w.token0 + min(t, w.tokens - 1);
    head = w.head0 + rho - t * a.share;
    return t < w.tokens;
}

// One wave's 16 NT rows: queries, running softmax and transposed output.  Lane l
// holds row c = l % 16 of each group of 16 and, with g = l / 16, of a 32-key block
// the scores of keys 8 g .. 8 g + 7 (S^T = K Q^T with the K rows of two 16-key
// MFMAs chosen so: row 4 g + v of MFMA u is key 8 g + 4 u + v): the lane's P is
// then the operand of O^T = V^T P^T as it stands, eight keys of one dim its
// other one.  Row 4 g + v of output MFMA j is dim VD (4 g + v) + j where a lane
// loads the VD = HD / 16 neighbouring dims VD c .. of eight keys itself (SPREAD),
// else dim 16 j + 4 g + v.
template <int HD, int QP, int NT, bool SPREAD>
struct Rows {
    static constexpr int NS = HD / 32, VD = HD / 16;
    // Parts of a weight.  bf16 queries: two, whose rest of 2^-16 is nothing beside the output's own
    // rounding, however many rows arrive together (one: a prompt of 2500 79 us, its error
    // against 64 bits 2.0e-3 where the output's rounding is 1.6e-3).
    static constexpr int PP = QP == 1 ? 2 : QP;
    bf16x8 q[NT][QP][NS];
    f32x4v acc[NT][VD];
    float m[NT], l[NT];
    f32x4v lv[QP == 1 ? NT : 1];   // bf16 weights: l, four times, as an MFMA sums it
    int qpos[NT];
    int g, c, see, most;      // the rows' lowest and highest position

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
            if constexpr (QP == 1) lv[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < VD; ++j) acc[t][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ static int dim(int g, int j, int v) {
        return SPREAD ? VD * (4 * g + v) + j : 16 * j + 4 * g + v;
    }
    __device__ __forceinline__ void lanes() {
        const int lane = thread_id() & 63;
        g = lane >> 4;
        c = lane & 15;
    }
    // Rows rho0 ..: read (raw, 16 bytes at a time), then split.
    static constexpr int kRaw = QP == 1 ? 1 : 2;
    __device__ __forceinline__ void read(const PagedAttnArgs& a, const Work& w, int rho0,
                                         f32x4v (&raw)[NT][NS][kRaw]) {
        see = w.last;
        most = -1;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            int token, head;
            const bool on = row_at(a, w, rho0 + 16 * t + c, token, head);
            qpos[t] = w.pos0 + (token - w.token0) * w.row_pos;
            see = min(see, qpos[t]);
            most = max(most, qpos[t]);
            const int64_t at = (int64_t)token * a.q_stride + (int64_t)head * HD + 8 * g;
            const f32x4v* x = QP == 1 ? reinterpret_cast<const f32x4v*>(static_cast<const uint16_t*>(a.q) + at)
                                      : reinterpret_cast<const f32x4v*>(static_cast<const float*>(a.q) + at);
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < kRaw; ++i) {
                    raw[t][s][i] = f32x4v{0.f, 0.f, 0.f, 0.f};
                    if (on) raw[t][s][i] = x[4 * kRaw * s + i];
                }
        }
    }
    __device__ __forceinline__ void split(const f32x4v (&raw)[NT][NS][kRaw]) {
        clear();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if constexpr (QP == 1) {
                    q[t][0][s] = __builtin_bit_cast(bf16x8, raw[t][s][0]);
                } else {
                    const f32x4v y = raw[t][s][0], z = raw[t][s][1];
                    const Parts8 r = parts8({y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]});
                    q[t][0][s] = r.h;
                    q[t][QP - 2][s] = r.m;
                    q[t][QP - 1][s] = r.l;
                }
            }
        for (int x = 1; x < 16; x <<= 1) {
            see = min(see, __shfl_xor(see, x));
            most = max(most, __shfl_xor(most, x));
        }
        see = __builtin_amdgcn_readfirstlane(see);
        most = __builtin_amdgcn_readfirstlane(most);
    }

    // Products of the parts of a K (or V) operand, KP of them, with the rows' QP, small
    // ones first: product p takes parts left(p) and right(p); for f32 on both sides the six
    // down to 2^-16 of the largest.  Those of one size (order(p)) are summed by themselves
    // where sums are short: an MFMA waits for the one before on the same sum.
    template <int KP>
    static constexpr int kProducts = KP == 1 ? QP : 6;
    static constexpr int kOrders = QP;
    template <int KP>
    static constexpr int left(int p) {
        constexpr int l[6] = {2, 0, 1, 1, 0, 0};
        return KP == 1 ? 0 : l[p];
    }
    template <int KP>
    static constexpr int right(int p) {
        constexpr int r[6] = {0, 2, 1, 0, 1, 0};
        return KP == 1 ? QP - 1 - p : r[p];
    }
    template <int KP>
    static constexpr int order(int p) { return left<KP>(p) + right<KP>(p); }

    // Scores of a 32-key block from K's parts x[u] of dims 32 i .., and the queries' (t, part)
    template <int KP, class Q>
    __device__ __forceinline__ static void scores(const bf16x8 (&x)[2][KP], Q&& query, f32x4v (&s)[kOrders][NT][2]) {
#pragma unroll
        for (int p = 0; p < kProducts<KP>; ++p)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    s[order<KP>(p)][t][u] = mfma(x[u][left<KP>(p)], query(t, right<KP>(p)), s[order<KP>(p)][t][u]);
    }
    __device__ __forceinline__ static void zero(f32x4v (&s)[kOrders][NT][2]) {
#pragma unroll
        for (int o = 0; o < kOrders; ++o)
#pragma unroll
            for (int t = 0; t < NT; ++t) s[o][t][0] = s[o][t][1] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ static void total(const f32x4v (&s)[kOrders][NT][2], f32x4v (&sum)[NT][2]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sum[t][u] = s[kOrders - 1][t][u];
#pragma unroll
                for (int o = kOrders - 2; o >= 0; --o) sum[t][u] += s[o][t][u];
            }
    }
    // Output MFMAs j0 .. j0 + N - 1 from V's parts x[j]
    template <int KP, int N>
    __device__ __forceinline__ void values(const bf16x8 (&x)[N][KP], int j0, const bf16x8 (&pp)[NT][PP]) {
#pragma unroll
        for (int p = 0; p < (KP == 1 ? PP : 6); ++p)
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    acc[t][j0 + j] = mfma(x[j][left<KP>(p)], pp[t][KP == 1 ? PP - 1 - p : right<KP>(p)], acc[t][j0 + j]);
    }

    // The running softmax over NB blocks of 32 keys from kb on: the scores s become the
    // weights' operands pp.  m, the score of weight 1, follows the maximum (and acc and l are
    // rescaled) only where that grew by more than kGrown in the exponent of 2: no weight
    // is above 2^kGrown, and all are rounded relative to themselves.
    static constexpr float kGrown = 8.f;
    template <int NB>
    __device__ __forceinline__ void softmax(const Work& w, int kb, f32x4v (&s)[NB][NT][2], float unit,
                                            bf16x8 (&pp)[NB][NT][PP]) {
        const bool whole = kb >= w.first && kb + 32 * NB - 1 <= see && kb + 32 * NB <= w.hi;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int top = min(min(qpos[t], w.last), w.hi - 1) - kb - 8 * g, low = w.first - kb - 8 * g;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        s[b][t][e >> 2][e & 3] =
                            32 * b + e >= low && 32 * b + e <= top ? s[b][t][e >> 2][e & 3] : -INFINITY;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float bm = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f32x4v x = s[b][t][0], y = s[b][t][1];
                bm = fmaxf(fmaxf(bm, x[0]), x[1]);
                bm = fmaxf(fmaxf(bm, x[2]), x[3]);
                bm = fmaxf(fmaxf(bm, y[0]), y[1]);
                bm = fmaxf(fmaxf(bm, y[2]), y[3]);
            }
            const float mn = fmaxf(m[t], quads_max(bm));
            if (__any((mn - m[t]) * unit > kGrown)) {   // (from -infinity: so it is)
                const float f = mn == -INFINITY ? 1.f : weight(m[t] - mn, unit);
                if constexpr (QP == 1)
                    lv[t] *= f;
                else
                    l[t] *= f;
#pragma unroll
                for (int j = 0; j < VD; ++j) acc[t][j] *= f;
                m[t] = mn;
            }
            const float mc = m[t] == -INFINITY ? 0.f : m[t];   // (no key seen yet: all weights 0)
            // (bf16 queries: one rounding more, of the row's largest exponent, against the 2^-8
            // of the output)
            const float mu = mc * unit;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = s[b][t][e >> 2][e & 3];
                    x[e] = QP == 1 ? __builtin_amdgcn_exp2f(fmaf(y, unit, -mu)) : weight(y - mc, unit);
                }
                if constexpr (QP == 1) {
                    const bf16x8 ones = __builtin_bit_cast(
                        bf16x8, make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u));
                    const Parts8 r = parts8(x);
                    pp[b][t][0] = r.h;
                    pp[b][t][PP - 1] = r.m;
#pragma unroll
                    for (int y = PP - 1; y >= 0; --y) lv[t] = mfma(ones, pp[b][t][y], lv[t]);
                } else {
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += x[e];
                    l[t] += sum;
                    const Parts8 r = parts8(x);
                    pp[b][t][0] = r.h;
                    pp[b][t][QP - 2] = r.m;
                    pp[b][t][QP - 1] = r.l;
                }
            }
        }
    }

    // l, a lane's own so far, of the whole row.
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (QP == 1)
                l[t] = lv[t][0];
            else
                l[t] = quads_add(l[t]);
        }
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
    // Keys lo .. lo + 31, lo + step .. for such a wave, row by row and key by key in
    // f32: positions that a row does not see are passed over.  tmp: HD floats of LDS.
    template <int KP>
    __device__ __forceinline__ void run_plain(const PagedAttnArgs& a, const Work& w, int rho0, int lo, int step,
                                           float unit, float* tmp) {
        constexpr int PL = HD / 64;
        const Cache<HD, KP> kv(a.p, w);
        const int lane = thread_id() & 63;
        bool bad = false;
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
                    const int64_t at = kv.at(kv.known(kv.page_of(k), bad), k) + PL * lane * kv.ES;
                    float s = 0.f, v[PL];
#pragma unroll
                    for (int i = 0; i < PL; ++i) {
                        const float kx = KP == 1 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(kv.k + at)[i])
                                                 : reinterpret_cast<const float*>(kv.k + at)[i];
                        v[i] = KP == 1 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(kv.v + at)[i])
                                       : reinterpret_cast<const float*>(kv.v + at)[i];
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
                        for (int v = 0; v < 4; ++v) acc[t][j][v] = tmp[dim(g, j, v)];
                }
            __threadfence_block();
        }
    }
};

// Few rows (at most 16): the four waves hold the same ones and take every fourth
// block of 32 keys, each straight from the cache into registers.  While one
// block is computed the next one's rows are on their way, K's from the moment the
// scores have used the last, V's from the end of the block, and the page numbers
// of the one after.
template <int HD, int QP, int KP>
struct Deep : Rows<HD, QP, 1, true> {
    typedef Rows<HD, QP, 1, true> R;
    static constexpr int NS = R::NS, VD = R::VD;
    using R::acc;
    using R::c;
    using R::g;
    typedef uint32_t words __attribute__((ext_vector_type(VD / 2)));
    uint4 kw[2][KP == 1 ? NS : 2 * NS];      // K of the lane's two rows
    words vw[KP == 1 ? 8 : 1];               // V of its eight
    float vf[KP == 3 ? 8 : 1][KP == 3 ? VD : 1];

    __device__ __forceinline__ void load_k(const Cache<HD, KP>& kv, int kb, int page) {
        const uint8_t* y = kv.k + kv.at(page, kb + 8 * (c >> 2) + (c & 3)) + 8 * kv.ES * g;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint4* x = reinterpret_cast<const uint4*>(y + 4 * u * kv.row);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                kw[u][KP == 1 ? i : 2 * i] = x[KP == 1 ? 4 * i : 8 * i];
                if constexpr (KP == 3) kw[u][2 * i + 1] = x[8 * i + 1];
            }
        }
    }
    __device__ __forceinline__ void load_v(const Cache<HD, KP>& kv, int kb, int page) {
        const uint8_t* x = kv.v + kv.at(page, kb + 8 * g) + VD * kv.ES * c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (KP == 1) {
                vw[e] = *reinterpret_cast<const words*>(x);
            } else {
#pragma unroll
                for (int i = 0; i < VD; i += 4) {
                    const f32x4v y = *reinterpret_cast<const f32x4v*>(x + 4 * i);
#pragma unroll
                    for (int z = 0; z < 4; ++z) vf[e][i + z] = y[z];
                }
            }
            x += kv.row;
        }
    }
    // V's rows that are not readable: 0
    __device__ __forceinline__ void clear_v(const Cache<HD, KP>& kv, int kb) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = kv.readable(kb + 8 * g + e);
            if constexpr (KP == 1) {
#pragma unroll
                for (int i = 0; i < VD / 2; ++i) vw[e][i] = in ? vw[e][i] : 0u;
            } else {
#pragma unroll
                for (int i = 0; i < VD; ++i) vf[e][i] = in ? vf[e][i] : 0.f;
            }
        }
    }
    // (the queries are read before the first block's rows and split while those are on
    // their way: loads come back in their order)
    // s_q: LDS of the wave's own, kQueries bytes: beside the rows of an f32 cache the queries'
    // parts leave too few registers for two workgroups per CU (104 spilled).
    static constexpr int kQueries = KP == 1 ? 0 : QP * NS * 1024;
    __device__ __forceinline__ void run(const PagedAttnArgs& a, const Work& w, int lo, int step, float unit,
                                        uint8_t* s_q) {
        const Cache<HD, KP> kv(a.p, w);
        this->lanes();
        bool bad = false;
        int pk0 = 0, pv0 = 0, pk1 = 0, pv1 = 0;
        if (lo < w.hi) {
            pk0 = kv.page_of(lo + 8 * (c >> 2));
            pv0 = kv.page_of(lo + 8 * g);
            if (lo + step < w.hi) {
                pk1 = kv.page_of(lo + step + 8 * (c >> 2));
                pv1 = kv.page_of(lo + step + 8 * g);
            }
        }
        f32x4v raw[1][NS][R::kRaw];
        this->read(a, w, 0, raw);
        if (lo < w.hi) {
            load_k(kv, lo, kv.known(pk0, bad));
            load_v(kv, lo, kv.known(pv0, bad));
        }
        this->split(raw);
        if constexpr (KP == 3) {
#pragma unroll
            for (int y = 0; y < QP; ++y)
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    *reinterpret_cast<bf16x8*>(s_q + 16 * (thread_id() & 63) + (y * NS + i) * 1024) = this->q[0][y][i];
        }
        const int hi = min(w.hi, min(this->most, w.last) + 1);
        if (lo < hi) {
            int pk, pv;
            for (int kb = lo; kb < hi; kb += step) {
                const int at = 16 * (thread_id() & 63);   // (the lane's queries: read anew for each block)
                const int nb = kb + step;
                pk = pk1;
                pv = pv1;
                if (nb + step < hi) {
                    pk1 = kv.page_of(nb + step + 8 * (c >> 2));
                    pv1 = kv.page_of(nb + step + 8 * g);
                }
                f32x4v part[QP][1][2], s[1][1][2];
                R::zero(part);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    bf16x8 x[2][KP];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if constexpr (KP == 1) {
                            x[u][0] = __builtin_bit_cast(bf16x8, kw[u][i]);
                        } else {
                            const f32x4v y = __builtin_bit_cast(f32x4v, kw[u][2 * i]);
                            const f32x4v z = __builtin_bit_cast(f32x4v, kw[u][2 * i + 1]);
                            const Parts8 r = parts8({y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]});
                            x[u][0] = r.h;
                            x[u][1] = r.m;
                            x[u][2] = r.l;
                        }
                    }
                    if constexpr (KP == 1) {
                        R::template scores<KP>(x, [&](int t, int y) { return this->q[t][y][i]; }, part);
                    } else {
                        bf16x8 qi[QP];
#pragma unroll
                        for (int y = 0; y < QP; ++y)
                            qi[y] = *reinterpret_cast<const bf16x8*>(s_q + at + (y * NS + i) * 1024);
                        R::template scores<KP>(x, [&](int, int y) { return qi[y]; }, part);
                    }
                }
                R::total(part, s[0]);
                if (nb < hi) load_k(kv, nb, kv.known(pk, bad));
                bf16x8 pp[1][1][R::PP];
                this->template softmax<1>(w, kb, s, unit, pp);
                if (kv.edge(kb, 32)) clear_v(kv, kb);
                constexpr int JG = KP == 1 ? 4 : 2;
#pragma unroll
                for (int j0 = 0; j0 < VD; j0 += JG) {
                    bf16x8 x[JG][KP];
#pragma unroll
                    for (int jj = 0; jj < JG; ++jj) {
                        const int j = j0 + jj;
                        if constexpr (KP == 1) {
                            uint32_t o[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[i] = __builtin_amdgcn_perm(vw[2 * i + 1][j >> 1], vw[2 * i][j >> 1],
                                                             j & 1 ? 0x07060302u : 0x05040100u);
                            x[jj][0] = __builtin_bit_cast(bf16x8, make_uint4(o[0], o[1], o[2], o[3]));
                        } else {
                            float y[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] = vf[e][j];
                            const Parts8 r = parts8(y);
                            x[jj][0] = r.h;
                            x[jj][1] = r.m;
                            x[jj][2] = r.l;
                        }
                    }
                    this->template values<KP>(x, j0, pp[0]);
                }
                if (nb < hi) load_v(kv, nb, kv.known(pv, bad));
            }
        }
        if (bad) flag_error(a.p.err, kErrPagedPage);
        this->close();
    }
};

// Many rows: the waves hold 16 NT rows each and share the keys, staged through LDS in
// pieces of SK.  The page numbers of the piece after the next are looked up while one
// is computed (lane l: of the piece's keys 8 (l % 16) ..).  The eight positions that share
// a page number are the same for a whole wave at every load, so that a load's address is
// one scalar base and a lane's constant offset.
template <int HD, int KP>
struct Stage;

// A bf16 cache: K and V row by row as the cache has them, copied by the loads themselves
// (no registers, no vector instruction), V's operands (eight keys of a dim) made by LDS reads
// that transpose, 4 keys x 16 dims at a time in 16 lanes.  A row's 16-byte units are placed
// so that the eight lanes of a K read, or the 32-byte pairs of the eight rows of 32 lanes
// of a V read, find theirs in different banks: the lane that copies a place takes the
// unit that belongs there.  (By way of registers, V's operands put together from words
// by v_perm: a prompt of 2500 positions 103 against 90 us.)
template <int HD>
struct Stage<HD, 1> {
    static constexpr int SK = 8192 / HD;                  // keys
    static constexpr int KU = HD / 8;                     // 16-byte units of a row
    static constexpr int kPlane = SK * HD * 2;            // bytes of K, of V
    static constexpr int kBytes = 2 * kPlane;
    static constexpr int kBuffers = 2;
    static constexpr int N = SK * KU / 256, KS = 256 / KU;   // copies of K (and V), positions of one
    static_assert(SK % 32 == 0 && SK <= 128 && N == 4, "a piece is whole 32-key blocks, in quarters");
    int pages, t, wave;
    uint32_t off, k_unit, v_unit;   // the lane's position in the wave's, its units at it, in bytes

    __device__ __forceinline__ static constexpr int k_turn(int key) {
        return ((key & 3) | ((key >> 3) & 3) << 2) & (KU - 1);
    }
    __device__ __forceinline__ static constexpr int v_turn(int key) {   // of pairs
        return HD == 64 ? ((key >> 1) & 1) | ((key >> 3) & 1) << 1 : (key & 3) | ((key >> 3) & 1) << 2;
    }
    __device__ __forceinline__ static int k_at(int key, int unit) { return (key * KU + (unit ^ k_turn(key))) * 16; }
    // Of the wave's keys key0 + 8 g .. + 7, dims 16 j + c.
    __device__ __forceinline__ static bf16x8 v_operand(const uint8_t* v, int key0, int j, int g, int c) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s16x4* lds_p;
        const int key = 8 * g + (c >> 2);
        const uint8_t* at = v + key0 * HD * 2 + key * HD * 2 + 32 * (j ^ v_turn(key)) + 8 * (c & 3);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at + 4 * HD * 2));
        return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void init(const Cache<HD, 1>& kv) {
        t = thread_id();
        wave = __builtin_amdgcn_readfirstlane(t >> 6);
        const int key = t / KU;
        off = (uint32_t)(key - 64 * wave / KU) * kv.row;
        k_unit = 16 * (t % KU ^ k_turn(key));
        v_unit = 16 * (t % KU ^ 2 * v_turn(key));
    }
    __device__ __forceinline__ void look(const Cache<HD, 1>& kv, int kb) {
        pages = kv.page_of(kb + 8 * (t & 15) % SK);
    }
    // Where the piece at kb is, by its pages (lane l: its group l % 16 of eight positions).
    __device__ __forceinline__ int64_t places(const Cache<HD, 1>& kv, int kb, bool& bad) const {
        return kv.at(kv.known(pages, bad), kb + 8 * (t & 15) % SK);
    }
    // A quarter of it to the buffer s: on its way until waited for.
    __device__ __forceinline__ void load(const Cache<HD, 1>& kv, int64_t at, int n, uint8_t* s) {
        const uint32_t lds = lds_addr(s) + 1024 * wave + 4096 * n;
        const int key = 64 * wave / KU + n * KS;   // the wave's first; (the lane's: its own turn, n's added)
        const int64_t base = Tile::lane64(at, key >> 3) + (uint32_t)(key & 7) * kv.row;
        lds_copy16(off + (k_unit ^ 16 * k_turn(n * KS)), kv.k + base, lds);
        lds_copy16(off + (v_unit ^ 32 * v_turn(n * KS)), kv.v + base, lds + kPlane);
    }
    // V's rows of the piece at kb (there, as far as the thread copied it) that are not
    // readable: 0
    __device__ __forceinline__ void clear_v(const Cache<HD, 1>& kv, int kb, uint8_t* s) const {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (!kv.readable(kb + t / KU + n * KS))
                *reinterpret_cast<uint4*>(s + kPlane + 16 * t + 4096 * n) = make_uint4(0, 0, 0, 0);
    }
};

// An f32 cache: K row by row as bf16 parts, V's parts transposed, eight keys of a dim
// together, both in 16-byte units placed so that the eight lanes an LDS read serves at
// once find theirs in different banks.  Each thread has 16 bytes of K at a time (a
// position's neighbouring dims) and VB dims of eight positions of V; the next piece is on
// its way into registers while one is computed.
template <int HD>
struct Stage<HD, 3> {
    static constexpr int SK = HD <= 128 ? 4096 / HD : 32;   // keys
    static constexpr int KU = HD / 8, VU = SK / 8;        // units of a K row, of a V row
    static constexpr int kPlane = SK * HD * 2;            // bytes of a part
    static constexpr int kBytes = 6 * kPlane;
    static constexpr int kBuffers = 1;
    static constexpr int VB = HD * SK / 2048;                   // dims of a thread's V block: 4 or 2
    static constexpr int NV = SK * HD / 8 / VB / 256;           // blocks of a thread
    static constexpr int CU = HD / 4;                           // 16-byte units of a position in the cache
    static constexpr int NK = SK * CU / 256;                    // loads of K
    static_assert(SK % 32 == 0 && SK <= 128 && NV >= 1 && NK >= 1, "a piece is whole 32-key blocks");
    typedef float vblock __attribute__((ext_vector_type(VB)));
    f32x4v kr[NK];
    float vr[NV][8][VB];
    int pages;
    // the thread, its wave, its offsets in a position of K and of V
    int t, wave;
    uint32_t k_off, v_off;

    __device__ __forceinline__ static int k_at(int key, int unit) {
        const int z = (key & 3) | ((key >> 3) & 3) << 2;
        return (key * KU + (unit ^ (z & (KU - 1)))) * 16;
    }
    __device__ __forceinline__ static int v_at(int d, int unit) {
        const int z = VU >= 8 ? d ^ (d >> 2) : (d >> 1) ^ (d >> 3);
        return (d * VU + (unit ^ (z & (VU - 1)))) * 16;
    }
    static constexpr int KS = 256 / CU;                   // positions of K the threads load at once
    __device__ __forceinline__ void init(const Cache<HD, 3>& kv) {
        t = thread_id();
        wave = __builtin_amdgcn_readfirstlane(t >> 6);
        k_off = (uint32_t)(t / CU - 64 * wave / CU) * kv.row + 16 * (t % CU);
        v_off = (uint32_t)(4 * VB * (t % (HD / VB)));
    }
    __device__ __forceinline__ void look(const Cache<HD, 3>& kv, int kb) {
        pages = kv.page_of(kb + 8 * (t & 15) % SK);
    }
    // The piece at kb, by its pages.
    __device__ __forceinline__ void load(const Cache<HD, 3>& kv, int kb, bool& bad) {
        // (lane l: where the group l % 16 of eight positions begins)
        const int64_t at = kv.at(kv.known(pages, bad), kb + 8 * (t & 15) % SK);
        const int key0 = 64 * wave / CU;   // the wave's first position of K
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int key = key0 + n * KS;
            kr[n] = *reinterpret_cast<const f32x4v*>(kv.k + (Tile::lane64(at, key >> 3) + (uint32_t)(key & 7) * kv.row) + k_off);
        }
        constexpr int kGroups = 64 * VB / HD > 1 ? 64 * VB / HD : 1;   // a wave's V blocks lie in so many
        static_assert(kGroups <= 2, "one group or two");
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int grp = (64 * wave + 256 * n) / (HD / VB);
            int64_t base = Tile::lane64(at, grp);
            if (kGroups == 2) {
                const int64_t other = Tile::lane64(at, grp + 1);
                base = (t & 63) >= HD / VB ? other : base;
            }
            const uint8_t* x = kv.v + base + v_off;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const vblock v = *reinterpret_cast<const vblock*>(x);
#pragma unroll
                for (int i = 0; i < VB; ++i) vr[n][e][i] = v[i];
                x += kv.row;
            }
        }
    }
    // V's rows of the piece at kb that are not readable: 0
    __device__ __forceinline__ void clear_v(const Cache<HD, 3>& kv, int kb) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = kv.readable(kb + (t + 256 * n) / (HD / VB) * 8 + e);
#pragma unroll
                for (int i = 0; i < VB; ++i) vr[n][e][i] = in ? vr[n][e][i] : 0.f;
            }
    }
    __device__ __forceinline__ void store(uint8_t* s) const {
#pragma unroll
        for (int n = 0; n < NK; ++n) {   // (half a unit of each part)
            const int key = t / CU + n * KS, unit = t % CU;
            uint2 h, m, l;
            parts4(kr[n], h, m, l);
            uint8_t* at = s + k_at(key, unit >> 1) + 8 * (unit & 1);
            *reinterpret_cast<uint2*>(at) = h;
            *reinterpret_cast<uint2*>(at + kPlane) = m;
            *reinterpret_cast<uint2*>(at + 2 * kPlane) = l;
        }
        uint8_t* sv = s + 3 * kPlane;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int b = t + 256 * n, grp = b / (HD / VB), d = VB * (b % (HD / VB));
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = vr[n][e][i];
                const Parts8 p = parts8(y);
                uint8_t* at = sv + v_at(d + i, grp);
                *reinterpret_cast<bf16x8*>(at) = p.h;
                *reinterpret_cast<bf16x8*>(at + kPlane) = p.m;
                *reinterpret_cast<bf16x8*>(at + 2 * kPlane) = p.l;
            }
        }
    }
};

template <int HD, int QP, int KP, int NT>
struct Wide : Rows<HD, QP, NT, false> {
    typedef Rows<HD, QP, NT, false> R;
    typedef Stage<HD, KP> S;
    static constexpr int NS = R::NS, VD = R::VD;
    // 32-key blocks a softmax takes at once: two halve its maxima and rescalings
    static constexpr int NB = S::SK >= 64 ? 2 : 1;

    // between(i): called in the course of it, i = 0 .. kBreaks - 1
    static constexpr int kBreaks = NB + 1;
    template <class F>
    __device__ __forceinline__ void blocks(const Work& w, int kb, int b0, float unit, const uint8_t* s_kv,
                                           F&& between) {
        const int g = this->g, c = this->c;
        f32x4v s[NB][NT][2];
        // (the SIMD's other wave's vector work fits between the MFMAs, not they between it)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4v part[QP][NT][2];
            R::zero(part);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                bf16x8 x[2][KP];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int y = 0; y < KP; ++y)
                        x[u][y] = *reinterpret_cast<const bf16x8*>(
                            s_kv + y * S::kPlane + S::k_at(32 * (b0 + b) + 8 * (c >> 2) + 4 * u + (c & 3), 4 * i + g));
                R::template scores<KP>(x, [&](int t, int y) { return this->q[t][y][i]; }, part);
            }
            R::total(part, s[b]);
            between(b);
        }
        __builtin_amdgcn_s_setprio(0);
        bf16x8 pp[NB][NT][R::PP];
        this->template softmax<NB>(w, kb, s, unit, pp);
        between(NB);
        __builtin_amdgcn_s_setprio(1);
        constexpr int JG = KP == 1 ? 4 : 2;
#pragma unroll
        for (int j0 = 0; j0 < VD; j0 += JG)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                bf16x8 x[JG][KP];
#pragma unroll
                for (int j = 0; j < JG; ++j)
#pragma unroll
                    for (int y = 0; y < KP; ++y) {
                        if constexpr (KP == 1)
                            x[j][y] = S::v_operand(s_kv + S::kPlane, 32 * (b0 + b), j0 + j, g, c);
                        else
                            x[j][y] = *reinterpret_cast<const bf16x8*>(
                                s_kv + (KP + y) * S::kPlane + S::v_at(16 * (j0 + j) + c, 4 * (b0 + b) + g));
                    }
                this->template values<KP>(x, j0, pp[b]);
            }
        __builtin_amdgcn_s_setprio(0);
    }
    // `rows`: whether the wave has some (those without take part in the staging)
    __device__ __forceinline__ void run(const PagedView& p, const Work& w, bool rows, float unit, uint8_t* s_kv) {
        const Cache<HD, KP> kv(p, w);
        const int hi = rows ? min(w.hi, min(this->most, w.last) + 1) : 0;
        bool bad = false;
        S st;
        st.init(kv);
        st.look(kv, w.lo);
        if constexpr (KP == 1) {
            int64_t at = st.places(kv, w.lo, bad);
#pragma unroll
            for (int n = 0; n < S::N; ++n) st.load(kv, at, n, s_kv);
            if (w.lo + S::SK < w.hi) st.look(kv, w.lo + S::SK);
            int turn = 0;
            for (int k0 = w.lo; k0 < w.hi; k0 += S::SK) {
                uint8_t* buf = s_kv + turn * S::kBytes;
                turn ^= 1;
                uint8_t* other = s_kv + turn * S::kBytes;
                wait_vm<0>();
                if (kv.edge(k0, S::SK)) st.clear_v(kv, k0, buf);
                const bool more = k0 + S::SK < w.hi;
                if (more) at = st.places(kv, k0 + S::SK, bad);
                __syncthreads();   // (the piece is there, and the other buffer read)
                // the next piece's copies, spread over this one's first blocks (at once a wave
                // waits 1000 of the piece's 5250 clocks to issue them)
                const auto rest = [&](int n0, int n1) {
                    if (!more) return;
#pragma unroll
                    for (int n = 0; n < S::N; ++n)
                        if (n >= n0 && n < n1) st.load(kv, at, n, other);
                };
                if (k0 + 2 * S::SK < w.hi) st.look(kv, k0 + 2 * S::SK);
                const bool on = k0 < hi;
                rest(0, on ? 1 : S::N);
                if (on)
                    blocks(w, k0, 0, unit, buf, [&](int i) { rest(i + 1, i + 1 < kBreaks ? i + 2 : S::N); });
#pragma unroll
                for (int b = NB; b < S::SK / 32; b += NB)
                    if (k0 + 32 * b < hi) blocks(w, k0 + 32 * b, b, unit, buf, [](int) {});
            }
        } else {
            st.load(kv, w.lo, bad);
            if (w.lo + S::SK < w.hi) st.look(kv, w.lo + S::SK);
            for (int k0 = w.lo; k0 < w.hi; k0 += S::SK) {
                __syncthreads();
                if (kv.edge(k0, S::SK)) st.clear_v(kv, k0);
                st.store(s_kv);
                __syncthreads();
                if (k0 + S::SK < w.hi) {
                    st.load(kv, k0 + S::SK, bad);
                    if (k0 + 2 * S::SK < w.hi) st.look(kv, k0 + 2 * S::SK);
                }
#pragma unroll
                for (int b = 0; b < S::SK / 32; b += NB)
                    if (k0 + 32 * b < hi) blocks(w, k0 + 32 * b, b, unit, s_kv, [](int) {});
            }
        }
        if (bad) flag_error(p.err, kErrPagedPage);
        this->close();
        __syncthreads();   // (s_kv is free again)
    }
};

// joins (m1, l1) with (m0, l0): the factors of both.  (Here and in mix the roundings are
// written out: the same wherever it is compiled.)
__device__ __forceinline__ void join(float& m0, float& l0, float m1, float l1, float unit, float& f0, float& f1) {
    const float mn = fmaxf(m0, m1), mc = mn == -INFINITY ? 0.f : mn;
    f0 = weight(m0 - mc, unit);
    f1 = weight(m1 - mc, unit);
    l0 = __builtin_fmaf(l0, f0, __fmul_rn(l1, f1));
    m0 = mn;
}
__device__ __forceinline__ f32x4v mix(f32x4v x, float f0, f32x4v y, float f1) {
    f32x4v o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(x[i], f0, __fmul_rn(y[i], f1));
    return o;
}

__device__ __forceinline__ void store4(const PagedAttnArgs& a, bool bf16, int64_t at, const float (&x)[4]) {
    if (bf16)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x[0], x[1], x[2], x[3]);
}

// Sixteen bytes to memory, past this XCD's L2 (sc1: for a workgroup on any XCD).  (The
// s_nop: a store of more than 8 bytes may still read its registers when the next
// instruction writes them, and the compiler does not see a store here.)
__device__ __forceinline__ void store4_coh(float* p, const float (&x)[4]) {
    const f32x4v v = {x[0], x[1], x[2], x[3]};
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" : : "v"(p), "v"(v) : "memory");
}
// Eight times sixteen bytes from there, waited for.
__device__ __forceinline__ void load8_coh(const float* const (&p)[8], f32x4v (&v)[8]) {
    asm volatile(
        "global_load_dwordx4 %0, %8, off sc1\n\tglobal_load_dwordx4 %1, %9, off sc1\n\t"
        "global_load_dwordx4 %2, %10, off sc1\n\tglobal_load_dwordx4 %3, %11, off sc1\n\t"
        "global_load_dwordx4 %4, %12, off sc1\n\tglobal_load_dwordx4 %5, %13, off sc1\n\t"
        "global_load_dwordx4 %6, %14, off sc1\n\tglobal_load_dwordx4 %7, %15, off sc1\n\t"
        "s_waitcnt vmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
        : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7])
        : "memory");
}

// Where a finished tile's rows go: divided by their sums to out, or as they are, with
// their maxima and sums, to a piece of the batch's rows (token, head) or, row by row, to
// a workgroup's slot, which another workgroup reads.
enum { kToOut, kToPiece, kToSlot };
template <int HD>
struct Sink {
    int to;
    float *o, *ml;            // [rows][HD], [rows][2]

    // dims d .. d + 3 of row rho
    __device__ __forceinline__ void put(const PagedAttnArgs& a, bool bf16, int rho, int token, int head, int d,
                                        float m, float l, float f, float x0, float x1, float x2, float x3) const {
        if (to == kToOut) {
            store4(a, bf16, (int64_t)token * a.out_stride + (int64_t)head * HD + d, {x0 * f, x1 * f, x2 * f, x3 * f});
        } else if (to == kToPiece) {
            const int64_t row = (int64_t)token * a.heads + head;
            *reinterpret_cast<float4*>(o + row * HD + d) = make_float4(x0, x1, x2, x3);
            if (d == 0) *reinterpret_cast<float2*>(ml + 2 * row) = make_float2(m, l);
        } else {
            store4_coh(o + rho * HD + d, {x0, x1, x2, x3});
            if (d == 0) {
                __hip_atomic_store(ml + 2 * rho, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(ml + 2 * rho + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
};

// Groups of 16 rows that a wave of Wide holds at most.  (f32 queries: three times the
// MFMAs per LDS read and three times the query registers)
template <int HD, int QP>
constexpr int tile_groups() { return HD <= 128 && QP == 1 ? 2 : 1; }
template <int HD, int QP>
constexpr int tile_rows() { return 64 * tile_groups<HD, QP>(); }
// floats of a workgroup's partial: o [R][HD], (m, l) [R]
template <int HD, int QP>
constexpr int64_t slot_floats() { return (int64_t)tile_rows<HD, QP>() * (HD + 2); }

// Workgroups that a CU holds (their registers).  (f32 cache, head_dim 128, eight turns of 1 to
// 30 tokens behind a prefix of 500: 39.3 us with one, 29.5 with two.)
constexpr int wgs_per_cu(int hd) { return hd <= 128 ? 2 : 1; }

// bytes of LDS: the stages of Wide; the four waves' results of Deep, or before them its
// queries and the plain path's four rows
template <int HD, int KP>
constexpr int work_lds() {
    return std::max({Stage<HD, KP>::kBuffers * Stage<HD, KP>::kBytes, (4 * 16 * HD + 128) * 4,
                     16 * HD + 4 * Deep<HD, 3, KP>::kQueries});
}

template <int HD, int QP, int KP>
__device__ __forceinline__ void few_rows(const PagedAttnArgs& a, const Work& w, float unit, uint8_t* s_buf,
                                         const Sink<HD>& sink) {
    constexpr int kWave = 16 * HD, VD = HD / 16;
    const int tid = thread_id(), wave = tid >> 6, lane = tid & 63;
    Deep<HD, QP, KP> r;
    // (the queries behind what run_plain of another wave may write)
    r.run(a, w, w.lo + 32 * wave, 128, unit, s_buf + 16 * HD + wave * r.kQueries);
    float* s = reinterpret_cast<float*>(s_buf);      // [4 waves][VD][64][4]
    float* s_ml = s + 4 * kWave;                     // [2][4][16]
    if (r.odd()) r.template run_plain<KP>(a, w, 0, w.lo + 32 * wave, 128, unit, s + wave * HD);
    // the waves' results of a row joined, wave i of four taking a quarter of its dims
    __syncthreads();
    if (lane < 16) {
        s_ml[16 * wave + lane] = r.m[0];
        s_ml[64 + 16 * wave + lane] = r.l[0];
    }
#pragma unroll
    for (int j = 0; j < VD; ++j) *reinterpret_cast<f32x4v*>(s + wave * kWave + (j * 64 + lane) * 4) = r.acc[0][j];
    __syncthreads();
    int token, head;
    const bool on = row_at(a, w, r.c, token, head);
    float f[4], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, s_ml[16 * k + r.c]);
    const float mc = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[k] = weight(s_ml[16 * k + r.c] - mc, unit);
        l = fmaf(s_ml[64 + 16 * k + r.c], f[k], l);
    }
    if (!on) return;
    // lane (g, c) of wave v: of row c the dims VD (4 g + v) .. + VD - 1
    const float inv = 1.0f / l;
#pragma unroll
    for (int j0 = 0; j0 < VD; j0 += 4) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i] = fmaf(s[k * kWave + ((j0 + i) * 64 + lane) * 4 + wave], f[k], x[i]);
        }
        sink.put(a, QP == 1, r.c, token, head, VD * (4 * r.g + wave) + j0, m, l, inv, x[0], x[1], x[2], x[3]);
    }
}

// Partials: the workgroups' slots; then, with a prefix, its pieces and one more for
// the rows' own positions, each [num_rows * heads][HD], and their (m, l).
template <int HD, int QP>
__device__ __forceinline__ Sink<HD> slot_of(const PagedAttnArgs& a, int i) {
    float* o = a.part + i * slot_floats<HD, QP>();
    return {kToSlot, o, o + (int64_t)tile_rows<HD, QP>() * HD};
}
// Workgroup p's piece of a tile that begins in workgroup `first` (it may have two pieces: of
// the tile that ends its share, and of the one that begins it).
template <int HD, int QP>
__device__ __forceinline__ Sink<HD> piece_slot(const PagedAttnArgs& a, int p, int first) {
    return slot_of<HD, QP>(a, p == first ? 2 * p + 1 : 2 * p);
}
template <int HD>
__device__ __forceinline__ Sink<HD> piece_of(const PagedAttnArgs& a, int i) {
    const int64_t rows = (int64_t)a.p.num_rows * a.heads;
    return {kToPiece, a.pre + i * rows * HD, a.pre + (a.splits + 1) * rows * HD + i * rows * 2};
}

template <int HD, int QP, class R>
__device__ __forceinline__ void many_out(const PagedAttnArgs& a, const Work& w, int rho0, const R& r,
                                         const Sink<HD>& sink) {
#pragma unroll
    for (int t = 0; t < (int)(sizeof(r.m) / sizeof(float)); ++t) {
        const int rho = rho0 + 16 * t + r.c;
        int token, head;
        if (!row_at(a, w, rho, token, head)) continue;
        const float f = 1.0f / r.l[t];
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
            sink.put(a, QP == 1, rho, token, head, 16 * j + 4 * r.g, r.m[t], r.l[t], f, r.acc[t][j][0],
                     r.acc[t][j][1], r.acc[t][j][2], r.acc[t][j][3]);
    }
}

// A tile that workgroups first .. last have a piece of, this one `mine`: the counter of
// those that have stored theirs (null: no such tile), and where the tile's rows go.
template <int HD>
struct Cut {
    uint32_t* counter;
    int first, last, mine;
    Sink<HD> done;
};

// True if a cut tile is done: all its other workgroups had ended, so that this one's rows
// need not go through memory (a prompt of 2500 positions, one part per weight, 83.9 -> 79.9 us).  Joined in the
// order of the pieces, as join_tile does.
template <int HD, int QP, int KP, int NT>
__device__ __forceinline__ bool many_rows(const PagedAttnArgs& a, const Work& w, float unit, uint8_t* s_buf,
                                          const Sink<HD>& sink, const Cut<HD>& cut) {
    const int wave = thread_id() >> 6, rho0 = wave * 16 * NT;
    const bool rows = rho0 < w.tokens * a.share;
    Wide<HD, QP, KP, NT> r;
    r.lanes();
    f32x4v raw[NT][HD / 32][Wide<HD, QP, KP, NT>::R::kRaw];
    r.read(a, w, rho0, raw);
    r.split(raw);
    r.run(a.p, w, rows, unit, s_buf);
    if (rows && r.odd())
        r.template run_plain<KP>(a, w, rho0, w.lo, 32, unit, reinterpret_cast<float*>(s_buf) + wave * HD);
    if (cut.counter) {
        uint32_t* s_there = reinterpret_cast<uint32_t*>(s_buf + 16 * HD);   // (behind run_plain's)
        if (threadIdx.x == 0)
            *s_there = __hip_atomic_load(cut.counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (*s_there == (uint32_t)(cut.last - cut.first)) {
            if (threadIdx.x == 0) __hip_atomic_store(cut.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (rows) {
                constexpr int VD = HD / 16, V = VD < 8 ? VD : 8;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int rho = rho0 + 16 * t + r.c;
                    float m = -INFINITY, l = 0.f;
#pragma unroll
                    for (int j0 = 0; j0 < VD; j0 += V) {
                        f32x4v o[V];
                        for (int p = cut.first; p <= cut.last; ++p) {
                            float mp = r.m[t], lp = r.l[t];
                            f32x4v y[8];
#pragma unroll
                            for (int k = 0; k < V; ++k) y[k] = r.acc[t][j0 + k];
                            if (p != cut.mine) {
                                const Sink<HD> slot = piece_slot<HD, QP>(a, p, cut.first);
                                const unsigned long long z =
                                    __hip_atomic_load(reinterpret_cast<unsigned long long*>(slot.ml + 2 * rho),
                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                                const float* at[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) at[k] = slot.o + rho * HD + 16 * (j0 + k % V) + 4 * r.g;
                                load8_coh(at, y);
                                mp = __uint_as_float((uint32_t)z);
                                lp = __uint_as_float((uint32_t)(z >> 32));
                            }
                            if (p == cut.first) {
                                m = mp;
                                l = lp;
#pragma unroll
                                for (int k = 0; k < V; ++k) o[k] = y[k];
                            } else {
                                float f0, f1;
                                join(m, l, mp, lp, unit, f0, f1);
#pragma unroll
                                for (int k = 0; k < V; ++k) o[k] = mix(o[k], f0, y[k], f1);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < V; ++k) r.acc[t][j0 + k] = o[k];
                    }
                    r.m[t] = m;
                    r.l[t] = l;
                }
                many_out<HD, QP>(a, w, rho0, r, cut.done);
            }
            return true;
        }
    }
    if (rows) many_out<HD, QP>(a, w, rho0, r, sink);
    return false;
}

template <int HD, int QP, int KP>
__device__ __forceinline__ bool compute(const PagedAttnArgs& a, const Work& w, float unit, uint8_t* s_buf,
                                        const Sink<HD>& sink, const Cut<HD>& cut) {
    const int n = w.tokens * a.share;
    if (n <= 16) {
        few_rows<HD, QP, KP>(a, w, unit, s_buf, sink);
        return false;
    }
    if (tile_groups<HD, QP>() == 1 || n <= 64) return many_rows<HD, QP, KP, 1>(a, w, unit, s_buf, sink, cut);
    if constexpr (tile_groups<HD, QP>() > 1)
        return many_rows<HD, QP, KP, tile_groups<HD, QP>()>(a, w, unit, s_buf, sink, cut);
    return false;
}

// The pieces of a tile that workgroups first .. last have written to their slots, joined.
// Few values: the threads that they leave share the pieces, eight loads of each in
// flight, and join theirs through LDS.  Many: eight values of a thread in flight, piece
// after piece.  Either way in an order that does not depend on who is last.
template <int HD, int QP>
__device__ __forceinline__ void join_tile(const PagedAttnArgs& a, const Work& w, int first, int last, float unit,
                                          uint8_t* s_buf, const Sink<HD>& sink) {
    constexpr int NV = tile_rows<HD, QP>() * HD / 4 / 256;
    const int rows = w.tokens * a.share, tid = thread_id(), values = rows * (HD / 4);
    const auto piece = [&](int p) { return piece_slot<HD, QP>(a, p, first); };
    const auto coh = [](const float* p) {
        return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    if (values <= 256) {
        const int groups = 256 / values, grp = tid / values, i = tid - grp * values;
        const int rho = i / (HD / 4), d = 4 * (i % (HD / 4));
        f32x4v o = {0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        if (grp < groups) {
            for (int p0 = first + 8 * grp; p0 <= last; p0 += 8 * groups) {
                const float* at[8];
                f32x4v y[8];
                float z[8], u[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const Sink<HD> slot = piece(min(p0 + k, last));
                    at[k] = slot.o + rho * HD + d;
                    z[k] = coh(slot.ml + 2 * rho);
                    u[k] = coh(slot.ml + 2 * rho + 1);
                }
                load8_coh(at, y);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (p0 + k > last) break;
                    float f0, f1;
                    join(m, l, z[k], u[k], unit, f0, f1);
                    o = mix(o, f0, y[k], f1);
                }
            }
        }
        float* s = reinterpret_cast<float*>(s_buf) + 8 * tid;
        *reinterpret_cast<f32x4v*>(s) = o;
        s[4] = m;
        s[5] = l;
        __syncthreads();
        int token, head;
        if (grp == 0 && row_at(a, w, rho, token, head)) {
            for (int k = 1; k < groups; ++k) {
                const float* y = reinterpret_cast<const float*>(s_buf) + 8 * (tid + k * values);
                float f0, f1;
                join(m, l, y[4], y[5], unit, f0, f1);
                o = mix(o, f0, *reinterpret_cast<const f32x4v*>(y), f1);
            }
            sink.put(a, QP == 1, rho, token, head, d, m, l, 1.0f / l, o[0], o[1], o[2], o[3]);
        }
        return;
    }
#pragma unroll 1
    for (int k0 = 0; k0 < NV && 256 * k0 < values; k0 += 8) {
        f32x4v o[8];
        float m[8], l[8];
        for (int p = first; p <= last; ++p) {
            const Sink<HD> slot = piece(p);
            const float* at[8];
            f32x4v y[8];
            float z[8], u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = tid + 256 * (k0 + k), rho = min(i / (HD / 4), rows - 1);
                at[k] = slot.o + rho * HD + 4 * (i % (HD / 4));
                z[k] = coh(slot.ml + 2 * rho);
                u[k] = coh(slot.ml + 2 * rho + 1);
            }
            load8_coh(at, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (p == first) {
                    o[k] = y[k];
                    m[k] = z[k];
                    l[k] = u[k];
                } else {
                    float f0, f1;
                    join(m[k], l[k], z[k], u[k], unit, f0, f1);
                    o[k] = mix(o[k], f0, y[k], f1);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = tid + 256 * (k0 + k), rho = i / (HD / 4);
            int token, head;
            if (rho < rows && row_at(a, w, rho, token, head))
                sink.put(a, QP == 1, rho, token, head, 4 * (i % (HD / 4)), m[k], l[k], 1.0f / l[k], o[k][0], o[k][1],
                         o[k][2], o[k][3]);
        }
    }
}

// The prefix, for all rows of the batch: workgroup = (tile of rows, kv head, piece of
// the prefix).
template <int HD, int QP, int KP>
__device__ __forceinline__ void prefix_piece(const PagedAttnArgs& a, int id, float unit, uint8_t* s_buf) {
    const PagedView& p = a.p;
    const int TT = tile_rows<HD, QP>() / a.share, tiles = (p.num_rows + TT - 1) / TT;
    const int head = id / tiles % p.kv_heads, piece = id / tiles / p.kv_heads;
    const int blocks = (p.prefix_len + 31) / 32;
    // the end of the rows: of the last sequence that is computed (the last start may be wrong)
    int* s_end = reinterpret_cast<int*>(s_buf);
    int rows = 0;
    for (int s = threadIdx.x; s < p.num_seqs; s += 256) {
        const int lo = p.row_start[s], hi = p.row_start[s + 1];
        if (seq_ok(p, lo, hi, p.kv_len[s]) && hi > lo) rows = max(rows, hi);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) rows = max(rows, __shfl_xor(rows, m));
    if ((threadIdx.x & 63) == 0) s_end[threadIdx.x >> 6] = rows;
    __syncthreads();
    rows = max(max(s_end[0], s_end[1]), max(s_end[2], s_end[3]));
    __syncthreads();   // (s_buf is the tile's)
    Work w;
    w.token0 = id % tiles * TT;
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
    w.uniform();
    compute<HD, QP, KP>(a, w, unit, s_buf, piece_of<HD>(a, piece), Cut<HD>{});
}

// The first workgroups take a share each of the line of the sequences' own positions, the
// others a piece each of the prefix.  A tile that several workgroups have a share of is
// joined by the last of them to end: their partials are stored past the L2s and complete
// before the workgroup is counted.
template <int HD, int QP, int KP>
__global__ __launch_bounds__(256, wgs_per_cu(HD)) void paged_attn_kernel(PagedAttnArgs a) {
    __shared__ int64_t s_cum[kPagedMaxSeqs + 1];
    __shared__ int64_t s_tmp[4];
    __shared__ int s_last;
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[work_lds<HD, KP>()];
    const PagedView& p = a.p;
    const float unit = a.scale * 1.44269504f;
    const int id = (int)blockIdx.x;
    if (id >= a.grid) {
        prefix_piece<HD, QP, KP>(a, id - a.grid, unit, s_buf);
        return;
    }
    Line ln;
    ln.cum = s_cum;
    ln.org = p.prefix_len & ~31;
    ln.TT = tile_rows<HD, QP>() / a.share;
    ln.kv_heads = p.kv_heads;
    make_line(p, ln, s_tmp, a.grid, id == 0);
    if (ln.total == 0) return;
    // neighbouring shares on one XCD (workgroup id mod 8)
    const int per = (ln.wgs + 7) / 8, wg = (id & 7) * per + (id >> 3);
    if ((id >> 3) >= per || wg >= ln.wgs) return;
    // (lane 0: the share's first place, lane 1: the next one's)
    const int lane = threadIdx.x & 63;
    int64_t x = ln.cut(wg + (lane == 1));
    const bool all = x >= ln.total;
    if (all) x = ln.total - 1;
    Tile t;
    ln.sequence(p, find_seq(p, ln, x), t);
    ln.find(x, t);
    x = all ? ln.total : ln.rounded(t, x);
    const int64_t x1 = Tile::lane64(x, 1);
    x = Tile::lane64(x, 0);
    t.of_lane(0);
    while (x < x1) {
        const int64_t end = min(t.end, x1);
        Work w;
        w.token0 = t.row0 + t.r * ln.TT;
        w.tokens = min(ln.TT, t.n - t.r * ln.TT);
        w.pos0 = t.base + t.r * ln.TT;
        w.row_pos = 1;
        w.head = t.head;
        w.head0 = t.head * a.share;
        w.lo = ln.org + ln.key(t, x);
        w.hi = ln.org + ln.key(t, end);
        w.first = p.prefix_len;
        w.last = w.pos0 + w.tokens - 1;
        w.table = p.pages + (int64_t)t.seq * p.table_stride;
        w.uniform();
        const Sink<HD> done = a.splits ? piece_of<HD>(a, a.splits) : Sink<HD>{kToOut, nullptr, nullptr};
        const bool whole = x == t.start && end == t.end;
        // the workgroups of a cut tile: from the one whose cut is its start (or rounded to
        // it) to the one with the last cut inside it
        int first = wg, last = wg;
        if (!whole) {
            if (x != t.start) first = ln.below(t.start + kTileKeys + kCut);
            if (end != t.end) last = ln.below(t.end);
        }
        const Cut<HD> cut{whole ? nullptr : a.counters + first, first, last, wg, done};
        const bool joined =
            compute<HD, QP, KP>(a, w, unit, s_buf, whole ? done : piece_slot<HD, QP>(a, wg, first), cut);
        if (!whole && !joined) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t before = __hip_atomic_fetch_add(a.counters + first, 1u, __ATOMIC_RELAXED,
                                                               __HIP_MEMORY_SCOPE_AGENT);
                s_last = before == (uint32_t)(last - first);
                if (s_last)
                    __hip_atomic_store(a.counters + first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s_last) join_tile<HD, QP>(a, w, first, last, unit, s_buf, done);
        }
        __syncthreads();   // (s_buf and s_last are the next tile's)
        x = end;
        if (x < x1) {
            if (x >= s_cum[t.seq + 1]) ln.sequence(p, find_seq(p, ln, x), t);
            ln.find(x, t);
            t.of_lane(0);
        }
    }
}

// A row's pieces of the prefix and its own part: out.  Workgroup = (token, some heads).
template <int HD, int QP>
__global__ __launch_bounds__(256) void paged_pieces_kernel(PagedAttnArgs a) {
    __shared__ int s_in;
    const PagedView& p = a.p;
    const float unit = a.scale * 1.44269504f;
    const int token = (int)blockIdx.x, tid = threadIdx.x;
    const int head = (int)blockIdx.y * (1024 / HD) + tid / (HD / 4), d = 4 * (tid % (HD / 4));
    const int64_t rows = (int64_t)p.num_rows * a.heads, row = (int64_t)token * a.heads + min(head, a.heads - 1);
    const Sink<HD> all = piece_of<HD>(a, 0);
    // (a row of a sequence that was computed)
    if (tid == 0) s_in = 0;
    __syncthreads();
    for (int s = tid; s < p.num_seqs; s += 256) {
        const int lo = p.row_start[s], hi = p.row_start[s + 1];
        if (token >= lo && token < hi && seq_ok(p, lo, hi, p.kv_len[s])) s_in = 1;
    }
    // (eight pieces in flight)
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 <= a.splits; s0 += 8) {
        float2 z[8];
        float4 y[8];
        float top = m;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t at = min(s0 + k, a.splits) * rows + row;
            z[k] = *reinterpret_cast<const float2*>(all.ml + 2 * at);
            y[k] = *reinterpret_cast<const float4*>(all.o + at * HD + d);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, z[k].x);
        const float mc = top == -INFINITY ? 0.f : top, f0 = weight(m - mc, unit);
        m = top;
        l *= f0;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= f0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (s0 + k > a.splits) break;   // (the last one again)
            const float f = weight(z[k].x - mc, unit);
            l = fmaf(z[k].y, f, l);
            o[0] = fmaf(y[k].x, f, o[0]);
            o[1] = fmaf(y[k].y, f, o[1]);
            o[2] = fmaf(y[k].z, f, o[2]);
            o[3] = fmaf(y[k].w, f, o[3]);
        }
    }
    __syncthreads();
    if (!s_in || head >= a.heads) return;
    const float f = 1.0f / l;
    store4(a, QP == 1, (int64_t)token * a.out_stride + (int64_t)head * HD + d,
           {o[0] * f, o[1] * f, o[2] * f, o[3] * f});
}

template <int HD, int QP, int KP>
void launch_attn(const PagedAttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((paged_attn_kernel<HD, QP, KP>), dim3((unsigned)(a.grid + a.prefix_wgs)), dim3(256), 0, st, a);
    if (a.splits)
        hipLaunchKernelGGL((paged_pieces_kernel<HD, QP>),
                           dim3((unsigned)a.p.num_rows, (unsigned)((a.heads + 1024 / HD - 1) / (1024 / HD))),
                           dim3(256), 0, st, a);
}

template <int HD>
void launch_attn_hd(const PagedAttnArgs& a, hipStream_t st) {
    if (a.x_bf16)
        launch_attn<HD, 1, 1>(a, st);
    else if (a.cache_bf16)
        launch_attn<HD, 3, 1>(a, st);
    else
        launch_attn<HD, 3, 3>(a, st);
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
    const int R = a.head_dim <= 128 && a.x_bf16 ? 128 : 64;   // tile_rows
    const int per = wgs_per_cu(a.head_dim);
    // With a prefix one workgroup per CU takes the sequences' own positions, as another
    // takes the prefix' at the same time, which computes while that one loads (two for
    // the own positions after the prefix': 64 steps of 20 to 600 positions behind 4096,
    // 45.6 us against 39.5; 8 turns behind 500, 41.3 against 40.2)
    a.grid = ((a.p.prefix_len ? 1 : per) * cus + 7) / 8 * 8;
    a.splits = a.prefix_wgs = 0;
    *own_floats = (int64_t)a.grid * 2 * R * (a.head_dim + 2);
    if (a.p.prefix_len == 0) return *own_floats;
    // about one workgroup per CU takes the prefix, pieces of at least 64 keys
    const int TT = R / a.share, tiles = (a.p.num_rows + TT - 1) / TT;
    const int64_t wgs = (int64_t)tiles * a.p.kv_heads;
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({a.p.prefix_len / 64, (cus + wgs - 1) / wgs, 32}));
    a.prefix_wgs = (int)(wgs * a.splits);
    return *own_floats + (int64_t)(a.splits + 1) * a.p.num_rows * a.heads * (a.head_dim + 2);
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
