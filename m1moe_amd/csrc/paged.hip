// paged.hip — a KV cache in pages for a batch of sequences: append (per-head
// q/k RMSNorm, RoPE and the store in one pass) and attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged.hpp"
#include "paged_attn.hpp"

namespace m1moe {

namespace {

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
    const int row0 = a.depth ? p.row_start[seq] : 0;
    if (tid < a.rotary / 2) {
        // (a drafted token: the position of its depth in the tree, not of its slot)
        const double at = a.depth ? (double)(pos - (row - row0)) + (double)a.depth[row] : (double)pos;
        const double ang = at * (double)a.inv_freq[tid];
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
    const auto grid = [&](int wgs) { return (wgs * cus + 7) / 8 * 8; };
    const auto slots = [&](int wgs) { return (int64_t)wgs * 2 * R * (a.head_dim + 2); };
    a.grid = grid(a.p.prefix_len ? 1 : per);
    a.splits = a.prefix_wgs = 0;
    *own_floats = slots(a.grid);
    if (a.p.prefix_len == 0) return *own_floats;
    // Pieces of at least 64 keys, so many that one workgroup per CU takes the prefix, and up to three
    // times as many where a last round would leave CUs without one (144 tiles on 256 CUs, 24 trees behind
    // 4096 positions: 98 us with 2 pieces, 84 with 3; 2100 rows, 32 heads over 8, bf16, 304 and 262).
    // That is weighed against a piece's rows, which are written and read once more: about 256 keys'
    // time a round (behind 500 positions 5 pieces of 800 such rows in place of 2: 54.8 us and 44.9).  By that
    // count more pieces have to save a twentieth, and past four rounds they do not (of 78 batches of 64 to
    // 2100 rows behind 500 and 4096 positions none is slower than with the fewest; 16 heads, f32 cache,
    // 24 turns behind 500, 65.8 us, would be 67.5).
    const int TT = R / a.share, tiles = (a.p.num_rows + TT - 1) / TT;
    const int64_t wgs = (int64_t)tiles * a.p.kv_heads, most = std::max(1, std::min(a.p.prefix_len / 64, 32));
    const int64_t least = std::min((cus + wgs - 1) / wgs, most);
    const auto keys = [&](int64_t s) {
        return (double)((wgs * s + cus - 1) / cus) * a.p.prefix_len / s + 256.0 * wgs * s / cus;
    };
    int64_t splits = least;
    for (int64_t s = least + 1; wgs <= 4 * (int64_t)cus && s <= std::min(3 * least, most); ++s)
        if (keys(s) < keys(splits) * (splits == least ? 0.95 : 1.0)) splits = s;
    a.splits = (int)splits;
    a.prefix_wgs = (int)(wgs * a.splits);
    // What is asked for never falls with the rows or the prefix, so that a program that has run its largest
    // batch captures any other of its model: the slots of a call without a prefix, and the most rows of
    // pieces that some batch of as many rows or fewer has: pieces x rows is at most most x rows, and
    // with wgs >= rows kv_heads / TT at most cus TT / kv_heads + rows for the fewest pieces, three times
    // that for as many more, which up to 4 cus workgroups have.
    const int64_t rows = a.p.num_rows, one = ((int64_t)cus * TT + a.p.kv_heads - 1) / a.p.kv_heads;
    const int64_t pieces = std::min(most * rows, std::max(one + rows, 3 * (one + std::min(rows, 4 * one))));
    return slots(grid(per)) + (pieces + rows) * a.heads * (a.head_dim + 2);
}

int launch_paged_attention(const PagedAttnArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    return launch_attention<false>(a, st);
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
