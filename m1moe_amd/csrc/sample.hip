// sample.hip — one token per row of logits from given random numbers:
// temperature, top-k, top-p and min-p.
//
// With a row's logits in descending order (ties to the lower index) every
// filter keeps a beginning of that order, and so does all of them together:
// the kept sum S is the smallest of theirs, and the drawn token is the first
// whose running sum reaches u S.  Nothing is sorted: each of these places is
// looked for by value.  The weights w = e^((x - max) / T) are computed in f64
// and rounded to whole multiples of 2^-44, so that their sums are integer sums:
// exact, whatever their order (2^18 logits of weight 1 stay below 2^63).
#include <hip/hip_runtime.h>

#include "device.hpp"
#include "paged.hpp"

namespace m1moe {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = 16;
constexpr int kBins = 2048;      // steps of a histogram
constexpr int kList = 256;       // a step of at most so many logits is ranked in pairs
constexpr int kUnit = 44;        // weights are whole multiples of 2^-44

// 2^t for t <= 0 in units of 2^-44 (0 below half a unit), and as it is.  2^f on
// [-1/2, 1/2] by its power series: the terms from ln2^13 f^13 / 13! on are below 2e-16.
__device__ __forceinline__ double exp2_f64(double t) {
    const double k = rint(t), f = t - k;
    double p = 2.5678435993488196e-11;
    p = fma(p, f, 4.44553827187081e-10);
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)k);
}

struct Scale {
    float top;       // the row's largest logit
    double c;        // log2(e) / T
    __device__ __forceinline__ double exponent(float x) const {   // <= 0; NaN or -inf: no weight
        return x == top ? 0.0 : ((double)x - (double)top) * c;
    }
    __device__ __forceinline__ bool some(float x) const { return exponent(x) >= -45.0; }
    __device__ __forceinline__ u64 units(float x) const {
        const double t = exponent(x);
        // (adding 2^52 leaves the rounded units in the low bits)
        const double y = exp2_f64(fmax(t, -60.0) + kUnit) + 4503599627370496.0;
        return t >= -45.0 ? (u64)__double_as_longlong(y) & ((1ull << 52) - 1) : 0ull;
    }
};

// The thread's logits: 4 (tid + 1024 j) .. + 3 for j = 0, 1, ..., NaN and those
// past the vocabulary as -inf; NV > 0: in registers, else read again each pass.
template <int NV>
struct Row {
    const float* x;
    int vocab;
    float4 v[NV > 0 ? NV : 1];

    __device__ __forceinline__ float4 load(int j) const {
        const int i = 4 * ((int)threadIdx.x + kThreads * j);
        float e[4];
        if (i + 3 < vocab) {
            const float4 y = *reinterpret_cast<const float4*>(x + i);
            e[0] = y.x;
            e[1] = y.y;
            e[2] = y.z;
            e[3] = y.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = i + k < vocab ? x[i + k] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = __builtin_isnan(e[k]) ? -INFINITY : e[k];
        return make_float4(e[0], e[1], e[2], e[3]);
    }
    __device__ __forceinline__ void init(const float* row, int n) {
        x = row;
        vocab = n;
        if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = load(j);
        }
    }
    __device__ __forceinline__ int chunks() const { return (vocab + 4 * kThreads - 1) / (4 * kThreads); }
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = 4 * ((int)threadIdx.x + kThreads * j);
                f(v[j].x, i);
                f(v[j].y, i + 1);
                f(v[j].z, i + 2);
                f(v[j].w, i + 3);
            }
        } else {
            for (int j = 0; j < chunks(); ++j) {
                const float4 y = load(j);
                const int i = 4 * ((int)threadIdx.x + kThreads * j);
                f(y.x, i);
                f(y.y, i + 1);
                f(y.z, i + 2);
                f(y.w, i + 3);
            }
        }
    }
};

// A histogram of the logits in [lo, hi], from hi down in kBins equal steps:
// where each step begins among the counts and units above (cnt and sum, with
// one more entry for the end).  f64 keeps the steps apart for any range.
struct Bins {
    u64 sum[kBins + 1];
    uint32_t cnt[kBins + 1];
};
struct Span {
    float lo, hi;
    double per;      // steps per logit
    __device__ __forceinline__ void set(float l, float h) {
        lo = l;
        hi = h;
        per = h > l ? (kBins - 1) / ((double)h - (double)l) : 0.0;
    }
    __device__ __forceinline__ bool in(float x) const { return x >= lo && x <= hi; }
    __device__ __forceinline__ int step(float x) const {
        return x == hi ? 0 : (int)(((double)hi - (double)x) * per);
    }
};

struct Shared {
    Bins top, sub;            // all logits with a weight; those of one step
    float lx[kList];          // one step's logits
    int li[kList];
    u64 lw[kList];
    u64 red[kWaves];
    uint32_t red32[kWaves];
    float redf[2][kWaves];
    int bin, n, at;
    uint32_t cnt;
    u64 sum, units;
    float x;
    uint32_t key_lo, key_hi;
};

// Whole numbers in the order of floats.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ float block_max(float v, float* red) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    v = wave_max(v);
    if (lane == 0) red[wave] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red[w]);
    __syncthreads();
    return m;
}

template <int NV>
__device__ __forceinline__ void histogram(const Row<NV>& row, const Scale& sc, const Span& sp, Bins& b, Shared& s) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int i = tid; i < kBins; i += kThreads) {
        b.sum[i] = 0;
        b.cnt[i] = 0;
    }
    __syncthreads();
    row.each([&](float x, int) {
        if (sp.in(x)) {
            const int k = sp.step(x);
            atomicAdd(&b.sum[k], sc.units(x));
            atomicAdd(&b.cnt[k], 1u);
        }
    });
    __syncthreads();
    // two neighbouring steps per thread, summed over the workgroup
    const u64 s0 = b.sum[2 * tid], s1 = b.sum[2 * tid + 1];
    const uint32_t c0 = b.cnt[2 * tid], c1 = b.cnt[2 * tid + 1];
    u64 ss = s0 + s1;
    uint32_t cc = c0 + c1;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const u64 o = __shfl_up(ss, m);
        const uint32_t q = __shfl_up(cc, m);
        if (lane >= m) {
            ss += o;
            cc += q;
        }
    }
    if (lane == 63) {
        s.red[wave] = ss;
        s.red32[wave] = cc;
    }
    __syncthreads();
    u64 bs = 0;
    uint32_t bc = 0;
    for (int w = 0; w < wave; ++w) {
        bs += s.red[w];
        bc += s.red32[w];
    }
    ss += bs;
    cc += bc;
    b.sum[2 * tid] = ss - s0 - s1;
    b.sum[2 * tid + 1] = ss - s1;
    b.cnt[2 * tid] = cc - c0 - c1;
    b.cnt[2 * tid + 1] = cc - c1;
    if (tid == kThreads - 1) {
        b.sum[kBins] = ss;
        b.cnt[kBins] = cc;
    }
    __syncthreads();
}

// A place in the order: the first logit at which the running count (by_count)
// or sum reaches `target` (1 <= target <= the whole), with the sum up to and with
// it; its index is looked for when `index`.
struct Found {
    u64 sum;
    float x;
    int index;
};

template <int NV>
__device__ Found find(const Row<NV>& row, const Scale& sc, const Span& all, Shared& s, bool by_count, u64 target,
                      bool index) {
    const int tid = threadIdx.x;
    Span sp = all;
    const Bins* b = &s.top;
    u64 above = 0;           // units and logits above the span
    uint32_t n_above = 0;
    while (true) {
        // the step that the place lies in
        const u64 want = by_count ? target - n_above : target - above;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = 2 * tid + i;
            const u64 lo = by_count ? b->cnt[k] : b->sum[k], hi = by_count ? b->cnt[k + 1] : b->sum[k + 1];
            if (lo < want && want <= hi) {
                s.bin = k;
                s.n = 0;
                s.key_lo = 0xFFFFFFFFu;
                s.key_hi = 0u;
            }
        }
        __syncthreads();
        const int bin = s.bin;
        const uint32_t n = b->cnt[bin + 1] - b->cnt[bin];
        above += b->sum[bin];
        n_above += b->cnt[bin];
        if (n <= kList) {
            row.each([&](float x, int i) {
                if (sp.in(x) && sp.step(x) == bin) {
                    const int at = atomicAdd(&s.n, 1);
                    s.lx[at] = x;
                    s.li[at] = i;
                    s.lw[at] = sc.units(x);
                }
            });
            __syncthreads();
            if (tid < (int)n) {
                const float x = s.lx[tid];
                const int i = s.li[tid];
                const u64 w = s.lw[tid];
                u64 sum = above + w;
                uint32_t cnt = n_above + 1;
                for (int j = 0; j < (int)n; ++j) {
                    const float y = s.lx[j];
                    if (y > x || (y == x && s.li[j] < i)) {
                        sum += s.lw[j];
                        ++cnt;
                    }
                }
                if (by_count ? cnt == target : sum >= target && sum - w < target) {
                    s.sum = sum;
                    s.x = x;
                    s.at = i;
                }
            }
            __syncthreads();
            const Found f{s.sum, s.x, s.at};
            __syncthreads();
            return f;
        }
        // narrower: from its smallest to its largest logit
        uint32_t klo = 0xFFFFFFFFu, khi = 0u;
        row.each([&](float x, int) {
            if (sp.in(x) && sp.step(x) == bin) {
                klo = min(klo, order_of(x));
                khi = max(khi, order_of(x));
            }
        });
        if (klo <= khi) {
            atomicMin(&s.key_lo, klo);
            atomicMax(&s.key_hi, khi);
        }
        __syncthreads();
        sp.set(of_order(s.key_lo), of_order(s.key_hi));
        __syncthreads();
        if (sp.lo == sp.hi) break;
        histogram(row, sc, sp, s.sub, s);
        b = &s.sub;
    }
    // all of them the same logit: the j-th of them by index
    const u64 w = sc.units(sp.hi);
    const u64 j = by_count ? target - n_above : (target - above + w - 1) / w;
    Found f{above + j * w, sp.hi, -1};
    if (!index) return f;
    u64 seen = 0;
    const int wave = tid >> 6, lane = tid & 63;
    for (int c = 0; c < row.chunks(); ++c) {
        const float4 y = row.load(c);
        const uint32_t e[4] = {y.x == sp.hi, y.y == sp.hi, y.z == sp.hi, y.w == sp.hi};
        uint32_t q = e[0] + e[1] + e[2] + e[3];
        const uint32_t mine = q;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(q, m);
            if (lane >= m) q += o;
        }
        if (lane == 63) s.red32[wave] = q;
        __syncthreads();
        u64 at = seen;
        for (int v = 0; v < kWaves; ++v) {
            if (v < wave) at += s.red32[v];
            seen += s.red32[v];
        }
        at += q - mine;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            at += e[k];
            if (e[k] && at == j) s.at = 4 * (tid + kThreads * c) + k;
        }
        __syncthreads();
        if (seen >= j) break;
    }
    f.index = s.at;
    __syncthreads();
    return f;
}

template <int NV>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int r = (int)blockIdx.x, tid = threadIdx.x;
    Row<NV> row;
    row.init(a.logits + (int64_t)r * a.stride, a.vocab);
    const float T = a.temperature ? a.temperature[r] : 1.f;
    float top = -INFINITY;
    row.each([&](float x, int) { top = fmaxf(top, x); });
    top = block_max(top, s.redf[0]);
    if (top == -INFINITY) {
        if (tid == 0) {
            a.tokens[r] = -1;
            if (a.probs) a.probs[r] = 0.f;
        }
        return;
    }
    if (!(T > 0.f)) {   // the largest, at its lowest index
        if (tid == 0) s.at = 0x7FFFFFFF;
        __syncthreads();
        int best = 0x7FFFFFFF;
        row.each([&](float x, int i) {
            if (x == top) best = min(best, i);
        });
        if (best != 0x7FFFFFFF) atomicMin(&s.at, best);
        __syncthreads();
        if (tid == 0) {
            a.tokens[r] = s.at;
            if (a.probs) a.probs[r] = 1.f;
        }
        return;
    }
    const Scale sc{top, 1.4426950408889634 / (double)T};
    float low = -INFINITY;   // (of the negated logits: the smallest with a weight)
    row.each([&](float x, int) {
        if (sc.some(x)) low = fmaxf(low, -x);
    });
    low = -block_max(low, s.redf[1]);
    Span all;
    all.set(low, top);
    histogram(row, sc, all, s.top, s);
    u64 kept = s.top.sum[kBins];
    const int k = a.top_k ? a.top_k[r] : 0;
    if (k > 0 && (uint32_t)k < s.top.cnt[kBins]) kept = find(row, sc, all, s, true, (u64)k, false).sum;
    const float mp = a.min_p ? a.min_p[r] : 0.f;
    u64 kept_m = kept;
    if (mp > 0.f) {
        // weights of at least min_p: whole steps above the one that holds the border,
        // and that one's logits
        const double border = fmin(log2((double)mp), 0.0);
        const double xb = (double)top + border / sc.c;
        if (tid == 0) s.units = 0;
        const int bin = !(xb > (double)low) ? kBins - 1
                                           : (int)fmin(((double)top - xb) * all.per, (double)(kBins - 1));
        __syncthreads();
        // (a step to either side: the border's own step is rounded another way)
        const int b0 = max(bin - 1, 0), b1 = min(bin + 1, kBins - 1);
        row.each([&](float x, int) {
            if (all.in(x)) {
                const int b = all.step(x);
                if (b >= b0 && b <= b1 && sc.exponent(x) >= border) atomicAdd(&s.units, sc.units(x));
            }
        });
        __syncthreads();
        kept_m = mp > 1.f ? 1ull << kUnit : s.top.sum[b0] + s.units;
    }
    const float tp = a.top_p ? a.top_p[r] : 1.f;
    if (tp < 1.f) {
        u64 want = (u64)ceil(fmax((double)tp, 0.0) * (double)kept);
        want = want < 1 ? 1 : want > kept ? kept : want;
        const u64 sum = find(row, sc, all, s, false, want, false).sum;
        kept = sum < kept ? sum : kept;
    }
    kept = kept_m < kept ? kept_m : kept;
    const float u = a.u[r];
    u64 want = (u64)ceil((u > 0.f ? fmin((double)u, 1.0) : 0.0) * (double)kept);
    want = want < 1 ? 1 : want > kept ? kept : want;
    const Found f = find(row, sc, all, s, false, want, true);
    if (tid == 0) {
        a.tokens[r] = f.index;
        if (a.probs)
            a.probs[r] = (float)(__builtin_ldexp(exp2_f64(sc.exponent(f.x)), kUnit) / (double)kept);
    }
}

}  // namespace

int launch_sample(const SampleArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)a.rows), block(kThreads);
    if (a.vocab <= 4 * kThreads * 4)
        hipLaunchKernelGGL(sample_kernel<4>, grid, block, 0, st, a);
    else if (a.vocab <= 4 * kThreads * 8)
        hipLaunchKernelGGL(sample_kernel<8>, grid, block, 0, st, a);
    else if (a.vocab <= 4 * kThreads * 13)
        hipLaunchKernelGGL(sample_kernel<13>, grid, block, 0, st, a);
    else
        hipLaunchKernelGGL(sample_kernel<0>, grid, block, 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace m1moe
