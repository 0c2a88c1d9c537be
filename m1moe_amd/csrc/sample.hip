// sample.hip — one token per row of logits from given random numbers:
// temperature, top-k, top-p and min-p.
//
// With a row's logits in descending order (ties to the lower index) every
// filter keeps a beginning of that order, and so does all of them together:
// the kept sum S is the smallest of theirs, and the drawn token is the first
// whose running sum reaches u S.  Nothing is sorted: each of these places is
// looked for by value, in a histogram and then among one step's logits.  The
// weights w = e^((x - max) / T) are computed in f64 and rounded to whole
// multiples of 2^-44, so that their sums are integer sums: exact, whatever their
// order (2^18 logits of weight 1 stay below 2^63).
//
// Bound by the chain of steps on a row: of the 28.7 us that one of 50304 at a temperature
// and a top-p takes from its first clock to its last (one run with clocks between the steps)
// 3.3 are its largest logit, 4.2 the histogram, 5.4 its joining and sums,
// 9.5 the end of the top-p and 6.3 the draw, each a pass over the row and a few barriers of 16
// waves; 64 rows with settings of their own and many equal logits take 46 us.  While rows
// are fewer than CUs several workgroups share a row's histogram, and the last of
// them to end adds the others' up and searches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "device.hpp"
#include "paged.hpp"

namespace m1moe {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;      // steps of a histogram
constexpr int kPer = kBins / kThreads;   // a thread's neighbouring steps
constexpr int kList = 256;       // a step of at most so many logits is ranked in pairs
constexpr int kFront = 1024;    // the order's beginning, kept aside where it is at most so long
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
    // Weights of smaller logits are 0 (the smallest of them may be, too).
    __device__ __forceinline__ float lowest() const {
        return top == INFINITY ? top : (float)((double)top - 45.5 / c);   // (-inf at an infinite T)
    }
    __device__ __forceinline__ u64 units(float x) const {
        const double t = exponent(x);
        // (adding 2^52 leaves the rounded units in the low bits)
        const double y = exp2_f64(fmax(t, -60.0) + kUnit) + 4503599627370496.0;
        return t >= -45.0 ? (u64)__double_as_longlong(y) & ((1ull << 52) - 1) : 0ull;
    }
};

// The thread's logits: the fours 4 (tid + 1024 j) .. + 3 for j = 0, 1, ... and one of
// the vocabulary's last, fewer than four.  NaN and -inf are in no range that is asked
// for.  Every pass reads them again, from the L2 after the first (kept in
// registers, with 512 threads, they leave too few for the f64 weights: 36.9 against
// 35.7 us for one row of 50304).
struct Row {
    const float* x;
    int vocab, fours;
    float last;

    // (past the end: the last four again)
    __device__ __forceinline__ float4 load(int j) const {
        return reinterpret_cast<const float4*>(x)[min((int)threadIdx.x + kThreads * j, fours - 1)];
    }
    __device__ __forceinline__ bool has(int j) const { return (int)threadIdx.x + kThreads * j < fours; }
    __device__ __forceinline__ void init(const float* row, int n) {
        x = row;
        vocab = n;
        fours = n >> 2;
        const int i = 4 * fours + (int)threadIdx.x;
        last = i < n ? x[i] : -INFINITY;
    }
    __device__ __forceinline__ int chunks() const { return (fours + kThreads - 1) / kThreads; }
    // f(four logits, the first one's index) of the thread's fours and, the last one with
    // three times -inf, of the rest; four loads in flight (eight: half as much code again,
    // 29.1 against 28.4 us for one row of 50304)
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        for (int j = 0; j < chunks(); j += 4) {
            float4 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = load(j + k);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (has(j + k)) f(y[k], 4 * ((int)threadIdx.x + kThreads * (j + k)));
        }
        f(make_float4(last, -INFINITY, -INFINITY, -INFINITY), 4 * fours + (int)threadIdx.x);
    }
    // f(logit, index) of those in [from, to], few of them (from above -inf)
    template <class F>
    __device__ __forceinline__ void each_in(float from, float to, F&& f) const {
        each([&](float4 y, int i) {
            const auto in = [&](float v) { return v >= from && v <= to; };
            if (!(in(y.x) | in(y.y) | in(y.z) | in(y.w))) return;
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
                const float t = y.x;
                y = make_float4(y.y, y.z, y.w, t);
                if (in(t)) f(t, i + e);
            }
        });
    }
    // f(logit) of the chunks first, first + step, ..., one by one (the weights of several
    // at once need more registers than there are), and of the last ones with chunk 0.
    template <class F>
    __device__ __forceinline__ void each_of(F&& f, int first, int step) const {
        if (first < chunks()) {
            float4 y = load(first);
            for (int j = first; j < chunks(); j += step) {
                float4 e = y;
                y = load(j + step);   // (on its way meanwhile)
                if (!has(j)) continue;
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const float t = e.x;
                    e = make_float4(e.y, e.z, e.w, t);
                    f(t);
                }
            }
        }
        if (first == 0) f(last);
    }
};

// A histogram of the logits in [lo, hi], from hi down in kBins equal steps:
// where each step begins among the counts and units above (cnt and sum, with
// one more entry for the end; counts only where top-k asks for them).  f64 keeps the steps apart for any range.
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
    // f32 bounds around the logits of steps a .. b, for a first glance: wider than they
    // can be off (a step's border by 2^-52 of hi and the range, an f32 by 2^-24).
    __device__ __forceinline__ void bounds(int a, int b, float& from, float& to) const {
        const double x0 = (double)hi - (b + 1) / per, x1 = (double)hi - a / per;
        const double eps = 1e-12 * (fabs((double)hi) + fabs((double)lo));
        from = per > 0.0 ? (float)(x0 - 1e-6 * fabs(x0) - eps) : lo;
        to = per > 0.0 ? (float)(x1 + 1e-6 * fabs(x1) + eps) : hi;
        from = fmaxf(from, lo);
        to = fminf(to, hi);
    }
};

struct Shared {
    Bins top, sub;            // all logits with a weight; those of one step
    float fx[kFront];         // the logits of the top steps, in any order, and their indexes
    int fi[kFront];
    int fn;
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

__device__ __forceinline__ void fill(const Row& row, const Scale& sc, const Span& sp, Bins& b, bool counts,
                                     int first, int step) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        b.sum[i] = 0;
        b.cnt[i] = 0;
    }
    __syncthreads();
    row.each_of([&](float x) {
        if (!sp.in(x)) return;
        const int k = sp.step(x);
        atomicAdd(&b.sum[k], sc.units(x));
        if (counts) atomicAdd(&b.cnt[k], 1u);
    }, first, step);
    __syncthreads();
}

// Turns the steps' sums and counts (of steps kPer tid ..) into what lies above each.
__device__ __forceinline__ void scan(Bins& b, const u64 (&sum)[kPer], const uint32_t (&cnt)[kPer], Shared& s) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    u64 ss = 0;
    uint32_t cc = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        ss += sum[i];
        cc += cnt[i];
    }
    const u64 s_own = ss;
    const uint32_t c_own = cc;
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
    ss -= s_own;
    cc -= c_own;
    for (int w = 0; w < wave; ++w) {
        ss += s.red[w];
        cc += s.red32[w];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        b.sum[kPer * tid + i] = ss;
        b.cnt[kPer * tid + i] = cc;
        ss += sum[i];
        cc += cnt[i];
    }
    if (tid == kThreads - 1) {
        b.sum[kBins] = ss;
        b.cnt[kBins] = cc;
    }
    __syncthreads();
}

__device__ __forceinline__ void histogram(const Row& row, const Scale& sc, const Span& sp, Bins& b, bool counts,
                                          Shared& s) {
    fill(row, sc, sp, b, counts, 0, 1);
    u64 sum[kPer];
    uint32_t cnt[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        sum[i] = b.sum[kPer * (int)threadIdx.x + i];
        cnt[i] = b.cnt[kPer * (int)threadIdx.x + i];
    }
    scan(b, sum, cnt, s);
}

// A row's histogram made by `parts` workgroups, part `mine` this one's: true in
// the last of them to end, which has the whole.  Stores and loads of the parts are
// coherent across the XCDs, and complete before the workgroup is counted.
__device__ __forceinline__ bool gather(Bins& b, bool counts, Shared& s, const SampleArgs& a, int row, int mine) {
    const int tid = threadIdx.x, parts = a.parts;
    u64* sums = a.part_sum + ((int64_t)row * parts) * kBins + tid;
    uint32_t* cnts = a.part_cnt + ((int64_t)row * parts) * kBins + tid;
    const auto put = [](auto* p, auto v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const auto get = [](const auto* p) {
        return __hip_atomic_load(const_cast<std::remove_const_t<std::remove_pointer_t<decltype(p)>>*>(p),
                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    u64 sum[kPer];
    uint32_t cnt[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {   // (neighbouring lanes, neighbouring words)
        sum[i] = b.sum[kPer * tid + i];
        cnt[i] = b.cnt[kPer * tid + i];
        put(sums + mine * kBins + i * kThreads, sum[i]);
        if (counts) put(cnts + mine * kBins + i * kThreads, cnt[i]);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
        const uint32_t before =
            __hip_atomic_fetch_add(a.counters + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s.bin = before == (uint32_t)parts - 1u;
        if (s.bin) put(a.counters + row, 0u);
    }
    __syncthreads();
    const bool last = s.bin != 0;
    __syncthreads();
    if (!last) return false;
#pragma unroll 4
    for (int c = 0; c < parts; ++c) {
        if (c == mine) continue;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            sum[i] += get(sums + c * kBins + i * kThreads);
            if (counts) cnt[i] += get(cnts + c * kBins + i * kThreads);
        }
    }
    scan(b, sum, cnt, s);
    return true;
}

// The logits of the steps down to `bin` of all, kept aside by the search for the end
// of the first top_k: the later places lie above it, and their searches need not read
// the row again.  (Where their number is not known before, as with top-p alone, keeping
// them costs more than a pass: 28.5 -> 31.6 us for one row.)
struct Front {
    int bin;         // -1: none
};

template <class F>
__device__ __forceinline__ void each_in(const Row& row, const Front& fr, const Shared& s, float from, float to,
                                        F&& f) {
    if (fr.bin < 0) {
        row.each_in(from, to, f);
        return;
    }
#pragma unroll
    for (int i = 0; i < kFront / kThreads; ++i) {
        const int at = (int)threadIdx.x + kThreads * i;
        if (at < s.fn && s.fx[at] >= from && s.fx[at] <= to) f(s.fx[at], s.fi[at]);
    }
}

// A place in the order: the first logit at which the running count (by_count)
// or sum reaches `target` (1 <= target <= the whole), with the sum up to and with
// it; its index is looked for when `index`.
struct Found {
    u64 sum;
    float x;
    int index;
};

__device__ __forceinline__ Found find(const Row& row, Front& fr, const Scale& sc, const Span& all, Shared& s,
                                      bool counts, bool by_count, u64 target, bool index) {
    const int tid = threadIdx.x;
    Span sp = all;
    const Bins* b = &s.top;
    u64 above = 0;           // units and logits above the span
    uint32_t n_above = 0;
    while (true) {
        // the step that the place lies in
        const u64 want = by_count ? target - n_above : target - above;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int k = kPer * tid + i;
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
        uint32_t n = b->cnt[bin + 1] - b->cnt[bin];   // (0 without counts)
        above += b->sum[bin];
        n_above += b->cnt[bin];
        float from, to;
        if (by_count && b == &s.top && n_above + n <= kFront) {
            if (tid == 0) s.fn = 0;
            __syncthreads();
            all.bounds(0, bin, from, to);
            row.each_in(from, to, [&](float x, int i) {
                if (all.step(x) > bin) return;
                const int at = atomicAdd(&s.fn, 1);
                s.fx[at] = x;
                s.fi[at] = i;
            });
            __syncthreads();
            fr.bin = bin;
        }
        sp.bounds(bin, bin, from, to);
        if (n <= kList) {
            each_in(row, fr, s, from, to, [&](float x, int i) {
                if (sp.step(x) == bin) {
                    const int at = atomicAdd(&s.n, 1);
                    if (at < kList) {
                        s.lx[at] = x;
                        s.li[at] = i;
                    }
                }
            });
            __syncthreads();
            n = s.n;
        }
        if (n <= kList) {
            if (tid < (int)n) s.lw[tid] = sc.units(s.lx[tid]);
            __syncthreads();
            // the lanes per logit of the step that there are, up to 64, share the others
            int shift = 2;
            static_assert(kThreads >> 2 == kList, "four lanes per logit of a full list");
            while (shift < 6 && (int)n << (shift + 1) <= kThreads) ++shift;
            const int lanes = 1 << shift, mine = tid >> shift;
            if (mine < (int)n) {
                const float x = s.lx[mine];
                const int i = s.li[mine];
                const u64 w = s.lw[mine];
                u64 sum = 0;
                uint32_t cnt = 0;
#pragma unroll 2
                for (int j = tid & (lanes - 1); j < (int)n; j += lanes) {
                    const float y = s.lx[j];
                    const bool before = y > x || (y == x && s.li[j] < i);
                    sum += before ? s.lw[j] : 0;
                    cnt += before;
                }
                for (int m = 1; m < lanes; m <<= 1) {
                    sum += __shfl_xor(sum, m);
                    cnt += __shfl_xor(cnt, m);
                }
                sum += above + w;
                cnt += n_above + 1;
                if ((tid & (lanes - 1)) == 0 && (by_count ? cnt == target : sum >= target && sum - w < target)) {
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
        each_in(row, fr, s, from, to, [&](float x, int) {
            if (sp.step(x) == bin) {
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
        histogram(row, sc, sp, s.sub, counts, s);
        b = &s.sub;
    }
    // all of them the same logit: the j-th of them by index
    const u64 w = sc.units(sp.hi);
    const u64 j = by_count ? target - n_above : (target - above + w - 1) / w;
    Found f{above + j * w, sp.hi, -1};
    if (!index) return f;
    u64 seen = 0;
    const int wave = tid >> 6, lane = tid & 63;
    for (int c = 0; c <= row.chunks(); ++c) {   // (the last ones after all fours)
        const bool end = c == row.chunks();
        const bool on = end || row.has(c);
        float4 y = make_float4(row.last, -INFINITY, -INFINITY, -INFINITY);
        if (!end) y = row.load(c);
        const uint32_t e[4] = {on && y.x == sp.hi, on && y.y == sp.hi, on && y.z == sp.hi, on && y.w == sp.hi};
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
            if (e[k] && at == j) s.at = end ? 4 * row.fours + tid : 4 * (tid + kThreads * c) + k;
        }
        __syncthreads();
        if (seen >= j) break;
    }
    f.index = s.at;
    __syncthreads();
    return f;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int r = (int)blockIdx.x / a.parts, part = (int)blockIdx.x % a.parts, tid = threadIdx.x;
    Row row;
    row.init(a.logits + (int64_t)r * a.stride, a.vocab);
    const float T = a.temperature ? a.temperature[r] : 1.f;
    float top = -INFINITY, low = -INFINITY;   // (low: of the negated logits)
    row.each([&](float4 y, int) {
        // (fmaxf passes over NaN)
        top = fmaxf(fmaxf(top, y.x), fmaxf(y.y, fmaxf(y.z, y.w)));
        const auto neg = [](float x) { return x == -INFINITY ? x : -x; };
        low = fmaxf(fmaxf(low, neg(y.x)), fmaxf(neg(y.y), fmaxf(neg(y.z), neg(y.w))));
    });
    top = block_max(top, s.redf[0]);
    low = -block_max(low, s.redf[1]);
    if (top == -INFINITY) {
        if (tid == 0 && part == 0) {
            a.tokens[r] = -1;
            if (a.probs) a.probs[r] = 0.f;
        }
        return;
    }
    if (!(T > 0.f)) {   // the largest, at its lowest index
        if (part) return;
        if (tid == 0) s.at = 0x7FFFFFFF;
        __syncthreads();
        int best = 0x7FFFFFFF;
        row.each_in(top, top, [&](float, int i) { best = min(best, i); });
        if (best != 0x7FFFFFFF) atomicMin(&s.at, best);
        __syncthreads();
        if (tid == 0) {
            a.tokens[r] = s.at;
            if (a.probs) a.probs[r] = 1.f;
        }
        return;
    }
    const Scale sc{top, 1.4426950408889634 / (double)T};
    Span all;
    all.set(fmaxf(low, sc.lowest()), top);
    const int k = a.top_k ? a.top_k[r] : 0;
    const bool counts = k > 0;
    if (a.parts == 1) {
        histogram(row, sc, all, s.top, counts, s);
    } else {
        fill(row, sc, all, s.top, counts, part, a.parts);
        if (!gather(s.top, counts, s, a, r, part)) return;
    }
    const float mp = a.min_p ? a.min_p[r] : 0.f, tp = a.top_p ? a.top_p[r] : 1.f, u = a.u[r];
    u64 kept = s.top.sum[kBins];
    // the end of the first top_k, of the fewest with top_p of what is left, the draw
    Front fr{-1};
    Found f{0, 0.f, 0};
#pragma unroll 1
    for (int phase = 0; phase < 3; ++phase) {
        if (phase == 0 && !(k > 0 && (uint32_t)k < s.top.cnt[kBins])) continue;
        if (phase == 1 && !(tp < 1.f)) continue;
        if (phase == 2 && mp > 0.f) {
            // weights of at least min_p: whole steps above the one that holds the border,
            // and the logits of that one (and, as it is rounded another way, of the steps
            // to either side).  A front holds its steps whole, and nothing behind it is kept:
            // of these steps those in the front count, and a border below all of it leaves
            // what is kept.
            const double border = fmin(log2((double)mp), 0.0);
            const double xb = (double)top + border / sc.c;
            const int bin = !(xb > (double)all.lo) ? kBins - 1
                                                  : (int)fmin(((double)top - xb) * all.per, (double)(kBins - 1));
            const int b0 = max(bin - 1, 0), b1 = min(bin + 1, fr.bin < 0 ? kBins - 1 : fr.bin);
            if (mp > 1.f) {
                kept = 1ull << kUnit;
            } else if (b0 <= b1) {
                if (tid == 0) s.units = 0;
                __syncthreads();
                float from, to;
                all.bounds(b0, b1, from, to);
                each_in(row, fr, s, from, to, [&](float x, int) {
                    const int b = all.step(x);
                    if (b >= b0 && b <= b1 && sc.exponent(x) >= border) atomicAdd(&s.units, sc.units(x));
                });
                __syncthreads();
                const u64 sum = s.top.sum[b0] + s.units;
                if (sum < kept) kept = sum;
            }
        }
        const double share = phase == 1 ? fmax((double)tp, 0.0) : u > 0.f ? fmin((double)u, 1.0) : 0.0;
        u64 want = (u64)ceil(share * (double)kept);
        want = want < 1 ? 1 : want > kept ? kept : want;
        f = find(row, fr, sc, all, s, counts, phase == 0, phase == 0 ? (u64)k : want, phase == 2);
        if (phase < 2 && f.sum < kept) kept = f.sum;
    }
    if (tid == 0) {
        a.tokens[r] = f.index;
        if (a.probs)
            a.probs[r] = (float)(__builtin_ldexp(exp2_f64(sc.exponent(f.x)), kUnit) / (double)kept);
    }
}

}  // namespace

// While the rows leave CUs idle, up to kMostParts workgroups per row, each with at
// least one chunk of its logits.  (One row of 50304: 40.7 us with one workgroup, 33.5 with 2,
// 30.0 with 4, 28.8 with 8, 29.2 with 16; 64 rows: 52.7 with one each, 47.6 with 4.)
int sample_parts(int rows, int vocab, int cus) {
    constexpr int kMostParts = 8;
    const int chunks = (vocab + 4 * kThreads - 1) / (4 * kThreads);
    return std::max(1, std::min({cus / rows, chunks, kMostParts}));
}
int64_t sample_part_words(int cus) { return (int64_t)cus * (3 * kBins + 1); }

int launch_sample(const SampleArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(a.rows * a.parts)), block(kThreads);
    hipLaunchKernelGGL(sample_kernel, grid, block, 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace m1moe
