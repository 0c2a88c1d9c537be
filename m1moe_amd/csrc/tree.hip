// tree.hip — trees of drafted tokens: who sees whom, and taking over those that the model
// agrees with.
#include <hip/hip_runtime.h>

#include "device.hpp"
#include "drafts.hpp"

namespace m1moe {

namespace {

// ---- plan ----------------------------------------------------------------------------
//
// sees(i) = {i} and sees(parent(i)), depth(i) = depth(parent(i)) + 1, by doubling: with
// up(i) the ancestor 2^r levels above i, sees(i) over these levels and depth(i) = the
// levels climbed,
//   sees'(i) = sees(i) | sees(up(i)), depth'(i) = depth(i) + depth(up(i)), up'(i) = up(up(i))
// until no row has an ancestor left above: as many rounds as the depth has bits.
//
// Workgroup = tree, a thread per row.  A few KB are read and written: bound by the launch and
// the chain start - parents - rounds (one tree of 26 rows and 64 of 1 to 64 alike 4.4 us, as
// fast as the calls are made).
template <int W>
__global__ __launch_bounds__(64 * W) void tree_plan_kernel(TreePlanArgs a) {
    constexpr int N = 64 * W;
    __shared__ int s_up[N], s_depth[N];
    __shared__ uint64_t s_sees[N][W];
    const int seq = (int)blockIdx.x, i = (int)threadIdx.x;
    const int lo = a.row_start[seq], hi = a.row_start[seq + 1], n = hi - lo;
    if (lo < 0 || hi < lo || hi > a.num_rows || n > N) {
        if (i == 0) flag_error(a.err, n > N && lo >= 0 && hi <= a.num_rows ? kErrTree : kErrPagedBatch);
        return;
    }
    int up = -1, depth = 0;
    uint64_t sees[W];
#pragma unroll
    for (int w = 0; w < W; ++w) sees[w] = w == i / 64 ? 1ull << (i & 63) : 0ull;
    if (i < n) {
        up = a.parents[lo + i];
        if (up < -1 || up >= i) {   // (counts as none)
            flag_error(a.err, kErrTree);
            up = -1;
        }
        depth = up >= 0;
    }
    while (__syncthreads_or(up >= 0)) {   // (and the last round's values are read)
        s_up[i] = up;
        s_depth[i] = depth;
#pragma unroll
        for (int w = 0; w < W; ++w) s_sees[i][w] = sees[w];
        __syncthreads();
        if (up >= 0) {
            const int u = up;
            up = s_up[u];
            depth += s_depth[u];
#pragma unroll
            for (int w = 0; w < W; ++w) sees[w] |= s_sees[u][w];
        }
    }
    if (i >= n) return;
#pragma unroll
    for (int w = 0; w < W; ++w) a.mask[(int64_t)(lo + i) * W + w] = sees[w];
    a.depth[lo + i] = depth;
}

// ---- accept --------------------------------------------------------------------------
//
// From row 0 on the way goes to the lowest child whose drafted token is the one drawn at
// the row.  The rows of the way, 0 = p_0 < p_1 < ..., move to the places 0, 1, .. behind
// the conversation: p_i >= i, so a place that is written is read by no later move, and a
// thread that reads its 16 bytes of eight rows before it writes them needs no second buffer.
//
// Workgroup = (tree, 4 KB of a position through all planes, the layers' k and v).  Every one walks
// for itself: the walk (a thread in LDS, a level at a time) takes less than a launch would.
// 32 trees of 8 to 64, 32 layers of 8 heads of 128 in bf16: 12.4 us, 2.7 TB/s, half of a large
// copy's rate; one tree, 16 layers: 5.9 us in a trace, the chain lengths - parents - walk - rows (7.6
// as fast as the calls are made).
__global__ __launch_bounds__(256) void tree_accept_kernel(TreeAcceptArgs a) {
    __shared__ int s_child[kTreeRows], s_drawn[kTreeRows], s_page[kTreeRows], s_path[kTreeRows], s_count;
    const PagedView& p = a.p;
    const int seq = (int)blockIdx.y, tid = (int)threadIdx.x;
    const bool first = blockIdx.x == 0;
    const int lo = p.row_start[seq], hi = p.row_start[seq + 1], len = p.kv_len[seq], n = hi - lo;
    const bool rows = lo >= 0 && hi >= lo && hi <= p.num_rows && len >= n &&
                      (int64_t)len <= (int64_t)p.table_stride << p.page_shift && (n == 0 || len - n >= p.prefix_len);
    const int base = len - n;
    if (!rows || n > kTreeRows || n == 0) {
        if (first && tid == 0) {
            if (!rows) flag_error(p.err, kErrPagedBatch);
            if (rows && n > kTreeRows) flag_error(p.err, kErrTree);
            a.accepted[seq] = 0;
            a.next[seq] = -1;
            a.past[seq] = len;
        }
        return;
    }
    int parent = -1, draft = 0;
    const bool on = tid < n;
    if (on) {
        parent = a.parents[lo + tid];
        draft = a.drafts[lo + tid];
        s_drawn[tid] = a.drawn[lo + tid];
        s_page[tid] = p.pages[(int64_t)seq * p.table_stride + ((base + tid) >> p.page_shift)];
        if (parent < -1 || parent >= tid) {   // (counts as none)
            if (first) flag_error(p.err, kErrTree);
            parent = -1;
        }
    }
    s_child[tid] = kTreeRows;
    __syncthreads();
    if (on && parent >= 0 && draft == s_drawn[parent]) atomicMin(&s_child[parent], tid);
    __syncthreads();
    if (tid == 0) {
        int at = 0, count = 0;
        do {
            s_path[count++] = at;
            at = s_child[at];
        } while (at < kTreeRows);
        s_count = count;
    }
    __syncthreads();
    const int count = s_count;
    if (first) {
        if (on) a.path[lo + tid] = tid < count ? s_path[tid] : -1;
        if (tid == 0) {
            a.accepted[seq] = count;
            a.next[seq] = s_drawn[s_path[count - 1]];
            a.past[seq] = base + count;
        }
    }
    const int all = (int)blockIdx.x * 256 + tid, plane = all / a.row_units, unit = all - plane * a.row_units;
    if (plane >= a.num_planes) return;
    uint4* cells = static_cast<uint4*>(a.planes[plane]);
    const auto cell = [&](int row) {
        const int pos = base + row;
        return (((int64_t)s_page[row] << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) * a.row_units + unit;
    };
    const auto known = [&](int row) { return (unsigned)s_page[row] < (unsigned)p.num_pages; };
    for (int i0 = 1; i0 < count; i0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(i0 + k, count - 1), from = s_path[i];
            if (known(from)) x[k] = cells[cell(from)];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k;
            if (i >= count) break;
            const int from = s_path[i];
            if (known(from) && known(i)) {
                if (from != i) cells[cell(i)] = x[k];
            } else if (first && tid == 0) {
                flag_error(p.err, kErrPagedPage);
            }
        }
    }
}

}  // namespace

int launch_tree_plan(const TreePlanArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)a.num_seqs);
    switch (a.words) {
        case 1: hipLaunchKernelGGL(tree_plan_kernel<1>, grid, dim3(64), 0, st, a); break;
        case 2: hipLaunchKernelGGL(tree_plan_kernel<2>, grid, dim3(128), 0, st, a); break;
        case 3: hipLaunchKernelGGL(tree_plan_kernel<3>, grid, dim3(192), 0, st, a); break;
        case 4: hipLaunchKernelGGL(tree_plan_kernel<4>, grid, dim3(256), 0, st, a); break;
        default: return (int)hipErrorInvalidValue;
    }
    return (int)hipGetLastError();
}

int launch_tree_accept(const TreeAcceptArgs& a, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)((a.num_planes * a.row_units + 255) / 256), (unsigned)a.p.num_seqs);
    hipLaunchKernelGGL(tree_accept_kernel, grid, dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace m1moe
