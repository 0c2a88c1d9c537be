// drafts.hpp — kernel arguments of the drafted tokens' trees (tree.hip) and of the
// products with 4-bit weights (q4.hip).
#pragma once

#include <cstdint>

#include "paged.hpp"

namespace m1moe {

constexpr int kTreeWords = 4;                 // most 64-bit words of a row's mask
constexpr int kTreeRows = 64 * kTreeWords;    // most rows of a tree
constexpr int kMostCaches = 64;               // caches of one accept

struct TreePlanArgs {
    int32_t num_seqs, num_rows, words;
    const int32_t *row_start, *parents;
    uint64_t* mask;
    int32_t* depth;
    uint32_t* err;
};

struct TreeAcceptArgs {
    PagedView p;              // (k and v: not used)
    void* planes[2 * kMostCaches];   // every cache's k and v
    int32_t num_planes;
    int32_t row_units;        // 16-byte units of a position
    const int32_t *parents, *drafts, *drawn;
    int32_t *path, *accepted, *next, *past;
};

struct Q4Args {
    const uint32_t* w;
    const uint16_t *scales, *biases;
    int32_t rows, cols, group;
    const void* x;
    int64_t x_stride;
    int32_t tokens;
    const void* residual;     // as y, or null
    void* y;
    int64_t y_stride;
    int32_t x_bf16, y_bf16;
    // set by matmul_q4_plan
    int32_t tiny;                  // less than a unit's groups
    int32_t grid, waves;           // workgroups, of so many waves
    int32_t wave_split, split;     // waves, and workgroups, that share a tile's columns
    int32_t grid_x, whole;         // tiles of rows of W; tiles that are not shared
    int32_t chunk, lds;            // units of columns staged at once, bytes of LDS
    int32_t part_split;            // workgroups that make a token's parts
    int64_t sums_at, down_at, part_at;   // floats of the workspace before these
    uint8_t *xparts, *xsums;       // x in parts, its groups' sums in parts
    float* down;                   // [tokens rounded up to 16]: what x was divided by
    float* part;                   // partials of split workgroups
    uint32_t* counters;            // of shared tiles, zero between launches
};

int launch_tree_plan(const TreePlanArgs& a, void* stream);
int launch_tree_attention(const PagedAttnArgs& a, void* stream);
int launch_tree_accept(const TreeAcceptArgs& a, void* stream);
int64_t matmul_q4_plan(Q4Args& a, int cus);   // the floats of workspace needed
int launch_matmul_q4(const Q4Args& a, void* stream);

}  // namespace m1moe
