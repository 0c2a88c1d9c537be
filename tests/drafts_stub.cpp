// The launchers that drafts.cpp calls and serving_stub.cpp does not have.
#include <cstdlib>

#include "drafts.hpp"

static long g_drafts = 0;
extern "C" long stub_drafts(void) { return g_drafts; }

namespace m1moe {
int launch_tree_plan(const TreePlanArgs&, void*) { return ++g_drafts, 0; }
int launch_tree_attention(const PagedAttnArgs& a, void*) {
    for (int i = 0; i < a.grid; ++i)
        if (a.counters[i]) abort();
    return ++g_drafts, 0;
}
int launch_tree_accept(const TreeAcceptArgs&, void*) { return ++g_drafts, 0; }
int64_t matmul_q4_plan(Q4Args& a, int cus) {
    a.split = 2;
    a.grid = 2 * cus;
    return 1000;
}
int launch_matmul_q4(const Q4Args& a, void*) {
    for (int i = 0; i < a.grid / a.split; ++i)
        if (a.counters[i]) abort();   // counters that were never cleared
    return ++g_drafts, 0;
}
}  // namespace m1moe
