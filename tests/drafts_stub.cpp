// The launchers that drafts.cpp calls and serving_stub.cpp does not have.
#include "drafts.hpp"

static long g_drafts = 0;
extern "C" long stub_drafts(void) { return g_drafts; }

namespace m1moe {
int launch_tree_plan(const TreePlanArgs&, void*) { return ++g_drafts, 0; }
int launch_tree_accept(const TreeAcceptArgs&, void*) { return ++g_drafts, 0; }
int launch_matmul_q4(const Q4Args&, int, void*) { return ++g_drafts, 0; }
}  // namespace m1moe
