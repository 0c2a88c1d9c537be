// tree_attn.hip — attention of trees of drafted tokens over the paged KV cache.
#include <hip/hip_runtime.h>

#include "drafts.hpp"
#include "paged_attn.hpp"

namespace m1moe {

int launch_tree_attention(const PagedAttnArgs& a, void* stream) {
    return launch_attention<true>(a, static_cast<hipStream_t>(stream));
}

}  // namespace m1moe
