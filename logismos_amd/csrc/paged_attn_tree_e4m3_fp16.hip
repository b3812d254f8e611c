// Attention of drafted tokens over a paged cache of e4m3 rows, fp16 queries (paged_attn_tree.hpp).
#include "paged_attn_tree.hpp"

namespace lg {

hipError_t tree_launch_e4m3_fp16(const TreeParams& p, int d, hipStream_t stream) {
    return tree_by_width<PackedF16, true>(p, d, stream);
}

}  // namespace lg
