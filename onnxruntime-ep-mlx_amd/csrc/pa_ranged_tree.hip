// pa_ranged_tree.hip — the kernels of pa_ranged.hpp for the nodes of drafted trees.
#include "pa_ranged.hpp"

namespace pa {

hipError_t launch_ranged_tree(const RangedParams& p, pa_dtype act, hipStream_t s) {
  if ((!p.tree_parents && (!p.tree_bits || p.tree_words <= 0)) || !p.tree_lag || p.groups || p.doc_starts)
    return hipErrorInvalidValue;
  return launch_kind<kRTree>(p, act, s);
}

}  // namespace pa
