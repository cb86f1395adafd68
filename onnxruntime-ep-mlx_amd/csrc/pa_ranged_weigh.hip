// pa_ranged_weigh.hip — the kernels of pa_ranged.hpp for rows whose probabilities are wanted again.
#include "pa_ranged.hpp"

namespace pa {

hipError_t launch_ranged_weigh(const RangedParams& p, pa_dtype act, hipStream_t s) {
  if (!p.row_stats || p.groups || p.doc_starts) return hipErrorInvalidValue;
  return launch_kind<kRWeigh>(p, act, s);
}

}  // namespace pa
