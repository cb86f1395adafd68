// pa_ranged.hip — the kernels of pa_ranged.hpp over ranges of keys.
#include "pa_ranged.hpp"

namespace pa {

bool ranged_supported(int head_dim, pa_dtype act, pa_dtype cache_dtype) {
  return (act == PA_DTYPE_FLOAT16 || act == PA_DTYPE_BFLOAT16) && cache_dtype == act &&
         (head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256);
}

hipError_t launch_ranged(const RangedParams& p, pa_dtype act, hipStream_t s) {
  return launch_kind<kRRanges>(p, act, s);
}

}  // namespace pa
