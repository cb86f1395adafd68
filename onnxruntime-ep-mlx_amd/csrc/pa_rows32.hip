// pa_rows32.hip — pa_rows32.hpp over pages of the activations' type.
#include "pa_rows32.hpp"

namespace pa {

hipError_t launch_rows32(const AttnParams& p, pa_dtype act, pa_dtype cache_dtype, hipStream_t s) {
  if (p.num_tokens <= 0 || p.batch <= 0) return hipSuccess;
  if (p.head_dim > 256 || p.v_head_dim != p.head_dim || p.linear_cap || !p.read_all_from_cache) return hipErrorInvalidValue;
  if (cache_dtype != act) return launch_rows32_coded(p, act, cache_dtype, s);
  switch (cache_dtype) {
    case PA_DTYPE_FLOAT16: return launch_head<TF16>(p, act, s);
    case PA_DTYPE_BFLOAT16: return launch_head<TBF16>(p, act, s);
    case PA_DTYPE_FLOAT32: return launch_head<TF32>(p, act, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
