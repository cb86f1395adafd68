// pa_rows32_coded.hip — pa_rows32.hpp over fp8, int8 and int4 pages.
#include "pa_rows32.hpp"

namespace pa {

hipError_t launch_rows32_coded(const AttnParams& p, pa_dtype act, pa_dtype cache_dtype, hipStream_t s) {
  switch (cache_dtype) {
    case PA_DTYPE_FP8_E4M3: return launch_head<Fp8Cache>(p, act, s);
    case PA_DTYPE_INT8: return launch_head<I8Cache>(p, act, s);
    case PA_DTYPE_INT4: return launch_head<I4Cache>(p, act, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
