// pa_weigh.hpp — which query rows count for a key's account.
#pragma once

#include "pa_ranged.hpp"

namespace pa {
namespace {

// Rows of a key: [lo, hi) of its sequence's rows (token * g + head) see it and count.
struct WRows {
  int lo, hi;
};
__device__ __forceinline__ WRows key_rows(const RangedParams& p, const RSeq& e, int key) {
  const int g = p.num_heads / p.kv_heads;
  int lo = p.observed > 0 ? max(e.nq - p.observed, 0) : 0, hi = e.nq;
  if (p.causal) lo = max(lo, key - e.past);
  if (p.window > 0) hi = (int)min((int64_t)hi, (int64_t)key - e.past + p.window);
  if (key >= e.total || lo >= hi) return WRows{INT32_MAX, 0};
  return WRows{lo * g, hi * g};
}

}  // namespace
}  // namespace pa
