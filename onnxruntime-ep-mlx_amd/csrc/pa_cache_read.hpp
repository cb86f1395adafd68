// pa_cache_read.hpp — elements of cache rows of every storage type, widened to fp32.
#pragma once

#include "pa_device.hpp"

namespace pa {
namespace {

// Element e of a cache row starting at storage index `base`, widened to fp32.  `scale` is the
// fp8 per-(block, kv-head) scale or the integer per-tensor / per-channel scale of element e.
template <typename CT>
struct CacheRead;

template <>
struct CacheRead<TF16> {
  __device__ static float at(const void* c, int64_t base, int e, float) {
    return f16_to_f32(reinterpret_cast<const uint16_t*>(c)[base + e]);
  }
};
template <>
struct CacheRead<TBF16> {
  __device__ static float at(const void* c, int64_t base, int e, float) {
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(c)[base + e]);
  }
};
template <>
struct CacheRead<TF32> {
  __device__ static float at(const void* c, int64_t base, int e, float) {
    return reinterpret_cast<const float*>(c)[base + e];
  }
};
struct Fp8Cache {};
template <>
struct CacheRead<Fp8Cache> {
  __device__ static float at(const void* c, int64_t base, int e, float scale) {
    return e4m3_to_f32(reinterpret_cast<const uint8_t*>(c)[base + e]) * scale;
  }
};
// Integer caches: QuantizedCache::decode (kv_cache.rs:222-256), code * scale in fp32.
struct I8Cache {};
template <>
struct CacheRead<I8Cache> {
  __device__ static float at(const void* c, int64_t base, int e, float scale) {
    return (float)reinterpret_cast<const int8_t*>(c)[base + e] * scale;
  }
};
struct I4Cache {};
template <>
struct CacheRead<I4Cache> {
  __device__ static float at(const void* c, int64_t base, int e, float scale) {
    const uint32_t byte = reinterpret_cast<const uint8_t*>(c)[base + (e >> 1)];
    return (float)((int)((byte >> ((e & 1) * 4)) & 15u) - 8) * scale;
  }
};

template <typename CT>
constexpr bool kIntCache = false;
template <>
constexpr bool kIntCache<I8Cache> = true;
template <>
constexpr bool kIntCache<I4Cache> = true;

}  // namespace
}  // namespace pa
