// pa_axes.hip — rotary positions of several axes on queries and keys, and the append into the pages.
//
// Frequency i of a head row is a pair of elements (a, b) that turns by the angle of its own axis'
// position: (a c - b s, b c + a s) with c, s = cos / sin [positions[axis(i)][t]][i].  Before that a
// row may be normalised, x / sqrt(mean(x^2) + eps) * w.  All of it in fp32 with one rounding to the
// activation dtype at the end (the tables may be fp32, which a rounding in between would waste);
// byte-coded pages encode that rounded row.
#include <algorithm>

#include "pa_append_rows.hpp"

#pragma clang fp contract(off)

namespace pa {
namespace {

template <typename TT>
__device__ __forceinline__ float table_at(const void* t, int64_t i, int f32) {
  return f32 ? reinterpret_cast<const float*>(t)[i] : ldv<TT>(t, i);
}

// Any element type, head size and alignment: one workgroup of four wavefronts per token and four of
// its rows (queries, keys, values in turn), one row per wavefront, held in LDS in fp32.
constexpr int kAxesMaxDim = 640;
template <typename TT, int CK>
__global__ __launch_bounds__(256) void axes_append_kernel(const AppendParams p, const AxisParams ax) {
  __shared__ float rows[4][kAxesMaxDim];
  const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int D = p.head_dim, half = p.rotary_half, off = p.rotary_offset;
  const int row0 = blockIdx.y * 4, r = row0 + wave;
  const int nq = p.num_heads, nqk = nq + p.kv_heads, nrows = nqk + p.kv_heads;
  if (t < p.cum[0] || t >= p.cum[p.batch]) return;  // of no sequence: left alone
  // The slot of the token's key and value rows, by the whole workgroup (last-writer rule)
  int64_t slot = -1;
  if (row0 + 4 > nq) {
    const SeqPos sp = seq_pos_of_token(p.cum, p.past, p.batch, t);
    const int64_t pos = (int64_t)max(sp.past, 0) + (t - sp.start);
    slot = p.slot_mapping ? (int64_t)p.slot_mapping[t] : slot_at(p, sp.b, pos);
    if (slot >= p.num_blocks * p.block_size) slot = -1;
    if (slot >= 0 && !p.slots_distinct) {
      bool later = false;
      if (p.slot_mapping) {
        for (int u = t + 1 + threadIdx.x; u < p.num_tokens; u += blockDim.x)
          if ((int64_t)p.slot_mapping[u] == slot) later = true;
        later = __syncthreads_or(later);
      } else {
        later = later_block_dup(p, sp.b, pos, slot);
      }
      if (later) slot = -1;
    }
  }
  const bool is_q = r < nq, is_v = r >= nqk, live = r < nrows && (is_q || slot >= 0);
  const int head = is_q ? r : is_v ? r - nqk : r - nq;
  float* row = rows[wave];
  if (live) {
    const void* src = is_q ? p.query : is_v ? p.value : p.key;
    const int64_t base = (int64_t)t * (is_q ? p.q_ld : is_v ? p.v_ld : p.k_ld) + (int64_t)head * D;
    const void* w = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
    float inv = 1.0f;
    if (w) {
      const float acc = sum_squares([&](int e) { return ldv<TT>(src, base + e); }, D, lane);
      inv = 1.0f / __builtin_sqrtf(acc / (float)D + p.norm_eps);
    }
    for (int e = lane; e < D; e += 64) {
      float v = ldv<TT>(src, base + e);
      if (w) v = v * inv * ldv<TT>(w, e);
      row[e] = v;
    }
  }
  __syncthreads();
  if (!live) return;
  // Element e of the finished row, rounded to T
  auto value = [&](int e) -> float {
    const int x = e - off;
    if (is_v || x < 0 || x >= 2 * half) return rnd<TT>(row[e]);
    const bool first = p.rotary_interleaved ? (x & 1) == 0 : x < half;
    const int i = p.rotary_interleaved ? x >> 1 : first ? x : x - half;
    const int64_t pos = ax.positions[ax.axis_of(i) * ax.ld + t];
    if (pos < 0 || pos >= p.rotary_positions) return rnd<TT>(row[e]);
    const float c = table_at<TT>(p.cos_cache, pos * half + i, ax.table_f32);
    const float s = table_at<TT>(p.sin_cache, pos * half + i, ax.table_f32);
    const float o = row[p.rotary_interleaved ? off + (x ^ 1) : first ? e + half : e - half];
    return rnd<TT>(first ? rot_sub32(row[e], c, o, s) : rot_add32(row[e], c, o, s));
  };
  if (is_q) {
    const int64_t base = ((int64_t)t * p.num_heads + head) * D;
    for (int e = lane; e < D; e += 64) stv<TT>(p.q_out, base + e, value(e));
    return;
  }
  const int Dc = CK == kCacheI4 ? (D + 1) >> 1 : D;
  const int64_t base = (slot * p.kv_heads + head) * Dc;
  void* cache = is_v ? p.value_cache : p.key_cache;
  const float* sc = is_v ? p.v_scale : p.k_scale;
  if constexpr (CK == kCacheT) {
    for (int e = lane; e < D; e += 64) stv<TT>(cache, base + e, value(e));
  } else if constexpr (CK == kCacheFp8) {
    const float s8 = sc[slot / p.block_size * p.kv_heads + head];
    for (int e = lane; e < D; e += 64)
      reinterpret_cast<uint8_t*>(cache)[base + e] =
          s8 == 0.0f ? 0 : (uint8_t)f32_to_e4m3_sat(value(e) / s8);
  } else {
    const bool pc = (is_v ? p.v_quant : p.k_quant) == PA_QUANT_PER_CHANNEL;
    auto code = [&](int e) {
      constexpr float top = CK == kCacheI4 ? 7.0f : 127.0f;
      return int_code(value(e), sc[pc ? (int64_t)head * D + e : 0], false, -top - 1.0f, top);
    };
    uint8_t* dst = reinterpret_cast<uint8_t*>(cache) + base;
    for (int j = lane; j < Dc; j += 64) {
      if constexpr (CK == kCacheI4)
        dst[j] = (uint8_t)((code(2 * j) + 8) | ((2 * j + 1 < D ? code(2 * j + 1) + 8 : 8) << 4));
      else
        dst[j] = (uint8_t)(int8_t)code(j);
    }
  }
}

template <typename TT>
hipError_t launch_t(const AppendParams& p, const AxisParams& ax, pa_dtype cache_dtype,
                    hipStream_t s) {
  const dim3 grid(p.num_tokens, (p.num_heads + 2 * p.kv_heads + 3) / 4), block(256);
  switch (cache_dtype) {
    case PA_DTYPE_FP8_E4M3:
      hipLaunchKernelGGL((axes_append_kernel<TT, kCacheFp8>), grid, block, 0, s, p, ax);
      break;
    case PA_DTYPE_INT8:
      hipLaunchKernelGGL((axes_append_kernel<TT, kCacheI8>), grid, block, 0, s, p, ax);
      break;
    case PA_DTYPE_INT4:
      hipLaunchKernelGGL((axes_append_kernel<TT, kCacheI4>), grid, block, 0, s, p, ax);
      break;
    default:
      hipLaunchKernelGGL((axes_append_kernel<TT, kCacheT>), grid, block, 0, s, p, ax);
      break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_axes_append(const AppendParams& p, const AxisParams& ax, pa_dtype act,
                              pa_dtype cache_dtype, hipStream_t s) {
  if (p.head_dim > kAxesMaxDim || p.num_heads + 2 * p.kv_heads > 4 * 65535) return hipErrorInvalidValue;
  switch (act) {
    case PA_DTYPE_FLOAT16: return launch_t<TF16>(p, ax, cache_dtype, s);
    case PA_DTYPE_BFLOAT16: return launch_t<TBF16>(p, ax, cache_dtype, s);
    case PA_DTYPE_FLOAT32: return launch_t<TF32>(p, ax, cache_dtype, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
