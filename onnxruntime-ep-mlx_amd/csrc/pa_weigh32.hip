// pa_weigh32.hip — the keys' accounts from scores made again (see pa_weigh.hip) for the types and heads of pa_rows32.hpp,
// in fp32 on matrix instructions, 32x32x2: a wavefront keeps 32 keys in registers, widened and scaled, a lane half a key,
// and walks over the query rows, 32 at a time in LDS for the workgroup's four.  A lane holds the scores of one key, made as the
// attention made them (the same products in the same order), so its sum crosses lanes once, at the end.
//
// Bound by the fp32 products, 64 of 64 cycles for 32 keys and rows at head 128, and what brings and widens keys for few rows: 32
// rows each of 8 sequences of 1568 - 5625 keys, 32 heads of 128 and 8 kv-heads, fp8 pages 119 us, matrix units busy 45 % of the time (365
// with the keys in LDS and no matrix instructions), fp32 at head 64 75 (283); all rows of a prompt of 2048 over fp8 pages 366.
#include "pa_rows32.hpp"
#include "pa_weigh.hpp"

namespace pa {
namespace {

template <typename CT, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void weigh_columns32_kernel(const WeighParams wp, int act) {
  constexpr int KP = DP + 4, BLOCK = 128;  // pitch of a row in LDS; keys of a workgroup
  __shared__ __attribute__((aligned(16))) float rows32[32 * KP];
  __shared__ __attribute__((aligned(16))) float consts[32];
  const RangedParams& p = wp.r;
  const int D = p.head_dim, g = p.num_heads / p.kv_heads, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, h = lane >> 5;
  const int blocks = (wp.max_keys + BLOCK - 1) / BLOCK, z = blockIdx.x / blocks, chunk = blockIdx.y;
  const int kb0 = (blockIdx.x - z * blocks) * BLOCK, b = z / p.kv_heads, kh = z - b * p.kv_heads;
  const RSeq e = r_seq(p, b);
  if (kb0 >= e.total) return;
  const int key = kb0 + 32 * wave + c;
  const int first = p.observed > 0 ? max(e.nq - p.observed, 0) * g : 0;
  const int64_t from = (int64_t)first + (int64_t)chunk * wp.chunk_rows;
  const int rb = (int)min(from, (int64_t)e.nq * g), re = (int)min(from + wp.chunk_rows, (int64_t)e.nq * g);
  // rows that some key of the workgroup counts, and of the wavefront
  const int last = min(kb0 + BLOCK, e.total) - 1;
  const int wg_lo = max(p.causal ? max(kb0 - e.past, 0) * g : 0, rb);
  const int wg_hi = p.window > 0 ? (int)min((int64_t)re, max((int64_t)last - e.past + p.window, (int64_t)0) * g) : re;
  WRows rows = key_rows(p, e, key);
  rows.hi = min(rows.hi, re);
  int some_lo = rows.lo, some_hi = rows.hi;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    some_lo = min(some_lo, __shfl_xor(some_lo, o, 64));
    some_hi = max(some_hi, __shfl_xor(some_hi, o, 64));
  }
  float acc = 0.0f;
  if (wg_lo < wg_hi) {
    const int Dc = std::is_same<CT, I4Cache>::value ? (D + 1) >> 1 : D;
    const Side<CT> ks{p.key_cache, wp.k_scale, (int64_t)kh * Dc, (int64_t)p.kv_heads * Dc, kh, p.kv_heads, D,
                      wp.k_quant == PA_QUANT_PER_CHANNEL};
    const int pos = min(key, e.total - 1), bi = pos / p.block_size;
    int64_t page = p.block_table[(int64_t)b * p.max_blocks + min(bi, p.max_blocks - 1)];
    page = min(max(page, (int64_t)0), p.num_blocks - 1);
    const int64_t slot = page * p.block_size + (pos - bi * p.block_size);
    // dims h DP / 2 .. of the lane's key (the order of a product's dims is free)
    f32x4 k[DP / 8];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) k[j] = ks.load(slot, page, h * (DP / 2) + 4 * j);
    const float* stats = p.row_stats + ((int64_t)kh * p.num_tokens + e.s0) * g;
    auto stage = [&](int r0, auto load) __attribute__((always_inline)) {
      constexpr int PER = DP / 4;
#pragma unroll 4
      for (int i = tid; i < 32 * PER; i += 256) {
        const int row = i / PER, d = 4 * (i - row * PER), r = min(r0 + row, wg_hi - 1), t = r / g;
        const int64_t base = ((int64_t)(e.s0 + t) * p.num_heads + kh * g + (r - t * g)) * D;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if ((D & 3) == 0) {
          if (d < D) x = load(base, d);
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (d + n < D) x[n] = act_load(p.q, base + d + n, act);
        }
        *reinterpret_cast<f32x4*>(&rows32[row * KP + d]) = x;
      }
    };
    for (int r0 = wg_lo; r0 < wg_hi; r0 += 32) {
      __syncthreads();  // the last tile's readers are done
      if (act == PA_DTYPE_FLOAT32) stage(r0, [&](int64_t base, int d) { return four<TF32>(p.q, base, d); });
      else if (act == PA_DTYPE_FLOAT16) stage(r0, [&](int64_t base, int d) { return four<TF16>(p.q, base, d); });
      else stage(r0, [&](int64_t base, int d) { return four<TBF16>(p.q, base, d); });
      if (tid < 32) consts[tid] = stats[min(r0 + tid, wg_hi - 1)];
      __syncthreads();
      if (r0 >= some_hi || r0 + 32 <= some_lo) continue;
      f32x16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < DP / 8; ++j) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(&rows32[c * KP + h * (DP / 2) + 4 * j]);
#pragma unroll
        for (int n = 0; n < 4; ++n) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[n], k[j][n], s, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i >> 2) + 4 * h + (i & 3);
        float x = s[i] * p.scale;
        if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
        const float w = exp2f(x * kLog2e - consts[r]);
        acc += r0 + r >= rows.lo && r0 + r < rows.hi ? w : 0.0f;
      }
    }
  }
  const float sum = acc + swap_half(acc);
  if (h == 0 && key < wp.part_ld) wp.part[((int64_t)chunk * p.batch * p.kv_heads + z) * wp.part_ld + key] = sum;
}

template <typename CT>
hipError_t launch_columns32(const WeighParams& p, pa_dtype act, hipStream_t s) {
  const int64_t wgs = (int64_t)p.r.batch * p.r.kv_heads * ((p.max_keys + 127) / 128);
  if (wgs > INT32_MAX || p.chunks > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs, p.chunks);
  if (p.r.head_dim <= 64) hipLaunchKernelGGL((weigh_columns32_kernel<CT, 64>), grid, dim3(256), 0, s, p, act);
  else if (p.r.head_dim <= 128) hipLaunchKernelGGL((weigh_columns32_kernel<CT, 128>), grid, dim3(256), 0, s, p, act);
  else hipLaunchKernelGGL((weigh_columns32_kernel<CT, 256>), grid, dim3(256), 0, s, p, act);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_weigh_columns32(const WeighParams& p, pa_dtype act, pa_dtype cache_dtype, hipStream_t s) {
  if (p.r.head_dim > 256) return hipErrorInvalidValue;
  switch (cache_dtype) {
    case PA_DTYPE_FP8_E4M3: return launch_columns32<Fp8Cache>(p, act, s);
    case PA_DTYPE_INT8: return launch_columns32<I8Cache>(p, act, s);
    case PA_DTYPE_INT4: return launch_columns32<I4Cache>(p, act, s);
    case PA_DTYPE_FLOAT16: return act == cache_dtype ? launch_columns32<TF16>(p, act, s) : hipErrorInvalidValue;
    case PA_DTYPE_BFLOAT16: return act == cache_dtype ? launch_columns32<TBF16>(p, act, s) : hipErrorInvalidValue;
    case PA_DTYPE_FLOAT32: return act == cache_dtype ? launch_columns32<TF32>(p, act, s) : hipErrorInvalidValue;
  }
  return hipErrorInvalidValue;
}

}  // namespace pa
