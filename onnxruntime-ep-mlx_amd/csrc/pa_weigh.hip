// pa_weigh.hip — what the keys of a paged cache weighed: w[key] = (key < past ? w[key] : 0) + sum over the rows
// that count (the last `observed` tokens of the sequence, the heads of the key's kv-head) of p = 2^(x - c), x the
// row's score in log2 units and c the constant of its softmax, which the attention left (row_stats).
//
// Few rows per sequence (decode): the attention left the scores, 4 bytes a row and key beside the 512 bytes of
// keys and values that it read for them, and fold_kernel sums them up.  Many rows: weigh_columns_kernel makes the
// scores again, key-stationary: a wavefront keeps 64 keys in registers (the B operand of 32x32x16 tiles) and walks
// over the query rows, so that a lane holds one key, its sum stays in a register and no sum crosses lanes or
// workgroups but for the fixed order of the chunks of rows, which fold_kernel adds.  Nothing is atomic: the same
// call gives the same bits.
#include "pa_cache_read.hpp"
#include "pa_ranged.hpp"

namespace pa {
namespace {

constexpr int kWKeys = 64;             // keys of a wavefront
constexpr int kWBlock = 4 * kWKeys;    // of a workgroup

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

// Score in log2 units of a raw product.
template <bool CAP>
__device__ __forceinline__ float w_score(float s, float sl, float ck) {
  return CAP ? half_tanh(s * ck) * sl : s * sl;
}

template <typename TT, int D, bool CAP>
__global__ __launch_bounds__(256) void weigh_columns_kernel(const WeighParams wp) {
  const RangedParams& p = wp.r;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int blocks = (wp.max_keys + kWBlock - 1) / kWBlock, z = blockIdx.x / blocks;
  const int kb0 = (blockIdx.x - z * blocks) * kWBlock, chunk = blockIdx.y;
  const int b = z / p.kv_heads, kh = z - b * p.kv_heads, g = p.num_heads / p.kv_heads;
  const RSeq e = r_seq(p, b);
  const int k0 = kb0 + wave * kWKeys;
  if (k0 >= e.total) return;
  const int first = p.observed > 0 ? max(e.nq - p.observed, 0) * g : 0;
  const int64_t from = (int64_t)first + (int64_t)chunk * wp.chunk_rows;
  const int rb = (int)min(from, (int64_t)e.nq * g), re = (int)min(from + wp.chunk_rows, (int64_t)e.nq * g);
  float acc[2] = {0.0f, 0.0f};
  WRows rows[2];
  int some_lo = INT32_MAX, some_hi = 0, all_lo = 0, all_hi = INT32_MAX;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    rows[kb] = key_rows(p, e, k0 + 32 * kb + c);
    some_lo = min(some_lo, rows[kb].lo);
    some_hi = max(some_hi, rows[kb].hi);
    all_lo = max(all_lo, rows[kb].lo);
    all_hi = min(all_hi, rows[kb].hi);
  }
  some_lo = max(half_min(some_lo), rb);
  some_hi = min(half_max(some_hi), re);
  all_lo = half_max(all_lo);
  all_hi = min(half_min(all_hi), re);
  if (some_lo < some_hi) {
    u32x4 k[2][D / 16];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const char* src = reinterpret_cast<const char*>(p.key_cache) +
                        (r_offset(p, b, kh, min(k0 + 32 * kb + c, e.total - 1), D) + 8 * h) * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) k[kb][ks] = ld16(src + 32 * ks);
    }
    const float* stats = p.row_stats + ((int64_t)kh * p.num_tokens + e.s0) * g;
    const float sl = CAP ? 2.0f * kLog2e * p.softcap : p.scale_log2, ck = CAP ? 2.0f * p.scale_log2 / p.softcap : 0.0f;
    for (int r0 = some_lo; r0 < some_hi; r0 += 32) {
      const int row = min(r0 + c, some_hi - 1), t = row / g;
      const char* src = reinterpret_cast<const char*>(p.q) +
                        (((int64_t)(e.s0 + t) * p.num_heads + kh * g + (row - t * g)) * D + 8 * h) * 2;
      f32x4 st[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) st[i][j] = stats[min(r0 + 8 * i + 4 * h + j, some_hi - 1)];
      f32x16 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const u32x4 a = ld16(src + 32 * ks) ^ p.qxor;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) s[kb] = mfma_r<TT>(a, k[kb][ks], s[kb]);
      }
      const bool whole = r0 >= all_lo && r0 + 32 <= all_hi;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __builtin_amdgcn_exp2f(w_score<CAP>(s[kb][i], sl, ck) - st[i >> 2][i & 3]);
          const int r = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
          acc[kb] += whole || (r >= rows[kb].lo && r < min(rows[kb].hi, re)) ? x : 0.0f;
        }
    }
  }
  float* dst = wp.part + ((int64_t)chunk * p.batch * p.kv_heads + z) * wp.part_ld;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const float sum = acc[kb] + half_swap(acc[kb]);
    const int key = k0 + 32 * kb + c;
    if (h == 0 && key < wp.part_ld) dst[key] = sum;
  }
}

// The same for every type and head size: 16 keys in LDS as fp32, 16 rows at a time.  Bound by LDS reads.
template <typename TT, typename CT>
__global__ __launch_bounds__(256) void weigh_columns_valu_kernel(const WeighParams wp) {
  constexpr int KB = 16;
  extern __shared__ float keys[];  // [KB][D + 1]
  __shared__ float sums[16][KB];
  const RangedParams& p = wp.r;
  const int D = p.head_dim, Dc = std::is_same<CT, I4Cache>::value ? (D + 1) >> 1 : D;
  const int blocks = (wp.max_keys + KB - 1) / KB, z = blockIdx.x / blocks;
  const int k0 = (blockIdx.x - z * blocks) * KB, chunk = blockIdx.y;
  const int b = z / p.kv_heads, kh = z - b * p.kv_heads, g = p.num_heads / p.kv_heads;
  const RSeq e = r_seq(p, b);
  if (k0 >= e.total) return;
  for (int i = threadIdx.x; i < KB * D; i += 256) {
    const int kk = i / D, d = i - kk * D, pos = min(k0 + kk, e.total - 1);
    int64_t page = p.block_table[(int64_t)b * p.max_blocks + min(pos / p.block_size, p.max_blocks - 1)];
    page = min(max(page, (int64_t)0), p.num_blocks - 1);
    const float ks = std::is_same<CT, Fp8Cache>::value ? wp.k_scale[page * p.kv_heads + kh]
                     : kIntCache<CT> ? wp.k_scale[wp.k_quant == PA_QUANT_PER_CHANNEL ? (int64_t)kh * D + d : 0]
                                     : 1.0f;
    const int64_t base = ((page * p.block_size + pos % p.block_size) * p.kv_heads + kh) * Dc;
    keys[kk * (D + 1) + d] = CacheRead<CT>::at(p.key_cache, base, d, ks);
  }
  __syncthreads();
  const int kk = threadIdx.x & (KB - 1), rl = threadIdx.x / KB;
  const int first = p.observed > 0 ? max(e.nq - p.observed, 0) * g : 0;
  const int64_t from = (int64_t)first + (int64_t)chunk * wp.chunk_rows;
  const WRows rows = key_rows(p, e, k0 + kk);
  const int re = (int)min(min(from + wp.chunk_rows, (int64_t)e.nq * g), (int64_t)rows.hi);
  const float* stats = p.row_stats + ((int64_t)kh * p.num_tokens + e.s0) * g;
  float acc = 0.0f;
  for (int64_t r = from + rl; r < re; r += 16) {
    if (r < rows.lo) continue;
    const int t = (int)(r / g);
    const typename TT::raw* q = reinterpret_cast<const typename TT::raw*>(p.q) +
                                ((int64_t)(e.s0 + t) * p.num_heads + kh * g + (int)(r - (int64_t)t * g)) * D;
    float x = 0.0f;
    for (int d = 0; d < D; ++d) x = __builtin_fmaf(TT::to_f32(q[d]), keys[kk * (D + 1) + d], x);
    x *= p.scale;
    if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
    acc += exp2f(x * kLog2e - stats[r]);
  }
  sums[rl][kk] = acc;
  __syncthreads();
  if (threadIdx.x < KB && k0 + kk < wp.part_ld) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += sums[i][kk];
    wp.part[((int64_t)chunk * p.batch * p.kv_heads + z) * wp.part_ld + k0 + kk] = sum;
  }
}

// The sums into the account, V keys per thread (four where pages hold a multiple of four).
template <int V>
__global__ __launch_bounds__(256) void fold_kernel(const WeighParams wp) {
  const RangedParams& p = wp.r;
  const int blocks = (wp.max_keys + 256 * V - 1) / (256 * V), z = blockIdx.x / blocks;
  const int b = z / p.kv_heads, kh = z - b * p.kv_heads, g = p.num_heads / p.kv_heads;
  const RSeq e = r_seq(p, b);
  const int64_t at = ((int64_t)(blockIdx.x - z * blocks) * 256 + threadIdx.x) * V;
  if (e.nq == 0 || at >= e.total || at + V > (p.scores ? p.score_ld : wp.part_ld)) return;
  const int key = (int)at;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  auto load = [&](const float* src, float (&x)[V]) {
    if constexpr (V == 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else {
      x[0] = src[0];
    }
  };
  if (p.scores) {
    WRows rows[V];
    int lo = INT32_MAX, hi = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      rows[i] = key_rows(p, e, key + i);
      lo = min(lo, rows[i].lo);
      hi = max(hi, rows[i].hi);
    }
    const int64_t first = ((int64_t)kh * p.num_tokens + e.s0) * g;
    for (int r = lo; r < hi; ++r) {
      float x[V];
      load(p.scores + (first + r) * p.score_ld + key, x);
      const float st = p.row_stats[first + r];
#pragma unroll
      for (int i = 0; i < V; ++i)
        sum[i] += r >= rows[i].lo && r < rows[i].hi ? __builtin_amdgcn_exp2f(x[i] - st) : 0.0f;
    }
  } else {
    for (int ch = 0; ch < wp.chunks; ++ch) {
      float x[V];
      load(wp.part + ((int64_t)ch * p.batch * p.kv_heads + z) * wp.part_ld + key, x);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += x[i];
    }
  }
  int64_t page = p.block_table[(int64_t)b * p.max_blocks + min(key / p.block_size, p.max_blocks - 1)];
  page = min(max(page, (int64_t)0), p.num_blocks - 1);
  float* w = wp.weights + (page * p.kv_heads + kh) * p.block_size + key % p.block_size;
  float old[V];
  load(w, old);
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = key + i < e.past ? old[i] + sum[i] : key + i < e.total ? sum[i] : old[i];
  if constexpr (V == 4)
    *reinterpret_cast<f32x4*>(w) = f32x4{sum[0], sum[1], sum[2], sum[3]};
  else
    w[0] = sum[0];
}

template <typename TT, int D>
void launch_columns(const WeighParams& p, dim3 grid, hipStream_t s) {
  if (p.r.softcap > 0.0f)
    hipLaunchKernelGGL((weigh_columns_kernel<TT, D, true>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((weigh_columns_kernel<TT, D, false>), grid, dim3(256), 0, s, p);
}
template <typename TT>
hipError_t launch_matrix(const WeighParams& p, dim3 grid, hipStream_t s) {
  switch (p.r.head_dim) {
    case 64: launch_columns<TT, 64>(p, grid, s); break;
    case 96: launch_columns<TT, 96>(p, grid, s); break;
    case 128: launch_columns<TT, 128>(p, grid, s); break;
    case 256: launch_columns<TT, 256>(p, grid, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}
template <typename TT>
hipError_t launch_valu(const WeighParams& p, pa_dtype cache_dtype, dim3 grid, hipStream_t s) {
  const size_t lds = (size_t)16 * (p.r.head_dim + 1) * sizeof(float);
  switch (cache_dtype) {
    case PA_DTYPE_FP8_E4M3: hipLaunchKernelGGL((weigh_columns_valu_kernel<TT, Fp8Cache>), grid, dim3(256), lds, s, p); break;
    case PA_DTYPE_INT8: hipLaunchKernelGGL((weigh_columns_valu_kernel<TT, I8Cache>), grid, dim3(256), lds, s, p); break;
    case PA_DTYPE_INT4: hipLaunchKernelGGL((weigh_columns_valu_kernel<TT, I4Cache>), grid, dim3(256), lds, s, p); break;
    default:
      if (cache_dtype != TT::code) return hipErrorInvalidValue;
      hipLaunchKernelGGL((weigh_columns_valu_kernel<TT, TT>), grid, dim3(256), lds, s, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_weigh(const WeighParams& p, pa_dtype act, pa_dtype cache_dtype, hipStream_t s) {
  const RangedParams& r = p.r;
  if (r.num_tokens <= 0 || r.batch <= 0) return hipSuccess;
  const int64_t z = (int64_t)r.batch * r.kv_heads;
  if (!r.row_stats || !p.weights || (!r.scores && (!p.part || p.chunks < 1 || p.chunks > 65535)) ||
      z * ((p.max_keys + 15) / 16) > INT32_MAX)
    return hipErrorInvalidValue;
  if (!r.scores) {
    const bool matrix = ranged_supported(r.head_dim, act, cache_dtype) && r.slots > 0;
    const int keys = matrix ? kWBlock : 16;
    const dim3 grid((unsigned)((p.max_keys + keys - 1) / keys * z), p.chunks);
    hipError_t e;
    if (matrix)
      e = act == PA_DTYPE_FLOAT16 ? launch_matrix<TF16>(p, grid, s) : launch_matrix<TBF16>(p, grid, s);
    else
      e = act == PA_DTYPE_FLOAT16    ? launch_valu<TF16>(p, cache_dtype, grid, s)
          : act == PA_DTYPE_BFLOAT16 ? launch_valu<TBF16>(p, cache_dtype, grid, s)
                                     : launch_valu<TF32>(p, cache_dtype, grid, s);
    if (e != hipSuccess) return e;
  }
  const bool four = r.block_size % 4 == 0 && (reinterpret_cast<uintptr_t>(p.weights) & 15) == 0;
  const unsigned per = four ? 1024 : 256;
  const dim3 grid((unsigned)((p.max_keys + per - 1) / per * z));
  if (four)
    hipLaunchKernelGGL((fold_kernel<4>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((fold_kernel<1>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace pa
