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
//
// What bounds it.  Scores: HBM; a step of 48 tokens, 32 heads, over 511 - 8190 keys writes and reads 27 MB of them, 31 - 33
// us more in the attention (194 for 162 without; its waits for keys count these stores, too) and 11.5 in fold_kernel.
// Columns: the exponentials' vector instructions beside the products, at two wavefronts per SIMD that overlap in part: 4095
// tokens after 600, 24 heads of 256 under a softcap, 133 GFLOP of products in 200 - 212 us (three transcendental
// instructions a score; vector and matrix units busy 53 and 27 % of the time); without LDS and a tile's lead 467.  Other types
// and heads up to 256: pa_weigh32.hip.  The last 32 rows of prompts of 3001 - 5001: 14.
#include "pa_cache_read.hpp"
#include "pa_weigh.hpp"

namespace pa {
namespace {

constexpr int kWKeys = 64;             // keys of a wavefront
constexpr int kWBlock = 4 * kWKeys;    // of a workgroup

// Forms of a score: as it is; under a softcap as a quotient, whose constant the exponent takes along, up to
// kCapNear, and beyond it by tanh to its own bits -- the attention's own arithmetic (r_softmax), so that what the two
// round alike cancels between a score and its row's constant.
enum WForm { kWPlain = 0, kWNear = 1, kWFar = 2 };
template <int FORM>
__device__ __forceinline__ float w_raw(float s, float ck) {
  if constexpr (FORM == kWNear) return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s * ck));
  if constexpr (FORM == kWFar) return half_tanh(s * ck);
  return s;
}

// Query rows in tiles of 32, which the workgroup's wavefronts share in LDS, two of them: the next one arrives while
// one is multiplied.  Blocks of keys over the same chunk of rows follow each other on one XCD, whose L2 then holds
// the rows.
template <typename TT, int D, int FORM>
__global__ __launch_bounds__(256, 2) void weigh_columns_kernel(const WeighParams wp) {
  using G = RGeom<D>;
  constexpr int TILE = 32 * G::PITCH, NI = 8 / G::RPI;  // bytes of a tile; loads of a wavefront's eight rows
  __shared__ __attribute__((aligned(1024))) char lds[2 * TILE];
  __shared__ __attribute__((aligned(16))) float consts[2][32];
  const RangedParams& p = wp.r;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int blocks = (wp.max_keys + kWBlock - 1) / kWBlock, seqs = p.batch * p.kv_heads;
  const int turn = blockIdx.x >> 3, group = (turn / blocks) * 8 + (blockIdx.x & 7);
  if (group >= seqs * wp.chunks) return;
  const int chunk = group / seqs, z = group - chunk * seqs, kb0 = (turn % blocks) * kWBlock;
  const int b = z / p.kv_heads, kh = z - b * p.kv_heads, g = p.num_heads / p.kv_heads;
  const RSeq e = r_seq(p, b);
  if (kb0 >= e.total) return;
  const int k0 = kb0 + wave * kWKeys;
  const int first = p.observed > 0 ? max(e.nq - p.observed, 0) * g : 0;
  const int64_t from = (int64_t)first + (int64_t)chunk * wp.chunk_rows;
  const int rb = (int)min(from, (int64_t)e.nq * g), re = (int)min(from + wp.chunk_rows, (int64_t)e.nq * g);
  // rows that some key of the workgroup counts, those that some and that all keys of the wavefront do
  const int last = min(kb0 + kWBlock, e.total) - 1;
  const int wg_lo = max(p.causal ? max(kb0 - e.past, 0) * g : 0, rb);
  const int wg_hi = p.window > 0 ? (int)min((int64_t)re, max((int64_t)last - e.past + p.window, (int64_t)0) * g) : re;
  WRows rows[2];
  int some_lo = INT32_MAX, some_hi = 0, all_lo = 0, all_hi = INT32_MAX;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    rows[kb] = key_rows(p, e, k0 + 32 * kb + c);
    some_lo = min(some_lo, rows[kb].lo);
    some_hi = max(some_hi, rows[kb].hi);
    all_lo = max(all_lo, rows[kb].lo);
    all_hi = min(all_hi, rows[kb].hi);
    rows[kb].hi = min(rows[kb].hi, re);
  }
  some_lo = half_min(some_lo);
  some_hi = half_max(some_hi);
  all_lo = half_max(all_lo);
  all_hi = min(half_min(all_hi), re);
  float acc[2] = {0.0f, 0.0f};
  if (wg_lo < wg_hi) {
    u32x4 k[2][D / 16];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const char* src = reinterpret_cast<const char*>(p.key_cache) +
                        (r_offset(p, b, kh, min(k0 + 32 * kb + c, e.total - 1), D) + 8 * h) * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) k[kb][ks] = ld16(src + 32 * ks) ^ p.qxor;
    }
    const float* stats = p.row_stats + ((int64_t)kh * p.num_tokens + e.s0) * g;
    const char* q0 = reinterpret_cast<const char*>(p.q) + ((int64_t)e.s0 * p.num_heads + kh * g) * D * 2;
    const uint32_t base = lds_address(lds) + wave * 8 * G::PITCH;
    // This lane's rows of the tile to be loaded next: token and head of the group, moved on by 32 rows a tile (a division
    // for each instead was a quarter of the loop's vector instructions); rows behind the last one repeat it.
    int tok[NI], head[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = wg_lo + wave * 8 + i * G::RPI + lane / G::CPR;
      tok[i] = r / g;
      head[i] = r - tok[i] * g;
    }
    const int dt = 32 / g, dh = 32 - dt * g, last_t = (wg_hi - 1) / g, last_h = wg_hi - 1 - last_t * g;
    const uint32_t row_bytes = D * 2, tok_bytes = (uint32_t)p.num_heads * row_bytes;
    auto load = [&](int buf) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int piece = (lane % G::CPR) ^ G::kx(wave * 8 + i * G::RPI + lane / G::CPR);
        if (D == 96 && piece >= 12) piece -= 8;
        const bool behind = tok[i] > last_t || (tok[i] == last_t && head[i] > last_h);
        const uint32_t t = behind ? last_t : tok[i], hd = behind ? last_h : head[i];
        dma_ptr(q0 + ((uint64_t)t * tok_bytes + hd * row_bytes + 16 * piece), base + buf * TILE + 1024 * i);
        tok[i] += dt;
        head[i] += dh;
        if (head[i] >= g) {
          head[i] -= g;
          ++tok[i];
        }
      }
    };
    const float sl = FORM == kWPlain ? p.scale_log2 : 2.0f * kLog2e * p.softcap;
    const float off = FORM == kWNear ? kLog2e * p.softcap : 0.0f;
    const float ck = FORM == kWPlain ? 0.0f : 2.0f * p.scale_log2 / p.softcap;
    if (threadIdx.x < 32) consts[0][threadIdx.x] = off - stats[min(wg_lo + (int)threadIdx.x, wg_hi - 1)];
    load(0);
    int buf = 0;
    for (int r0 = wg_lo; r0 < wg_hi; r0 += 32, buf ^= 1) {
      wait_loads<0>();
      wait_lds_reads();
      barrier();
      const bool more = r0 + 32 < wg_hi;
      float next = 0.0f;
      if (more) {
        if (threadIdx.x < 32) next = stats[min(r0 + 32 + (int)threadIdx.x, wg_hi - 1)];
        load(buf ^ 1);
      }
      if (r0 < some_hi && r0 + 32 > some_lo) {
        const char* row = lds + buf * TILE + c * G::PITCH;
        const int x = G::kx(c) ^ h;
        f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
        constexpr int A = D / 16 % 4 ? 3 : 4;  // operands read a group of products ahead
        u32x4 a[2][A];
        auto read = [&](int gi) {
#pragma unroll
          for (int i = 0; i < A; ++i)
            a[gi & 1][i] = *reinterpret_cast<const u32x4*>(row + (((2 * (gi * A + i)) ^ x) << 4));
        };
        read(0);
#pragma unroll
        for (int gi = 0; gi < D / 16 / A; ++gi) {
          if (gi + 1 < D / 16 / A) read(gi + 1);
          r_order();
#pragma unroll
          for (int i = 0; i < A; ++i)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] = mfma_r<TT>(a[gi & 1][i], k[kb][gi * A + i], s[kb]);
          r_order();
        }
        f32x4 st[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) st[i] = *reinterpret_cast<const f32x4*>(&consts[buf][8 * i + 4 * h]);
        auto sum = [&](auto masked) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            f32x4 part = {0.0f, 0.0f, 0.0f, 0.0f};
            const int lo = rows[kb].lo - r0 - 4 * h, hi = rows[kb].hi - r0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(w_raw<FORM>(s[kb][i], ck), sl, st[i >> 2][i & 3]));
              const int r = 8 * (i >> 2) + (i & 3);
              part[i & 3] += !decltype(masked)::value || (r >= lo && r < hi) ? w : 0.0f;
            }
            acc[kb] += (part[0] + part[1]) + (part[2] + part[3]);
          }
        };
        if (r0 >= all_lo && r0 + 32 <= all_hi) sum(std::false_type{});
        else sum(std::true_type{});
      }
      if (more && threadIdx.x < 32) consts[buf ^ 1][threadIdx.x] = off - next;
    }
  }
  float* dst = wp.part + ((int64_t)chunk * seqs + z) * wp.part_ld;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const float sum = acc[kb] + half_swap(acc[kb]);
    const int key = k0 + 32 * kb + c;
    if (h == 0 && key < wp.part_ld) dst[key] = sum;
  }
}

// The same for heads beyond 256, of every type: 16 keys in LDS as fp32, 16 rows at a time.  Bound by LDS reads.
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
  // (the entries come in while the sums are made)
  const int64_t named = p.block_table[(int64_t)b * p.max_blocks + min(key / p.block_size, p.max_blocks - 1)];
  const int64_t page = min(max(named, (int64_t)0), p.num_blocks - 1);
  float* w = wp.weights + (page * p.kv_heads + kh) * p.block_size + key % p.block_size;
  float old[V];
  load(w, old);
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
    for (int r0 = lo; r0 < hi; r0 += 4) {  // (four rows in flight)
      float x[4][V], st[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t row = first + min(r0 + k, hi - 1);
        load(p.scores + row * p.score_ld + key, x[k]);
        st[k] = p.row_stats[row];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          sum[i] += r0 + k >= rows[i].lo && r0 + k < rows[i].hi ? __builtin_amdgcn_exp2f(x[k][i] - st[k]) : 0.0f;
    }
  } else {
    const float* part = wp.part + (int64_t)z * wp.part_ld + key;
    const int64_t step = (int64_t)p.batch * p.kv_heads * wp.part_ld;
    for (int c0 = 0; c0 < wp.chunks; c0 += 8) {  // (eight chunks in flight)
      float x[8][V];
#pragma unroll
      for (int k = 0; k < 8; ++k) load(part + min(c0 + k, wp.chunks - 1) * step, x[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += c0 + k < wp.chunks ? x[k][i] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = key + i < e.past ? old[i] + sum[i] : key + i < e.total ? sum[i] : old[i];
  if (page != named) return;  // no page: nobody's entries
  if constexpr (V == 4)
    *reinterpret_cast<f32x4*>(w) = f32x4{sum[0], sum[1], sum[2], sum[3]};
  else
    w[0] = sum[0];
}

template <typename TT, int D>
void launch_columns(const WeighParams& p, dim3 grid, hipStream_t s) {
  if (p.r.softcap > kCapNear)
    hipLaunchKernelGGL((weigh_columns_kernel<TT, D, kWFar>), grid, dim3(256), 0, s, p);
  else if (p.r.softcap > 0.0f)
    hipLaunchKernelGGL((weigh_columns_kernel<TT, D, kWNear>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((weigh_columns_kernel<TT, D, kWPlain>), grid, dim3(256), 0, s, p);
}
template <typename TT>
hipError_t launch_matrix(const WeighParams& p, hipStream_t s) {
  const int64_t groups = (int64_t)p.r.batch * p.r.kv_heads * p.chunks, blocks = (p.max_keys + kWBlock - 1) / kWBlock;
  const int64_t all = (groups + 7) / 8 * 8 * blocks;
  if (all > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)all);
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
    const dim3 grid((unsigned)((p.max_keys + 15) / 16 * z), p.chunks);
    hipError_t e;
    if (matrix)
      e = act == PA_DTYPE_FLOAT16 ? launch_matrix<TF16>(p, s) : launch_matrix<TBF16>(p, s);
    else if (r.head_dim <= 256)
      e = launch_weigh_columns32(p, act, cache_dtype, s);
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
