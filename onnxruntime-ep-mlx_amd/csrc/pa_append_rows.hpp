// pa_append_rows.hpp — row arithmetic and slot rules shared by the append kernels: rounding helpers,
// the cache slot of a position, the last-writer rule, integer codes, 16-bit pairs and the row norm's
// sum in its fixed order.  Contraction into FMA is off from here on to the end of the file that
// includes it: every product and sum of a row is rounded on its own.
#pragma once

#include "pa_device.hpp"

#pragma clang fp contract(off)

namespace pa {
namespace {

// gqa_rope_f32 terms: fp32 products and their sum or difference, each rounded on its own (the
// pragma above keeps them apart; the HIP __f*_rn helpers are compiled outside it, and their
// products and sums were fused -- down to one fp16 rounding of a*c - b*s through v_fma_mix).
__device__ __forceinline__ float rot_sub32(float a, float c, float b, float s) {
  const float x = a * c, y = b * s;
  return x - y;
}
__device__ __forceinline__ float rot_add32(float a, float c, float b, float s) {
  const float x = a * c, y = b * s;
  return x + y;
}

// a * b rounded to fp32 before anything else rounds it: without the barrier the compiler joins the
// product of a norm and its rounding to fp16 into one v_fma_mixlo_f16 here and there, whose single
// rounding differs from the two of the reference's graph about once in 25,000 elements.
__device__ __forceinline__ float mul32(float a, float b) {
  float x = a * b;
  asm("" : "+v"(x));
  return x;
}

template <typename TT>
__device__ __forceinline__ float ldv(const void* p, int64_t i) {
  return TT::to_f32(reinterpret_cast<const typename TT::raw*>(p)[i]);
}
template <typename TT>
__device__ __forceinline__ void stv(void* p, int64_t i, float v) {
  reinterpret_cast<typename TT::raw*>(p)[i] = TT::from_f32(v);
}
template <typename TT>
__device__ __forceinline__ float rnd(float v) {
  return TT::to_f32(TT::from_f32(v));
}

// Cache slot of logical position `logical` of sequence b; -1 when its block-table entry is
// out of range.
__device__ __forceinline__ int64_t slot_at(const AppendParams& p, int b, int64_t logical) {
  const int64_t bi = logical / p.block_size;
  if (bi < 0 || bi >= p.max_blocks) return -1;
  const int64_t blk = p.block_table[(int64_t)b * p.max_blocks + bi];
  if (blk < 0 || blk >= p.num_blocks) return -1;
  return blk * p.block_size + logical % p.block_size;
}


// Last-writer rule without a slot mapping: whether a later token writes `slot` (block blk =
// slot / bs, offset slot % bs) of token position `pos` in sequence b.  A later token u can only
// be a new position of sequence b (after pos) or of a later sequence whose block-table entry
// for u's block is blk, at offset slot % bs of that block -- so the workgroup scans the
// block-table entries that cover the new positions of sequences b.. (O(T / bs + B) per token)
// instead of every later token.  Called by the whole workgroup (256 threads).
__device__ bool later_block_dup(const AppendParams& p, int b, int64_t pos, int64_t slot) {
  constexpr int NT = 256;
  __shared__ int pre[NT + 1];   // prefix of block-entry counts over a chunk of sequences
  __shared__ int k0s[NT];       // first block index of each sequence's new positions
  __shared__ int64_t ps_s[NT];  // first new position (past, clamped at 0)
  __shared__ int n_s[NT];       // new-token count
  __shared__ int wsum[NT / 64];
  const int tid = threadIdx.x;
  const int64_t bs = p.block_size;
  const int64_t blk = slot / bs, off = slot % bs;
  bool dup = false;
  for (int base = b; base < p.batch; base += NT) {
    const int sq = base + tid;
    int k0 = 0, nk = 0, n = 0;
    int64_t ps = 0;
    if (sq < p.batch) {
      n = p.cum[sq + 1] - p.cum[sq];
      ps = (int64_t)max(p.past[sq], 0);
      if (n > 0) {
        const int64_t k1 = min((ps + n - 1) / bs, (int64_t)p.max_blocks - 1);
        k0 = (int)min(ps / bs, (int64_t)p.max_blocks);
        nk = k1 >= k0 ? (int)(k1 - k0 + 1) : 0;
      }
    }
    k0s[tid] = k0;
    ps_s[tid] = ps;
    n_s[tid] = n;
    // Inclusive scan of nk: wave scans, then the totals of the earlier wavefronts.
    int x = nk;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if ((tid & 63) >= o) x += y;
    }
    if ((tid & 63) == 63) wsum[tid >> 6] = x;
    __syncthreads();
    for (int w = 0; w < (tid >> 6); ++w) x += wsum[w];
    pre[tid + 1] = x;
    if (tid == 0) pre[0] = 0;
    __syncthreads();
    const int total = pre[NT];
    for (int j = tid; j < total; j += NT) {
      int lo = 0, hi = NT - 1;  // sequence i of entry j: pre[i] <= j < pre[i + 1]
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= j) lo = mid; else hi = mid - 1;
      }
      const int sq2 = base + lo;
      const int k = k0s[lo] + (j - pre[lo]);
      if ((int64_t)p.block_table[(int64_t)sq2 * p.max_blocks + k] == blk) {
        const int64_t pp = (int64_t)k * bs + off;
        if (pp >= ps_s[lo] && pp < ps_s[lo] + n_s[lo] && (sq2 > b || pp > pos)) dup = true;
      }
    }
    __syncthreads();  // the next chunk rewrites the tables
  }
  return __syncthreads_or(dup);
}

// Cache storage kinds of the append kernel.
enum CacheKind { kCacheT = 0, kCacheFp8 = 1, kCacheI8 = 2, kCacheI4 = 3 };

// Integer code of x (QuantizedCache::encode, kv_cache.rs:170-199): paged caches divide by the
// scale and store 0 for a zero scale; GroupQueryAttention caches multiply by the fp32
// reciprocal with a zero scale read as 1.  Then clip to the code range and round half to even
// (the clip bounds are integers, so clip-then-round equals round-then-clip).  NaN -> 0.
__device__ __forceinline__ int int_code(float x, float s, bool reciprocal, float lo, float hi) {
  float y;
  if (reciprocal) {
    const float r = 1.0f / (s == 0.0f ? 1.0f : s);
    y = x * r;
  } else {
    y = s == 0.0f ? 0.0f : x / s;
  }
  if (y != y) return 0;
  return (int)__builtin_rintf(fminf(fmaxf(y, lo), hi));
}

// Two elements of T in one word.  pack2 rounds to nearest even, as TT::from_f32 does (bf16: one
// v_cvt_pk_bf16_f32, equal to the integer rounding for every fp32 pattern, NaNs included).
template <typename TT>
struct Pair;
template <>
struct Pair<TF16> {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static float lo(uint32_t w) { return TF16::to_f32((uint16_t)w); }
  __device__ __forceinline__ static float hi(uint32_t w) { return TF16::to_f32((uint16_t)(w >> 16)); }
  __device__ __forceinline__ static uint32_t pack2(float a, float b) {
    return (uint32_t)TF16::from_f32(a) | ((uint32_t)TF16::from_f32(b) << 16);
  }
  // v c -+ w s, each operation rounded to fp16.  fp16 arithmetic gives the bits of an fp32
  // operation rounded to fp16: products of two fp16 values are exact in fp32, and a sum or
  // difference of two that falls near a rounding boundary of fp16 is exact there too.
  __device__ __forceinline__ static uint32_t rope(uint32_t v, uint32_t w, uint32_t c, uint32_t s,
                                                  bool first) {
    const f16x2 x = __builtin_bit_cast(f16x2, v) * __builtin_bit_cast(f16x2, c);
    const f16x2 y = __builtin_bit_cast(f16x2, w) * __builtin_bit_cast(f16x2, s);
    return __builtin_bit_cast(uint32_t, first ? x - y : x + y);
  }
};
template <>
struct Pair<TBF16> {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static float lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
  __device__ __forceinline__ static float hi(uint32_t w) {
    return __builtin_bit_cast(float, w & 0xffff0000u);
  }
  __device__ __forceinline__ static uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
  __device__ __forceinline__ static uint32_t rope(uint32_t v, uint32_t w, uint32_t c, uint32_t s,
                                                  bool first) {
    const uint32_t x = pack2(lo(v) * lo(c), hi(v) * hi(c));
    const uint32_t y = pack2(lo(w) * lo(s), hi(w) * hi(s));
    return first ? pack2(lo(x) - lo(y), hi(x) - hi(y)) : pack2(lo(x) + lo(y), hi(x) + hi(y));
  }
};
// x * inv rounded to T, times the weight, rounded to T (process_row's norm).
template <typename TT>
__device__ __forceinline__ uint32_t norm2(uint32_t x, float inv, uint32_t w) {
  using P = Pair<TT>;
  const uint32_t y = P::pack2(mul32(P::lo(x), inv), mul32(P::hi(x), inv));
  return P::pack2(P::lo(y) * P::lo(w), P::hi(y) * P::hi(w));
}

// Sum of squares of one row held as 8 elements per lane, RL lanes per row (RL = 8, 16 or 32, rows
// aligned to RL lanes), in the order of sum_squares: virtual lane v = e % 64 folds its elements
// e = v, v + 64, ... with fused multiply-adds -- lane group of 8 by lane group of 8, the running
// fold passed 8 lanes on -- then the XOR butterfly over virtual distances 32, 16, 8 (real lanes 4,
// 2, 1) and 4, 2, 1 (inside a lane).  Both partners of a butterfly pair add the same two values, so
// the sum has the same bits as sum_squares'.
template <int RL>
__device__ __forceinline__ float row_sum_squares(const float (&x)[8], int lane) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = __builtin_fmaf(x[i], x[i], 0.0f);
#pragma unroll
  for (int f = 1; f < RL / 8; ++f) {
    const bool mine = ((lane & (RL - 1)) >> 3) == f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float before = __shfl(a[i], (lane - 8) & 63, 64);
      if (mine) a[i] = __builtin_fmaf(x[i], x[i], before);
    }
  }
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += __shfl_xor(a[i], o, 64);
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < o) a[i] += a[i + o];
  return __shfl(a[0], lane | (RL - 1), 64);  // the last fold's lanes hold the whole row
}

}  // namespace
}  // namespace pa
