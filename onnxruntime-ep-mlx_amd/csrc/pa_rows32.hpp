// pa_rows32.hpp — attention of drafted trees and of rows that are weighed over every type and head size up to 256 that
// pa_ranged.hpp does not take: fp32, fp8 / int8 / int4 pages, heads other than 64 / 96 / 128 / 256, caches at odd addresses.
//
// A wavefront keeps 32 rows (token, head of the group) of one sequence and kv-head; a workgroup (four wavefronts, or one
// where a sequence has no more than 32 rows) brings 32 keys and values at a time into LDS as fp32, each code widened and
// scaled as the VALU kernel does it, and both products run on fp32 matrix instructions, 32x32x2, as in pa_ranged.hpp
// transposed: S^T = K Q^T, whose lanes hold one row and 16 keys, and O^T = V^T P^T, which takes the probabilities as they
// lie.  So everything is fp32, as on the VALU kernel, whose partial rows and merge it shares (chunks of keys over
// the grid); but a key is read once for 32 or 128 rows, and a row's sums cross lanes once.
//
// Values that are not finite lie in LDS as zeros and are added for the rows that see them (rare).
//
// Bound, where a sequence has few rows, by the chain of a tile (rows into LDS, products, softmax: 7.6 us at head 128 with
// one wavefront per SIMD, its products 3.4; matrix units busy 27 % of the time); where it has many, by the fp32 products, 128
// of 64 cycles a tile and wavefront at head 128, which two wavefronts per SIMD keep busy 42 % of the time beside the softmax
// and the widening of keys.  8 sequences of 1568 - 5625 keys, 32 heads of 128 and 8 kv-heads, fp8 pages: one token each 103 us
// a call (about 490 on the VALU kernel; 244 with four elements a load and none ahead), trees of 32 nodes 270 (11400; 339 in one
// build with the other's registers); head 80 in bf16 96 (372) and 257 (9400); fp32 at head 64 63 (281) and 167 (6990).  Chunks
// half as long: 112 and 303.  A prompt of 2048 over fp8 pages 520.
#pragma once

#include "pa_cache_read.hpp"

namespace pa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float swap_half(float x) {  // lane l ^ 32's x
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// Elements d .. d + 3 of a cache row that begins at storage index `base`, widened (unscaled).
template <typename CT>
__device__ __forceinline__ f32x4 four(const void* c, int64_t base, int d) {
  f32x4 x;
  if constexpr (std::is_same<CT, TF32>::value) {
    __builtin_memcpy(&x, reinterpret_cast<const float*>(c) + base + d, 16);
  } else if constexpr (std::is_same<CT, Fp8Cache>::value) {
    uint32_t w;
    __builtin_memcpy(&w, reinterpret_cast<const uint8_t*>(c) + base + d, 4);
    x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  } else if constexpr (std::is_same<CT, I8Cache>::value) {
    uint32_t w;
    __builtin_memcpy(&w, reinterpret_cast<const int8_t*>(c) + base + d, 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)(int8_t)(w >> (8 * k));
  } else if constexpr (std::is_same<CT, I4Cache>::value) {
    uint16_t w;
    __builtin_memcpy(&w, reinterpret_cast<const uint8_t*>(c) + base + (d >> 1), 2);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)((int)((w >> (4 * k)) & 15) - 8);
  } else {
    uint16_t w[4];
    __builtin_memcpy(w, reinterpret_cast<const uint16_t*>(c) + base + d, 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = CT::to_f32(w[k]);
  }
  return x;
}

// Elements of 16 bytes of a cache row, and these widened (unscaled).
template <typename CT>
constexpr int kPiece = std::is_same<CT, TF32>::value                                             ? 4
                       : std::is_same<CT, TF16>::value || std::is_same<CT, TBF16>::value         ? 8
                       : std::is_same<CT, I4Cache>::value                                        ? 32
                                                                                                 : 16;
template <typename CT>
__device__ __forceinline__ void widen(u32x4 w, float (&x)[kPiece<CT>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<CT, TF32>::value) {
      const uint32_t u = w[i];  // (a copy: the cast of a vector's element takes the first one)
      x[i] = __builtin_bit_cast(float, u);
    } else if constexpr (std::is_same<CT, Fp8Cache>::value) {
      x[4 * i] = __builtin_amdgcn_cvt_f32_fp8(w[i], 0);
      x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(w[i], 1);
      x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(w[i], 2);
      x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(w[i], 3);
    } else if constexpr (std::is_same<CT, I8Cache>::value) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = (float)(int8_t)(w[i] >> (8 * k));
    } else if constexpr (std::is_same<CT, I4Cache>::value) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[8 * i + k] = (float)((int)((w[i] >> (4 * k)) & 15) - 8);
    } else {
      x[2 * i] = CT::to_f32((uint16_t)w[i]);
      x[2 * i + 1] = CT::to_f32((uint16_t)(w[i] >> 16));
    }
  }
}

// One side of a cache, of one kv-head.
template <typename CT>
struct Side {
  const void* cache;
  const float* scale;
  int64_t head;    // storage index of the head in a row
  int64_t row;     // storage units of a row
  int kh, kv, D;
  bool channel;
  // Elements d .. d + 3 (zeros from D on) of the row in slot `slot` of page `page`.
  __device__ __forceinline__ f32x4 load(int64_t slot, int64_t page, int d) const {
    const int64_t base = slot * row + head;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    const float one = std::is_same<CT, Fp8Cache>::value ? scale[page * kv + kh] : kIntCache<CT> && !channel ? scale[0] : 1.0f;
    if ((D & 3) == 0) {
      if (d < D) {
        x = four<CT>(cache, base, d);
        if (kIntCache<CT> && channel) {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] *= scale[kh * D + d + k];
        } else if (std::is_same<CT, Fp8Cache>::value || kIntCache<CT>) {
          x *= one;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < D) x[k] = CacheRead<CT>::at(cache, base, d + k, channel ? scale[kh * D + d + k] : one);
    }
    return x;
  }
};

// An element of the activations, of whatever type they are.
__device__ __forceinline__ float act_load(const void* x, int64_t i, int act) {
  if (act == PA_DTYPE_FLOAT32) return reinterpret_cast<const float*>(x)[i];
  const uint16_t u = reinterpret_cast<const uint16_t*>(x)[i];
  return act == PA_DTYPE_FLOAT16 ? f16_to_f32(u) : bf16_to_f32(u);
}
__device__ __forceinline__ void act_store(void* x, int64_t i, int act, float v) {
  if (act == PA_DTYPE_FLOAT32) reinterpret_cast<float*>(x)[i] = v;
  else reinterpret_cast<uint16_t*>(x)[i] = act == PA_DTYPE_FLOAT16 ? f32_to_f16_rne(v) : f32_to_bf16_rne(v);
}

template <typename CT, int DP, int NT>
__global__ __launch_bounds__(NT, DP <= 64 || (NT == 256 && DP <= 128) ? 2 : 1) void rows32_kernel(const AttnParams p, int row_blocks, int act) {
  constexpr int KP = DP + 4, VP = DP + 8, ND = DP / 32;  // pitches of a key's and a value's row in LDS
  __shared__ __attribute__((aligned(16))) float keys[32 * KP], values[32 * VP];
  __shared__ int odd, ends[8];
  __shared__ int2 slots[2][32];  // slot and page of a tile's keys, the next tile's beside it
  constexpr int WAVES = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  // chunks of different sequences side by side: 8 or 16 chunks of one would each go to an XCD of their own, the last of
  // which only the longest sequences have (trees of 32 nodes 282 us for 297 over int8, 259 for 265 at head 80)
  const int seqs = p.batch * p.kv_heads, rest = blockIdx.x / seqs, z = blockIdx.x - rest * seqs;
  const int split = rest / row_blocks, blk = rest - split * row_blocks, b = z / p.kv_heads, kh = z - b * p.kv_heads;
  const int g = p.num_heads / p.kv_heads, D = p.head_dim;
  const int cap = (int)min((int64_t)p.max_blocks * p.block_size, (int64_t)(INT32_MAX / 2));
  const int s0 = min(max(p.cum[b], 0), p.num_tokens);
  const int nq = min(min(max(p.cum[b + 1], s0), p.num_tokens) - s0, cap);
  const int past = min(max(p.past[b], 0), cap - nq), total = past + nq;
  const int64_t start64 = (int64_t)split * p.chunk;
  if (start64 >= total || (int64_t)blk * 32 * WAVES >= (int64_t)nq * g) return;
  // (the last chunk goes to the sequence's end: contexts beyond the call's bound)
  const int start = (int)start64, end = split == p.max_splits - 1 ? total : (int)min(start64 + p.chunk, (int64_t)total);
  const int r = blk * 32 * WAVES + 32 * wave + c;
  const bool valid = r < nq * g;
  const int qi = valid ? r / g : 0, t = s0 + qi, head = kh * g + (valid ? r - qi * g : 0);
  int hi = valid ? min(p.causal ? past + qi + 1 : total, end) : 0, lo = start;
  if (p.window > 0) lo = max(lo, past + qi - (p.tree_lag ? p.tree_lag[t] : 0) - p.window + 1);
  if (lo >= hi) lo = hi = 0;
  const bool any = lo < hi;
  // keys that some row of the workgroup sees
  int first = any ? lo : INT32_MAX, last = hi;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    first = min(first, __shfl_xor(first, o, 64));
    last = max(last, __shfl_xor(last, o, 64));
  }
  if (WAVES > 1) {
    if (lane == 0) {
      ends[2 * wave] = first;
      ends[2 * wave + 1] = last;
    }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) {
      first = min(first, ends[2 * w]);
      last = max(last, ends[2 * w + 1]);
    }
  }
  first = __builtin_amdgcn_readfirstlane(first);
  last = __builtin_amdgcn_readfirstlane(last);
  // dims h DP / 2 .. of the row's query (the order of a product's dims is free)
  float q[DP / 2];
  const int64_t row0 = ((int64_t)t * p.num_heads + head) * D;
  auto queries = [&](auto load) __attribute__((always_inline)) {  // (all loads in flight: no branch among them)
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) q[s] = load(row0 + min(h * (DP / 2) + s, D - 1));
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) q[s] = h * (DP / 2) + s < D ? q[s] : 0.0f;
  };
  if (act == PA_DTYPE_FLOAT32)
    queries([&](int64_t i) { return reinterpret_cast<const float*>(p.q)[i]; });
  else if (act == PA_DTYPE_FLOAT16)
    queries([&](int64_t i) { return f16_to_f32(reinterpret_cast<const uint16_t*>(p.q)[i]); });
  else
    queries([&](int64_t i) { return bf16_to_f32(reinterpret_cast<const uint16_t*>(p.q)[i]); });
  f32x16 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.0f;
  float m = kNegInf, l = 0.0f;
  // the scores of rows that count, as in pa_ranged.hpp
  float* scores = p.scores && any && qi >= (p.observed > 0 ? nq - p.observed : 0)
                      ? p.scores + stat_row(p, t, head) * p.score_ld
                      : nullptr;
  const int Dc = std::is_same<CT, I4Cache>::value ? (D + 1) >> 1 : D;
  const Side<CT> ks{p.key_cache, p.k_scale, (int64_t)kh * Dc, (int64_t)p.kv_heads * Dc, kh, p.kv_heads, D,
                    p.k_quant == PA_QUANT_PER_CHANNEL},
      vs{p.value_cache, p.v_scale, (int64_t)kh * Dc, (int64_t)p.kv_heads * Dc, kh, p.kv_heads, D,
         p.v_quant == PA_QUANT_PER_CHANNEL};
  // (keys that no row sees repeat the nearest that some do; a cache has less than 2^31 slots)
  auto place = [&](int t0) {
    const int pos = min(max(t0 + tid, first), last - 1), bi = pos / p.block_size;
    int page = p.block_table[(int64_t)b * p.max_blocks + min(bi, p.max_blocks - 1)];
    page = min(max(page, 0), (int)p.num_blocks - 1);
    return int2{page * p.block_size + (pos - bi * p.block_size), page};
  };
  const int begin = first & ~31;
  int buf = 0;
  // Rows of whole 16 bytes: a thread keeps to row tid % 32 of the tile and takes every NT / 32nd piece of it, R of a round
  // of keys and of values; the first round of a tile is on its way while the last tile is multiplied, the table's entry a
  // tile earlier.  Other rows: four elements at a time.
  constexpr int E = kPiece<CT>, stride = NT / 32, ALL = (DP / E + stride - 1) / stride, R = ALL < 4 ? ALL : 4;
  const int bytes = D * 16 / E, np = bytes / 16, own = tid & 31, piece0 = tid >> 5;
  const bool pieces = (D * 16) % (16 * E) == 0;
  u32x4 kr[R], vr[R];
  float kone = 1.0f, vone = 1.0f;
  auto place_own = [&](int t0) {
    const int pos = min(max(t0 + own, first), last - 1), bi = pos / p.block_size;
    int page = p.block_table[(int64_t)b * p.max_blocks + min(bi, p.max_blocks - 1)];
    page = min(max(page, 0), (int)p.num_blocks - 1);
    return int2{page * p.block_size + (pos - bi * p.block_size), page};
  };
  auto fetch = [&](int2 at, int r) {
    const int64_t row = ((int64_t)at.x * p.kv_heads + kh) * bytes;
    const char *kc = reinterpret_cast<const char*>(p.key_cache) + row, *vc = reinterpret_cast<const char*>(p.value_cache) + row;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if ((r * R + j) * stride >= np) break;
      const int piece = min((r * R + j) * stride + piece0, np - 1);
      __builtin_memcpy(&kr[j], kc + 16 * piece, 16);
      __builtin_memcpy(&vr[j], vc + 16 * piece, 16);
    }
    if (std::is_same<CT, Fp8Cache>::value && r == 0) {
      kone = p.k_scale[(int64_t)at.y * p.kv_heads + kh];
      vone = p.v_scale[(int64_t)at.y * p.kv_heads + kh];
    }
  };
  if (kIntCache<CT>) {
    if (!ks.channel) kone = p.k_scale[0];
    if (!vs.channel) vone = p.v_scale[0];
  }
  auto stash = [&](int r) {  // whether a value is not finite
    bool strange = false;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int piece = (r * R + j) * stride + piece0;
      if (piece >= np) break;
      float x[E];
      auto scaled = [&](const Side<CT>& side, float one) {
        if (kIntCache<CT> && side.channel) {
#pragma unroll
          for (int k = 0; k < E; ++k) x[k] *= side.scale[kh * D + piece * E + k];
        } else if (kIntCache<CT> || std::is_same<CT, Fp8Cache>::value) {
#pragma unroll
          for (int k = 0; k < E; ++k) x[k] *= one;
        }
      };
      widen<CT>(kr[j], x);
      scaled(ks, kone);
#pragma unroll
      for (int k = 0; k < E; k += 4)
        *reinterpret_cast<f32x4*>(&keys[own * KP + piece * E + k]) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
      widen<CT>(vr[j], x);
      scaled(vs, vone);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (!(fabsf(x[k]) < -kNegInf)) {
          strange = true;
          x[k] = 0.0f;
        }
#pragma unroll
      for (int k = 0; k < E; k += 4)
        *reinterpret_cast<f32x4*>(&values[own * VP + piece * E + k]) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
    }
    return strange;
  };
  int2 at{0, 0}, ahead{0, 0};
  if (pieces) {
    for (int i = tid; i < 32 * (DP - D); i += NT) {
      const int kk = i / (DP - D), d = D + i - kk * (DP - D);
      keys[kk * KP + d] = values[kk * VP + d] = 0.0f;
    }
    if (begin < last) {
      at = place_own(begin);
      fetch(at, 0);
      ahead = place_own(begin + 32);
    }
  } else if (tid < 32 && begin < last) {
    slots[0][tid] = place(begin);
  }
  for (int t0 = begin; t0 < last; t0 += 32, buf ^= 1) {
    if (tid == 0) odd = 0;
    __syncthreads();  // the last tile's readers are done
    bool strange = false;
    constexpr int PER = DP / 4, N = 4;  // fours of a row; of a thread in flight
    if (pieces) {
      if (tid < 32) slots[buf][tid] = at;
      strange = stash(0);
#pragma unroll 1
      for (int r = 1; r * R * stride < np; ++r) {
        fetch(at, r);
        strange |= stash(r);
      }
    } else if (tid < 32 && t0 + 32 < last) {
      slots[buf ^ 1][tid] = place(t0 + 32);
    }
    for (int i0 = pieces ? 32 * PER : tid; i0 < 32 * PER; i0 += N * NT) {
      f32x4 kv[N], vv[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = min(i0 + j * NT, 32 * PER - 1), kk = i / PER;
        const int2 at = slots[buf][kk];
        kv[j] = ks.load(at.x, at.y, 4 * (i - kk * PER));
        vv[j] = vs.load(at.x, at.y, 4 * (i - kk * PER));
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = i0 + j * NT, kk = i / PER, d = 4 * (i - kk * PER);
        if (i >= 32 * PER) continue;
        *reinterpret_cast<f32x4*>(&keys[kk * KP + d]) = kv[j];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (!(fabsf(vv[j][k]) < -kNegInf)) {
            strange = true;
            vv[j][k] = 0.0f;
          }
        *reinterpret_cast<f32x4*>(&values[kk * VP + d]) = vv[j];
      }
    }
    if (strange) odd = 1;
    __syncthreads();
    if (pieces && t0 + 32 < last) {
      at = ahead;
      fetch(at, 0);
      ahead = place_own(t0 + 64);
    }
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&keys[c * KP + h * (DP / 2) + 4 * j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[k], q[4 * j + k], s, 0, 0, 0);
    }
    uint32_t bits = ~0u;
    if (p.tree_bits && t0 + 32 > past) bits = tree_window(p.tree_bits + (int64_t)t * p.tree_words, p.tree_words, t0 - past);
    bits >>= 4 * h;
    float mx = kNegInf;
    uint32_t seen = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = 8 * (i >> 2) + (i & 3), key = t0 + 4 * h + k;
      float x = s[i] * p.scale;
      if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
      const bool sees = key >= lo && key < hi && ((bits >> k) & 1u);
      seen |= sees ? 1u << i : 0u;
      s[i] = sees ? x * kLog2e : kNegInf;
      mx = fmaxf(mx, s[i]);
    }
    if (scores && t0 + 32 <= p.score_ld) {
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4*>(scores + t0 + 2 * i + 4 * h) = f32x4{s[i], s[i + 1], s[i + 2], s[i + 3]};
    }
    mx = fmaxf(mx, swap_half(mx));
    const float mn = fmaxf(m, mx), ms = mn == kNegInf ? 0.0f : mn;
    // (not below fp32's smallest, that infinite sums stay what they are)
    const float a = m == kNegInf ? 0.0f : fmaxf(exp2f(m - ms), 0x1p-126f);
    if (__any(mn != m)) {
      const float f = m == kNegInf ? 1.0f : a;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= f;
      l *= f;
    }
    m = mn;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2f(s[i] - ms);
      l += s[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float* row = &values[(8 * (i >> 2) + 4 * h + (i & 3)) * VP + c];
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(row[32 * n], s[i], o[n], 0, 0, 0);
    }
    if (odd) {
      // what is not finite, in the place of the keys
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < 32 * PER; i += NT) {
        const int kk = i / PER, d = 4 * (i - kk * PER);
        const int2 at = slots[buf][kk];
        f32x4 v = vs.load(at.x, at.y, d);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fabsf(v[k]) < -kNegInf ? 0.0f : v[k];
        *reinterpret_cast<f32x4*>(&keys[kk * KP + d]) = v;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // key 8 (i / 4) + 4 half + i % 4, whose weight that half of the wavefront holds
          const float mine = (seen >> i) & 1u ? fmaxf(s[i], 0x1p-126f) : 0.0f, other = swap_half(mine);
          const float w = half == h ? mine : other;
          const float* row = &keys[(8 * (i >> 2) + 4 * half + (i & 3)) * KP + 4 * h];
          if (w == 0.0f) continue;  // not seen
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[n][e] = __builtin_fmaf(row[32 * n + 8 * (e >> 2) + (e & 3)], w, o[n][e]);
        }
    }
  }
  l += swap_half(l);
  if (!valid) return;
  if (start == 0 && end == total) {
    const float sink = p.head_sink ? act_load(p.head_sink, head, act) * kLog2e : kNegInf, f = finalize_factor(m, l, sink);
    if (p.row_stats && h == 0) p.row_stats[stat_row(p, t, head)] = softmax_stat(m, l, sink);
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
        if (d < D) act_store(p.out, row0 + d, act, o[n][i] * f);
      }
  } else if (p.part_o) {
    const int64_t row = ((int64_t)t * p.num_heads + head) * p.max_splits + split;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
        if (d < D) p.part_o[row * D + d] = o[n][i];
      }
    if (h == 0) {
      p.part_ml[2 * row] = m;
      p.part_ml[2 * row + 1] = l;
    }
  }
}

template <typename CT>
hipError_t launch_head(const AttnParams& p, pa_dtype act, hipStream_t s) {
  const int64_t rows = (int64_t)p.max_query_len * (p.num_heads / p.kv_heads), z = (int64_t)p.batch * p.kv_heads;
  const int per = rows <= 32 ? 32 : 128;
  const int64_t blocks = (rows + per - 1) / per, all = blocks * z * p.max_splits;
  if (all > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)all);
  auto go = [&](auto dp, auto nt) {
    hipLaunchKernelGGL((rows32_kernel<CT, decltype(dp)::value, decltype(nt)::value>), grid, dim3(nt), 0, s, p, (int)blocks, act);
  };
  auto with = [&](auto nt) {
    if (p.head_dim <= 64) go(std::integral_constant<int, 64>{}, nt);
    else if (p.head_dim <= 128) go(std::integral_constant<int, 128>{}, nt);
    else go(std::integral_constant<int, 256>{}, nt);
  };
  if (per == 32) with(std::integral_constant<int, 64>{});
  else with(std::integral_constant<int, 256>{});
  return hipGetLastError();
}

}  // namespace
}  // namespace pa
