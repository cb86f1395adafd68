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

// Any element type, head size and alignment, and slots that may be shared: one workgroup of four
// wavefronts per token and four of its rows (queries, keys, values in turn), one row per wavefront, held in
// LDS in fp32.  Bound by its chain of loads and, on prompts, by a position and two table loads per element
// and the search for later writers: 6.3 us for one token of 32 and 8 heads of 128, 7.9 for 64 tokens of 24
// and 4 heads of 256 (axes_rows_kernel 5.4, 6.6), 323 for prompts that the other appends in 45.
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

// 16-bit activations, rows of whole 16-byte pieces and distinct slots (axes_rows_takes has the conditions): a
// head row lies in RL lanes, eight elements each (head 96: 12 of 16), and a wavefront walks `passes` groups of
// 64 / RL rows of one token -- its queries, keys and values in turn -- the next groups' rows in flight while one is
// turned and stored.  What depends on the token alone is fetched once per wavefront: the slot, the axes'
// positions and the lane's eight cosines and sines (F32T: from fp32 tables), one 16-byte piece of a table row per axis, of which every
// element keeps its own axis' (a piece may hold several: sections end anywhere, and axes may take turns).  The
// partner's piece comes from its lane.
// Bound by HBM on prompts (45 us where a copy of their bytes takes 33), by its chain of loads (cum -> table ->
// store, positions -> tables) on decode steps (5.4 us for one token, 6.6 for 64).
constexpr int kAxesDepth = 2;  // groups of rows in flight
template <typename TT, int CK, int RL, bool F32T>
__global__ __launch_bounds__(256) void axes_rows_kernel(const AppendParams p, const AxisParams ax, int slices,
                                                        int passes) {
  using raw = typename TT::raw;
  using P = Pair<TT>;
  const int lane = threadIdx.x & 63;
  const int wid = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = wid / slices, sl = wid - t * slices;
  if (t >= p.num_tokens) return;  // whole wavefront
  const int D = p.head_dim, off = p.rotary_offset, half = p.rotary_half;
  const int nq = p.num_heads, nqk = nq + p.kv_heads, nrows = nqk + p.kv_heads;
  const int e = 8 * (lane & (RL - 1)), x0 = e - off;  // the lane's elements of every row
  const bool mine = e < D, turns = mine && x0 >= 0 && x0 < 2 * half;
  const int pe = p.rotary_interleaved ? e : x0 < half ? e + half : e - half;  // partner piece
  struct Piece {
    int row;
    u32x4 x;
  };
  auto load = [&](int pass) __attribute__((always_inline)) {
    Piece c;
    c.row = (sl * passes + pass) * (64 / RL) + lane / RL;
    c.x = u32x4{0u, 0u, 0u, 0u};
    if (pass < passes && c.row < nrows && mine) {
      const raw* src = c.row < nq ? reinterpret_cast<const raw*>(p.query) + (int64_t)t * p.q_ld + c.row * D
                       : c.row < nqk
                           ? reinterpret_cast<const raw*>(p.key) + (int64_t)t * p.k_ld + (c.row - nq) * D
                           : reinterpret_cast<const raw*>(p.value) + (int64_t)t * p.v_ld + (c.row - nqk) * D;
      c.x = *reinterpret_cast<const u32x4*>(src + e);
    } else {
      c.row = INT32_MAX;
    }
    return c;
  };
  // The lane's frequencies: i0 .. (eight, or four of pairs side by side)
  const int i0 = p.rotary_interleaved ? x0 / 2 : x0 < half ? x0 : x0 - half;
  int64_t ids[PA_MAX_AXES];
#pragma unroll
  for (int a = 0; a < PA_MAX_AXES; ++a) {
    ids[a] = ax.positions[min(a, ax.axes - 1) * ax.ld + t];
    if (ids[a] >= p.rotary_positions) ids[a] = -1;
  }
  Piece ring[kAxesDepth];
#pragma unroll
  for (int i = 0; i < kAxesDepth; ++i) ring[i] = load(i);
  const SeqPos sp = seq_pos_of_token(p.cum, p.past, p.batch, t);
  if (t < p.cum[0] || t >= p.cum[p.batch]) return;  // of no sequence: left alone

  // An element comes out as inv * (x A + partner B): A = weight * cosine, B = -+ partner's weight * sine; unturned
  // ones (bit k of `still`) as inv * x * weight.
  float ca[8], sa[8];
  uint32_t still = 0xff;
  {
    int axis[8];
    int m = ax.interleaved ? i0 % ax.axes : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (ax.interleaved) {
        int bound = ax.bound[0];
#pragma unroll
        for (int a = 1; a < PA_MAX_AXES; ++a) bound = m == a ? ax.bound[a] : bound;
        axis[k] = i0 + k < bound ? m : 0;
        m = m + 1 == ax.axes ? 0 : m + 1;
      } else {
        axis[k] = ax.axis_of(i0 + k);
      }
      ca[k] = 1.0f;
      sa[k] = 0.0f;
    }
    const bool four = p.rotary_interleaved;
    // every axis' pieces in flight together (axes that are not there repeat the last)
    constexpr int W = F32T ? 8 : 4;
    uint32_t tc[PA_MAX_AXES][W], ts[PA_MAX_AXES][W];
#pragma unroll
    for (int a = 0; a < PA_MAX_AXES; ++a) {
      const int64_t at = (max(ids[a], (int64_t)0) * half + (turns ? i0 : 0)) * (F32T ? 4 : 2);
      const char* ct = reinterpret_cast<const char*>(p.cos_cache) + at;
      const char* st = reinterpret_cast<const char*>(p.sin_cache) + at;
      const int next = four ? 0 : F32T ? 16 : 8;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (F32T) {
          const u32x4 c = *reinterpret_cast<const u32x4*>(ct + j * next), x = *reinterpret_cast<const u32x4*>(st + j * next);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            tc[a][4 * j + k] = c[k];
            ts[a][4 * j + k] = x[k];
          }
        } else {
          const u32x2 c = *reinterpret_cast<const u32x2*>(ct + j * next), x = *reinterpret_cast<const u32x2*>(st + j * next);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            tc[a][2 * j + k] = c[k];
            ts[a][2 * j + k] = x[k];
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t c = tc[0][F32T ? k : k / 2], x = ts[0][F32T ? k : k / 2];
      int64_t id = ids[0];
#pragma unroll
      for (int a = 1; a < PA_MAX_AXES; ++a) {
        c = axis[k] == a ? tc[a][F32T ? k : k / 2] : c;
        x = axis[k] == a ? ts[a][F32T ? k : k / 2] : x;
        id = axis[k] == a ? ids[a] : id;
      }
      if (turns && id >= 0) {
        ca[k] = F32T ? __builtin_bit_cast(float, c) : (k & 1) ? P::hi(c) : P::lo(c);
        sa[k] = F32T ? __builtin_bit_cast(float, x) : (k & 1) ? P::hi(x) : P::lo(x);
        still &= ~(1u << k);
      }
    }
    if (four) {  // frequency k turns elements 2 k and 2 k + 1
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        ca[2 * k + 1] = ca[2 * k] = ca[k];
        sa[2 * k + 1] = sa[k];
        sa[2 * k] = -sa[k];
      }
      uint32_t two = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) two |= ((still >> k) & 1) * (3u << (2 * k));
      still = two;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) sa[k] = x0 < half ? -sa[k] : sa[k];
    }
  }
  // weights of queries and keys
  float qa[8], qb[8], ka[8], kb[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    qa[k] = ka[k] = ca[k];
    qb[k] = kb[k] = sa[k];
  }
  if (p.q_norm && mine) {
    const raw* nq_w = reinterpret_cast<const raw*>(p.q_norm);
    const raw* nk_w = reinterpret_cast<const raw*>(p.k_norm);
    const int pp = turns ? pe : e;
    const u32x4 g0 = *reinterpret_cast<const u32x4*>(nq_w + e), h0 = *reinterpret_cast<const u32x4*>(nq_w + pp);
    const u32x4 g1 = *reinterpret_cast<const u32x4*>(nk_w + e), h1 = *reinterpret_cast<const u32x4*>(nk_w + pp);
    const int sw = p.rotary_interleaved ? 1 : 0;  // (the partner of element k is then k ^ 1 of the same piece)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      auto el = [](const u32x4& v, int i) { return (i & 1) ? P::hi(v[i >> 1]) : P::lo(v[i >> 1]); };
      qa[k] *= el(g0, k);
      ka[k] *= el(g1, k);
      qb[k] *= sw ? el(h0, k ^ 1) : el(h0, k);
      kb[k] *= sw ? el(h1, k ^ 1) : el(h1, k);
    }
  }
  const bool plain = !turns && !p.q_norm;  // a copy
  const bool whole = __all(still == 0 || !turns);

  const int64_t pos = (int64_t)max(sp.past, 0) + (t - sp.start);
  int64_t slot = p.slot_mapping ? (int64_t)p.slot_mapping[t] : slot_at(p, sp.b, pos);
  if (slot >= p.num_blocks * p.block_size) slot = -1;
  constexpr int EB = CK == kCacheI4 ? 4 : CK == kCacheT ? 16 : 8;  // cache bytes per piece
  const int64_t blk = (CK == kCacheFp8 && slot >= 0) ? (int64_t)((uint32_t)slot / (uint32_t)p.block_size) : 0;

  const float rd = 1.0f / (float)D;
  const int partner = (lane & ~(RL - 1)) + (turns ? pe / 8 : 0);
  auto row_group = [&](const Piece& c) __attribute__((always_inline)) {
    const bool is_q = c.row < nq, is_v = c.row >= nqk;
    float v[8], w[8], inv = 1.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = P::lo(c.x[k]);
      v[2 * k + 1] = P::hi(c.x[k]);
    }
    if (p.rotary_interleaved) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = v[k ^ 1];
    } else {  // every lane takes part
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = __shfl(c.x[k], partner, 64);
        w[2 * k] = P::lo(x);
        w[2 * k + 1] = P::hi(x);
      }
    }
    if (p.q_norm) {  // every lane takes part in the exchanges
      float acc = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc = __builtin_fmaf(v[k], v[k], acc);
#pragma unroll
      for (int o = RL / 2; o >= 1; o >>= 1) acc += __shfl_xor(acc, o, 64);
      inv = __builtin_amdgcn_rsqf(__builtin_fmaf(acc, rd, p.norm_eps));  // (about one unit in the last place)
    }
    if (c.row >= nrows) return;
    if (turns && whole) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = inv * __builtin_fmaf(v[k], is_q ? qa[k] : ka[k], w[k] * (is_q ? qb[k] : kb[k]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float own = v[k] * (is_q ? qa[k] : ka[k]);
        v[k] = inv * (turns && !((still >> k) & 1) ? own + w[k] * (is_q ? qb[k] : kb[k]) : own);
      }
    }
    u32x4 y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = P::pack2(v[2 * k], v[2 * k + 1]);
    if (is_v || plain) y = c.x;
    if (is_q) {
      *reinterpret_cast<u32x4*>(reinterpret_cast<raw*>(p.q_out) + ((int64_t)t * p.num_heads + c.row) * D + e) = y;
      return;
    }
    if (slot < 0) return;
    const int kh = is_v ? c.row - nqk : c.row - nq;
    char* dst = reinterpret_cast<char*>(is_v ? p.value_cache : p.key_cache) +
                ((slot * p.kv_heads + kh) * (D / 8) + e / 8) * EB;
    if constexpr (CK == kCacheT) {
      *reinterpret_cast<u32x4*>(dst) = y;
    } else {
      const float* sc = is_v ? p.v_scale : p.k_scale;
      const bool pc = (is_v ? p.v_quant : p.k_quant) == PA_QUANT_PER_CHANNEL;
      uint32_t code[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = (k & 1) ? P::hi(y[k >> 1]) : P::lo(y[k >> 1]);
        if constexpr (CK == kCacheFp8) {
          const float s8 = sc[blk * p.kv_heads + kh];
          code[k] = s8 == 0.0f ? 0u : f32_to_e4m3_sat(f / s8);
        } else {
          constexpr float top = CK == kCacheI4 ? 7.0f : 127.0f;
          const int i = int_code(f, sc[pc ? (int64_t)kh * D + e + k : 0], false, -top - 1.0f, top);
          code[k] = CK == kCacheI4 ? (uint32_t)(i + 8) : (uint32_t)(uint8_t)(int8_t)i;
        }
      }
      if constexpr (CK == kCacheI4) {
        uint32_t o = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) o |= (code[2 * k] | (code[2 * k + 1] << 4)) << (8 * k);
        *reinterpret_cast<uint32_t*>(dst) = o;
      } else {
        u32x2 o = u32x2{0u, 0u};
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k >> 2] |= (code[k] & 0xffu) << (8 * (k & 3));
        *reinterpret_cast<u32x2*>(dst) = o;
      }
    }
  };
  for (int pass = 0; pass < passes; pass += kAxesDepth) {
#pragma unroll
    for (int i = 0; i < kAxesDepth; ++i) {
      const Piece c = ring[i];
      if (pass + i >= passes) break;
      ring[i] = load(pass + i + kAxesDepth);
      row_group(c);
    }
  }
}

// The calls that axes_rows_kernel takes: distinct slots by the caller's word, whole 16-byte pieces everywhere
// (head size, rotary range, row strides, every base address; code rows to their 8 or 4 bytes).
bool axes_rows_takes(const AppendParams& p, const AxisParams& ax, pa_dtype act, pa_dtype cache_dtype) {
  if (act != PA_DTYPE_FLOAT16 && act != PA_DTYPE_BFLOAT16) return false;
  if (!p.slots_distinct || p.head_dim % 8 != 0 || p.head_dim > 512) return false;
  if (p.rotary_offset % 8 != 0 || p.rotary_half % (p.rotary_interleaved ? 4 : 8) != 0) return false;
  const uintptr_t a16 = (uintptr_t)p.query | (uintptr_t)p.key | (uintptr_t)p.value | (uintptr_t)p.q_out |
                        (uintptr_t)p.cos_cache | (uintptr_t)p.sin_cache | (uintptr_t)p.q_norm |
                        (uintptr_t)p.k_norm | (uintptr_t)(p.q_ld * 2) | (uintptr_t)(p.k_ld * 2) |
                        (uintptr_t)(p.v_ld * 2);
  const uintptr_t ac = (uintptr_t)p.key_cache | (uintptr_t)p.value_cache;
  const uintptr_t cb = cache_dtype == act ? 15 : cache_dtype == PA_DTYPE_INT4 ? 3 : 7;
  return (a16 & 15) == 0 && (ac & cb) == 0;
}

constexpr int64_t kAxesWaves = 4096;
template <typename TT, int CK, int RL>
void launch_rows(const AppendParams& p, const AxisParams& ax, hipStream_t s) {
  const int64_t rows = (int64_t)p.num_heads + 2 * p.kv_heads;
  const int64_t per = (rows * RL + 63) / 64;  // passes per token
  // As many passes per wavefront as still leave about kAxesWaves wavefronts; every token takes one at least.
  const int64_t want = (kAxesWaves + p.num_tokens - 1) / p.num_tokens;
  const int passes = (int)std::max<int64_t>(per / want, 1);
  const int slices = (int)((per + passes - 1) / passes);
  const dim3 grid((unsigned)(((int64_t)p.num_tokens * slices + 3) / 4));
  if (ax.table_f32)
    hipLaunchKernelGGL((axes_rows_kernel<TT, CK, RL, true>), grid, dim3(256), 0, s, p, ax, slices, passes);
  else
    hipLaunchKernelGGL((axes_rows_kernel<TT, CK, RL, false>), grid, dim3(256), 0, s, p, ax, slices, passes);
}
template <typename TT, int CK>
void launch_rows_ck(const AppendParams& p, const AxisParams& ax, hipStream_t s) {
  if (p.head_dim <= 64) launch_rows<TT, CK, 8>(p, ax, s);
  else if (p.head_dim <= 128) launch_rows<TT, CK, 16>(p, ax, s);
  else if (p.head_dim <= 256) launch_rows<TT, CK, 32>(p, ax, s);
  else launch_rows<TT, CK, 64>(p, ax, s);
}
template <typename TT>
hipError_t launch_rows_t(const AppendParams& p, const AxisParams& ax, pa_dtype cache_dtype, hipStream_t s) {
  switch (cache_dtype) {
    case PA_DTYPE_FP8_E4M3: launch_rows_ck<TT, kCacheFp8>(p, ax, s); break;
    case PA_DTYPE_INT8: launch_rows_ck<TT, kCacheI8>(p, ax, s); break;
    case PA_DTYPE_INT4: launch_rows_ck<TT, kCacheI4>(p, ax, s); break;
    default: launch_rows_ck<TT, kCacheT>(p, ax, s); break;
  }
  return hipGetLastError();
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
  if (axes_rows_takes(p, ax, act, cache_dtype))
    return act == PA_DTYPE_FLOAT16 ? launch_rows_t<TF16>(p, ax, cache_dtype, s)
                                   : launch_rows_t<TBF16>(p, ax, cache_dtype, s);
  switch (act) {
    case PA_DTYPE_FLOAT16: return launch_t<TF16>(p, ax, cache_dtype, s);
    case PA_DTYPE_BFLOAT16: return launch_t<TBF16>(p, ax, cache_dtype, s);
    case PA_DTYPE_FLOAT32: return launch_t<TF32>(p, ax, cache_dtype, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
