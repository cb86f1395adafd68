// pa_upkeep.hip — rows that move within the pages of a cache: those of a drafted tree's accepted path, and those
// that eviction leaves.
//
// Both write row i from row kept[i], kept rising (kept[i] >= i), in the same pages.  Read in rising order, a row
// that is overwritten has been read: rows below i have passed, and of the rows from i on only those of the same
// round are read before the round is written.
//
// Accepting moves a few whole tokens of every sequence: a thread keeps to its 16 bytes of the token's row and takes
// the rows in turn, eight loads in flight.  Evicting moves thousands of rows of single kv-heads, which stay by
// different positions: the bytes of a head's row are independent of each other, so a workgroup takes 64 of them (of
// keys or of values), or all of them where the heads are many, for all rows, hundreds per round with a barrier between
// its loads and its stores; to other pages no round waits for another.
#include <algorithm>

#include "pa_device.hpp"

namespace pa {
namespace {

// U bytes that move at once.
template <int U>
struct Unit;
template <>
struct Unit<16> {
  typedef u32x4 type;
};
template <>
struct Unit<4> {
  typedef uint32_t type;
};
template <>
struct Unit<1> {
  typedef uint8_t type;
};

// Slot (page * block_size + row) of position pos of sequence b, and its page.  A table's entry that names no page reads
// the nearest one and writes nothing.
struct Slot {
  int64_t slot;
  int64_t page;
  bool there;
};
__device__ __forceinline__ Slot slot_of(const RowsParams& c, const int32_t* table, int max_blocks, int b, int pos) {
  const int bi = c.bs_shift >= 0 ? pos >> c.bs_shift : pos / c.block_size;
  const int64_t named = table[(int64_t)b * max_blocks + min(bi, max_blocks - 1)];
  const int64_t page = min(max(named, (int64_t)0), c.num_blocks - 1);
  return Slot{page * c.block_size + (pos - bi * c.block_size), page, page == named};
}

// fp8 codes written for another page's scale: the value that they stand for, encoded as the append does.
__device__ __forceinline__ uint32_t recode(uint32_t code, float from, float to) {
  const float x = e4m3_to_f32(code) * from;
  return to == 0.0f ? 0u : f32_to_e4m3_sat(x / to);
}
template <int U>
__device__ __forceinline__ typename Unit<U>::type recode_unit(typename Unit<U>::type v, float from, float to) {
  if (from == to) return v;
  if constexpr (U == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int k = 0; k < 32; k += 8) w |= recode((v[i] >> k) & 255u, from, to) << k;
      v[i] = w;
    }
    return v;
  } else if constexpr (U == 4) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 32; k += 8) w |= recode((v >> k) & 255u, from, to) << k;
    return w;
  } else {
    return (uint8_t)recode(v, from, to);
  }
}

// ------------------------------------------------------------------------------------ accepted paths
// Bound by its chain: metadata, the walk (one LDS read and ballot a node), then for eight rows at a time their table entries and the
// rows: one tree of 26 nodes 6.3 us, 64 of 30 - 64 nodes with 4 heads of 256, a workgroup to each, 18; 64 paths of 8 rows on average, 8
// heads of 128 13, over fp8 pages, whose codes are encoded anew, 56.
//
// The path: from row 0 to the first child whose drafted token is the model's choice at its parent, and so on.  Every
// workgroup of a sequence walks it for itself, a wavefront over 64 rows at a time; the first writes it down.
template <int U>
__global__ __launch_bounds__(256) void accept_kernel(const AcceptParams p) {
  typedef typename Unit<U>::type unit;
  __shared__ int16_t agree[PA_MAX_TREE_NODES];  // parent of a row whose token is that parent's choice, else -1
  __shared__ int16_t path[PA_MAX_TREE_NODES];
  __shared__ int count;
  const RowsParams& c = p.c;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int s0 = min(max(p.cum[b], 0), p.num_tokens);
  const int cap = (int)min((int64_t)c.max_blocks * c.block_size, (int64_t)(INT32_MAX / 2));
  const int n = min(min(max(p.cum[b + 1], s0), p.num_tokens) - s0, min(cap, PA_MAX_TREE_NODES));
  const int past = min(max(p.past[b], 0), cap - n);
  const int most = min(p.max_path, n);
  if (p.parents) {
    for (int r = tid; r < n; r += 256) {
      const int up = p.parents[s0 + r];
      agree[r] = (int16_t)(up >= 0 && up < r && p.tokens[s0 + r] == p.targets[s0 + up] ? up : -1);
    }
    __syncthreads();
    if (tid < 64) {
      int node = n > 0 ? 0 : -1, len = 0;
      while (node >= 0 && len < most) {
        if (lane == 0) path[len] = (int16_t)node;
        ++len;
        int next = -1;
        for (int r0 = (node + 1) & ~63; r0 < n && next < 0; r0 += 64) {
          const int r = r0 + lane;
          const uint64_t hit = __ballot(r > node && r < n && agree[min(r, n - 1)] == node);
          if (hit) next = r0 + __builtin_ctzll(hit);
        }
        node = next;
      }
      if (lane == 0) count = len;
    }
  } else {
    const int len = min(max(p.path_lens[b], 0), most);
    for (int i = tid; i < len; i += 256) path[i] = (int16_t)min(max(p.path[(int64_t)b * p.max_path + i], 0), n - 1);
    if (tid == 0) count = len;
  }
  __syncthreads();
  const int len = count;
  if (p.parents && blockIdx.x == 0) {
    for (int i = tid; i < p.max_path; i += 256) p.path[(int64_t)b * p.max_path + i] = i < len ? path[i] : -1;
    if (tid == 0) {
      p.path_lens[b] = len;
      if (p.next_tokens) p.next_tokens[b] = len > 0 ? p.targets[s0 + path[len - 1]] : -1;
    }
  }
  if (p.weights && blockIdx.x == 0)
    for (int i = tid; i < len * c.kv_heads; i += 256) {
      const int r = i / c.kv_heads, kh = i - r * c.kv_heads;
      const Slot d = slot_of(c, c.block_table, c.max_blocks, b, past + r);
      if (d.there) p.weights[(d.page * c.kv_heads + kh) * c.block_size + (d.slot - d.page * c.block_size)] = 0.0f;
    }
  // rows of whole tokens, keys then values
  const int64_t row = (int64_t)c.kv_heads * c.head_bytes;
  const int64_t x = ((int64_t)blockIdx.x * 256 + tid) * U;
  if (x >= 2 * row) return;
  const bool value = x >= row;
  const int64_t at = value ? x - row : x;
  char* cache = value ? c.value_cache : c.key_cache;
  const float* scale = value ? c.v_scale : c.k_scale;
  const int kh = (int)(at / c.head_bytes);
  constexpr int N = 8;
  for (int i0 = 0; i0 < len; i0 += N) {
    unit v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = min(i0 + k, len - 1);
      const Slot s = slot_of(c, c.block_table, c.max_blocks, b, past + path[i]);
      v[k] = *reinterpret_cast<const unit*>(cache + s.slot * row + at);
      if (c.fp8) {
        const Slot d = slot_of(c, c.block_table, c.max_blocks, b, past + i);
        v[k] = recode_unit<U>(v[k], scale[s.page * c.kv_heads + kh], scale[d.page * c.kv_heads + kh]);
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = i0 + k;
      if (i >= len || path[i] == i) continue;
      const Slot d = slot_of(c, c.block_table, c.max_blocks, b, past + i);
      if (d.there) *reinterpret_cast<unit*>(cache + d.slot * row + at) = v[k];
    }
  }
}

// ------------------------------------------------------------------------------------ eviction
// Weights as integers of the same order: -0 like +0, NaN above all.
__device__ __forceinline__ uint32_t weight_order(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return ~0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEThreads = 1024, kEWaves = kEThreads / 64, kEBins = 2048;

// Of the n keys of a (sequence, kv-head) more than the budget: the `need` heaviest between the first and the last
// that stay anyway.  Three rounds of counting, 11, 11 and 10 bits of the weights from the top, find the weight of the
// last one that stays; of those that weigh as much the lowest positions do.  The wavefronts then number what stays in
// stretches of their own.  HELD weights stay in LDS, more are read again in every round.
// Bound by latency, 8 us, and its passes over LDS, 0.7 us for 1000 keys (9000 keys of 128 heads 15.7; a weight to a lane at a time 17.2;
// 32768 of 8 heads 31).  Where the weights do not stay in LDS, by their loads and the tables' in every pass (131072 keys of 8 heads 320).
template <int HELD>
__global__ __launch_bounds__(kEThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t held[HELD];
  __shared__ uint32_t bins[kEBins];
  __shared__ uint32_t part[kEWaves];
  __shared__ uint32_t found[2];
  __shared__ uint32_t above[kEWaves], same[kEWaves];
  const RowsParams& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / c.kv_heads, kh = blockIdx.x - b * c.kv_heads;
  const int cap = (int)min((int64_t)c.max_blocks * c.block_size, (int64_t)(INT32_MAX / 2));
  const int n = min(max(p.lens[b], 0), min(cap, p.max_keys));
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  if (kh == 0 && tid == 0) p.lens_out[b] = min(n, p.budget);
  if (n <= p.budget) {
    for (int i = tid; i < p.budget; i += kEThreads) kept[i] = i < n ? i : -1;
    return;
  }
  for (int i = tid; i < p.sinks; i += kEThreads) kept[i] = i;
  for (int i = tid; i < p.recent; i += kEThreads) kept[p.budget - p.recent + i] = n - p.recent + i;
  uint32_t need = p.budget - p.sinks - p.recent;
  if (need == 0) return;
  const int first = p.sinks, end = n - p.recent;  // the weights of positions [first, end), lowest order elsewhere
  const bool hold = end <= HELD;
  auto load = [&](int i) {
    const Slot s = slot_of(c, c.block_table, c.max_blocks, b, i);
    const int64_t off = s.slot - s.page * c.block_size;
    return p.weights + (s.page * c.kv_heads + kh) * c.block_size + off;
  };
  if (hold) {
    // four at a time where pages hold a multiple of four, eight loads in flight
    if (p.four) {
      for (int i0 = 4 * tid; i0 < end; i0 += 8 * 4 * kEThreads) {
        f32x4 w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[k] = *reinterpret_cast<const f32x4*>(load(min(i0 + 4 * kEThreads * k, (end - 1) & ~3)));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = i0 + 4 * kEThreads * k;
          if (i < end)
            *reinterpret_cast<u32x4*>(held + i) = u32x4{weight_order(w[k][0]), weight_order(w[k][1]),
                                                        weight_order(w[k][2]), weight_order(w[k][3])};
        }
      }
    } else {
      for (int i = tid; i < end; i += kEThreads) held[i] = weight_order(*load(i));
    }
  }
  // weights i .. i + 3 (i a multiple of four; what lies outside [first, end) may be anything)
  auto quad = [&](int i) {
    if (hold) return *reinterpret_cast<const u32x4*>(held + min(i, HELD - 4));
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = weight_order(*load(min(i + k, end - 1)));
    return w;
  };
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t digit = round == 2 ? 1023u : 2047u;
    for (int i = tid; i < kEBins; i += kEThreads) bins[i] = 0;
    __syncthreads();
    for (int i = (first & ~3) + 4 * tid; i < end; i += 4 * kEThreads) {
      const u32x4 w = quad(i);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k >= first && i + k < end && (w[k] & mask) == prefix) atomicAdd(&bins[(w[k] >> shift) & digit], 1u);
    }
    __syncthreads();
    // bins from the top: thread t holds 2047 - 2 t and the one below
    const uint32_t hi = bins[kEBins - 1 - 2 * tid], lo = bins[kEBins - 2 - 2 * tid];
    uint32_t sum = hi + lo;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(sum, o, 64);
      if (lane >= o) sum += u;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    uint32_t before = sum - hi - lo;
    for (int w = 0; w < wave; ++w) before += part[w];
    if (before < need && need <= before + hi + lo) {
      const bool upper = need <= before + hi;
      found[0] = kEBins - 1 - 2 * tid - (upper ? 0 : 1);
      found[1] = need - before - (upper ? 0 : hi);
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= digit << shift;
    need = found[1];  // of the weights with this prefix
    __syncthreads();
  }
  // `need` of the weights that equal prefix stay, and all above it
  const int stretch = ((end - (first & ~3) + kEWaves - 1) / kEWaves + 255) & ~255;  // four weights to a lane at a time
  const int i0 = (first & ~3) + wave * stretch, i1 = min(i0 + stretch, end);
  int na = 0, ns = 0;
  for (int i = i0 + 4 * lane; i < i1; i += 256) {
    const u32x4 w = quad(i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = i + k >= first && i + k < i1;
      na += in && w[k] > prefix ? 1 : 0;
      ns += in && w[k] == prefix ? 1 : 0;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    na += __shfl_xor(na, o, 64);
    ns += __shfl_xor(ns, o, 64);
  }
  if (lane == 0) {
    above[wave] = na;
    same[wave] = ns;
  }
  __syncthreads();
  uint32_t ba = 0, bs = 0;
  for (int w = 0; w < wave; ++w) {
    ba += above[w];
    bs += same[w];
  }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int i = i0 + 4 * lane; i - 4 * lane < i1; i += 256) {
    const u32x4 w = quad(min(i, (end - 1) & ~3));
    uint32_t ra = ba, rs = bs;  // of those that stay before this lane's four, and so on
    bool a[4], e[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = i + k >= first && i + k < i1;
      a[k] = in && w[k] > prefix;
      e[k] = in && w[k] == prefix;
      const uint64_t ma = __ballot(a[k]), me = __ballot(e[k]);
      ra += __builtin_popcountll(ma & below);
      rs += __builtin_popcountll(me & below);
      ba += __builtin_popcountll(ma);
      bs += __builtin_popcountll(me);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (a[k] || (e[k] && rs < need)) kept[first + ra + min(rs, need)] = i + k;
      ra += a[k] ? 1 : 0;
      rs += e[k] ? 1 : 0;
    }
  }
}

// A head's rows that stay, of keys, of values (slices of W bytes of each) or the weights: in place all of them, a
// round of 2048 after the other; to other pages one round to a workgroup, of whole rows.
// Bound by HBM: 2048 of up to 9000 rows of 8 heads of 16 sequences, 268 MB read and written, to other pages in 58 us
// (4.6 TB/s; a copy of 1 GiB 5.2; in rounds of 64 KB 75 us, with stores that stay in the cache 62).  In place by its rounds:
// 1, 4 and 16 sequences of 9000 keys 8, 18 and 75 us (in rounds of 256 whole rows the last took 126).  fp8 rows, half the bytes, by their
// encoding: 16 sequences 118 us in place and 160 to other pages.
template <bool INPLACE>
struct Round {  // threads, rows in flight of each
  static constexpr int THREADS = INPLACE ? 1024 : 256, DEPTH = INPLACE ? 8 : 4;
};
template <int U, int W, bool INPLACE>
__global__ __launch_bounds__(Round<INPLACE>::THREADS) void evict_move_kernel(const EvictParams p) {
  typedef typename Unit<U>::type unit;
  constexpr int kMThreads = Round<INPLACE>::THREADS, kMDepth = Round<INPLACE>::DEPTH;
  const RowsParams& c = p.c;
  const int tid = threadIdx.x, slices = (c.head_bytes + W - 1) / W, parts = 2 * slices + 1;
  // a head's slices, which share lines, all on one XCD (every eighth workgroup) and one after the other
  const int group = blockIdx.x / (8 * parts), turn = blockIdx.x - group * 8 * parts;
  const int part = turn >> 3, z = 8 * group + (turn & 7);
  if (z >= c.batch * c.kv_heads) return;
  const int b = z / c.kv_heads, kh = z - b * c.kv_heads;
  const int cap = (int)min((int64_t)c.max_blocks * c.block_size, (int64_t)(INT32_MAX / 2));
  const int n = min(max(p.lens[b], 0), min(cap, p.max_keys)), rows = min(n, p.budget);
  if (INPLACE && n <= p.budget) return;
  const int32_t* kept = p.kept + (int64_t)z * p.budget;
  const int32_t* to = INPLACE ? c.block_table : p.table_out;
  const int to_blocks = INPLACE ? c.max_blocks : p.max_blocks_out;
  constexpr int PER = W / U, ROWS = kMThreads / PER;  // units of a slice, rows at once
  const bool weights = part == 2 * slices;
  const int step = (weights ? kMThreads : ROWS) * kMDepth;
  const int first = INPLACE ? 0 : (int)blockIdx.y * step, next = INPLACE ? step : (int)gridDim.y * step;
  if (weights) {
    for (int i0 = first; i0 < rows; i0 += next) {
      float w[kMDepth];
#pragma unroll
      for (int k = 0; k < kMDepth; ++k) {
        const Slot s = slot_of(c, c.block_table, c.max_blocks, b, max(kept[min(i0 + k * kMThreads + tid, rows - 1)], 0));
        w[k] = p.weights[(s.page * c.kv_heads + kh) * c.block_size + (s.slot - s.page * c.block_size)];
      }
      if (INPLACE) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < kMDepth; ++k) {
        const int i = i0 + k * kMThreads + tid;
        if (i >= rows) continue;
        const Slot d = slot_of(c, to, to_blocks, b, i);
        if (d.there) p.weights[(d.page * c.kv_heads + kh) * c.block_size + (d.slot - d.page * c.block_size)] = w[k];
      }
    }
    return;
  }
  const bool value = part >= slices;
  char* cache = value ? c.value_cache : c.key_cache;
  const float* scale = value ? c.v_scale : c.k_scale;
  const int at = ((value ? part - slices : part) * PER + tid % PER) * U;
  const bool mine = at < c.head_bytes;
  const int64_t row = (int64_t)c.kv_heads * c.head_bytes, off = (int64_t)kh * c.head_bytes + (mine ? at : 0);
  for (int i0 = first; i0 < rows; i0 += next) {
    unit v[kMDepth];
    int from[kMDepth];
#pragma unroll
    for (int k = 0; k < kMDepth; ++k) from[k] = max(kept[min(i0 + k * ROWS + tid / PER, rows - 1)], 0);
#pragma unroll
    for (int k = 0; k < kMDepth; ++k) {
      const Slot s = slot_of(c, c.block_table, c.max_blocks, b, from[k]);
      v[k] = *reinterpret_cast<const unit*>(cache + s.slot * row + off);
      if (c.fp8) {
        const Slot d = slot_of(c, to, to_blocks, b, min(i0 + k * ROWS + tid / PER, rows - 1));
        v[k] = recode_unit<U>(v[k], scale[s.page * c.kv_heads + kh], scale[d.page * c.kv_heads + kh]);
      }
    }
    if (INPLACE) {  // every row of the round has been read
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kMDepth; ++k) {
      const int i = i0 + k * ROWS + tid / PER;
      if (!mine || i >= rows || (INPLACE && from[k] == i)) continue;
      const Slot d = slot_of(c, to, to_blocks, b, i);
      if (!d.there) continue;
      unit* dst = reinterpret_cast<unit*>(cache + d.slot * row + off);
      if (INPLACE) *dst = v[k];
      else __builtin_nontemporal_store(v[k], dst);
    }
  }
}
template <int U, int W, bool INPLACE>
hipError_t launch_move_in(const EvictParams& p, hipStream_t s) {
  const int64_t parts = 2 * ((p.c.head_bytes + W - 1) / W) + 1;
  const int64_t wgs = ((int64_t)p.c.batch * p.c.kv_heads + 7) / 8 * 8 * parts;
  constexpr int step = Round<INPLACE>::THREADS / (W / U) * Round<INPLACE>::DEPTH;
  const int rows = std::min(p.budget, p.max_keys);
  const int rounds = INPLACE ? 1 : std::min((rows + step - 1) / step, 65535);
  if (wgs > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((evict_move_kernel<U, W, INPLACE>), dim3((unsigned)wgs, (unsigned)rounds),
                     dim3(Round<INPLACE>::THREADS), 0, s, p);
  return hipGetLastError();
}
template <int U>
hipError_t launch_move(const EvictParams& p, hipStream_t s) {
  // (odd rows too: bytes, 64 of a row at once)
  return p.table_out ? launch_move_in<U, U == 16 ? 256 : 64, false>(p, s) : launch_move_in<U, 64, true>(p, s);
}

// Bytes that rows of both caches allow at once.
int unit_of(const RowsParams& c) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(c.key_cache) | reinterpret_cast<uintptr_t>(c.value_cache) |
                      (uintptr_t)c.head_bytes;
  return x % 16 == 0 ? 16 : x % 4 == 0 ? 4 : 1;
}

}  // namespace

hipError_t launch_accept(const AcceptParams& p, hipStream_t s) {
  if (p.c.batch <= 0 || p.max_path <= 0) return hipSuccess;
  const int64_t row = 2 * (int64_t)p.c.kv_heads * p.c.head_bytes;
  const int u = unit_of(p.c);
  const dim3 grid((unsigned)((row / u + 255) / 256), p.c.batch);
  if (p.c.batch > 65535) return hipErrorInvalidValue;
  if (u == 16) hipLaunchKernelGGL((accept_kernel<16>), grid, dim3(256), 0, s, p);
  else if (u == 4) hipLaunchKernelGGL((accept_kernel<4>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((accept_kernel<1>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_evict(const EvictParams& p, hipStream_t s) {
  if (p.c.batch <= 0) return hipSuccess;
  const int64_t z = (int64_t)p.c.batch * p.c.kv_heads;
  const int u = unit_of(p.c);
  if (p.max_keys <= 8192)
    hipLaunchKernelGGL((evict_select_kernel<8192>), dim3((unsigned)z), dim3(kEThreads), 0, s, p);
  else
    hipLaunchKernelGGL((evict_select_kernel<32768>), dim3((unsigned)z), dim3(kEThreads), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return u == 16 ? launch_move<16>(p, s) : u == 4 ? launch_move<4>(p, s) : launch_move<1>(p, s);
}

}  // namespace pa
