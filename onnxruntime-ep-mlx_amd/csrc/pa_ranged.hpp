// pa_ranged.hpp — paged attention whose rows each see a range of keys (documents, prefixes, windows,
// causality), with a bias by distance, and prefixes that a group of sequences shares, on gfx950 matrix
// cores; and its kinds (RKind): nodes of drafted trees, and rows whose probabilities are wanted again.
//
// Row r of a sequence (or of a group, for its shared prefix) is query token r / g and head kh g + r % g
// of kv-head kh.  It sees keys [lo, hi); with x = softcap(scale q.k) log2(e) - slope |i - j| the output
// is sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m), m a maximum that moves only when a score exceeds it by
// more than 2^8.
//
// Work.  Sources: every group (all its rows against the shared keys, read through its first sequence's
// table) and every sequence (its rows against the keys behind the shared ones).  An item is a block of
// rows of one source and kv-head, its cost the 64-key tiles that the block may see and a few more for its
// start and end.  Sources of more than 32 rows (prompts, shared prefixes) are wide: blocks of 128 rows, a
// workgroup each.  The others (decode) are narrow: one block, a wavefront each.  The grid is shared out
// between both kinds by their tiles.  A kind's tiles form a flat list, cut into equal stretches whatever
// item borders lie inside: an item that meets several workers leaves (m, l, O) of each in fp32 and the
// merge joins them, as it joins a row's shared and own keys.  Where it costs no more (r_share), workgroups
// take whole wide items instead, in turns, each sequence's longest first and the sequences in their order,
// every other turn backwards; or, where documents hide what items cost, from queues.  The plan is a scan over
// the lengths that every workgroup makes for itself, from the device's metadata.
//
// Both products run transposed on 32x32x16 tiles, so that a lane holds one query row:
//   S^T[key][row] = K Q^T   (A: 32 keys x 16 dims from LDS, B: the queries in registers)
//   O^T[dim][row] = V^T P^T (A: 32 dims x 16 keys by transposing LDS reads, B: the probabilities as the
//                            score product leaves them)
// A row's maximum and sum need one exchange between the lane halves, and its range, slope and position
// are scalars of the lane.  Probabilities enter the second product in two parts of the activation type
// (off by at most 2^-17 of themselves in bf16, 2^-20 in fp16, as in the streaming decode: one part
// alone erred as much as the output's own rounding), two products against one read of the values; scores,
// statistics and sums are fp32.
//
// Wide items: four wavefronts of 32 rows each on the same 64-key tile (32 keys at head 256), staged by
// direct loads from the pages into two LDS buffers, one barrier per tile.  Narrow items: a wavefront with a
// 32-key tile of its own in LDS, the next keys in flight while the values are multiplied, no barrier.
//
// Masked keys weigh exactly zero, but zero times an infinite value is NaN in the product: rows whose sums of
// values come out not finite are computed again, a wavefront's together and one key at a time, which skips what
// they do not see.  Tiles read no key outside [first visible, last visible] of their rows (such places repeat a
// visible one), so pages behind a sequence's end or before its window may hold anything.
//
// Drafted trees (kRTree): a node's keys end with its own, and a word of its bits for every 32 new rows masks what lies
// among them; only tiles with new rows look at it.  Weighed rows (kRWeigh): the constant m + log2(l) of a row goes beside
// its output, and narrow items leave their scores (pa_weigh.hip).
//
// What bounds it (GPU times of a call, merge included).  Prompts of 8192: 32 heads of 128 in 746 us, 737
// TFLOP/s of the two products, 1105 with the second part of the probabilities, the softmax's vector instructions
// behind them in turn; 64 heads of 64 in 945 us (twice the scores per product), 16 heads of 256 in 767.  64
// sequences of up to 8192 keys, one token each: 212 us, 5.8 TB/s from HBM.  A tree of 257 nodes after 60001 keys, 32 heads
// of 128: 413 - 451 us by the card, 611 TFLOP/s at the best (nine blocks of rows of which the last holds four); 16 trees of
// 40 - 64 nodes, 28 heads, 84 - 90.  Small calls: 5 us of dependent
// loads and the scan before the first item, 2 us to its first tile, 3 us per launch.
#pragma once

#include <algorithm>

#include "pa_tiles.hpp"

namespace pa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

// What a kernel is built for: ranges of keys alone; nodes of trees, whose range of keys reaches from the window's
// edge to the node itself and which see of the new rows in it those that their bits name; ranges whose rows leave
// the constant of their softmax (row_stats), and on narrow items their scores.
enum RKind { kRRanges = 0, kRTree = 1, kRWeigh = 2 };

constexpr int kRTile = 64;     // keys per unit of cost
constexpr int kRWide = 128;    // rows of a block of four wavefronts
constexpr int kRNarrow = 32;   // rows of a block whose wavefronts split the keys
constexpr int kRChunk = 256;   // sources scanned at a time, one per thread
// What an item's start and end cost, in tiles (8 instead: 64 samples of a prompt of 8176 41 us for 39).
constexpr int kRStart = 4;
// What partial rows and their merge cost, in tiles of every worker: 3, 8 and 20 gave 826, 836 and 748 us over a
// prompt of 8192, 236, 214 and 213 over six prompts of 1001 - 2500 at head 64; 25 each for 40 samples of 1500.
constexpr float kRCut = 20.0f;
// ... of drafted trees, whose few rows the merge joins in the 4 us that its launch takes anyway (a tree of 26 nodes after
// 700 keys: 34 us with 10 or 20, 25 with 2 or 5; 24 trees of 9 - 33 nodes at head 64 45 with any).
constexpr float kRCutTree = 5.0f;
// Time of a tile where a workgroup has its CU to itself (1.0 instead: 1024 tokens over 1000 keys 70 us for
// 62, over 3000 115 for 109).
constexpr float kRAlone = 0.65f;
// Time of a wide tile on a workgroup over a narrow one's on a wavefront, in the sharing out of workgroups (1, 2 and 3:
// 64 samples of a prompt of 8176 40, 45 and 44 us for 39; 40 samples of 1500 26, 25 and 25 for 25).
constexpr float kRWideCost = 1.5f;
// Least weight of a key that a row sees, beside fp32's smallest: infinite values show however little they weigh.
constexpr float kRTiny = 0x1p-126f;
// Rows up to which the merge gives each a workgroup, a wavefront; workgroups of the merge of more.
constexpr int64_t kRJoinWide = 1024, kRJoinRows = 16384;
constexpr int kRMergeGrid = 2048;

template <typename TT>
__device__ __forceinline__ f32x16 mfma_r(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (TT::code == PA_DTYPE_FLOAT16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float half_swap(float x) {  // lane l ^ 32's x
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x),
                                                  __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// Eight probabilities as the sum of two parts in T.
struct RPair {
  u32x4 hi, lo;
};
template <typename TT>
__device__ __forceinline__ RPair split_pair(const float (&x)[8]) {
  typename TT::vec8 h, l;
  TT::split8(x, h, l);
  return RPair{__builtin_bit_cast(u32x4, h), __builtin_bit_cast(u32x4, l)};
}
template <typename TT>
__device__ __forceinline__ u32x2 pack4(float a, float b, float c, float d) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef decltype(__builtin_shufflevector(typename TT::vec8{}, typename TT::vec8{}, 0, 1)) vec2;
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, vec2)),
               __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{c, d}, vec2))};
}

// x, hidden from the compiler: what follows from it would otherwise be computed at the kernel's start for every path
// there is, and keep registers there that the tile loops need.
__device__ __forceinline__ int hidden(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Direct LDS loads of 16 bytes per lane to M0 + 16 * lane, as inline assembly so that the compiler's
// memory counters do not see them and nothing waits for them but the tile loops (wait_loads).  The
// immediate offset counts for both addresses.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int N, bool NT>
__device__ __forceinline__ void dma_rows(const char* base, const uint32_t* off, uint32_t lds) {
  static_assert(N == 2 || N == 4, "two or four KiB");
  if constexpr (N == 4 && NT)
    asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4 nt\n\t"
                 "global_load_lds_dwordx4 %1, %4 offset:1024 nt\n\t"
                 "global_load_lds_dwordx4 %2, %4 offset:2048 nt\n\tglobal_load_lds_dwordx4 %3, %4 offset:3072 nt"
                 :
                 : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(lds)
                 : "memory", "m0");
  else if constexpr (N == 4)
    asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\t"
                 "global_load_lds_dwordx4 %1, %4 offset:1024\n\t"
                 "global_load_lds_dwordx4 %2, %4 offset:2048\n\tglobal_load_lds_dwordx4 %3, %4 offset:3072"
                 :
                 : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(lds)
                 : "memory", "m0");
  else if constexpr (NT)
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2 nt\n\t"
                 "global_load_lds_dwordx4 %1, %2 offset:1024 nt"
                 :
                 : "v"(off[0]), "v"(off[1]), "s"(base), "s"(lds)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\t"
                 "global_load_lds_dwordx4 %1, %2 offset:1024"
                 :
                 : "v"(off[0]), "v"(off[1]), "s"(base), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma_ptr(const char* ptr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(ptr), "s"(lds)
               : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N vector loads are outstanding
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A barrier that waits for nothing itself: the tile loops' loads are waited for by hand, and what was read from
// LDS has been used.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Maximum of v over lanes 0 .. 31 in lane 31, over lanes 32 .. 63 in lane 63.
__device__ __forceinline__ int half_top(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // row_mirror
  return max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));  // row_bcast:15
}
// Over the 32 rows of a wavefront (both halves alike).
__device__ __forceinline__ int half_max(int v) { return __builtin_amdgcn_readlane(half_top(v), 31); }
__device__ __forceinline__ int half_min(int v) { return -half_max(-v); }

// A table entry at a wave-uniform place, through the scalar cache (no kernel writes the tables).
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  return *(cptr)(uintptr_t)p;
}

// ------------------------------------------------------------------------------------ the plan
struct RSeq {
  int s0, nq, past, total;
};
__device__ __forceinline__ RSeq r_seq(const RangedParams& p, int b) {
  RSeq q;
  const int c0 = p.cum[b], c1 = p.cum[b + 1], pb = p.past[b];
  const int cap = (int)min((int64_t)p.max_blocks * p.block_size, (int64_t)(INT32_MAX / 2));
  q.s0 = min(max(c0, 0), p.num_tokens);
  q.nq = min(min(max(c1, q.s0), p.num_tokens) - q.s0, cap);
  q.past = min(max(pb, 0), cap - q.nq);
  q.total = q.past + q.nq;
  return q;
}
// Sequences of group gi and the keys that they share: none in a group of one sequence, at most the
// keys of its first.
struct RGroup {
  int b0, b1, prefix;
};
__device__ __forceinline__ RGroup r_group(const RangedParams& p, int gi) {
  RGroup q;
  q.b0 = min(max(p.group_cum[gi], 0), p.batch);
  q.b1 = min(max(p.group_cum[gi + 1], q.b0), p.batch);
  q.prefix = q.b1 - q.b0 < 2 ? 0 : min(max(p.shared_lens[gi], 0), r_seq(p, q.b0).total);
  return q;
}
// Group of sequence b, -1 if none: the last one that begins at or before b.
__device__ __forceinline__ int group_of(const RangedParams& p, int b) {
  int lo = 0, hi = p.groups;
  while (hi - lo > 4) {
    const int mid = (lo + hi) >> 1;
    if (p.group_cum[mid] <= b) lo = mid; else hi = mid;
  }
  int n = lo;  // (a few loads at once end the search in one round trip)
#pragma unroll
  for (int k = 0; k < 4; ++k) n += lo + k < hi && p.group_cum[lo + k] <= b ? 1 : 0;
  return n > 0 && b < p.group_cum[n] ? n - 1 : -1;
}

// A group's rows against the keys it shares, or a sequence's against its own.
struct RSource {
  int first;      // its first tile in its kind's flat list
  int item;       // its first item there
  int tok0, rows; // first token, rows (tokens * g) of one kv-head
  int b0, b1;     // its sequences; b0's table names the pages
  int ka, kb;     // its keys
  int base;       // tiles of block 0 (see r_before)
  int shared;     // keys that the sequence shares
  int group;      // its group; -1 - group for the group's own source
};
__device__ __forceinline__ bool r_wide(const RSource& s) { return s.rows > kRNarrow; }
__device__ __forceinline__ int r_blocks(const RSource& s) {
  return r_wide(s) ? (s.rows + kRWide - 1) / kRWide : s.rows > 0;
}
// Places of one kv-head before block i, kRStart and the tiles of each: all of the source's (constant), or growing with the rows' positions
// under a causal mask -- base + 2 i / g each, close to what block i can see, in closed form.
__device__ __forceinline__ int r_before(const RSource& s, int i, int g, bool grows) {
  return i * s.base + (grows ? (int)((int64_t)i * (i - 1) / g) : 0);
}
__device__ __forceinline__ bool r_grows(const RangedParams& p, const RSource& s) {
  return p.causal && !p.prefix_lens && s.group >= -1 && r_wide(s);
}
// Source i: groups, then sequences (first and item are the scan's).
__device__ __forceinline__ RSource r_source(const RangedParams& p, int i) {
  RSource s{};
  s.group = -1;
  const int g = p.num_heads / p.kv_heads;
  if (i >= p.groups + p.batch) return s;
  const bool seq = i >= p.groups;
  const int b = i - p.groups, gi = seq ? (p.groups ? group_of(p, b) : -1) : i;
  const RGroup q = gi >= 0 ? r_group(p, gi) : RGroup{0, 0, 0};
  int end;
  if (!seq) {
    s.group = -2 - gi;
    if (q.prefix == 0) return s;
    s.b0 = q.b0;
    s.b1 = q.b1;
    s.tok0 = r_seq(p, q.b0).s0;
    const RSeq last = r_seq(p, q.b1 - 1);
    s.rows = max(last.s0 + last.nq - s.tok0, 0) * g;
    end = s.kb = s.shared = q.prefix;
  } else {
    const RSeq e = r_seq(p, b);
    s.group = gi;
    s.b0 = b;
    s.b1 = b + 1;
    s.tok0 = e.s0;
    s.rows = e.nq * g;
    s.shared = s.ka = min(q.prefix, e.total);
    if (p.window > 0) s.ka = max(s.ka, min(e.past - p.window + 1, e.total));
    end = s.kb = e.total;
    if (r_grows(p, s)) end = min(end, e.past + (kRWide + g - 1) / g);  // the last position of block 0
  }
  // (an item without keys keeps a tile, whose worker writes its empty rows)
  s.base = kRStart + max((end + kRTile - 1) / kRTile - s.ka / kRTile, 1);
  return s;
}

// Per kind (wide, narrow): items in the upper, tiles in the lower bits.
constexpr int kRItemShift = 40;
struct RScan {
  RSource src[kRChunk];
  int64_t wt[4][2];
  int red[8];
  int most[4];
  int next;  // from the queue
};
struct RTotals {
  int tiles[2], items[2];  // wide, narrow
  int most;                // places of the largest wide item
};
__device__ __forceinline__ int pick(const int (&x)[2], int kind) { return kind ? x[1] : x[0]; }
__device__ __forceinline__ int64_t scan64(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
// Sources base .. base + 255 with their places in the flat lists into sh.src; t: tiles and items before
// them, moved past them.  Called by all 256 threads.
__device__ __forceinline__ void scan_chunk(const RangedParams& p, int base, RScan& sh, RTotals& t) {
  const int tid = hidden(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  RSource s = r_source(p, base + tid);
  const int blocks = r_blocks(s), kind = r_wide(s) ? 0 : 1, g = p.num_heads / p.kv_heads;
  const bool grows = r_grows(p, s);
  const int largest = kind ? 0 : r_before(s, blocks, g, grows) - r_before(s, blocks - 1, g, grows);
  const int64_t mine = ((int64_t)(blocks * p.kv_heads) << kRItemShift) +
                       (int64_t)p.kv_heads * r_before(s, blocks, g, grows);
  const int top = max(half_max(largest), __builtin_amdgcn_readlane(half_top(largest), 63));
  int64_t before[2], all[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) before[k] = scan64(kind == k ? mine : 0, lane);
  __syncthreads();  // the last chunk's readers are done
  if (lane == 63) {
    sh.wt[wave][0] = before[0];
    sh.wt[wave][1] = before[1];
    sh.most[wave] = top;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (kind == k) before[k] -= mine;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before[k] += sh.wt[w][k];
      all[k] += sh.wt[w][k];
    }
  }
  constexpr int64_t low = ((int64_t)1 << kRItemShift) - 1;
  const int64_t b = before[0] * (1 - kind) + before[1] * kind;
  s.first = (kind ? t.tiles[1] : t.tiles[0]) + (int)(b & low);
  s.item = (kind ? t.items[1] : t.items[0]) + (int)(b >> kRItemShift);
  sh.src[tid] = s;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    t.tiles[k] += uniform((int)(all[k] & low));
    t.items[k] += uniform((int)(all[k] >> kRItemShift));
  }
  t.most = uniform(max(t.most, max(max(sh.most[0], sh.most[1]), max(sh.most[2], sh.most[3]))));
  __syncthreads();
}
// Who takes what: workgroups [0, wide) the wide items, the wavefronts of the others the narrow ones; tiles
// per worker of each kind (0: whole items).
struct RShare {
  int wide, per[2];
};
template <int KIND>
__device__ __forceinline__ RShare r_share(const RangedParams& p, const RTotals& t) {
  RShare r;
  const float cost = kRWideCost * (float)t.tiles[0];
  r.wide = t.tiles[0] == 0 ? 0
           : t.tiles[1] == 0
               ? p.slots
               : min(max((int)((float)p.slots * (cost / (cost + (float)t.tiles[1]))), 1), p.slots - 1);
  const int waves = max((p.slots - r.wide) * 4, 1);
  // Whole wide items, or equal stretches of their tiles.  Whole, a worker takes the largest item, or its share
  // of all in turns: items of equal cost as many as there are turns, of evenly spread costs little over an even
  // share; an item that has its CU to itself runs faster.  Stretches take an even share and what the partial rows
  // and their merge cost (kRCut tiles; little where shared prefixes leave them anyway).  Documents hide what items
  // cost, and go whole.
  const float even = (float)t.tiles[0] / (float)max(r.wide, 1), avg = (float)t.tiles[0] / (float)max(t.items[0], 1);
  const int turns = (t.items[0] + r.wide - 1) / max(r.wide, 1);
  const float spread = fminf(fmaxf((float)t.most / fmaxf(avg, 1.0f) - 1.0f, 0.0f), 1.0f);
  const float whole =
      turns <= 1 ? t.most * (2 * t.items[0] <= r.wide && p.per_cu > 1 ? kRAlone : 1.0f)
                 : fmaxf((float)t.most, avg * turns * (1.0f - spread) + 1.05f * even * spread);
  const bool take = p.whole || (p.doc_starts && 2 * t.items[0] >= r.wide) ||
                    whole <= even + (p.groups ? 0.25f : 1.0f) * (KIND == kRTree ? kRCutTree : kRCut);
  r.per[0] = take || t.items[0] == 0 ? 0 : max((t.tiles[0] + r.wide - 1) / max(r.wide, 1), p.least[0]);
  r.per[1] = p.whole || t.items[1] == 0 ? 0 : max((t.tiles[1] + waves - 1) / waves, p.least[1]);
  return r;
}
// One item: block blk of source s and kv-head kh, its number and places in the flat list: kRStart for its start
// and end, then its tiles.
struct RItem {
  int blk, kh, item, at, size;
};
__device__ __forceinline__ RItem r_item(const RangedParams& p, const RSource& s, int blk, int kh) {
  const int g = p.num_heads / p.kv_heads;
  const bool grows = r_grows(p, s);
  RItem r;
  r.blk = blk;
  r.kh = kh;
  r.item = s.item + blk * p.kv_heads + kh;
  const int f = r_before(s, blk, g, grows);
  r.size = r_before(s, blk + 1, g, grows) - f;
  r.at = s.first + f * p.kv_heads + kh * r.size;
  return r;
}
// Worker of tile x of an item; what lies behind its counted tiles belongs to its last worker.  (Whole items: 0, for
// their places in the workspace go by the item alone.)
__device__ __forceinline__ int r_worker(int per, const RItem& q, int x) {
  return per > 0 ? (q.at + min(kRStart + x, q.size - 1)) / per : 0;
}

// The range [lo, hi) of token t at position pos of sequence b (total keys).
struct RRange {
  int lo, hi;
};
template <int KIND>
__device__ __forceinline__ RRange r_range(const RangedParams& p, int t, int pos, int b, int total, int lag) {
  int hi = p.causal ? pos + 1 : total;
  if (p.causal && p.prefix_lens) hi = max(hi, p.prefix_lens[b]);
  int lo = p.window > 0 ? pos - p.window + 1 : 0;
  // (a node's place in its text goes by its depth; ancestors in the window lie above that place, for none has more
  // ancestors than rows before it)
  if (KIND == kRTree && p.window > 0) lo -= lag;
  if (p.doc_starts) lo = max(lo, p.doc_starts[t]);
  return RRange{max(lo, 0), min(hi, total)};
}

// First partial row of a worker's part of an item.  With shared prefixes every part may be one of several of a
// row: place worker + item (the parts of an item follow each other and the next begins with the worker where it
// ends).  Otherwise only a worker's first and last items meet others: two places each.
__device__ __forceinline__ int64_t r_slot(const RangedParams& p, int kind, int worker, int item, bool head) {
  const int64_t slot = p.groups > 0 ? (int64_t)worker + item : 2 * (int64_t)worker + (head ? 1 : 0);
  return kind == 0 ? slot * kRWide : p.part_narrow + slot * p.narrow_rows;
}

// A worker's part of an item: keys [k0, k1).
struct RUnit {
  RSource s;
  bool group;
  int kh, row0;    // first row of the block
  int k0, k1;
  bool head;       // the item's first part
  int64_t slot;    // its first partial row
};
__device__ __forceinline__ int r_token_seq(const RangedParams& p, int lo, int hi, int t) {
  while (hi - lo > 1) {  // the last of sequences lo .. hi - 1 that begins at or before t
    const int mid = (lo + hi) >> 1;
    if (p.cum[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}
// A row of a unit's block: its token, head and position, the keys of the unit that it sees; how: kRAny (some),
// kRSingle (all that it sees at all), kRZero (it sees nothing at all and this unit writes that).
struct RInfo {
  int t, h, pos, lo, hi, how;
  // kRTree: key of the sequence's first new row, and the new rows that the row sees, by bits: in memory, or of small
  // trees here
  int past;
  const uint32_t* bits;
  uint64_t mask;
};
constexpr int kRAny = 1, kRSingle = 2, kRZero = 4;
__device__ __forceinline__ RInfo r_place(const RangedParams& p, const RUnit& u, int rl) {
  const int g = p.num_heads / p.kv_heads, r = u.row0 + rl;
  const bool valid = r < u.s.rows;
  RInfo q;
  q.t = u.s.tok0 + (valid ? r / g : 0);
  q.h = u.kh * g + (valid ? r % g : 0);
  return q;
}
// A tree of at most 64 nodes, one to a lane of the wavefront: the bits of node `node` and how far behind its row its
// place in the text is.  Lines of ancestors double, six times at most.  (For a kernel of its own, before this one, a tree
// of 26 nodes waited 5 us, 16 of 40 - 64 8.)
struct RNode {
  uint64_t mask;
  int lag;
};
__device__ __forceinline__ RNode small_tree(const RangedParams& p, int tok0, int nodes, int node) {
  const int lane = hidden(threadIdx.x & 63);
  int up = lane < nodes ? p.tree_parents[tok0 + lane] : -1;
  up = up >= 0 && up < lane ? up : -1;
  uint64_t line = (uint64_t)1 << lane;
  while (__any(up >= 0)) {  // line: 2^k nodes, up: the one behind them
    const int from = max(up, 0), next = __shfl(up, from, 64);
    const uint64_t more = __shfl((unsigned long long)line, from, 64);
    if (up >= 0) {
      line |= more;
      up = next;
    }
  }
  const int depth = __builtin_popcountll(line) - 1;
  if (p.window > 0)
    while (__builtin_popcountll(line) > p.window) line &= line - 1;  // the farthest ancestors are the lowest rows
  const int at = min(node, 63);
  const uint64_t mask = __shfl((unsigned long long)line, at, 64);
  const int lag = node - __shfl(depth, at, 64);
  return RNode{node < 64 ? mask : 0, lag};
}
template <int KIND>
__device__ __forceinline__ void r_keys(const RangedParams& p, const RUnit& u, int rl, RInfo& q) {
  const int g = p.num_heads / p.kv_heads;
  const bool valid = u.row0 + rl < u.s.rows;
  int b = u.s.b0, total = u.s.kb, shared = u.s.shared, lag = 0;
  if (u.group) {
    b = r_token_seq(p, u.s.b0, u.s.b1, q.t);
    const RSeq e = r_seq(p, b);
    q.pos = e.past + (q.t - e.s0);
    total = e.total;
    shared = min(shared, total);
  } else {
    q.pos = total - u.s.rows / g + (q.t - u.s.tok0);
    if constexpr (KIND == kRTree) {
      q.past = total - u.s.rows / g;
      if (p.tree_parents) {
        const RNode node = small_tree(p, u.s.tok0, u.s.rows / g, q.t - u.s.tok0);
        q.mask = node.mask;
        lag = node.lag;
        if (p.window > 0 && valid) p.tree_lag[q.t] = lag;  // for the merge
      } else {
        q.bits = p.tree_bits + (int64_t)q.t * p.tree_words;
        if (p.window > 0) lag = p.tree_lag[q.t];
      }
    }
  }
  const RRange x = r_range<KIND>(p, q.t, q.pos, b, total, lag);
  const int a = max(x.lo, u.group ? 0 : shared), z = min(x.hi, u.group ? shared : total);
  q.lo = max(a, u.k0);
  q.hi = min(z, u.k1);
  q.how = 0;
  if (valid && q.lo < q.hi) {
    const bool other = u.group ? x.hi > max(x.lo, shared) : x.lo < min(x.hi, shared);
    q.how = kRAny | (a >= u.k0 && z <= u.k1 && !other ? kRSingle : 0);
  }
  if (valid && !u.group && x.lo >= x.hi && u.head) q.how |= kRZero;
}

template <typename TT>
__device__ __forceinline__ float r_sink(const RangedParams& p, int h) {
  return p.head_sink ? TT::to_f32(reinterpret_cast<const typename TT::raw*>(p.head_sink)[h]) * kLog2e
                     : kNegInf;
}

// Element offset of key / value row `pos` of kv-head kh in the pages that table row b names.
__device__ __forceinline__ int64_t r_offset(const RangedParams& p, int b, int kh, int pos, int D) {
  const int bi = min(pos / p.block_size, p.max_blocks - 1);
  int64_t page = p.block_table[(int64_t)b * p.max_blocks + bi];
  page = min(max(page, (int64_t)0), p.num_blocks - 1);
  return ((page * p.block_size + pos % p.block_size) * p.kv_heads + kh) * D;
}

// ------------------------------------------------------------------------------------ the tiles
// LDS rows of one tile: PITCH bytes each, 16-byte pieces exchanged by an XOR with the row so that the
// operand reads of 16 lanes meet 16 different bank groups.  Keys are read a row per lane: piece ^ row.
// Values are read transposed, four rows of 32 dims at a time: pieces in fours, exchanged by row % 4.
// Head 96 keeps rows of 256 bytes (its last four pieces are read twice and used once).
template <int D>
struct RGeom {
  static constexpr int PITCH = D == 96 ? 256 : 2 * D;
  static constexpr int CPR = PITCH / 16;     // pieces per row
  static constexpr int RPI = 64 / CPR;       // rows per load instruction
  // Keys of a wide tile, two of which are buffered.  (Tiles of 32 keys, four deep: 626 us for 554 over a
  // prompt of 8192 at head 128, four deep at head 256 664 for 647, with one part of the probabilities: what is
  // loaded a tile ahead is there in time.)
  static constexpr int KT = D > 128 ? 32 : 64;
  static constexpr int WIDE = 2 * 2 * KT * PITCH;
  static constexpr int NARROW = 4 * 2 * 32 * PITCH;   // four wavefronts' tiles of 32 keys
  static constexpr int LDS = WIDE > NARROW ? WIDE : NARROW;
  __device__ static int kx(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
  __device__ static int vx(int row) { return D == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); }
};

// A wavefront's loads of tile rows: groups of GR rows (16; 8 where a wavefront has no more of a tile), each in
// one page where pages hold a power of two of at least 16 rows.
template <int D, int GR>
struct RFeed {
  using G = RGeom<D>;
  static constexpr int NI = GR / G::RPI;          // load instructions per group and side
  static constexpr int NB = NI < 4 ? NI : 4;      // ... per base
  static constexpr int kBias = 1024 * (NB - 1);   // (offsets stay positive: the immediate goes up, they go down)
  const char *kc, *vc;
  const int32_t* bt;
  uint32_t rowb;       // bytes of a cache row
  int pages, last;     // pages of the pool, last entry of the table
  int kmin, kmax;      // keys that may be read
  int bs, sh;          // block size, its logarithm if it is a power of two of at least 16, else -1
  uint32_t ko[NI], vo[NI];

  __device__ __forceinline__ uint32_t piece(int row, int lane, bool value) const {
    int c = (lane % G::CPR) ^ (value ? G::vx(row) : G::kx(row));
    if (D == 96 && c >= 12) c -= 8;
    return 16 * c;
  }
  // Group rows r0 .. (its place in the tile modulo 16) of this lane.
  __device__ __forceinline__ void begin(const RangedParams& p, int b, int kh, int r0, int lane) {
    bt = p.block_table + (int64_t)b * p.max_blocks;
    rowb = (uint32_t)p.kv_heads * D * 2;
    const int64_t hoff = (int64_t)kh * D * 2 - kBias;
    kc = reinterpret_cast<const char*>(p.key_cache) + hoff;
    vc = reinterpret_cast<const char*>(p.value_cache) + hoff;
    pages = (int)p.num_blocks;
    last = p.max_blocks - 1;
    bs = p.block_size;
    sh = p.bs_shift;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = i * G::RPI + lane / G::CPR;
      ko[i] = row * rowb + piece(r0 + row, lane, false) + kBias - 1024 * (i % NB);
      vo[i] = row * rowb + piece(r0 + row, lane, true) + kBias - 1024 * (i % NB);
    }
  }
  // Page of the group at key pos, or of the nearest group that may be read.
  __device__ __forceinline__ int page(int pos) const {
    const int x = min(max(pos, kmin), kmax - 1);
    return sh >= 0 ? min(max(scalar_load(bt + min(x >> sh, last)), 0), pages - 1) : 0;
  }
  // Loads of one group at key pos, page pg: keys and / or values of its rows.
  template <bool KEYS, bool VALUES, bool NT>
  __device__ __forceinline__ void load(int pos, int pg, uint32_t kl, uint32_t vl, int r0, int lane0) const {
    if (sh >= 0 && pos >= kmin && pos + GR <= kmax) {
      const uint64_t off = (uint64_t)(((uint32_t)pg << sh) + (uint32_t)(pos & (bs - 1))) * rowb;
#pragma unroll
      for (int i = 0; i < NI; i += NB) {
        if constexpr (KEYS) dma_rows<NB, NT>(kc + off, ko + i, kl + 1024 * i);
        if constexpr (VALUES) dma_rows<NB, NT>(vc + off, vo + i, vl + 1024 * i);
      }
    } else if (sh >= 0) {
      // an edge: rows that must not be read repeat the nearest that may
      const int lane = hidden(lane0);
      const int x = min(max(pos, kmin), kmax - 1) & ~(GR - 1);
      const uint64_t off = (uint64_t)(((uint32_t)pg << sh) + (uint32_t)(x & (bs - 1))) * rowb;
#pragma unroll
      for (int i = 0; i < NI; i += NB) {
        uint32_t k[NB], v[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int row = (i + j) * G::RPI + lane / G::CPR;
          const uint32_t at = (uint32_t)(min(max(pos + row, kmin), kmax - 1) - x) * rowb + kBias - 1024 * j;
          k[j] = at + piece(r0 + row, lane, false);
          v[j] = at + piece(r0 + row, lane, true);
        }
        if constexpr (KEYS) dma_rows<NB, NT>(kc + off, k, kl + 1024 * i);
        if constexpr (VALUES) dma_rows<NB, NT>(vc + off, v, vl + 1024 * i);
      }
    } else {
      // pages of any size: lane r finds the page of row r
      const int lane = hidden(lane0);
      const int mine = min(max(pos + (lane & (GR - 1)), kmin), kmax - 1), bi = mine / bs;
      const int slot = min(max(bt[min(bi, last)], 0), pages - 1) * bs + (mine - bi * bs);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * G::RPI + lane / G::CPR;
        const uint64_t off = (uint64_t)(uint32_t)__shfl(slot, row, 64) * rowb + kBias;
        if constexpr (KEYS) dma_ptr(kc + off + piece(r0 + row, lane, false), kl + 1024 * i);
        if constexpr (VALUES) dma_ptr(vc + off + piece(r0 + row, lane, true), vl + 1024 * i);
      }
    }
  }
};

// A wavefront's 32 rows: lane l holds row l % 32, half h = l / 32 of the keys of a tile and of the dims.
template <typename TT, int D>
struct RState {
  u32x4 q[D / 16];
  f32x16 o[D / 32];
  float m, l;
  int lo, hi;  // keys that the row sees in this unit
  int pos;
  float slope;  // in units of the scores it is taken from (r_softmax)
  float* scores;         // kRWeigh: the row's scores, or null
};

// Bits of keys t0 .. t0 + 31 of a row's mask over the new rows, the first of which is key `past`; the keys before
// them are all seen.
__device__ __forceinline__ uint32_t tree_mask(const RangedParams& p, const RInfo& q, int n) {  // n = t0 - past
  if (n <= -32) return ~0u;
  if (p.tree_parents) return (uint32_t)(n < 0 ? (q.mask << -n) | ((1u << -n) - 1u) : n < 64 ? q.mask >> n : 0);
  return tree_window(q.bits, p.tree_words, n);
}

// Matrix products run in groups, whose operands are read from LDS while the group before multiplies: reads and
// products keep their order (the compiler alone reuses one operand's registers and waits for every read), vector
// and scalar instructions may move.
__device__ __forceinline__ void r_order() { __builtin_amdgcn_sched_barrier(0x0406); }

// Scores of 32 KB keys: raw products.
template <typename TT, int D, int KB>
__device__ __forceinline__ void r_scores(const RState<TT, D>& st, const char* kt, int lane,
                                         f32x16 (&s)[KB]) {
  using G = RGeom<D>;
  constexpr int N = D / 16 * KB, A = N % 4 ? 3 : 4;  // products, of a group
  static_assert(N % A == 0, "whole groups");
  const int c = lane & 31, h = lane >> 5;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
  const char* row = kt + c * G::PITCH;
  const int x = G::kx(c) ^ h;
  u32x4 k[2][A];
  auto read = [&](int g) {
#pragma unroll
    for (int i = 0; i < A; ++i) {
      const int ks = (g * A + i) / KB, kb = (g * A + i) % KB;
      k[g & 1][i] = *reinterpret_cast<const u32x4*>(row + (((2 * ks) ^ x) << 4) + kb * 32 * G::PITCH);
    }
  };
  read(0);
#pragma unroll
  for (int g = 0; g < N / A; ++g) {
    if (g + 1 < N / A) read(g + 1);
    r_order();
#pragma unroll
    for (int i = 0; i < A; ++i) s[(g * A + i) % KB] = mfma_r<TT>(k[g & 1][i], st.q[(g * A + i) / KB], s[(g * A + i) % KB]);
    r_order();
  }
}

// Forms of a score: as it is, less a slope times the distance, softcapped (and less that).
enum RForm { kRPlain = 0, kRSlope = 1, kRCap = 2 };

// tanh(y) / 2 of z = 2 y log2(e).  Near zero by its series, elsewhere from 1 - 2 / (1 + exp(2 y)), which holds its own bits there.
__device__ __forceinline__ float half_tanh(float z) {
  const float y = z * (0.5f / kLog2e);
  const float far = 0.5f + __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(z));
  return fabsf(y) < 0.25f ? y * half_tanh_series(y * y) : far;
}

// Bias, mask, the lazy maximum and the probabilities of 32 KB keys at t0, in two parts per 16 keys.
template <typename TT, int D, int KB, int FORM, int KIND>
__device__ __forceinline__ void r_softmax(const RangedParams& p, RState<TT, D>& st, f32x16 (&s)[KB],
                                          int t0, bool low, bool high, bool before, int lane, RPair (&pr)[2 * KB],
                                          bool tree, const uint32_t (&tw)[KB]) {
  const int h = lane >> 5;
  // A score in log2 units is s * sl + off.  kRCap: softcap tanh(y), whose last product the exponent's FMA makes.
  // Up to kCapNear s keeps the quotient of softcap (1 - 2 / (1 + exp(2 y))): its error, a few steps of 2^-24 of the
  // softcap, stays below 2^-16, the probabilities' own.  Beyond it s is tanh(y) / 2 to its own bits.
  const float sl = FORM == kRCap ? 2.0f * kLog2e * p.softcap : p.scale_log2;
  float off = 0.0f;
  if constexpr (FORM == kRCap) {
    const float ck = 2.0f * p.scale_log2 / p.softcap;
    if (p.softcap <= kCapNear) {
      off = kLog2e * p.softcap;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[kb][i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[kb][i] * ck));
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = half_tanh(s[kb][i] * ck);
    }
  }
  if (FORM == kRSlope || (FORM == kRCap && p.slopes)) {
    const float far = (float)(st.pos - t0 - 4 * h);
    if (before) {
      // no key behind the row (that it sees): the distance is far less the key's place
      off = __builtin_fmaf(-st.slope * far, sl, off);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[kb][i] = __builtin_fmaf(st.slope, (float)(32 * kb + 8 * (i >> 2) + (i & 3)), s[kb][i]);
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[kb][i] = __builtin_fmaf(fabsf(far - (float)(32 * kb + 8 * (i >> 2) + (i & 3))), -st.slope, s[kb][i]);
    }
  }
  if (low) {  // some row's keys begin inside the tile
    const int lo = st.lo - t0 - 4 * h;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) >= lo ? s[kb][i] : kNegInf;
  }
  if (high) {  // ... end inside it
    const int hi = st.hi - t0 - 4 * h;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) < hi ? s[kb][i] : kNegInf;
  }
  if constexpr (KIND == kRTree) {
    if (tree) {  // new rows in the tile
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t m = tw[kb] >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = (m >> (8 * (i >> 2) + (i & 3))) & 1u ? s[kb][i] : kNegInf;
      }
    }
  }
  if constexpr (KIND == kRWeigh && KB == 1) {
    if (st.scores && t0 + 32 <= p.score_ld) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        f32x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __builtin_fmaf(s[0][i + k], sl, off);
        *reinterpret_cast<f32x4*>(st.scores + t0 + 2 * i + 4 * h) = x;
      }
    }
  }
  float mx = s[0][0];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(s[kb][i], s[kb][i + 1]), mx);
  // (the halves' keys are four apart, and off with them)
  mx = FORM == kRPlain ? mx * sl : __builtin_fmaf(mx, sl, off);
  mx = fmaxf(mx, half_swap(mx));
  if (__any(mx > st.m + 8.0f)) {
    const float mn = fmaxf(st.m, mx);
    const float a = mn == kNegInf ? 1.0f : exp2f(st.m - mn);
    st.l *= a;
    st.m = mn;
#pragma unroll
    for (int n = 0; n < D / 32; ++n) st.o[n] *= a;
  }
  const float ms = st.m == kNegInf ? 0.0f : st.m - off;
#pragma unroll
  for (int t = 0; t < 2 * KB; ++t) {
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][8 * (t & 1) + i], sl, -ms));
    pr[t] = split_pair<TT>(e);
    st.l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
  }
}

// O^T += V^T P^T over 32 KB keys.
template <typename TT, int D, int KB>
struct RValues {
  using G = RGeom<D>;
  static constexpr int NB = D / 32, N = 2 * KB * NB, A = NB == 3 ? 3 : 4;  // products, of a group
  static_assert(N % A == 0, "whole groups");
  const char* row;
  int vx, sub;
  u32x4 v[2][A];
  __device__ __forceinline__ void read(int g) {
#pragma unroll
    for (int k = 0; k < A; ++k) {
      const int t = (g * A + k) / NB, n = (g * A + k) % NB;
      const char* a = row + ((((4 * n) ^ vx) + sub) << 4);
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(a + t * 16 * G::PITCH));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(a + (t * 16 + 8) * G::PITCH));
      const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
      v[g & 1][k] = u32x4{w0[0], w0[1], w1[0], w1[1]};
    }
  }
  // Reads the first group.
  __device__ __forceinline__ RValues(const char* vt, int lane) {
    const int h = lane >> 5, dh = (lane >> 4) & 1, i = lane & 15;
    // rows 4 h + i / 4 (+ 8) of each 16 keys, dims 32 n + 16 dh + 4 (i % 4) .. + 3
    row = vt + (4 * h + (i >> 2)) * G::PITCH + 8 * (i & 1);
    vx = G::vx(4 * h + (i >> 2));
    sub = 2 * dh + ((i & 3) >> 1);
    read(0);
    r_order();
  }
  __device__ __forceinline__ void multiply(RState<TT, D>& st, const RPair (&pr)[2 * KB]) {
#pragma unroll
    for (int g = 0; g < N / A; ++g) {
      if (g + 1 < N / A) read(g + 1);
      r_order();
#pragma unroll
      for (int k = 0; k < A; ++k)
        st.o[(g * A + k) % NB] = mfma_r<TT>(v[g & 1][k], pr[(g * A + k) / NB].hi, st.o[(g * A + k) % NB]);
#pragma unroll
      for (int k = 0; k < A; ++k)
        st.o[(g * A + k) % NB] = mfma_r<TT>(v[g & 1][k], pr[(g * A + k) / NB].lo, st.o[(g * A + k) % NB]);
      r_order();
    }
  }
};

template <typename TT, int D>
__device__ __forceinline__ void r_queries(const RangedParams& p, const RInfo& q, int lane, RState<TT, D>& st) {
  const char* src = reinterpret_cast<const char*>(p.q) + ((int64_t)q.t * p.num_heads + q.h) * D * 2 +
                    16 * (lane >> 5);
  // Rows beyond the block repeat its first and are not written.  A negative scale goes into the queries'
  // signs (p.scale_log2 has its magnitude).
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) st.q[ks] = ld16(src + 32 * ks) ^ p.qxor;
  st.slope = p.slopes ? p.slopes[q.h] * p.slope_unit : 0.0f;
}
template <typename TT, int D>
__device__ __forceinline__ void r_init(const RInfo& q, RState<TT, D>& st) {
#pragma unroll
  for (int n = 0; n < D / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) st.o[n][i] = 0.0f;
  st.m = kNegInf;
  st.l = 0.0f;
  st.lo = (q.how & kRAny) ? q.lo : 0;
  st.hi = (q.how & kRAny) ? q.hi : 0;
  st.pos = q.pos;
  st.scores = nullptr;
}

// Keys below it lie before every row of the wavefront that sees them (see r_softmax).
template <int FORM>
__device__ __forceinline__ int r_near(const RangedParams& p, const RInfo& q) {
  if (FORM == kRPlain || !p.slopes) return 0;
  return p.causal && !p.prefix_lens ? INT32_MAX : half_min((q.how & kRAny) ? q.pos : INT32_MAX);
}

// ------------------------------------------------------------------------------------ a unit
// The wavefront's rows, final where the unit has all their keys, else as partial rows; returns those that came
// out not finite, which want slow_rows.
template <typename TT, int D, int KIND>
__device__ __forceinline__ uint32_t r_store(const RangedParams& p, const RUnit& u, const RInfo& q, int rl,
                                            const RState<TT, D>& st, float sink, int lane) {
  const int h = lane >> 5;
  const bool any = q.how & kRAny;
  const float l = st.l + half_swap(st.l);
  float sum = 0.0f;  // NaN if an output is not finite
#pragma unroll
  for (int n = 0; n < D / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(st.o[n][i], 0.0f, sum);
  if ((q.how & kRZero) || (any && (q.how & kRSingle))) {
    // (zeros outright: an empty row went through the tiles that the others see, and what it summed may be anything)
    const bool none = q.how & kRZero;
    if constexpr (KIND == kRWeigh)
      if (h == 0) p.row_stats[stat_row(p, q.t, q.h)] = none ? -kNegInf : softmax_stat(st.m, l, sink);
    const float fct = fmaxf(finalize_factor(st.m, l, sink), kRTiny);
    auto four = [&](int n, int i) {
      auto x = [&](int k) { return none ? 0.0f : st.o[n][4 * i + k] * fct; };
      return pack4<TT>(x(0), x(1), x(2), x(3));
    };
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + ((int64_t)q.t * p.num_heads + q.h) * D + 8 * h;
    // (the halves exchange every other four dims, so that each stores eight at a time)
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const u32x2 a = four(n, i), b = four(n, i + 1);
        const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
        *reinterpret_cast<u32x4*>(dst + 32 * n + 8 * i) = u32x4{x[0], y[0], x[1], y[1]};
      }
  } else if (any) {
    const int64_t row = u.slot + rl;
    if (row < p.part_rows) {
#pragma unroll
      for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(p.part_o + row * D + 32 * n + 8 * i + 4 * h) =
              f32x4{st.o[n][4 * i], st.o[n][4 * i + 1], st.o[n][4 * i + 2], st.o[n][4 * i + 3]};
      if (h == 0) p.part_ml[row] = float2{st.m, l};
    }
  }
  // (A sum that is NaN has seen a score that is NaN or infinite: its row is NaN, as it came out.)
  const uint64_t odd = __ballot(any && sum != 0.0f && l == l);
  return (uint32_t)(odd | (odd >> 32));
}

// The rows of `odd` again, a key at a time for all of them, so that a key that a row does not see takes no part
// in it whatever its value; written like the others.  About 1 us per key: a prompt of 8192 with one
// infinite value 37 ms for 0.9 (row by row 800).
template <typename TT, int D, int KIND>
__device__ __forceinline__ void slow_rows(const RangedParams& p, const RUnit& u, RInfo q, int rl, uint32_t odd) {
  const int lane = hidden(threadIdx.x & 63), h = lane >> 5;
  if (!((odd >> (lane & 31)) & 1)) q.how = 0;
  RState<TT, D> st;
  r_queries<TT, D>(p, q, lane, st);
  r_init<TT, D>(q, st);
  const float sink = r_sink<TT>(p, q.h), slope = p.slopes ? p.slopes[q.h] : 0.0f, scale = fabsf(p.scale);
  const bool any = q.how & kRAny;
  const int k0 = half_min(any ? q.lo : INT32_MAX), k1 = half_max(any ? q.hi : 0);
#pragma unroll 1
  for (int j = k0; j < k1; ++j) {
    const int64_t at = r_offset(p, u.s.b0, u.kh, j, D);
    const uint16_t* kr = reinterpret_cast<const uint16_t*>(p.key_cache) + at + 8 * h;
    const uint16_t* vr = reinterpret_cast<const uint16_t*>(p.value_cache) + at + 4 * h;
    float x = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(kr + 16 * ks);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x = __builtin_fmaf(TT::to_f32((uint16_t)k[i]), TT::to_f32((uint16_t)st.q[ks][i]), x);
        x = __builtin_fmaf(TT::to_f32((uint16_t)(k[i] >> 16)), TT::to_f32((uint16_t)(st.q[ks][i] >> 16)), x);
      }
    }
    x = (x + half_swap(x)) * scale;
    if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
    x = (x - slope * fabsf((float)(q.pos - j))) * kLog2e;
    bool seen = j >= st.lo && j < st.hi && x != kNegInf;
    if constexpr (KIND == kRTree) seen = seen && (tree_mask(p, q, j - q.past) & 1u);
    const float mn = seen ? fmaxf(st.m, x) : st.m, ms = mn == kNegInf ? 0.0f : mn;
    const float a = st.m == kNegInf ? 0.0f : fmaxf(exp2f(st.m - ms), kRTiny);
    const float w = seen ? fmaxf(exp2f(x - ms), kRTiny) : 0.0f;
    st.l = st.l * a + (h == 0 ? w : 0.0f);  // (the halves' sums are added)
    st.m = mn;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(vr + 32 * n + 2 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = TT::to_f32((uint16_t)(v[e >> 1] >> (16 * (e & 1))));
          st.o[n][i + e] = st.o[n][i + e] * a + (seen ? w * y : 0.0f);
        }
      }
  }
  r_store<TT, D, KIND>(p, u, q, rl, st, sink, lane);
}

// A block of 128 rows, by the whole workgroup: wavefront w takes rows 32 w .. 32 w + 31 of every tile.
template <typename TT, int D, int FORM, int KIND>
__device__ __forceinline__ uint32_t wide_unit(const RangedParams& p, const RUnit& u, char* lds, RScan& sh,
                                              RInfo& q) {
  using G = RGeom<D>;
  constexpr int KB = G::KT / 32, SIDE = G::KT * G::PITCH;
  const int wave = uniform(threadIdx.x >> 6), lane = hidden(threadIdx.x & 63);
  const int rl = 32 * wave + (lane & 31);
  RState<TT, D> st;
  q = r_place(p, u, rl);
  r_queries<TT, D>(p, q, lane, st);
  const float sink = r_sink<TT>(p, q.h);
  r_keys<KIND>(p, u, rl, q);
  const bool any = q.how & kRAny;
  r_init<TT, D>(q, st);
  // keys that some / every row of the wavefront sees, and some row of the workgroup
  const int wlo = half_min(any ? q.lo : INT32_MAX), whi = half_max(any ? q.hi : 0);
  const int flo = half_max(any ? q.lo : 0), fhi = half_min(any ? q.hi : INT32_MAX);
  const int near = r_near<FORM>(p, q);
  const int past = KIND == kRTree ? uniform(q.past) : 0;
  __syncthreads();  // the last unit's readers are done
  if (lane == 0) {
    sh.red[2 * wave] = wlo;
    sh.red[2 * wave + 1] = whi;
  }
  __syncthreads();
  constexpr int GR = G::KT / 4;  // a wavefront's rows of a tile
  RFeed<D, GR> f;
  f.begin(p, u.s.b0, u.kh, wave * GR & 15, lane);
  f.kmin = uniform(min(min(sh.red[0], sh.red[2]), min(sh.red[4], sh.red[6])));
  f.kmax = uniform(max(max(sh.red[1], sh.red[3]), max(sh.red[5], sh.red[7])));
  if (f.kmin < f.kmax) {
    const int tb = f.kmin / G::KT, te = (f.kmax + G::KT - 1) / G::KT;
    const uint32_t base = lds_address(lds) + wave * GR * G::PITCH;
    int pg = f.page(tb * G::KT + wave * GR);  // of the tile to be loaded next
    // iteration t loads tile t + 1 and multiplies tile t (none in the first)
    for (int t = tb - 1; t < te; ++t) {
      if (t >= tb) wait_loads<0>();
      barrier();
      // (at once: between the products they cost more, 735 us for 627 over a prompt of 8192 at head 256,
      // with one part of the probabilities)
      if (t + 1 < te) {
        const uint32_t put = base + ((t + 1 - tb) & 1) * 2 * SIDE;
        const int pos = (t + 1) * G::KT + wave * GR;
        f.template load<true, true, false>(pos, pg, put, put + SIDE, wave * GR & 15, lane);
        pg = f.page(pos + G::KT);
      }
      const int t0 = t * G::KT;
      if (t < tb || t0 >= whi || t0 + G::KT <= wlo) continue;
      const char* buf = lds + ((t - tb) & 1) * 2 * SIDE;
      f32x16 s[KB];
      RPair pr[2 * KB];
      uint32_t tw[KB];
      const bool tree = KIND == kRTree && t0 + G::KT > past;
      if constexpr (KIND == kRTree) {
        if (tree) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) tw[kb] = tree_mask(p, q, t0 + 32 * kb - past);
        }
      }
      r_scores<TT, D, KB>(st, buf, lane, s);
      RValues<TT, D, KB> v(buf + SIDE, lane);
      r_softmax<TT, D, KB, FORM, KIND>(p, st, s, t0, t0 < flo, t0 + G::KT > fhi, t0 + G::KT <= near, lane, pr, tree,
                                       tw);
      v.multiply(st, pr);
    }
  }
  return r_store<TT, D, KIND>(p, u, q, rl, st, sink, lane);
}

// At most 32 rows, by one wavefront on 32-key tiles in `mine`.
template <typename TT, int D, int FORM, int KIND>
__device__ __forceinline__ uint32_t narrow_unit(const RangedParams& p, const RUnit& u, char* mine, RInfo& q) {
  using G = RGeom<D>;
  constexpr int SIDE = 32 * G::PITCH, NI = 32 / G::RPI;
  const int lane = hidden(threadIdx.x & 63), rl = lane & 31;
  RState<TT, D> st;
  q = r_place(p, u, rl);
  r_queries<TT, D>(p, q, lane, st);
  const float sink = r_sink<TT>(p, q.h);
  r_keys<KIND>(p, u, rl, q);
  const bool any = q.how & kRAny;
  r_init<TT, D>(q, st);
  RFeed<D, 16> f;
  f.begin(p, u.s.b0, u.kh, 0, lane);
  f.kmin = half_min(any ? q.lo : INT32_MAX);
  f.kmax = half_max(any ? q.hi : 0);
  const int flo = half_max(any ? q.lo : 0), fhi = half_min(any ? q.hi : INT32_MAX);
  const int near = r_near<FORM>(p, q);
  const int past = KIND == kRTree ? uniform(q.past) : 0;
  if constexpr (KIND == kRWeigh) {
    // the scores of rows that count
    const int g = p.num_heads / p.kv_heads, tokens = u.s.rows / g;
    st.scores = p.scores && any && q.t - u.s.tok0 >= (p.observed > 0 ? tokens - p.observed : 0)
                    ? p.scores + stat_row(p, q.t, q.h) * p.score_ld
                    : nullptr;
  }
  if (f.kmin < f.kmax) {
    const int tb = f.kmin / 32, te = (f.kmax + 31) / 32;
    const uint32_t base = lds_address(mine);
    wait_lds_reads();
    int p0 = f.page(tb * 32), p1 = f.page(tb * 32 + 16);  // pages of the tile to be loaded next
    constexpr int HALF = 16 * G::PITCH;
    // iteration t loads tile t + 1 and multiplies tile t (none in the first)
    for (int t = tb - 1; t < te; ++t) {
      const bool more = t + 1 < te, have = t >= tb;
      const int t0 = t * 32;
      f32x16 s[1];
      RPair pr[2];
      uint32_t tw[1];
      const bool tree = KIND == kRTree && have && t0 + 32 > past;
      if (tree) tw[0] = tree_mask(p, q, t0 - past);
      if (have) {
        wait_loads<NI>();  // the keys; the values are younger
        r_scores<TT, D, 1>(st, mine, lane, s);
        wait_lds_reads();
      }
      if (more) {
        f.template load<true, false, true>(t0 + 32, p0, base, 0, 0, lane);
        f.template load<true, false, true>(t0 + 48, p1, base + HALF, 0, 0, lane);
      }
      if (have) {
        r_softmax<TT, D, 1, FORM, KIND>(p, st, s, t0, t0 < flo, t0 + 32 > fhi, t0 + 32 <= near, lane, pr, tree,
                                         tw);
        if (more)
          wait_loads<NI>();
        else
          wait_loads<0>();
        RValues<TT, D, 1>(mine + SIDE, lane).multiply(st, pr);
        wait_lds_reads();
      }
      if (more) {
        f.template load<false, true, true>(t0 + 32, p0, 0, base + SIDE, 0, lane);
        f.template load<false, true, true>(t0 + 48, p1, 0, base + SIDE + HALF, 0, lane);
        p0 = f.page(t0 + 64);
        p1 = f.page(t0 + 80);
      }
    }
  }
  return r_store<TT, D, KIND>(p, u, q, rl, st, sink, lane);
}

// WIDE: the batch may have wide items.
// Workgroups per CU: two by LDS and registers, three at head 64, one at head 256.
template <typename TT, int D, int FORM, bool WIDE, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : D == 64 ? 3 : 2))) void
ranged_kernel(const RangedParams p) {
  constexpr int kMine = 2 * 32 * RGeom<D>::PITCH;  // a wavefront's tile
  __shared__ __attribute__((aligned(1024))) char
      lds[WIDE && RGeom<D>::WIDE > 4 * kMine ? RGeom<D>::WIDE : 4 * kMine];
  __shared__ RScan sh;
  const int n = p.groups + p.batch, chunks = (n + kRChunk - 1) / kRChunk;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // Pass 0 adds up tiles and items of all sources, pass 1 walks them; both at once if one chunk has them all.
  RTotals t{}, tb{};
  RShare r{};
  int me = 0, per = 0, kind = 0, at = 0, end = 0, stride = 0, turn = 0;
  bool queued = false;
  for (int c = chunks > 1 ? -chunks : 0; c < chunks; ++c) {
    const int base = (c < 0 ? c + chunks : c) * kRChunk;
    tb = t;
    scan_chunk(p, base, sh, t);
    if (c < -1) continue;
    if (c == -1 || chunks == 1) {
      r = r_share<KIND>(p, t);
      kind = (int)blockIdx.x < r.wide ? 0 : 1;
      queued = p.queue && kind == 0 && r.per[0] == 0;
      me = kind ? ((int)blockIdx.x - r.wide) * 4 + wave : (int)blockIdx.x;
      per = kind ? r.per[1] : r.per[0];
      // my stretch of tiles, or my first item
      at = per > 0 ? me * per : me;
      end = per > 0 ? min(at + per, pick(t.tiles, kind)) : pick(t.items, kind);
      stride = kind ? (p.slots - r.wide) * 4 : r.wide;
      // the sources' places, for the merge
      if (blockIdx.x == 0 && threadIdx.x == 0) p.table[0] = RTable{{r.per[0], r.per[1]}};
      if (c == -1) {
        t = RTotals{};
        continue;
      }
    }
    if (blockIdx.x == 0 && base + (int)threadIdx.x < n) {
      const RSource s = sh.src[threadIdx.x];
      p.table[1 + base + threadIdx.x] =
          RTable{{s.first, s.item, s.tok0, s.rows, s.b0, s.b1, s.ka, s.kb, s.base, s.shared, s.group, 0}};
    }
    // The parts of mine that this chunk's sources hold
    for (;;) {
      if (per > 0) {
        if (at >= min(end, pick(t.tiles, kind))) break;
      } else if (queued) {
        if (at >= t.items[0]) break;
      } else {
        // whole items in turns; wide ones alternately up and down the list, in runs of eight (neighbours share
        // keys, and runs keep them on their XCD)
        bool found = false;
        for (; turn * stride < end && !found; ++turn) {
          const bool back = kind == 0 && (turn & 1) && (stride & 7) == 0;
          at = turn * stride + (back ? (stride - 8 - (me & ~7)) + (me & 7) : me);
          found = at >= pick(tb.items, kind) && at < pick(t.items, kind);
        }
        if (!found) {
          turn = 0;  // (the next chunk looks from the first turn on)
          break;
        }
      }
      // its source: every lane looks at a few
      int si = 0;
      for (int b0 = 0; b0 < min(kRChunk, n - base); b0 += 64) {
        const RSource& s = sh.src[b0 + (threadIdx.x & 63)];
        const int blocks = r_blocks(s);
        const int first = per > 0 ? s.first : s.item;
        const int size = p.kv_heads * (per > 0 ? r_before(s, blocks, p.num_heads / p.kv_heads, r_grows(p, s)) : blocks);
        const uint64_t hit = __ballot(b0 + (int)(threadIdx.x & 63) < n - base && r_wide(s) == (kind == 0) &&
                                      at >= first && at - first < size);
        if (hit) {
          si = b0 + __builtin_ctzll(hit);
          break;
        }
      }
      RUnit u;
      const RSource sl = sh.src[si];
      u.s = RSource{uniform(sl.first), uniform(sl.item), uniform(sl.tok0), uniform(sl.rows),
                    uniform(sl.b0),    uniform(sl.b1),   uniform(sl.ka),   uniform(sl.kb),
                    uniform(sl.base),  uniform(sl.shared), uniform(sl.group)};
      u.group = u.s.group < -1;
      const int g = p.num_heads / p.kv_heads;
      int blk, kh;
      if (per > 0) {
        // the last block that begins at or before the place
        const int rel = at - u.s.first;
        const bool grows = r_grows(p, u.s);
        int lo = 0, hi = r_blocks(u.s);
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (p.kv_heads * r_before(u.s, mid, g, grows) <= rel) lo = mid; else hi = mid;
        }
        blk = lo;
        const int f = r_before(u.s, blk, g, grows);
        kh = (rel - p.kv_heads * f) / (r_before(u.s, blk + 1, g, grows) - f);
      } else {
        blk = r_blocks(u.s) - 1 - (at - u.s.item) / p.kv_heads;  // the rows that see most keys first
        kh = (at - u.s.item) % p.kv_heads;
      }
      blk = uniform(blk);
      kh = uniform(kh);
      const RItem it = r_item(p, u.s, blk, kh);
      u.kh = kh;
      u.row0 = blk * kRWide;
      const int x0 = per > 0 ? at - it.at : 0, kt = u.s.ka / kRTile;
      const int x1 = per > 0 ? min(it.size, end - it.at) : it.size;
      if (per > 0) at = it.at + x1;
      if (x1 <= kRStart) continue;  // (the places of its start alone)
      u.head = x0 <= kRStart;
      u.k0 = u.head ? 0 : (kt + x0 - kRStart) * kRTile;
      u.k1 = x1 == it.size ? INT32_MAX : (kt + x1 - kRStart) * kRTile;
      u.slot = r_slot(p, kind, per > 0 ? me : 0, it.item, u.head);
      RInfo q;
      uint32_t odd;
      bool wide = false;
      if constexpr (WIDE) wide = kind == 0;
      // The next one from the queue: eight queues, of every eighth item each, so that neighbours, which share keys,
      // keep their XCDs.
      const int queues = (r.wide & (kRQueues - 1)) == 0 ? kRQueues : 1, mine = me & (queues - 1);
      int ticket = 0;
      if (queued && threadIdx.x == 0) ticket = atomicAdd(p.queue + mine * kRQueueStep, 1);
      if (wide)
        odd = wide_unit<TT, D, FORM, KIND>(p, u, lds, sh, q);
      else
        odd = narrow_unit<TT, D, FORM, KIND>(p, u, lds + wave * kMine, q);
      // rows that came out not finite, again
      if (odd) slow_rows<TT, D, KIND>(p, u, q, (wide ? 32 * wave : 0) + (lane & 31), odd);
      if (queued) {
        if (threadIdx.x == 0) sh.next = r.wide + queues * ticket + mine;
        __syncthreads();
        at = uniform(sh.next);
      }
    }
  }
}

// ------------------------------------------------------------------------------------ the merge
// Rows whose keys several workers took: their (m, l, O) joined.  A row's pieces are those of the workers from the
// one that holds its first key to the one that holds its last, for the shared keys and for its own.
struct RPieces {
  int n;             // pieces
  int64_t first;     // the first one's partial row
  int64_t next, step;  // piece k > 0: next + k * step
};
struct RJoin {
  RPieces a, b;      // of the shared and of its own keys
  __device__ __forceinline__ int64_t row(int k) const {
    const RPieces& q = k < a.n ? a : b;
    const int y = k < a.n ? k : k - a.n;
    return y == 0 ? q.first : q.next + y * q.step;
  }
};
template <int KIND>
__device__ __forceinline__ RJoin r_join(const RangedParams& p, int t, int h, int b, const int (&per)[2]) {
  const int g = p.num_heads / p.kv_heads, kh = h / g;
  auto source = [&](int i) {
    const RTable e = p.table[1 + i];
    return RSource{e.v[0], e.v[1], e.v[2], e.v[3], e.v[4], e.v[5], e.v[6], e.v[7], e.v[8], e.v[9], e.v[10]};
  };
  const RSource own = source(p.groups + b);
  const RRange r = r_range<KIND>(p, t, own.kb - own.rows / g + (t - own.tok0), b, own.kb,
                                 KIND == kRTree && p.window > 0 ? p.tree_lag[t] : 0);
  auto pieces = [&](const RSource& e, int a, int z) {
    const int kind = r_wide(e) ? 0 : 1, pr = pick(per, kind);
    const int rr = (t - e.tok0) * g + h - kh * g, blk = kind ? 0 : rr / kRWide, kt = e.ka / kRTile;
    const RItem it = r_item(p, e, blk, kh);
    const int w0 = r_worker(pr, it, a / kRTile - kt), w1 = r_worker(pr, it, (z - 1) / kRTile - kt);
    const int rl = rr - blk * kRWide;
    RPieces q;
    q.n = w1 - w0 + 1;
    q.first = r_slot(p, kind, w0, it.item, w0 == r_worker(pr, it, 0)) + rl;
    q.next = r_slot(p, kind, w0, it.item, false) + rl;
    q.step = r_slot(p, kind, w0 + 1, it.item, false) + rl - q.next;
    if (q.first >= p.part_rows || q.next + (q.n - 1) * q.step >= p.part_rows) q.n = 0;  // (metadata beyond its bounds)
    return q;
  };
  RJoin j{};
  const int sh_hi = min(r.hi, own.shared), own_lo = max(r.lo, own.shared);
  if (r.lo < sh_hi) j.a = pieces(source(own.group), r.lo, sh_hi);
  if (own_lo < r.hi) j.b = pieces(own, own_lo, r.hi);
  return j;
}
// (m, l) and four elements of a row from the pieces, and the join of two of them.
struct RSum {
  float m, l;
  f32x4 o;
  __device__ __forceinline__ void meet(float m2, float l2, f32x4 o2) {
    const float mn = fmaxf(m, m2);
    const float wa = m == kNegInf ? 0.0f : fmaxf(exp2f(m - mn), kRTiny);
    const float wb = m2 == kNegInf ? 0.0f : fmaxf(exp2f(m2 - mn), kRTiny);
    // (pieces whose scores are all NaN have no maximum, but a sum)
    l = (l == l ? l * wa : l) + (l2 == l2 ? l2 * wb : l2);
    o = o * wa + o2 * wb;
    m = mn;
  }
};
constexpr int kRDepth = 4;
// Pieces k0, k0 + stride, ... of a row, several in flight.
__device__ __forceinline__ RSum r_pieces(const RangedParams& p, const RJoin& j, int k0, int stride, int D, int d0) {
  RSum s{kNegInf, 0.0f, f32x4{0.f, 0.f, 0.f, 0.f}};
  const int n = j.a.n + j.b.n;
  for (int i0 = k0; i0 < n; i0 += stride * kRDepth) {
    float2 ml[kRDepth];
    f32x4 o[kRDepth];
#pragma unroll
    for (int i = 0; i < kRDepth; ++i) {
      const int64_t row = j.row(min(i0 + i * stride, n - 1));
      ml[i] = p.part_ml[row];
      o[i] = *reinterpret_cast<const f32x4*>(p.part_o + row * D + d0);
    }
    float mn = s.m;
#pragma unroll
    for (int i = 0; i < kRDepth; ++i)
      if (i0 + i * stride < n) mn = fmaxf(mn, ml[i].x);
    const float a = s.m == kNegInf ? 0.0f : fmaxf(exp2f(s.m - mn), kRTiny);
    s.l = s.l == s.l ? s.l * a : s.l;
    s.o *= a;
#pragma unroll
    for (int i = 0; i < kRDepth; ++i)
      if (i0 + i * stride < n) {
        const float w = ml[i].x == kNegInf ? 0.0f : fmaxf(exp2f(ml[i].x - mn), kRTiny);
        s.l += ml[i].y == ml[i].y ? ml[i].y * w : ml[i].y;
        s.o += o[i] * w;
      }
    s.m = mn;
  }
  return s;
}
template <typename TT, int KIND>
__device__ __forceinline__ void r_finish(const RangedParams& p, const RSum& s, int64_t t, int h, int D, int d0) {
  const float f = s.l == s.l ? fmaxf(finalize_factor(s.m, s.l, r_sink<TT>(p, h)), kRTiny) : s.l;
  if constexpr (KIND == kRWeigh)
    if (d0 == 0) p.row_stats[stat_row(p, t, h)] = softmax_stat(s.m, s.l, r_sink<TT>(p, h));
  *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + (t * p.num_heads + h) * D + d0) =
      pack4<TT>(s.o[0] * f, s.o[1] * f, s.o[2] * f, s.o[3] * f);
}

// Few rows: NW wavefronts per row, whose groups of lanes (16 bytes of the row per lane) take pieces in turn and meet
// through lane exchanges and, with four wavefronts, LDS.  Bound by its chain of loads.
template <typename TT, int D, int NW, int KIND>
__global__ __launch_bounds__(256) void ranged_join_kernel(const RangedParams p) {
  constexpr int LP = D == 96 ? 32 : D / 4, NG = 64 / LP * NW;
  __shared__ f32x4 sh_o[NW > 1 ? 4 : 1][LP];
  __shared__ float2 sh_ml[NW > 1 ? 4 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int64_t row = (int64_t)blockIdx.x * (4 / NW) + (NW > 1 ? 0 : wave);
  const int t = uniform((int)(row / p.num_heads)), h = uniform((int)(row % p.num_heads));
  if (t >= p.num_tokens) return;
  const int per[2] = {p.table[0].v[0], p.table[0].v[1]};
  const int c0 = p.cum[0], c1 = p.cum[p.batch];
  const int b = uniform(seq_of_token(p.cum, p.batch, t));
  if (t < c0 || t >= c1 || (per[0] == 0 && per[1] == 0 && p.groups == 0)) return;
  const RJoin j = r_join<KIND>(p, t, h, b, per);
  if (j.a.n + j.b.n < 2) return;
  const int d0 = 4 * min(lane % LP, D / 4 - 1);
  RSum s = r_pieces(p, j, (NW > 1 ? wave * (64 / LP) : 0) + lane / LP, NG, D, d0);
#pragma unroll
  for (int o = LP; o < 64; o <<= 1)
    s.meet(__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64),
           f32x4{__shfl_xor(s.o[0], o, 64), __shfl_xor(s.o[1], o, 64), __shfl_xor(s.o[2], o, 64),
                 __shfl_xor(s.o[3], o, 64)});
  if constexpr (NW > 1) {
    if (lane < LP) sh_o[wave][lane] = s.o;
    if (lane == 0) sh_ml[wave] = float2{s.m, s.l};
    __syncthreads();
    if (wave > 0 || lane >= LP) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) s.meet(sh_ml[w].x, sh_ml[w].y, sh_o[w][lane]);
  }
  if (lane < D / 4) r_finish<TT, KIND>(p, s, t, h, D, d0);
}

// Many rows: workgroups take 32 rows (token, head of the group) of a kv-head at a time; thread k finds the pieces of
// row k, then groups of lanes sum a row each.
template <typename TT, int D, int KIND>
__global__ __launch_bounds__(256) void ranged_merge_kernel(const RangedParams p, int blocks) {
  constexpr int LP = D == 96 ? 32 : D / 4, NG = 256 / LP, RM = 32;
  __shared__ RJoin join[RM];
  __shared__ int2 place[RM];
  const int per[2] = {p.table[0].v[0], p.table[0].v[1]};
  if (per[0] == 0 && per[1] == 0 && p.groups == 0) return;
  const int tid = threadIdx.x, g = p.num_heads / p.kv_heads;
  for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int kh = blk % p.kv_heads;
    if (tid < RM) {
      const int64_t gr = (int64_t)(blk / p.kv_heads) * RM + tid;
      const int t = (int)min(gr / g, (int64_t)p.num_tokens), h = kh * g + (int)(gr % g);
      RJoin j{};
      if (t < p.num_tokens && t >= p.cum[0] && t < p.cum[p.batch])
        j = r_join<KIND>(p, t, h, r_token_seq(p, 0, p.batch, t), per);
      join[tid] = j;
      place[tid] = int2{t, h};
    }
    __syncthreads();
    const int d0 = 4 * min(tid % LP, D / 4 - 1);
    for (int k = tid / LP; k < RM; k += NG) {
      const RJoin j = join[k];
      if (j.a.n + j.b.n < 2) continue;
      const RSum s = r_pieces(p, j, 0, 1, D, d0);
      if (tid % LP < D / 4) r_finish<TT, KIND>(p, s, place[k].x, place[k].y, D, d0);
    }
    __syncthreads();
  }
}

[[maybe_unused]] __global__ __launch_bounds__(64) void ranged_queue_kernel(const RangedParams p) {
  if (threadIdx.x < kRQueues) p.queue[threadIdx.x * kRQueueStep] = 0;
}

template <typename TT, int D, int FORM, int KIND>
void launch_f(const RangedParams& p, hipStream_t s) {
  if (p.wide)
    hipLaunchKernelGGL((ranged_kernel<TT, D, FORM, true, KIND>), dim3(p.slots), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((ranged_kernel<TT, D, FORM, false, KIND>), dim3(p.slots), dim3(256), 0, s, p);
}

template <typename TT, int D, int KIND>
hipError_t launch_d(const RangedParams& p, hipStream_t s) {
  const dim3 block(256);
  if (KIND == kRRanges && p.queue) hipLaunchKernelGGL(ranged_queue_kernel, dim3(1), dim3(64), 0, s, p);
  if (p.softcap > 0.0f) {
    launch_f<TT, D, kRCap, KIND>(p, s);
  } else if (!p.slopes) {
    launch_f<TT, D, kRPlain, KIND>(p, s);
  } else {
    if constexpr (KIND == kRRanges)  // (the other kinds take no slopes)
      launch_f<TT, D, kRSlope, KIND>(p, s);
    else
      return hipErrorInvalidValue;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.merge) return e;
  const int64_t rows = (int64_t)p.num_tokens * p.num_heads;
  if (rows <= kRJoinWide) {
    hipLaunchKernelGGL((ranged_join_kernel<TT, D, 4, KIND>), dim3((unsigned)rows), block, 0, s, p);
  } else if (rows <= kRJoinRows) {
    hipLaunchKernelGGL((ranged_join_kernel<TT, D, 1, KIND>), dim3((unsigned)((rows + 3) / 4)), block, 0, s, p);
  } else {
    const int blocks = (int)((rows / p.kv_heads + 31) / 32 * p.kv_heads);
    hipLaunchKernelGGL((ranged_merge_kernel<TT, D, KIND>), dim3((unsigned)std::min(blocks, kRMergeGrid)), block, 0, s,
                       p, blocks);
  }
  return hipGetLastError();
}

template <typename TT, int KIND>
hipError_t launch_t(const RangedParams& p, hipStream_t s) {
  switch (p.head_dim) {
    case 64: return launch_d<TT, 64, KIND>(p, s);
    case 96: return launch_d<TT, 96, KIND>(p, s);
    case 128: return launch_d<TT, 128, KIND>(p, s);
    case 256: return launch_d<TT, 256, KIND>(p, s);
    default: return hipErrorInvalidValue;
  }
}

template <int KIND>
hipError_t launch_kind(const RangedParams& p, pa_dtype act, hipStream_t s) {
  if (p.num_tokens <= 0 || p.batch <= 0) return hipSuccess;
  if (p.slots <= 0 || !p.table) return hipErrorInvalidValue;
  return act == PA_DTYPE_FLOAT16 ? launch_t<TF16, KIND>(p, s) : launch_t<TBF16, KIND>(p, s);
}

}  // namespace
}  // namespace pa
