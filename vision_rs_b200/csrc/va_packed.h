// Work lists of the packed-sequence attention: what the plan kernel writes and
// the forward and backward kernels read (va_packed_plan.cu, va_packed_attn.cu,
// va_packed_attn_bwd.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace va {

constexpr int kPackBlock = 128;   // keys (and rows of a tile) a step
// The largest part of a tile is at least so many key blocks (forward) or query steps (dK/dV); a tile a little longer is cut
// in two, so parts are at least half of that.  Measured (graph replays, plan built before): 4 single tokens, 32/8 heads of 128,
// over 7, 8, 9 and 11 blocks 13.5, 14.1, 15.3 and 17.0 us, 15.3, 17.0, 18.4 and 21.9 with no part below the constant; 64
// tokens, whose tiles fill the GPU uncut, over 8 and 11 blocks 64.9 and 82.0 us against 50.8 and 66.6.  Backward of 2
// documents of 50 steps, 16 heads of 128: 361 against 378.
constexpr int kMinKeyBlocks = 6, kMinQuerySteps = 32;
constexpr int kMaxSeqs = 1 << 20;
constexpr int kPlanSeqs = 2048;   // sequences whose tile counts fit the plan kernel's shared memory

// One unit of forward or dQ work: up to `tokens` queries of one sequence
// against its key blocks [kb0, kb1).  Query t of the unit sees keys
// j ≤ see + t (not causal: all `lk` of them).
struct alignas(16) QItem {
  int q0, tokens;   // first query (row of the packed tensor) and their number
  int k0, lk;       // the sequence's first key (row of the packed tensor) and its length
  int see;          // causal: last key that query 0 sees
  int kb0, kb1;     // key blocks
  int slot;         // partial result's slot, -1: the unit is the whole tile and writes the output
  int slot0, parts; // the tile's first slot and number of parts
  int counter;      // the tile's arrival counter
  int pad;
};
// One unit of dK/dV work: up to 128 keys of one sequence and key head against
// steps [h0, h1) of those that see them: step h is 64 queries of head h / nh of
// the group, nh steps a head from the first that sees a key of the unit on.
struct alignas(16) KItem {
  int k0, keys;     // first key (row of the packed tensor) and their number
  int j0;           // its index in the sequence
  int q0, lq, lk;   // the sequence's first query (row) and lengths
  int h0, h1;
  int slot, slot0, parts, counter;  // as a QItem's
};

// Sizes that host and device agree on, from the call's sizes alone.
struct PackedShape {
  int num_seqs, total_q, total_k, heads, kv_heads, dim, causal, training;
  int group;        // query heads a key head
  // Forward: rows of a 128-row tile are the queries of one head, two tiles a
  // unit (few = 0), or (query, head of the group) pairs, one tile a unit
  // with its keys split over units (few = 1).
  int few;
  int tile_rows;    // few: rows of a tile that hold anything, 128 or 32
  int q_tile;       // queries a forward unit
  int units;        // heads (or key heads) that each forward unit is run for
  int max_tiles, max_items, max_slots, split_budget;
  int max_dq_items, max_dkv_tiles, max_dkv_items, dkv_budget;
  // byte offsets in the plan
  size_t items, dq_items, dkv_items, counters, dkv_counters, scratch, part_o, part_lse, part_dkv, rows, do_norm,
      v_norm, total;
};

// Header words of the plan, one of each for the three lists: the number of
// units, and whether the sequences' offsets had to be clamped.
enum { kHdrItems = 0, kHdrDq = 1, kHdrDkv = 2, kHdrBad = 4 };

inline size_t pk_align(size_t x) { return (x + 255) & ~(size_t)255; }

inline PackedShape packed_shape(int num_seqs, int total_q, int total_k, int heads, int kv_heads, int dim, int causal,
                                int training) {
  PackedShape s{};
  s.num_seqs = num_seqs, s.total_q = total_q, s.total_k = total_k;
  s.heads = heads, s.kv_heads = kv_heads, s.dim = dim, s.causal = causal, s.training = training;
  s.group = heads / kv_heads;
  // One tile of (query, head) rows a unit when the sequences' queries are few on
  // average, or when units of 256 queries would leave SMs idle.
  const long long big = ((long long)total_q / 256 + num_seqs) * heads;
  s.few = (long long)total_q * s.group <= 128LL * num_seqs || big < 148 ? 1 : 0;
  // Single tokens and the like: 32 rows a tile leave shared memory for a third K or V block on its way.
  s.tile_rows = s.few && s.group <= 32 && (long long)total_q * s.group <= 32LL * num_seqs ? 32 : kPackBlock;
  s.q_tile = s.few ? s.tile_rows / s.group : 2 * kPackBlock;
  s.units = s.few ? kv_heads : heads;
  s.max_tiles = (int)std::min<long long>((total_q + s.q_tile - 1) / s.q_tile + (long long)num_seqs, total_q);
  // Parts over the number of tiles: about two units for each place a CTA has on the GPU (forward), one an SM (dK/dV, whose
  // parts are larger to join: 507 us for a causal step of 10 k tokens against 516 with half as many more and 520 with
  // twice, in short bursts; under sustained load the step takes 546), and no more than the longest possible tiles allow (none where no tile can pass the smallest part).
  auto budget = [](int most, long long tiles, long long longest, int smallest) {
    return longest <= smallest ? 0 : (int)std::min<long long>(most, (tiles * longest + smallest - 1) / smallest);
  };
  s.split_budget =
      s.few ? budget((592 + s.units - 1) / s.units, s.max_tiles, ((long long)total_k + 127) / 128, kMinKeyBlocks) : 0;
  s.max_items = s.max_tiles + s.split_budget;
  s.max_slots = 2 * s.split_budget;
  s.max_dq_items = training ? (int)std::min<long long>((total_q + 127) / 128 + (long long)num_seqs, total_q) : 0;
  s.max_dkv_tiles = training ? (int)std::min<long long>((total_k + 127) / 128 + (long long)num_seqs, total_k) : 0;
  s.dkv_budget = training ? budget((148 + kv_heads - 1) / kv_heads, s.max_dkv_tiles,
                                   ((long long)total_q + 63) / 64 * s.group, kMinQuerySteps)
                          : 0;
  s.max_dkv_items = s.max_dkv_tiles + s.dkv_budget;
  size_t o = 256;
  s.items = o, o += pk_align((size_t)s.max_items * sizeof(QItem));
  s.dq_items = o, o += pk_align((size_t)s.max_dq_items * sizeof(QItem));
  s.dkv_items = o, o += pk_align((size_t)s.max_dkv_items * sizeof(KItem));
  s.counters = o, o += pk_align(s.few ? (size_t)s.max_tiles * s.units * 4 : 0);
  s.dkv_counters = o, o += pk_align((size_t)s.max_dkv_tiles * kv_heads * 4);
  s.scratch = o, o += pk_align(num_seqs > kPlanSeqs ? (size_t)3 * (num_seqs + 1) * 4 : 0);
  s.part_o = o, o += pk_align((size_t)s.max_slots * s.units * s.tile_rows * dim * 4);
  s.part_lse = o, o += pk_align((size_t)s.max_slots * s.units * s.tile_rows * 4);
  s.part_dkv = o, o += pk_align((size_t)2 * s.dkv_budget * kv_heads * 2 * kPackBlock * dim * 4);
  // training: (lse·log2 e, Δ) a query and head, ‖dO_i‖ and ‖V_j‖ (the f16 backward's)
  s.rows = o, o += pk_align(training ? (size_t)total_q * heads * 8 : 0);
  s.do_norm = o, o += pk_align(training ? (size_t)total_q * heads * 4 : 0);
  s.v_norm = o, o += pk_align(training ? (size_t)total_k * kv_heads * 4 : 0);
  s.total = o;
  return s;
}

// The plan's arithmetic (host and device).  Sums over tiles may need 64 bits: the dK/dV steps of one document of 2^20 tokens
// with 32 query heads over one key head already add up to 2^31 (packed_sums_wide).
#ifdef __CUDACC__
#define VA_PACKED_FN __host__ __device__ __forceinline__
#else
#define VA_PACKED_FN inline
#endif
using PackedSum = long long;
VA_PACKED_FN int pk_min(int a, int b) { return a < b ? a : b; }
VA_PACKED_FN int pk_max(int a, int b) { return a > b ? a : b; }
// Key blocks that the queries [i0, i0 + n) of a sequence see.
VA_PACKED_FN int key_blocks(int lq, int lk, int i0, int n, int causal) {
  const int end = causal ? pk_min(lk, pk_max(0, lk - (lq - i0 - n))) : lk;
  return (end + kPackBlock - 1) / kPackBlock;
}
// Steps of 64 queries, over the heads of a group, that see any of the keys from j0 on.
VA_PACKED_FN int query_steps(int lq, int lk, int j0, int causal, int group) {
  const int first = causal ? pk_max(0, j0 - (lk - lq)) / 64 : 0;
  return pk_max(0, (lq + 63) / 64 - first) * group;
}
// Largest part of a tile, for `blocks` blocks in all: Σ ceil(b / part) ≤ tiles + blocks / part ≤ tiles + budget.
VA_PACKED_FN int part_blocks(PackedSum blocks, int budget, int smallest) {
  if (!budget) return 1 << 30;
  const PackedSum part = (blocks + budget - 1) / budget;
  return part > (1 << 30) ? 1 << 30 : pk_max((int)part, smallest);
}
VA_PACKED_FN int part_count(int blocks, int part) { return pk_max(1, (blocks + part - 1) / part); }  // blocks < 2^27

// Whether a sum over tiles can pass 31 bits, whatever the offsets say (each sequence's are clamped to the totals; a list
// has at most its room of tiles).
inline bool packed_sums_wide(const PackedShape& s) {
  const double seqs = s.num_seqs, q = s.total_q, k = s.total_k, most = 2147483647.0;
  if (seqs * (q / s.q_tile + 1) > most || s.max_tiles * (k / kPackBlock + 1) > most) return true;
  return s.training && (seqs * (std::max(q, k) / kPackBlock + 1) > most ||
                        s.max_dkv_tiles * (q / 64 + 1) * s.group > most || s.max_dq_items * (k / kPackBlock + 1) > most);
}

int packed_status_read(int* out, cudaStream_t st);
int packed_status_clear(cudaStream_t st);
int packed_bwd_status_read(int* out, cudaStream_t st);
int packed_bwd_status_clear(cudaStream_t st);
// Tensor map over [rows, heads, dim] (strides in elements) in boxes of 64 dims × box_heads × box_rows.
int packed_map(CUtensorMap* m, const void* base, bool bf16, int rows, int heads, int dim, long long row_stride,
               long long head_stride, int box_heads, int box_rows, const char* what);
// Argument checks shared by the entry points (VA_OK or an error that is set).
int packed_check(int num_seqs, int total_q, int total_k, int heads, int kv_heads, int dim, int training);

}  // namespace va
