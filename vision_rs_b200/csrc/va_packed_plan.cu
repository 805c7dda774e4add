// The plan of a packed-sequence attention: from the sequences' offsets (on the
// device) to the lists of work units that the attention kernels walk, without
// a copy to the host.  One launch, one block for each list:
//
//   list 0  forward units,  list 1  dQ units,  list 2  dK/dV units (training)
//
// A block counts its tiles (prefix sum over the sequences), sums their key
// (or query) blocks, cuts long tiles into parts where that evens the load (at
// most `budget` parts more than tiles), and writes the units sorted
// by their size, longest first (a counting sort over 256 size classes), so
// that the last blocks of the attention's grid are its shortest.  Units of a
// class may come in any order: each writes results of its own.
//
// Offsets that decrease or pass the packed tensors' ends are clamped (no
// access leaves the tensors) and reported in the header.  5–6 µs, most of it
// the launch and the dependent loads; the attention's launch overlaps its end.
#include <limits.h>

#include "va_common.cuh"
#include "va_packed.h"

namespace va {
namespace {

constexpr int kPlanThreads = 512, kClasses = 256;

struct Seq {
  int q0, lq, k0, lk;
};

__device__ __forceinline__ Seq load_seq(const int* cu_q, const int* cu_k, const int* used_k, int num_seqs, int b,
                                       int total_q, int total_k, int* bad) {
  const int a0 = cu_q[b], a1 = cu_q[b + 1], c0 = cu_k[b], c1 = cu_k[b + 1];
  Seq s;
  s.q0 = min(max(a0, 0), total_q);
  s.lq = max(min(max(a1, 0), total_q) - s.q0, 0);
  s.k0 = min(max(c0, 0), total_k);
  s.lk = max(min(max(c1, 0), total_k) - s.k0, 0);
  if (used_k) {  // keys in use of the rows reserved
    const int n = min(max(used_k[b], 0), s.lk);
    if (n != used_k[b]) *bad = 1;
    if (s.k0 != c0 || s.lk != c1 - c0) *bad = 1;
    s.lk = n;
  } else if (s.lk != c1 - c0) {
    *bad = 1;
  }
  if (s.q0 != a0 || s.lq != a1 - a0 || s.k0 != c0 || (b == 0 && (a0 != 0 || c0 != 0))) *bad = 1;
  if (b == num_seqs - 1 && (a1 != total_q || c1 != total_k)) *bad = 1;  // rows of no sequence would stay unwritten
  return s;
}

// Exclusive sum over the block's threads; *total: of all.
template <typename T> __device__ T block_scan(T v, T* total) {
  __shared__ T warp_sum[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous call's readers are done
  if (lane == 31) warp_sum[w] = x;
  __syncthreads();
  T before = 0, all = 0;
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    const T t = warp_sum[i];
    if (i < w) before += t;
    all += t;
  }
  *total = all;
  return before + x - v;
}

struct PlanArgs {
  const int *cu_q, *cu_k, *used_k;
  uint8_t* plan;
  PackedShape s;
};

// Tile t of a list: its sequence and index in it.  first[b] = tiles before sequence b (first[num_seqs] = all).
__device__ __forceinline__ int seq_of_tile(const int* first, int num_seqs, int t) {
  int lo = 0, hi = num_seqs;  // the last b with first[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sum: int, or PackedSum where packed_sums_wide says so (0.3–0.5 µs more).
template <typename Sum> __global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(PlanArgs a) {
  __shared__ int hist[kClasses], cursor[kClasses];
  __shared__ int bad, full, most, first_smem[kPlanSeqs + 1];
  const PackedShape& s = a.s;
  let_next_start();
  wait_for_previous();
  const int list = blockIdx.x, tid = threadIdx.x;
  int* hdr = reinterpret_cast<int*>(a.plan);
  // tiles before each sequence
  int* first = s.num_seqs <= kPlanSeqs
                   ? first_smem
                   : reinterpret_cast<int*>(a.plan + s.scratch) + (size_t)list * (s.num_seqs + 1);
  const int tile = list == 0 ? s.q_tile : kPackBlock;
  if (tid == 0) bad = 0, full = 0, most = 0;
  for (int c = tid; c < kClasses; c += kPlanThreads) hist[c] = 0;
  __syncthreads();

  Sum sum_tiles = 0;
  for (int b0 = 0; b0 < s.num_seqs; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < s.num_seqs) {
      const Seq q = load_seq(a.cu_q, a.cu_k, a.used_k, s.num_seqs, b, s.total_q, s.total_k, &bad);
      n = ((list == 2 ? q.lk : q.lq) + tile - 1) / tile;
    }
    Sum sum;
    const Sum before = block_scan<Sum>(n, &sum);
    if (b < s.num_seqs) first[b] = (int)min(sum_tiles + before, (Sum)INT_MAX);
    sum_tiles += sum;
  }
  if (tid == 0) first[s.num_seqs] = (int)min(sum_tiles, (Sum)INT_MAX);
  __syncthreads();
  // offsets that run backwards could name more rows than there are: keep to the lists' room
  const int room = list == 0 ? s.max_tiles : list == 1 ? s.max_dq_items : s.max_dkv_tiles;
  if (sum_tiles > room && tid == 0) bad = 1;
  const int tiles = (int)min(sum_tiles, (Sum)room);

  Seq own_seq{};  // the thread's first tile, which every pass below asks for
  int own_i0 = 0, own_blocks = -1;
  auto tile_of = [&](int t, Seq* q, int* i0) -> int {  // its key blocks or query steps
    if (t == tid && own_blocks >= 0) {
      *q = own_seq, *i0 = own_i0;
      return own_blocks;
    }
    const int b = seq_of_tile(first, s.num_seqs, t);
    *q = load_seq(a.cu_q, a.cu_k, a.used_k, s.num_seqs, b, s.total_q, s.total_k, &bad);
    *i0 = (t - first[b]) * tile;
    const int n = list == 2 ? query_steps(q->lq, q->lk, *i0, s.causal, s.group)
                            : key_blocks(q->lq, q->lk, *i0, min(tile, q->lq - *i0), s.causal);
    if (t == tid) own_seq = *q, own_i0 = *i0, own_blocks = n;
    return n;
  };

  Sum mine = 0;
  int mine_most = 0;
  for (int t = tid; t < tiles; t += kPlanThreads) {
    Seq q;
    int i0;
    const int n = tile_of(t, &q, &i0);
    mine += n;
    mine_most = max(mine_most, n);
  }
  atomicMax(&most, mine_most);
  Sum blocks;
  block_scan<Sum>(mine, &blocks);
  const int budget = list == 0 ? s.split_budget : list == 2 ? s.dkv_budget : 0;
  const int chunk = part_blocks(blocks, budget, list == 0 ? kMinKeyBlocks : kMinQuerySteps);
  const int top = max(1, min(most, chunk));
  // the lists' room: part_blocks keeps to it, and what would pass it all the same (offsets that change meanwhile) is left out
  const int room_items = list == 0 ? s.max_items : list == 1 ? s.max_dq_items : s.max_dkv_items;
  const int room_slots = list == 0 ? s.max_slots : list == 2 ? 2 * s.dkv_budget : 0;

  auto size_class = [&](int n, int parts) {
    return max(0, kClasses - 1 - (int)((long long)(n / parts) * (kClasses - 1) / top));
  };
  int slots = 0, items = 0;
  for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
    const int t = t0 + tid;
    if (t < tiles) {
      Seq q;
      int i0;
      const int n = tile_of(t, &q, &i0), p = part_count(n, chunk);
      atomicAdd(&hist[size_class(n, p)], p);
    }
  }
  __syncthreads();
  {
    int sum;
    const int n = tid < kClasses ? hist[tid] : 0, before = block_scan<int>(n, &sum);
    if (tid < kClasses) cursor[tid] = before;
    items = sum;
  }
  __syncthreads();
  for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
    const int t = t0 + tid;
    Seq q{};
    int i0 = 0, n = 0, p = 0;
    if (t < tiles) {
      n = tile_of(t, &q, &i0);
      p = part_count(n, chunk);
    }
    int sum;
    const int slot0 = slots + block_scan<int>(p > 1 ? p : 0, &sum);
    slots += sum;
    if (t >= tiles) continue;
    int at = atomicAdd(&cursor[size_class(n, p)], p);
    if (at < 0 || at > room_items - p || (p > 1 && (slot0 < 0 || slot0 > room_slots - p))) {
      full = 1;
      continue;
    }
    if (list == 2) {
      KItem* out = reinterpret_cast<KItem*>(a.plan + s.dkv_items);
      for (int k = 0; k < p; ++k, ++at)
        out[at] = KItem{q.k0 + i0, min(tile, q.lk - i0), i0, q.q0, q.lq, q.lk,
                        (int)((long long)n * k / p), (int)((long long)n * (k + 1) / p),
                        p > 1 ? slot0 + k : -1, slot0, p, t};
      continue;
    }
    QItem* out = reinterpret_cast<QItem*>(a.plan + (list == 0 ? s.items : s.dq_items));
    for (int k = 0; k < p; ++k, ++at)
      out[at] = QItem{q.q0 + i0, min(tile, q.lq - i0), q.k0, q.lk, i0 + q.lk - q.lq,
                      (int)((long long)n * k / p), (int)((long long)n * (k + 1) / p),
                      p > 1 ? slot0 + k : -1, slot0, p, t, 0};
  }
  if (budget) {  // arrival counters of the split tiles
    int* cnt = reinterpret_cast<int*>(a.plan + (list == 0 ? s.counters : s.dkv_counters));
    const long long cells = (long long)tiles * (list == 0 ? s.units : s.kv_heads);
    for (long long i = tid; i < cells; i += kPlanThreads) cnt[i] = 0;
  }
  __syncthreads();
  if (tid == 0) {
    hdr[list] = full ? 0 : items;  // a list with holes is not walked
    hdr[kHdrBad + list] = bad | full;
  }
}


}  // namespace

int packed_check(int num_seqs, int total_q, int total_k, int heads, int kv_heads, int dim, int training) {
  VA_CHECK_ARG(num_seqs > 0 && num_seqs <= kMaxSeqs && total_q >= 0 && total_k >= 0,
               "packed attention: %d sequences, %d queries, %d keys", num_seqs, total_q, total_k);
  VA_CHECK_ARG(total_q <= (1 << 30) && total_k <= (1 << 30), "packed attention: more than 2^30 tokens");
  VA_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= kPackBlock && heads <= 4096,
               "packed attention: %d query heads over %d key heads", heads, kv_heads);
  // the backward counts a key head's (query, head) rows in 32 bits
  VA_CHECK_ARG(!training || (long long)total_q * (heads / kv_heads) < (1LL << 32) - (1 << 16),
               "packed attention: training with %d queries of %d heads a key head", total_q, heads / kv_heads);
  VA_CHECK_ARG(dim >= 8 && dim <= 128 && dim % 8 == 0, "packed attention: head size %d (a multiple of 8 up to 128)",
               dim);
  return VA_OK;
}

}  // namespace va

using namespace va;

extern "C" {

size_t va_packed_plan_bytes(int num_seqs, int total_q, int total_k, int num_heads, int num_kv_heads, int head_dim,
                            int causal, int training) {
  if (packed_check(num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim, training)) return 0;
  return packed_shape(num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim, causal != 0, training != 0).total;
}

int va_packed_plan_build(const int32_t* cu_q, const int32_t* cu_k, const int32_t* used_k, int num_seqs, int total_q, int total_k,
                         int num_heads, int num_kv_heads, int head_dim, int causal, int training, void* plan,
                         size_t plan_bytes, va_stream_t stream) {
  if (int rc = packed_check(num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim, training)) return rc;
  VA_CHECK_ARG(cu_q && cu_k, "packed plan: null offsets");
  VA_CHECK_ARG(!(used_k && training), "packed plan: reserved rows have no gradient, train without used_k");
  PlanArgs a{cu_q, cu_k, used_k, static_cast<uint8_t*>(plan),
             packed_shape(num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim, causal != 0, training != 0)};
  if (!plan || plan_bytes < a.s.total)
    return set_error(VA_ERR_WORKSPACE, "packed plan: %zu < %zu bytes", plan_bytes, a.s.total);
  if (reinterpret_cast<uintptr_t>(plan) & 255)
    return set_error(VA_ERR_ALIGN, "packed plan: the buffer needs 256-byte alignment");
  auto kernel = packed_sums_wide(a.s) ? packed_plan_kernel<PackedSum> : packed_plan_kernel<int>;
  return launch_behind("packed plan", kernel, training ? 3 : 1, kPlanThreads, 0, (cudaStream_t)stream, a);
}

int va_packed_plan_status(const void* plan, int training, int* bad_offsets, va_stream_t stream) {
  VA_CHECK_ARG(plan && bad_offsets, "packed plan status: null pointer");
  int bad[3] = {0, 0, 0};
  const int lists = training ? 3 : 1;
  cudaError_t e = cudaMemcpyAsync(bad, static_cast<const int*>(plan) + kHdrBad, lists * sizeof(int),
                                  cudaMemcpyDeviceToHost, (cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "packed plan status: %s", cudaGetErrorString(e));
  *bad_offsets = bad[0] | bad[1] | bad[2];
  return VA_OK;
}

}  // extern "C"
