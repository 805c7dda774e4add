// Gradient of the packed-sequence attention (tcgen05 + TMEM + TMA).  With
// P = exp(scale·q·k − lse) and Δ_i = dO_i·O_i, per head:
//
//   dV_j = Σ_i P_ij dO_i,   dS = P ⊙ (dO Vᵀ − Δ),
//   dQ_i = scale Σ_j dS_ij k_j,   dK_j = scale Σ_i dS_ij q_i
//
// (dK and dV summed over the query heads that share the key head).  Three
// launches, no atomics, so the results do not depend on scheduling:
//
//   row kernel   (lse·log2 e, Δ) of every query and head
//   dQ kernel    a CTA per (128 queries, head) walks the keys in steps of 64:
//                S = Q·Kᵀ, dP = dO·Vᵀ with Q and dO as TMEM operands, dS in
//                TMEM, dQ += dS·K
//   dK/dV kernel a CTA per (128 keys, key head) walks the group's heads and
//                their queries in steps of 64: Sᵀ = K·Qᵀ and dPᵀ = V·dOᵀ in
//                TMEM, Pᵀ and dSᵀ back into the same columns in 16 bits, then
//                dV += Pᵀ·dO, dK += dSᵀ·Q with the TMEM operand; long ranges are
//                split over CTAs and joined by the last, in order
//
// S and dP are computed twice (7 products instead of 5); the one-kernel form
// would add f32 dQ partials to memory from every key tile, in an order that
// changes from run to run, or write and read all of them.  Two score buffers
// (three at 64 dims) and as many groups of warps alternate, so the MMAs of one
// step run under the exponentials of another.  Steps are 64 wide because dV,
// dK (256 columns) and two buffers of S and dP (4 × 64) fill the 512 TMEM
// columns at 128 dims.
//
// Measured (B200): 4 documents of 1025–4095 tokens, 12/3 heads of 128, causal,
// bf16: 546 µs for plan, forward and backward under sustained load (CUDA
// events).  Shares under a profiler (single cold launches): row sums 15 µs, dQ
// 170, dK/dV 251; their 3 and 4 products take 88 and 117 µs at 1,647 TFLOP/s.
// The tensor pipe is 45% busy in dQ and 39% in dK/dV (402 blocks): a buffer's
// chain scores → P and dS → products is covered only in part by the other
// buffer.  With one warp to issue both kinds of products and dK/dV's tiles not
// yet split: dQ 220 µs, dK/dV 349.
//
// P and dS are 16-bit operands.  f16 has few exponents, so there P carries
// 2^15 and dS a power of two chosen for its row (key or query) such that the
// largest possible |dS| stays below 2^15: |dO_i·V_j| ≤ ‖dO_i‖·‖V_j‖; the f32
// sums are scaled back at the end.  bf16 needs neither.  Sequences and rows of
// at most 128 keys keep P's and dS's remainders as second operands.
//
// What a row does not see stays out of its gradient, whatever it holds: scores
// of hidden pairs and of other sequences' rows are masked by selection.  As
// 0 · NaN is NaN, the rows of the summed operand past the sequence's end are
// zeroed, and in steps with hidden pairs the score groups look through it while
// the score MMAs run and leave out what is not finite.  A query or a key that is
// not finite reaches what depends on it through P and dS all the same; a dO
// value is given back to dV of the keys that its row sees.  Measured: backward
// of the 4 documents below 422.5 → 426 µs (a warp of its own for it: 436, the
// gradients' issuing warp: 443).
#include <cudaTypedefs.h>

#include <type_traits>

#include "va_common.cuh"
#include "va_packed.h"
#include "va_sm100.cuh"

namespace va {
using namespace sm100;

__device__ int g_packed_bwd_status;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kHalf = 64;     // queries (or keys) a step
// Sequences of at most this many 64-row steps hold P and dS as two 16-bit words, value and remainder, and multiply by both:
// there the second products cost nothing that is measured, and the gradients are exact to their own rounding.
constexpr int kFineSteps = 2;
constexpr float kPShift = 15.0f;     // f16: P is held times 2^15

// Groups of four warps that take the score steps in turn, each with a buffer of S and dP (64 + 64 columns) of its own: as
// many as fit the 512 TMEM columns beside the accumulators (and Q and dO).  At 64 dims, where the exponentials and not the
// MMAs set the pace, the third hides the others' latencies.
template <int DP> struct BwdCfg {
  static constexpr int kGroups = DP == 64 ? 3 : 2;
  static constexpr int kSoft = kGroups * 128;         // threads of the score groups
  static constexpr int kWarps = kGroups * 4;          // their warps; then 1 TMA, 1 issues the scores' MMAs, 1 the gradients'
  static constexpr int kThreads = kSoft + 96;
  static constexpr int kStages = DP == 64 ? 6 : 4;    // ring of 64-row (Q, dO) or (K, V) pairs
  static constexpr uint32_t kColAcc = kGroups * 128;  // score buffer b at 128·b (S, then dP); accumulators from here
};

template <int DP> struct BwdSmem {
  using C = BwdCfg<DP>;
  static constexpr int kTile = kPackBlock * DP * 2, kStep = kHalf * DP * 2;
  uint8_t a[2][kTile];               // K and V of the keys, or Q and dO of the queries: per 64 dims 128 rows × 128 bytes
  uint8_t ring[C::kStages][2][kStep];   // per 64 dims 64 rows × 128 bytes
  float4 stats[C::kGroups][2][2][kHalf / 4];  // dK/dV: −lse·log2 e and −Δ of the step's queries, per group, two steps
  float red[C::kWarps];
  float row_part[2][kPackBlock];     // dQ: Σ P·dP over a group's keys
  uint64_t a_full, a_ready, full[C::kStages], empty[C::kStages];
  uint64_t s_full[C::kGroups], p_full[C::kGroups], g_done[C::kGroups], fin;
  uint32_t tmem_base;
  int abort, last;
  int loose;    // something that is not finite was left out of a step's tiles (dK/dV: it may be dO's)
  int scanned;  // f16: how far the score warps are with the norms that bound dS, before their first step
};
constexpr unsigned kScanChunk = 4096;  // turns of that loop between two updates of `scanned`

struct BwdArgs {
  uint8_t* plan;
  PackedShape s;
  void *dq, *dk, *dv;
  long long dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
  float scale;
  const uint16_t* d_out;
  long long do_row, do_head;
};

// A score group's share of `bytes` of a step's tiles (the thread's cells of 16 bytes, in whatever order the swizzle has
// them): whether they hold anything that is not finite, and the tiles without that.
template <bool BF16, int BYTES> __device__ __forceinline__ bool holds_loose(const uint8_t* tile, int t) {
  uint32_t any = 0;
#pragma unroll 4
  for (int i = t; i < BYTES / 16; i += 128) {
    const uint4 x = reinterpret_cast<const uint4*>(tile)[i];
    any |= not_finite2<BF16>(x.x) | not_finite2<BF16>(x.y) | not_finite2<BF16>(x.z) | not_finite2<BF16>(x.w);
  }
  return any != 0;
}
template <bool BF16, int BYTES> __device__ __noinline__ void drop_loose(uint8_t* tile, int t, int* flag) {
  for (int i = t; i < BYTES / 16; i += 128) {
    uint4* p = reinterpret_cast<uint4*>(tile) + i;
    const uint4 x = *p;
    *p = make_uint4(finite2<BF16>(x.x), finite2<BF16>(x.y), finite2<BF16>(x.z), finite2<BF16>(x.w));
  }
  fence_proxy_async_smem();
  *(volatile int*)flag = 1;
}

// The score warps never leave a loop early: a wait that gives up is passed over, as are the thread's later ones, so that
// every thread meets every one of these barriers and the lanes of a warp stay together at its TMEM instructions.  The
// result is not written then.
// All score groups meet.
template <int N> __device__ __forceinline__ void scores_sync() { asm volatile("bar.sync 4, %0;" ::"n"(N) : "memory"); }
// The four warps of one meet.
__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(g + 1) : "memory"); }

// Largest power of two p with bound·p < 2^15 (1 for a bound of zero; the exponent is kept within ±60).
__device__ __forceinline__ float pow2_below(float bound) {
  if (!(bound > 0.0f) || !(bound < INFINITY)) return 1.0f;
  const int e = min(60, max(-60, 14 - ilogbf(bound)));
  return __int_as_float((127 + e) << 23);
}

// Zeroes rows [used, 16·ceil(used/16)) of a 64-row tile, whole warp.
template <int DP> __device__ __forceinline__ void zero_tail(uint8_t* tile, int used, int lane) {
  const int n = ((used + 15) / 16 * 16 - used) * (DP / 8);
  for (int i = lane; i < n; i += 32) {
    const int r = used + i / (DP / 8), c = i % (DP / 8);
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kHalf * 128 + sw128_off(r, c & 7)) = make_uint4(0, 0, 0, 0);
  }
}

// Set-up shared by both kernels: barriers and TMEM.
template <int DP> __device__ __forceinline__ uint32_t bwd_setup(BwdSmem<DP>& sm, int tid, int warp) {
  if (tid == 0) {
    mbar_init(&sm.a_full, 1);
    mbar_init(&sm.a_ready, 256);
    for (int i = 0; i < BwdCfg<DP>::kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int b = 0; b < BwdCfg<DP>::kGroups; ++b) {
      mbar_init(&sm.s_full[b], 1);
      mbar_init(&sm.p_full[b], 128);
      mbar_init(&sm.g_done[b], 1);
    }
    mbar_init(&sm.fin, 2);
    sm.abort = 0;
    sm.loose = 0;
    sm.scanned = 0;
    fence_mbar_init();
  }
  if (warp == BwdCfg<DP>::kWarps) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return sm.tmem_base;
}

// 16 accumulator columns of the thread's row → out[c .. c+16) times f (rows that are stored, dims below dim).
template <bool BF16>
__device__ __forceinline__ void store16(uint32_t taddr, bool zero, float f, bool mine, uint16_t* out, int c, int dim) {
  uint32_t o[16] = {};
  if (!zero) {
    tmem_ld16(taddr + c, o);
    tmem_ld_wait();
    reg_fence(o);
  }
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = zero ? 0u : pack2<BF16>(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f);
  if (mine) {
    *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
    if (c + 8 < dim) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
  __syncwarp();
}

// Producer: the ring's steps, each two 64-row tiles.  at(h, &head, &row) says where step h begins.
template <int DP, typename At>
__device__ __forceinline__ void produce(BwdSmem<DP>& sm, const CUtensorMap* m0, const CUtensorMap* m1, int n, At at) {
  constexpr int NB = DP / 64, kStages = BwdCfg<DP>::kStages;
  int issued = 0;
  for (int h = 0; h < n; ++h) {
    const int st = h % kStages;
    if (h >= kStages && !mbar_wait_behind(&sm.empty[st], (h / kStages - 1) & 1, &sm.abort, &sm.scanned, &g_packed_bwd_status, 1))
      break;
    int head, row;
    at(h, &head, &row);
    mbar_arrive_expect_tx(&sm.full[st], 2 * BwdSmem<DP>::kStep);
    for (int b = 0; b < NB; ++b) {
      tma_load_3d(sm.ring[st][0] + b * kHalf * 128, m0, &sm.full[st], b * 64, head, row);
      tma_load_3d(sm.ring[st][1] + b * kHalf * 128, m1, &sm.full[st], b * 64, head, row);
    }
    ++issued;
  }
  // loads issued here land (bounded) before the CTA can exit, also when it was another role that gave up
  for (int h = max(0, issued - kStages); h < issued; ++h) {
    const long long c0 = clock64();
    while (!mbar_try_wait(&sm.full[h % kStages], (h / kStages) & 1) && clock64() - c0 < kSpinCycles) {
    }
  }
  const long long c0 = clock64();
  while (!mbar_try_wait(&sm.a_full, 0) && clock64() - c0 < kSpinCycles) {
  }
}

// The issuing warps stay converged with uniform values (operands that differ
// between lanes cost ~60 cycles an MMA); one elected lane issues.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_packed_bwd_status, where));
}
// For what comes after the score warps' scan of the norms.
template <typename Smem> __device__ __forceinline__ bool wait_scores(Smem& sm, uint64_t* bar, uint32_t parity, int where) {
  return __all_sync(0xffffffffu, mbar_wait_behind(bar, parity, &sm.abort, &sm.scanned, &g_packed_bwd_status, where));
}
template <typename Smem> __device__ __forceinline__ void issue_end(Smem& sm, uint32_t lead) {
  mma_commit_p(&sm.fin, lead);  // every MMA issued here completes before the CTA tears down
  const long long c0 = clock64();
  while (!mbar_try_wait(&sm.fin, 0) && clock64() - c0 < kSpinCycles) {
  }
}

// ── (lse·log2 e, Δ) and, for f16, the norms that bound dS ───────────────────
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

// 16 lanes a row, four rows in flight.  blockIdx.y below heads: Δ of a query head's tokens; the rest (f16): ‖V_j‖ of a key head's.
constexpr int kRowsBlock = 64;
template <bool BF16>
__global__ void __launch_bounds__(256)
packed_rows_kernel(const uint16_t* __restrict__ out, const uint16_t* __restrict__ d_out, long long do_row,
                   long long do_head, const uint16_t* __restrict__ v, long long v_row, long long v_head,
                   const float* __restrict__ lse, float2* __restrict__ pairs, float* __restrict__ do_norm,
                   float* __restrict__ v_norm, int total_q, int total_k, int heads, int dim) {
  let_next_start();
  wait_for_previous();
  const bool is_q = (int)blockIdx.y < heads;
  const int h = is_q ? blockIdx.y : blockIdx.y - heads, total = is_q ? total_q : total_k;
  const int t0 = blockIdx.x * kRowsBlock + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 8;
  if ((int)blockIdx.x * kRowsBlock >= total) return;
  uint4 ua[4], ub[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long t = t0 + u * 16;
    ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
    if (t < total && c < dim) {
      if (is_q) ua[u] = *reinterpret_cast<const uint4*>(out + (t * heads + h) * dim + c);
      ub[u] = *reinterpret_cast<const uint4*>(is_q ? d_out + t * do_row + h * do_head + c : v + t * v_row + h * v_head + c);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = t0 + u * 16;
    float a[8], b[8], dot = 0.0f, sq = 0.0f;
    unpack8<BF16>(ua[u], a);
    unpack8<BF16>(ub[u], b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dot = fmaf(a[i], b[i], dot);
      if constexpr (!BF16) sq = fmaf(b[i], b[i], sq);
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if constexpr (!BF16) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    }
    if (t < total && (threadIdx.x & 15) == 0) {
      const long long at = (long long)h * total + t;
      if (is_q) {
        pairs[at] = make_float2(lse[at] * kLog2e, dot);
        if constexpr (!BF16) do_norm[at] = sqrtf(sq);
      } else if constexpr (!BF16) {
        v_norm[at] = sqrtf(sq);
      }
    }
  }
}

// dO values that were left out of a unit's product, to dV of the thread's key, whose row it has stored.  (Not inlined: the
// kernel's loops need its registers.)
template <bool BF16>
__device__ __noinline__ void give_back(const BwdArgs& a, const KItem* item, int kvh, int key) {
  const PackedShape& ps = a.s;
  const KItem it = *item;
  const int off = it.lk - it.lq, j = it.j0 + key, hb0 = ps.causal ? max(0, it.j0 - off) / kHalf : 0;
  const int nh = (it.lq + kHalf - 1) / kHalf - hb0, last = it.j0 + it.keys - 1 - off;
  auto value = [](uint16_t w) { return BF16 ? __uint_as_float((uint32_t)w << 16) : __half2float(__ushort_as_half(w)); };
  uint16_t* out = static_cast<uint16_t*>(a.dv) + (it.k0 + key) * a.dv_row + kvh * a.dv_head;
  float* part = reinterpret_cast<float*>(a.plan + ps.part_dkv) +
                (((long long)it.slot * ps.kv_heads + kvh) * 2 * kPackBlock + key) * ps.dim;
  for (int h = it.h0; h < it.h1; ++h) {
    const int i0 = (hb0 + h % nh) * kHalf;
    if (it.lq > kFineSteps * kHalf && !(ps.causal && last > i0)) continue;
    for (int i = ps.causal ? max(i0, j - off) : i0; i < min(i0 + kHalf, it.lq); ++i) {
      const uint16_t* row = a.d_out + (it.q0 + i) * a.do_row + (kvh * ps.group + h / nh) * a.do_head;
      for (int c = 0; c < ps.dim; ++c) {
        const float x = value(row[c]);
        if (fabsf(x) < INFINITY) continue;
        if (it.slot < 0) out[c] = (uint16_t)pack2<BF16>(value(out[c]) + x, 0.0f);
        else part[c] += x;
      }
    }
  }
}

// ── dK and dV ────────────────────────────────────────────────────────────────
template <int DP, bool BF16, bool CAUSAL>
__global__ void __launch_bounds__(BwdCfg<DP>::kThreads, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ BwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<DP>& sm = *reinterpret_cast<BwdSmem<DP>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using C = BwdCfg<DP>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kColAcc = C::kColAcc;
  const PackedShape& ps = a.s;
  let_next_start();
  wait_for_previous();
  const int unit = blockIdx.x / ps.kv_heads, kvh = blockIdx.x - unit * ps.kv_heads;
  if (unit >= reinterpret_cast<const int*>(a.plan)[kHdrDkv]) return;
  const KItem it = reinterpret_cast<const KItem*>(a.plan + ps.dkv_items)[unit];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int dim16 = (ps.dim + 15) & ~15;
  // 64-query blocks of a head from the first that sees a key of the tile, and the unit's steps (block b0 of head g0 first)
  const int hb0 = CAUSAL ? max(0, it.j0 - (it.lk - it.lq)) / kHalf : 0, nh = max(0, (it.lq + kHalf - 1) / kHalf - hb0);
  const int n = it.h1 - it.h0, g0 = nh > 0 ? it.h0 / nh : 0, b0 = it.h0 - g0 * nh;
  const bool fine = it.lq <= kFineSteps * kHalf;
  const uint32_t tmem = bwd_setup<DP>(sm, tid, warp);

  if (warp == C::kWarps) {
    if (lane == 0 && n > 0) {
      constexpr int NB = DP / 64;
      mbar_arrive_expect_tx(&sm.a_full, 2 * BwdSmem<DP>::kTile);
      for (int b = 0; b < NB; ++b) {
        tma_load_3d(sm.a[0] + b * kPackBlock * 128, &map_k, &sm.a_full, b * 64, kvh, it.k0);
        tma_load_3d(sm.a[1] + b * kPackBlock * 128, &map_v, &sm.a_full, b * 64, kvh, it.k0);
      }
      int g = g0, b = b0;
      produce<DP>(sm, &map_q, &map_do, n, [&](int, int* head, int* row) {
        *head = kvh * ps.group + g;
        *row = it.q0 + (hb0 + b) * kHalf;
        if (++b == nh) b = 0, ++g;
      });
    }
    __syncwarp();
  } else if (warp == C::kWarps + 1) {
    // ── Sᵀ = K·Qᵀ and dPᵀ = V·dOᵀ of step h into buffer h mod groups, once the products of its last step are done ──
    if (n > 0) {
      const uint32_t lead = elect_lead(), tm = uniform(tmem);
      const int steps = uniform(n), blocks = uniform(nh), tail = uniform(it.lq - (hb0 + nh - 1) * kHalf);
      const uint32_t id_s = idesc_f32acc(kPackBlock, kHalf, BF16 ? AB_BF16 : AB_F16, false, false);
      const uint64_t dk = sdesc(smem_u32(sm.a[0]), 16, 1024, SW_128B), dv = sdesc(smem_u32(sm.a[1]), 16, 1024, SW_128B);
      const uint64_t dq0 = sdesc(smem_u32(sm.ring[0][0]), 16, 1024, SW_128B);
      constexpr int kABlk = (kPackBlock * 128) >> 4, kBBlk = (kHalf * 128) >> 4, kTileStep = BwdSmem<DP>::kStep >> 4;
      int buf = 0;       // score buffer of the step
      uint32_t par = 0;  // parity of its use
      auto next_buffer = [&] {
        if (++buf == C::kGroups) buf = 0, par ^= 1;
      };
      bool ok = wait_all(&sm.a_full, 0, &sm.abort, 2);
      int b = uniform(b0);
      for (int h = 0; ok && h < steps; ++h) {
        const int st = h % kStages;
        if (!(ok = wait_all(&sm.full[st], (h / kStages) & 1, &sm.abort, 3))) break;
        if (++b == blocks) {  // the last block of a head: rows past the sequence's end
          b = 0;
          if (tail & 15) {
            zero_tail<DP>(sm.ring[st][0], tail, lane);
            zero_tail<DP>(sm.ring[st][1], tail, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        if (h >= C::kGroups && !(ok = wait_scores(sm, &sm.g_done[buf], par ^ 1, 6))) break;
        tc_fence_after();
        const uint64_t bq = dq0 + (uint64_t)(st * 2 * kTileStep), bo = bq + kTileStep;
        const uint32_t ts = tm + buf * 128;
        auto one = [&](int s) {
          const uint64_t oa = (uint64_t)((s >> 2) * kABlk + (s & 3) * 2), ob = (uint64_t)((s >> 2) * kBBlk + (s & 3) * 2);
          mma_ss_p(ts, dk + oa, bq + ob, id_s, s > 0 ? 1u : 0u, lead);
          mma_ss_p(ts + kHalf, dv + oa, bo + ob, id_s, s > 0 ? 1u : 0u, lead);
        };
        if (dim16 == DP) {
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) one(s);
        } else {
          for (int s = 0; s < dim16 / 16; ++s) one(s);
        }
        mma_commit_p(&sm.s_full[buf], lead);
        next_buffer();
      }
      issue_end(sm, lead);
    }
    __syncwarp();
  } else if (warp == C::kWarps + 2) {
    // ── dV += Pᵀ·dO, dK += dSᵀ·Q ──
    if (n > 0) {
      const bool uniform_fine = uniform(fine);
      const uint32_t lead = elect_lead(), tm = uniform(tmem);
      const int steps = uniform(n), blocks = uniform(nh), tail = uniform(it.lq - (hb0 + nh - 1) * kHalf);
      const uint32_t id_g = idesc_f32acc(kPackBlock, dim16, BF16 ? AB_BF16 : AB_F16, false, true);
      const uint64_t dq0 = sdesc(smem_u32(sm.ring[0][0]), kHalf * 128, 1024, SW_128B);
      constexpr int kTileStep = BwdSmem<DP>::kStep >> 4;
      int buf = 0;       // score buffer of the step
      uint32_t par = 0;  // parity of its use
      auto next_buffer = [&] {
        if (++buf == C::kGroups) buf = 0, par ^= 1;
      };
      bool ok = true;
      int b = uniform(b0);
      for (int h = 0; h < steps; ++h) {
        const int st = h % kStages;
        int ks = kHalf / 16;
        if (++b == blocks) b = 0, ks = min(ks, (tail + 15) >> 4);
        if (!(ok = wait_scores(sm, &sm.p_full[buf], par, 4))) break;
        tc_fence_after();
        const uint64_t gq = dq0 + (uint64_t)(st * 2 * kTileStep), go = gq + kTileStep;
        const uint32_t tp = tm + buf * 128;
        auto one = [&](int s) {
          const uint32_t acc = (h > 0 || s > 0) ? 1u : 0u;
          mma_ts_p(tm + kColAcc, tp + s * 8, go + (uint64_t)(s * (2048 >> 4)), id_g, acc, lead);
          mma_ts_p(tm + kColAcc + DP, tp + kHalf + s * 8, gq + (uint64_t)(s * (2048 >> 4)), id_g, acc, lead);
        };
        if (ks == kHalf / 16 && !uniform_fine) {
#pragma unroll
          for (int s = 0; s < kHalf / 16; ++s) one(s);
        } else {
          for (int s = 0; s < ks; ++s) one(s);
          for (int s = 0; uniform_fine && s < ks; ++s) {
            mma_ts_p(tm + kColAcc, tp + 32 + s * 8, go + (uint64_t)(s * (2048 >> 4)), id_g, 1u, lead);
            mma_ts_p(tm + kColAcc + DP, tp + kHalf + 32 + s * 8, gq + (uint64_t)(s * (2048 >> 4)), id_g, 1u, lead);
          }
        }
        mma_commit_p(&sm.g_done[buf], lead);
        mma_commit_p(&sm.empty[st], lead);
        next_buffer();
      }
      issue_end(sm, lead);
    }
    __syncwarp();
  } else {
    // ── scores: group g takes steps h ≡ g (mod groups), thread = key ──
    const int g = warp >> 2, key = tid - g * 128;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + g * 128;
    const float2* pairs = reinterpret_cast<const float2*>(a.plan + ps.rows);
    const float scale2 = a.scale * kLog2e;
    const bool mine = key < it.keys;
    float mult = 1.0f;
    if constexpr (!BF16) {  // |dS_ij| ≤ max_i ‖dO_i‖ · ‖V_j‖ + max_i |Δ_i|
      const float* norms = reinterpret_cast<const float*>(a.plan + ps.do_norm);
      float top_n = 0.0f, top_d = 0.0f;
      const unsigned head_rows = nh * kHalf;  // head_rows · group < 2^32 (packed_check)
      const long long all = (long long)head_rows * ps.group;
      for (long long i0 = 0; i0 < all; i0 += C::kSoft * kScanChunk) {
        const unsigned end = (unsigned)min(all, i0 + C::kSoft * kScanChunk);
        for (unsigned i = (unsigned)i0 + tid; i < end; i += C::kSoft) {
          const int gh = i / head_rows, q = hb0 * kHalf + (int)(i - gh * head_rows);
          if (q >= it.lq) continue;
          const long long at = (long long)(kvh * ps.group + gh) * ps.total_q + it.q0 + q;
          const float nq = norms[at], dq = fabsf(pairs[at].y);
          // (a row that is not finite sets no scale: the keys that it sees get NaN, the others do not depend on it)
          if (nq < INFINITY) top_n = fmaxf(top_n, nq);
          if (dq < INFINITY) top_d = fmaxf(top_d, dq);
        }
        if (tid == 0) *(volatile int*)&sm.scanned = (int)(i0 / (C::kSoft * kScanChunk)) + 1;
      }
      for (int o = 16; o; o >>= 1) {
        top_n = fmaxf(top_n, __shfl_xor_sync(0xffffffffu, top_n, o));
        top_d = fmaxf(top_d, __shfl_xor_sync(0xffffffffu, top_d, o));
      }
      float* red = reinterpret_cast<float*>(sm.stats);
      if (lane == 0) red[warp] = top_n, red[C::kWarps + warp] = top_d;
      scores_sync<C::kSoft>();
      for (int i = 0; i < C::kWarps; ++i) top_n = fmaxf(top_n, red[i]), top_d = fmaxf(top_d, red[C::kWarps + i]);
      scores_sync<C::kSoft>();
      const float vn = mine ? reinterpret_cast<const float*>(a.plan + ps.v_norm)[(long long)kvh * ps.total_k + it.k0 + key] : 0.0f;
      mult = pow2_below(top_n * vn + top_d);
    }
    const float mult_p = BF16 ? 1.0f : mult * 3.0517578125e-05f;  // dS from P·2^15
    const int off = it.lk - it.lq, j = it.j0 + key;
    auto hides_queries = [&](int i0) { return CAUSAL && it.j0 + it.keys - 1 - off > i0; };  // from some key of the tile
    bool ok = true;
    // (lse, Δ) of a step's query, fetched a step ahead by the group's first 64 threads
    int fg = g0, fb = b0;  // head and block of the step that is fetched next
    auto advance = [&](int by) {
      fb += by;
      while (fb >= nh) fb -= nh, ++fg;
    };
    auto fetch = [&](int h) -> float2 {
      float2 f = make_float2(INFINITY, 0.0f);  // past the sequence: P = 2^−∞
      if (h < n && key < kHalf) {
        const int i = (hb0 + fb) * kHalf + key;
        if (i < it.lq) f = pairs[(long long)(kvh * ps.group + fg) * ps.total_q + it.q0 + i];
        if constexpr (!BF16) f.x -= kPShift;
      }
      return f;
    };
    if (n > 0) advance(g);
    float2 ahead = fetch(g);
    int block = fb;
    for (int h = g, k = 0; h < n; h += C::kGroups, ++k) {
      if (key < kHalf) {
        reinterpret_cast<float*>(sm.stats[g][k & 1][0])[key] = -ahead.x;
        reinterpret_cast<float*>(sm.stats[g][k & 1][1])[key] = -ahead.y;
      }
      group_sync(g);
      const int i0 = (hb0 + block) * kHalf;
      advance(C::kGroups);
      ahead = fetch(h + C::kGroups);
      block = fb;
      // queries [lo, hi) of the step see this key
      const int lo = CAUSAL ? j - off - i0 : 0, hi = it.lq - i0;
      const bool hides = hides_queries(i0), whole = hi >= kHalf && !hides;
      bool loose = false;
      // (fine: a weight's remainder may be zero or negative, and times infinity that is not the weight's product)
      if (CAUSAL && (hides || fine)) {
        ok = ok && mbar_wait(&sm.full[h % kStages], (h / kStages) & 1, &sm.abort, &g_packed_bwd_status, 10);
        loose = holds_loose<BF16, 2 * BwdSmem<DP>::kStep>(sm.ring[h % kStages][0], key);
      }
      ok = ok && mbar_wait(&sm.s_full[g], k & 1, &sm.abort, &g_packed_bwd_status, 8);
      if (loose) drop_loose<BF16, 2 * BwdSmem<DP>::kStep>(sm.ring[h % kStages][0], key, &sm.loose);
      tc_fence_after();
      const float4 *nl = sm.stats[g][k & 1][0], *nd = sm.stats[g][k & 1][1];
      // 16 queries at a time: their statistics are read while the scores come
      struct Chunk {
        uint32_t s[16], d[16];
      };
      struct Stats {
        float4 l[4], e[4];
      };
      auto fetch16 = [&](int c, Chunk& x) {
        tmem_ld16(ts + c * 16, x.s);
        tmem_ld16(ts + kHalf + c * 16, x.d);
      };
      auto stats16 = [&](int c) {
        Stats x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.l[i] = nl[c * 4 + i], x.e[i] = nd[c * 4 + i];
        return x;
      };
      auto scores16 = [&](int c, const Chunk& x, const Stats& y, auto masked, auto with_rest) {
        uint32_t pp[8], pd[8], rp[8], rd[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 &lf = y.l[i >> 1], &ef = y.e[i >> 1];
          float p0, p1, d0 = __uint_as_float(x.d[2 * i]), d1 = __uint_as_float(x.d[2 * i + 1]);
          ffma2(p0, p1, __uint_as_float(x.s[2 * i]), __uint_as_float(x.s[2 * i + 1]), scale2, scale2,
                i & 1 ? lf.z : lf.x, i & 1 ? lf.w : lf.y);
          fadd2(d0, d1, i & 1 ? ef.z : ef.x, i & 1 ? ef.w : ef.y);
          p0 = ex2(p0);
          p1 = ex2(p1);
          fmul2(d0, d1, p0, p1);
          if constexpr (decltype(masked)::value) {
            const int q0 = c * 16 + 2 * i, q1 = q0 + 1;
            const bool v0 = q0 >= lo && q0 < hi, v1 = q1 >= lo && q1 < hi;
            p0 = v0 ? p0 : 0.0f;
            d0 = v0 ? d0 : 0.0f;
            p1 = v1 ? p1 : 0.0f;
            d1 = v1 ? d1 : 0.0f;
          }
          if constexpr (!BF16) fmul2(d0, d1, mult_p, mult_p);
          pp[i] = pack2<BF16>(p0, p1);
          pd[i] = pack2<BF16>(d0, d1);
          if constexpr (decltype(with_rest)::value) {
            rp[i] = pack2_rest<BF16>(pp[i], p0, p1);
            rd[i] = pack2_rest<BF16>(pd[i], d0, d1);
          }
        }
        tmem_st8(ts + c * 8, pp);
        tmem_st8(ts + kHalf + c * 8, pd);
        if constexpr (decltype(with_rest)::value) {
          tmem_st8(ts + 32 + c * 8, rp);
          tmem_st8(ts + kHalf + 32 + c * 8, rd);
        }
      };
      auto arrived = [&](Chunk& x) {
        reg_fence(x.s);
        reg_fence(x.d);
      };
      auto scores = [&](auto masked) {
#pragma unroll
        for (int c = 0; c < kHalf / 16; ++c) {
          Chunk x;
          fetch16(c, x);
          const Stats y = stats16(c);
          tmem_ld_wait();
          arrived(x);
          scores16(c, x, y, masked, std::false_type{});
        }
      };
      if (fine) {  // the remainders of chunk c take the columns of scores c / 2 + 2: those are read first
        Chunk even, odd;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          Chunk x, &later = c ? odd : even;
          fetch16(c, x);
          fetch16(c + 2, later);
          tmem_ld_wait();
          arrived(x);
          arrived(later);
          scores16(c, x, stats16(c), std::true_type{}, std::true_type{});
        }
        scores16(2, even, stats16(2), std::true_type{}, std::true_type{});
        scores16(3, odd, stats16(3), std::true_type{}, std::true_type{});
      } else if (__all_sync(0xffffffffu, whole)) {
        scores(std::false_type{});
      } else {
        scores(std::true_type{});
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_full[g]);
    }
    if (n > 0) ok = ok && mbar_wait(&sm.fin, 0, &sm.abort, &g_packed_bwd_status, 9);
    if (__all_sync(0xffffffffu, ok && !*(volatile int*)&sm.abort) && g < 2) {  // group 0 stores dV, group 1 dK
      tc_fence_after();
      const uint32_t acc = tmem + lanes + kColAcc + g * DP;
      const float f = g == 0 ? (BF16 ? 1.0f : 3.0517578125e-05f) : 1.0f / mult;
      if (it.slot < 0) {
        const long long row = it.k0 + key;
        uint16_t* out = g == 0 ? static_cast<uint16_t*>(a.dv) + row * a.dv_row + kvh * a.dv_head
                               : static_cast<uint16_t*>(a.dk) + row * a.dk_row + kvh * a.dk_head;
        for (int c = 0; c < dim16; c += 16)
          store16<BF16>(acc, n == 0, g == 0 ? f : f * a.scale, mine, out, c, ps.dim);
      } else {
        float* out = reinterpret_cast<float*>(a.plan + ps.part_dkv) +
                     ((((long long)it.slot * ps.kv_heads + kvh) * 2 + g) * kPackBlock + key) * ps.dim;
        for (int c = 0; c < dim16; c += 16) {
          uint32_t o[16];
          tmem_ld16(acc + c, o);
          tmem_ld_wait();
          reg_fence(o);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            if (mine && c + i < ps.dim)
              *reinterpret_cast<float4*>(out + c + i) =
                  make_float4(__uint_as_float(o[i]) * f, __uint_as_float(o[i + 1]) * f, __uint_as_float(o[i + 2]) * f,
                              __uint_as_float(o[i + 3]) * f);
          __syncwarp();
        }
      }
      if (g == 0 && mine && *(volatile int*)&sm.loose)
        give_back<BF16>(a, reinterpret_cast<const KItem*>(a.plan + ps.dkv_items) + unit, kvh, key);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarps) tmem_dealloc(tmem, 512);

  if (it.slot < 0) return;
  // ── the last of a tile's parts to arrive adds them in their order (one whose wait gave up arrives too: this call's result
  // is void, the counter is whole for the next) ──
  if (tid == 0) {
    __threadfence();
    int* cnt = reinterpret_cast<int*>(a.plan + ps.dkv_counters) + (long long)it.counter * ps.kv_heads + kvh;
    sm.last = atomicAdd(cnt, 1) == it.parts - 1;
    if (sm.last) *cnt = 0;  // for the next call with this plan
    __threadfence();
  }
  __syncthreads();
  if (!sm.last) return;
  const int vecs = ps.dim / 4;
  const long long part_step = (long long)ps.kv_heads * 2 * kPackBlock * ps.dim;
  const int all = 2 * it.keys * vecs;
  constexpr int kTogether = 4;  // vectors of a thread that are in flight together
  for (int i0 = tid; i0 < all; i0 += kTogether * C::kThreads) {
    float4 sum[kTogether];
    const float* src[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int i = min(i0 + u * C::kThreads, all - 1), which = i / (it.keys * vecs), rest = i - which * it.keys * vecs;
      const int r = rest / vecs, c = (rest - r * vecs) * 4;
      src[u] = reinterpret_cast<const float*>(a.plan + ps.part_dkv) +
               ((((long long)it.slot0 * ps.kv_heads + kvh) * 2 + which) * kPackBlock + r) * ps.dim + c;
      sum[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k = 0; k < it.parts; ++k) {
      float4 v[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) v[u] = __ldcg(reinterpret_cast<const float4*>(src[u] + k * part_step));
#pragma unroll
      for (int u = 0; u < kTogether; ++u) sum[u].x += v[u].x, sum[u].y += v[u].y, sum[u].z += v[u].z, sum[u].w += v[u].w;
    }
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int i = i0 + u * C::kThreads;
      if (i >= all) continue;
      const int which = i / (it.keys * vecs), rest = i - which * it.keys * vecs, r = rest / vecs, c = (rest - r * vecs) * 4;
      const float f = which ? a.scale : 1.0f;
      const long long row = it.k0 + r;
      uint16_t* out = which ? static_cast<uint16_t*>(a.dk) + row * a.dk_row + kvh * a.dk_head
                            : static_cast<uint16_t*>(a.dv) + row * a.dv_row + kvh * a.dv_head;
      *reinterpret_cast<uint2*>(out + c) =
          make_uint2(pack2<BF16>(sum[u].x * f, sum[u].y * f), pack2<BF16>(sum[u].z * f, sum[u].w * f));
    }
  }
}

// ── dQ ───────────────────────────────────────────────────────────────────────
template <int DP, bool BF16, bool CAUSAL>
__global__ void __launch_bounds__(BwdCfg<DP>::kThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                 const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ BwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<DP>& sm = *reinterpret_cast<BwdSmem<DP>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using C = BwdCfg<DP>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kColAcc = C::kColAcc;
  const PackedShape& ps = a.s;
  let_next_start();
  wait_for_previous();
  const int unit = blockIdx.x / ps.heads, head = blockIdx.x - unit * ps.heads, kvh = head / ps.group;
  if (unit >= reinterpret_cast<const int*>(a.plan)[kHdrDq]) return;
  const QItem it = reinterpret_cast<const QItem*>(a.plan + ps.dq_items)[unit];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int dim16 = (ps.dim + 15) & ~15;
  const int see_end = CAUSAL ? min(it.lk, max(0, it.see + it.tokens)) : it.lk;  // one past the last key that is seen
  const int n = (see_end + kHalf - 1) / kHalf;
  constexpr uint32_t kColQ = kColAcc + DP, kColDO = kColQ + DP / 2;
  const uint32_t tmem = bwd_setup<DP>(sm, tid, warp);

  if (warp == C::kWarps) {
    if (lane == 0 && n > 0) {
      constexpr int NB = DP / 64;
      mbar_arrive_expect_tx(&sm.a_full, 2 * BwdSmem<DP>::kTile);
      for (int b = 0; b < NB; ++b) {
        tma_load_3d(sm.a[0] + b * kPackBlock * 128, &map_q, &sm.a_full, b * 64, head, it.q0);
        tma_load_3d(sm.a[1] + b * kPackBlock * 128, &map_do, &sm.a_full, b * 64, head, it.q0);
      }
      produce<DP>(sm, &map_k, &map_v, n, [&](int h, int* hd, int* row) {
        *hd = kvh;
        *row = it.k0 + h * kHalf;
      });
    }
    __syncwarp();
  } else if (warp == C::kWarps + 1) {
    // ── S = Q·Kᵀ and dP = dO·Vᵀ of step h into buffer h mod groups, once dQ is done with its last step's ──
    if (n > 0) {
      const uint32_t lead = elect_lead(), tm = uniform(tmem);
      const int steps = uniform(n), tail = uniform(see_end - (n - 1) * kHalf);
      const uint32_t id_s = idesc_f32acc(kPackBlock, kHalf, BF16 ? AB_BF16 : AB_F16, false, false);
      const uint64_t dk0 = sdesc(smem_u32(sm.ring[0][0]), 16, 1024, SW_128B);
      constexpr int kBBlk = (kHalf * 128) >> 4, kTileStep = BwdSmem<DP>::kStep >> 4;
      int buf = 0;       // score buffer of the step
      uint32_t par = 0;  // parity of its use
      auto next_buffer = [&] {
        if (++buf == C::kGroups) buf = 0, par ^= 1;
      };
      bool ok = wait_scores(sm, &sm.a_ready, 0, 12);
      for (int h = 0; ok && h < steps; ++h) {
        const int st = h % kStages;
        if (!(ok = wait_all(&sm.full[st], (h / kStages) & 1, &sm.abort, 13))) break;
        if (h == steps - 1 && (tail & 15)) {
          zero_tail<DP>(sm.ring[st][0], tail, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (h >= C::kGroups && !(ok = wait_scores(sm, &sm.g_done[buf], par ^ 1, 16))) break;
        tc_fence_after();
        const uint64_t bk = dk0 + (uint64_t)(st * 2 * kTileStep), bv = bk + kTileStep;
        const uint32_t ts = tm + buf * 128;
        auto one = [&](int s) {
          const uint64_t ob = (uint64_t)((s >> 2) * kBBlk + (s & 3) * 2);
          mma_ts_p(ts, tm + kColQ + s * 8, bk + ob, id_s, s > 0 ? 1u : 0u, lead);
          mma_ts_p(ts + kHalf, tm + kColDO + s * 8, bv + ob, id_s, s > 0 ? 1u : 0u, lead);
        };
        if (dim16 == DP) {
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) one(s);
        } else {
          for (int s = 0; s < dim16 / 16; ++s) one(s);
        }
        mma_commit_p(&sm.s_full[buf], lead);
        next_buffer();
      }
      issue_end(sm, lead);
    }
    __syncwarp();
  } else if (warp == C::kWarps + 2) {
    // ── dQ += dS·K ──
    if (n > 0) {
      const uint32_t lead = elect_lead(), tm = uniform(tmem);
      const int steps = uniform(n), tail = uniform(see_end - (n - 1) * kHalf);
      const uint32_t id_g = idesc_f32acc(kPackBlock, dim16, BF16 ? AB_BF16 : AB_F16, false, true);
      const uint64_t dk0 = sdesc(smem_u32(sm.ring[0][0]), kHalf * 128, 1024, SW_128B);
      constexpr int kTileStep = BwdSmem<DP>::kStep >> 4;
      int buf = 0;       // score buffer of the step
      uint32_t par = 0;  // parity of its use
      auto next_buffer = [&] {
        if (++buf == C::kGroups) buf = 0, par ^= 1;
      };
      bool ok = true;
      for (int h = 0; h < steps; ++h) {
        const int st = h % kStages, ks = h == steps - 1 ? (tail + 15) >> 4 : kHalf / 16;
        if (!(ok = wait_scores(sm, &sm.p_full[buf], par, 14))) break;
        tc_fence_after();
        const uint64_t gk = dk0 + (uint64_t)(st * 2 * kTileStep);
        auto one = [&](int s) {
          mma_ts_p(tm + kColAcc, tm + buf * 128 + s * 8, gk + (uint64_t)(s * (2048 >> 4)), id_g,
                   (h > 0 || s > 0) ? 1u : 0u, lead);
        };
        if (ks == kHalf / 16 && steps > kFineSteps) {
#pragma unroll
          for (int s = 0; s < kHalf / 16; ++s) one(s);
        } else {
          for (int s = 0; s < ks; ++s) one(s);
          for (int s = 0; steps <= kFineSteps && s < ks; ++s)
            mma_ts_p(tm + kColAcc, tm + buf * 128 + kHalf + s * 8, gk + (uint64_t)(s * (2048 >> 4)), id_g, 1u, lead);
        }
        mma_commit_p(&sm.g_done[buf], lead);
        mma_commit_p(&sm.empty[st], lead);
        next_buffer();
      }
      issue_end(sm, lead);
    }
    __syncwarp();
  } else {
    const int g = warp >> 2, row = tid - g * 128;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + g * 128;
    const bool mine = row < it.tokens;
    const int see = !mine ? 0 : CAUSAL ? min(it.lk, it.see + row + 1) : it.lk;
    float2 stat = make_float2(INFINITY, 0.0f);
    const long long at = (long long)head * ps.total_q + it.q0 + row;
    if (mine) stat = reinterpret_cast<const float2*>(a.plan + ps.rows)[at];
    float mult = 1.0f;
    if constexpr (!BF16) {  // |dS_ij| ≤ ‖dO_i‖ · max_j ‖V_j‖ + |Δ_i|
      const float* vn = reinterpret_cast<const float*>(a.plan + ps.v_norm) + (long long)kvh * ps.total_k + it.k0;
      float top = 0.0f;
      for (int i0 = 0; i0 < see_end; i0 += C::kSoft * kScanChunk) {
        const int end = min(see_end, i0 + (int)(C::kSoft * kScanChunk));
        for (int i = i0 + tid; i < end; i += C::kSoft) top = fmaxf(top, vn[i] < INFINITY ? vn[i] : 0.0f);
        if (tid == 0) *(volatile int*)&sm.scanned = i0 / (int)(C::kSoft * kScanChunk) + 1;
      }
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) sm.red[warp] = top;
      scores_sync<C::kSoft>();
      for (int i = 0; i < C::kWarps; ++i) top = fmaxf(top, sm.red[i]);
      if (mine) mult = pow2_below(reinterpret_cast<const float*>(a.plan + ps.do_norm)[at] * top + fabsf(stat.y));
    }
    const float scale2 = a.scale * kLog2e;
    bool ok = true;
    if (n > 0 && g < 2) {
      // group 0 moves Q, group 1 dO from shared memory to TMEM: a thread its row
      ok = mbar_wait(&sm.a_full, 0, &sm.abort, &g_packed_bwd_status, 17);
#pragma unroll
      for (int b = 0; b < DP / 64; ++b) {
        uint32_t u[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(sm.a[g] + b * kPackBlock * 128 + sw128_off(row, c));
          u[4 * c] = w.x, u[4 * c + 1] = w.y, u[4 * c + 2] = w.z, u[4 * c + 3] = w.w;
        }
        tmem_st32(tmem + lanes + (g == 0 ? kColQ : kColDO) + b * 32, u);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.a_ready);
    }
    if (n > 0 && n <= kFineSteps) {
      // Rows that see at most 128 keys: all their scores are in the two buffers, so Δ_i = Σ_j P_ij dP_ij is summed from
      // them.  dO·O carries the rounding of the stored O, which matters here (O is an average of few values): it
      // would add as much error to dQ and dK as the rounding of dS.  The dK/dV kernel reads the better Δ too.
      float t = 0.0f;
      if (g < n) {
        ok = ok && mbar_wait(&sm.s_full[g], 0, &sm.abort, &g_packed_bwd_status, 20);
        tc_fence_after();
        const int limit = see - g * kHalf;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32], d[32];
          tmem_ld32(ts + c * 32, s);
          tmem_ld32(ts + kHalf + c * 32, d);
          tmem_ld_wait();
          reg_fence(s);
          reg_fence(d);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float p = ex2(fmaf(__uint_as_float(s[i]), scale2, -stat.x)) * __uint_as_float(d[i]);
            t += c * 32 + i < limit ? p : 0.0f;
          }
        }
      }
      if (g < 2) sm.row_part[g][row] = t;
      scores_sync<C::kSoft>();
      ok = ok && !*(volatile int*)&sm.abort;
      stat.y = sm.row_part[0][row] + sm.row_part[1][row];
      if (mine && ok && g == 0) reinterpret_cast<float2*>(a.plan + ps.rows)[at].y = stat.y;
    }
    for (int h = g, k = 0; h < n; h += C::kGroups, ++k) {
      bool loose = false;
      if (CAUSAL && (h + 1) * kHalf > it.see + 1) {  // keys that some query of the tile does not see
        ok = ok && mbar_wait(&sm.full[h % kStages], (h / kStages) & 1, &sm.abort, &g_packed_bwd_status, 11);
        loose = holds_loose<BF16, BwdSmem<DP>::kStep>(sm.ring[h % kStages][0], row);
      }
      ok = ok && mbar_wait(&sm.s_full[g], k & 1, &sm.abort, &g_packed_bwd_status, 18);
      if (loose) drop_loose<BF16, BwdSmem<DP>::kStep>(sm.ring[h % kStages][0], row, &sm.loose);
      tc_fence_after();
      const int limit = see - h * kHalf;
      auto scores = [&](auto masked, auto fine) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32], d[32];
          tmem_ld32(ts + c * 32, s);
          tmem_ld32(ts + kHalf + c * 32, d);
          tmem_ld_wait();
          reg_fence(s);
          reg_fence(d);
          uint32_t pd[16], rest[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float p0, p1, d0 = __uint_as_float(d[i]), d1 = __uint_as_float(d[i + 1]);
            ffma2(p0, p1, __uint_as_float(s[i]), __uint_as_float(s[i + 1]), scale2, scale2, -stat.x, -stat.x);
            fadd2(d0, d1, -stat.y, -stat.y);
            fmul2(d0, d1, ex2(p0), ex2(p1));
            if constexpr (decltype(masked)::value) {
              d0 = c * 32 + i < limit ? d0 : 0.0f;
              d1 = c * 32 + i + 1 < limit ? d1 : 0.0f;
            }
            if constexpr (!BF16) fmul2(d0, d1, mult, mult);
            pd[i >> 1] = pack2<BF16>(d0, d1);
            if constexpr (decltype(fine)::value) rest[i >> 1] = pack2_rest<BF16>(pd[i >> 1], d0, d1);
          }
          tmem_st16(ts + c * 16, pd);
          if constexpr (decltype(fine)::value) tmem_st16(ts + kHalf + c * 16, rest);
        }
      };
      if (n <= kFineSteps) scores(std::true_type{}, std::true_type{});
      else if (__all_sync(0xffffffffu, limit >= kHalf)) scores(std::false_type{}, std::false_type{});
      else scores(std::true_type{}, std::false_type{});
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_full[g]);
    }
    if (n > 0) ok = ok && mbar_wait(&sm.fin, 0, &sm.abort, &g_packed_bwd_status, 19);
    if (__all_sync(0xffffffffu, ok && !*(volatile int*)&sm.abort)) {  // each group stores half of the 16-column chunks
      tc_fence_after();
      uint16_t* out = static_cast<uint16_t*>(a.dq) + (it.q0 + row) * a.dq_row + head * a.dq_head;
      for (int c = g * 16; c < dim16; c += C::kGroups * 16)
        store16<BF16>(tmem + lanes + kColAcc, n == 0, a.scale / mult, mine, out, c, ps.dim);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarps) tmem_dealloc(tmem, 512);
}

template <typename K> int set_smem(K kernel, int smem) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e == cudaSuccess ? VA_OK : set_error(VA_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
}

struct BwdMaps {
  CUtensorMap q_tile, do_tile, k_tile, v_tile, q_step, do_step, k_step, v_step;
};

template <int DP, bool BF16, bool CAUSAL> int launch_bwd(const BwdMaps& m, const BwdArgs& a, cudaStream_t st) {
  constexpr int smem = (int)sizeof(BwdSmem<DP>) + 1024;
  static PerDeviceOnce once;
  if (int rc = once.run([&]() -> int {
        if (int rc = set_smem(packed_dkv_kernel<DP, BF16, CAUSAL>, smem)) return rc;
        return set_smem(packed_dq_kernel<DP, BF16, CAUSAL>, smem);
      }))
    return rc;
  const long long g1 = (long long)a.s.max_dkv_items * a.s.kv_heads, g2 = (long long)a.s.max_dq_items * a.s.heads;
  VA_CHECK_ARG(g1 < (1LL << 31) && g2 < (1LL << 31), "packed attention backward: too many units");
  if (g2 > 0) {
    if (int rc = launch_behind("packed attention dQ", packed_dq_kernel<DP, BF16, CAUSAL>, (unsigned)g2, BwdCfg<DP>::kThreads, smem, st,
                               m.q_tile, m.do_tile, m.k_step, m.v_step, a))
      return rc;
  }
  if (g1 > 0) {
    if (int rc = launch_behind("packed attention dK/dV", packed_dkv_kernel<DP, BF16, CAUSAL>, (unsigned)g1, BwdCfg<DP>::kThreads, smem, st,
                               m.q_step, m.do_step, m.k_tile, m.v_tile, a))
      return rc;
  }
  return VA_OK;
}

template <bool BF16>
int packed_bwd(const void* d_out, const void* q, const void* k, const void* v, const void* out, const float* lse,
               void* dq, void* dk, void* dv, const int64_t* strides, int num_seqs, int total_q, int total_k, int heads,
               int kv_heads, int dim, int causal, int training, float scale, void* plan, size_t plan_bytes,
               cudaStream_t st) {
  if (int rc = packed_check(num_seqs, total_q, total_k, heads, kv_heads, dim, 1)) return rc;
  VA_CHECK_ARG(training, "packed attention backward: the plan must be built for training");
  VA_CHECK_ARG(scale > 0.0f && scale < INFINITY, "packed attention: the scale must be positive and finite");
  VA_CHECK_ARG(strides && (total_q == 0 || (d_out && q && out && lse && dq)) && (total_k == 0 || (k && v && dk && dv)),
               "packed attention backward: null pointer");
  BwdArgs a{};
  a.plan = static_cast<uint8_t*>(plan);
  a.s = packed_shape(num_seqs, total_q, total_k, heads, kv_heads, dim, causal != 0, 1);
  if (!plan || plan_bytes < a.s.total)
    return set_error(VA_ERR_WORKSPACE, "packed attention backward: plan of %zu < %zu bytes", plan_bytes, a.s.total);
  if (reinterpret_cast<uintptr_t>(plan) & 255)
    return set_error(VA_ERR_ALIGN, "packed attention backward: the plan needs 256-byte alignment");
  a.dq = dq, a.dk = dk, a.dv = dv, a.scale = scale;
  a.d_out = static_cast<const uint16_t*>(d_out), a.do_row = strides[6], a.do_head = strides[7];
  a.dq_row = strides[8], a.dq_head = strides[9], a.dk_row = strides[10], a.dk_head = strides[11];
  a.dv_row = strides[12], a.dv_head = strides[13];
  for (int i = 8; i < 14; ++i)
    if (strides[i] % 8) return set_error(VA_ERR_ALIGN, "packed attention backward: gradients need strides of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return set_error(VA_ERR_ALIGN, "packed attention backward: out and the gradients need 16-byte alignment");
  BwdMaps m;
  // a side without rows is never read: its maps may be any valid ones
  const void *mq = total_q ? q : k, *mo = total_q ? d_out : k, *mk = total_k ? k : q, *mv = total_k ? v : q;
  if (total_q == 0 && total_k == 0) return VA_OK;
  const int hq = total_q ? heads : kv_heads, hk = total_k ? kv_heads : heads;
  const int nq = total_q ? total_q : total_k, nk = total_k ? total_k : total_q;
  const int64_t* sq = total_q ? strides : strides + 2;
  const int64_t* so = total_q ? strides + 6 : strides + 2;
  const int64_t* sk = total_k ? strides + 2 : strides;
  const int64_t* sv = total_k ? strides + 4 : strides;
  for (int step = 0; step < 2; ++step) {
    const int rows = step ? kHalf : kPackBlock;
    if (int rc = packed_map(step ? &m.q_step : &m.q_tile, mq, BF16, nq, hq, dim, sq[0], sq[1], 1, rows, "q")) return rc;
    if (int rc = packed_map(step ? &m.do_step : &m.do_tile, mo, BF16, nq, hq, dim, so[0], so[1], 1, rows, "grad_out"))
      return rc;
    if (int rc = packed_map(step ? &m.k_step : &m.k_tile, mk, BF16, nk, hk, dim, sk[0], sk[1], 1, rows, "k")) return rc;
    if (int rc = packed_map(step ? &m.v_step : &m.v_tile, mv, BF16, nk, hk, dim, sv[0], sv[1], 1, rows, "v")) return rc;
  }
  {
    // queries' heads, and for f16 the key heads
    const int tokens = BF16 ? total_q : std::max(total_q, total_k), y = (total_q ? heads : 0) + (BF16 ? 0 : kv_heads);
    if (tokens > 0)
      if (int rc = launch_behind("packed attention backward rows", packed_rows_kernel<BF16>,
                                 dim3((tokens + kRowsBlock - 1) / kRowsBlock, y), 256, 0, st,
                                 static_cast<const uint16_t*>(out), static_cast<const uint16_t*>(d_out), strides[6],
                                 strides[7], static_cast<const uint16_t*>(v), strides[4], strides[5], lse,
                                 reinterpret_cast<float2*>(a.plan + a.s.rows),
                                 reinterpret_cast<float*>(a.plan + a.s.do_norm),
                                 reinterpret_cast<float*>(a.plan + a.s.v_norm), total_q, total_k, total_q ? heads : 0, dim))
        return rc;
  }
  auto go = [&](auto dp) -> int {
    return causal ? launch_bwd<dp, BF16, true>(m, a, st) : launch_bwd<dp, BF16, false>(m, a, st);
  };
  return dim <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace

int packed_bwd_status_read(int* out, cudaStream_t st) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_packed_bwd_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "device status read: %s", cudaGetErrorString(e));
  return VA_OK;
}

int packed_bwd_status_clear(cudaStream_t st) {
  static const int zero = 0;
  cudaError_t e = cudaMemcpyToSymbolAsync(g_packed_bwd_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "device status clear: %s", cudaGetErrorString(e));
  return VA_OK;
}

}  // namespace va

using namespace va;

#define VA_PACKED_BWD(sfx, T, BF)                                                                                    \
  int va_packed_attention_bwd_##sfx(const T* grad_out, const T* q, const T* k, const T* v, const T* out,             \
                                    const float* lse, T* grad_q, T* grad_k, T* grad_v, const int64_t* strides,       \
                                    int num_seqs, int total_q, int total_k, int num_heads, int num_kv_heads,         \
                                    int head_dim, int causal, int training, float softmax_scale, void* plan,         \
                                    size_t plan_bytes, va_stream_t stream) {                                         \
    return packed_bwd<BF>(grad_out, q, k, v, out, lse, grad_q, grad_k, grad_v, strides, num_seqs, total_q, total_k,  \
                          num_heads, num_kv_heads, head_dim, causal, training, softmax_scale, plan, plan_bytes,      \
                          (cudaStream_t)stream);                                                                     \
  }

extern "C" {
VA_PACKED_BWD(bf16, va_bf16, true)
VA_PACKED_BWD(f16, void, false)
}  // extern "C"
