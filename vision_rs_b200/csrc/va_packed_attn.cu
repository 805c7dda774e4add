// Attention over packed sequences of different lengths (tcgen05 + TMEM + TMA):
//
//   O_i = Σ_j P_ij v_j,  P_ij = exp(scale·q_i·k_j − lse_i),
//   lse_i = log Σ_j exp(scale·q_i·k_j)
//
// over the keys j of query i's own sequence (causal: j ≤ i + lk − lq), query
// head h reading key head h / group.  One pass over the keys with a running
// maximum and sum (f32); a row that sees no key gets O = 0 and lse = −∞.
//
// A CTA takes one unit of the plan (va_packed_plan.cu) for one head:
//   TILES = 2: 256 queries of one head as two 128-row tiles that share the
//     K/V stream (whole prompts, training);
//   TILES = 1: one tile whose rows are (query, head of the group) pairs, so
//     the query heads of a key head read its keys once, over a part of the
//     keys; two CTAs an SM.  The last CTA of a tile's parts to arrive joins
//     them in the parts' order (single tokens, few queries).
// Warps: 4 a tile for the softmax (a thread owns a row), 1 a tile to issue its
// MMAs, 1 TMA producer.  Per 64-key step: S = Q·Kᵀ into one of the tile's two
// score buffers in TMEM, the row's p = 2^(s − reference) back into the same
// columns as 16-bit P, O += P·V with P as the TMEM operand; the scores of step
// h + 2 follow step h's product into its buffer while the softmax is on h + 1.
// The reference only follows the row maximum when it grows by more than 2^8,
// so O is rarely rescaled.  P is held in the inputs' 16-bit type (rows of at
// most 128 keys: with its remainder as a second operand); its rounding adds
// about as much error as that of the output.  Sums, maxima and O stay f32.
//
// O is summed by the tensor core, which drops what lies about 2^-25 below the
// running sum: with n equal weights and values of one sign an unsplit tile's
// output is low by about n·2^-27.5 (measured: 0.06% at 2^17 keys, 0.6% at 2^20,
// 2.4% at 2^22); values around zero and tiles in parts show nothing.
//
// Measured (sustained; B200): prompts of 2049 and 8191 tokens, 16/2 heads of
// 128, causal, 296 µs = 0.99 PFLOP/s (254 µs before the power limit acts;
// floor 177): bound by issuing the MMAs and by the shared-memory reads of the
// N = 64 score MMAs.  16 images of 257–1601 tokens, 6 heads of 64, 64 µs (floor
// 21, the exponentials): bound by the softmax's latencies between them.  64
// single tokens over 17–8192 keys, 32/8 heads of 128, 219 µs = 4.9 TB/s (189
// before the power limit acts): HBM.
// An earlier form took 339 µs for the prompts where this one took 264 (short
// bursts): one 128-key score buffer a tile, one issuing warp for both tiles, an
// election for each MMA, scalar f32 arithmetic.  What each of these costs by
// itself was not measured.
//
// What a row does not see stays out of it, whatever it holds (another
// sequence's rows in a box, unused rows of a cache, later keys): scores of such
// keys are replaced, not added to, and as 0 · NaN would be NaN, the V blocks
// that hold them are checked (by a warp of its own, or by the producer of a
// one-tile unit): rows past the unit's last key become zeros, values that are
// not finite are left out of the product and given back to the rows that do
// see them.  The MMAs stop at the last 16-key group in use.
#include <cudaTypedefs.h>

#include <type_traits>

#include "va_common.cuh"
#include "va_packed.h"
#include "va_sm100.cuh"

namespace va {
using namespace sm100;

__device__ int g_packed_status;

namespace {

constexpr int kHalf = 64;  // keys of a score step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleAt = 8.0f;  // the reference follows the maximum once it is 2^8 ahead
// Rows of at most this many 64-key steps hold P as two 16-bit words, value and remainder, and multiply V by both: there the
// second product costs nothing that is measured, and the output is exact to its own rounding.
constexpr int kFineSteps = 2;
constexpr int kMaxChecked = 3;        // V blocks with keys that some row of a unit does not see: at most 256 rows' diagonal
constexpr float kF16Shift = 7.0f;   // f16: P is held times 2^7 (at most 2^15), so small ones keep their bits

// DP: head size in shared memory and TMEM (64 or 128; the TMA boxes fill what is past `dim` with zeros).
// ROWS: rows of a tile that hold anything (32 or 128; the MMAs always take 128, the others' results go nowhere).
template <int DP, int TILES, int ROWS> struct FwdCfg {
  static constexpr int kSlotBytes = kPackBlock * DP * 2;
  static constexpr int kQBytes = ROWS * DP * 2;
  static constexpr int kSlots = TILES == 2 ? (DP == 128 ? 4 : 8) : (DP == 128 ? 2 : 5) + (ROWS == 32 ? 1 : 0);
  static constexpr int kThreads = TILES == 2 ? 384 : 192;
  static constexpr int kCtas = TILES == 2 ? 1 : 2;  // an SM
  static constexpr uint32_t kTmemCols = TILES == 2 ? 512 : 256;
  static constexpr uint32_t kColS = 0, kColO = TILES * 128;  // tile m: scores at 128·m and 128·m + 64, O at kColO + DP·m
};

template <int DP, int TILES, int ROWS> struct FwdSmem {
  using C = FwdCfg<DP, TILES, ROWS>;
  uint8_t q[TILES][C::kQBytes];         // per 64 dims: ROWS rows × 128 bytes, SW128 (the MMAs read on into kv)
  uint8_t kv[C::kSlots][C::kSlotBytes];
  uint64_t q_full, kv_full[C::kSlots], kv_empty[C::kSlots];
  uint64_t s_full[TILES][2], p_full[TILES][2], o_done[TILES][2], v_sent[kMaxChecked], v_ready[kMaxChecked], fin;
  uint32_t tmem_base;
  int abort;
  int sent;  // blocks that the producer has sent
  int last;
  int loose;  // a checked V block held something that is not finite
};

struct FwdArgs {
  const uint8_t* plan;
  PackedShape s;
  const uint16_t* v;
  long long v_row, v_head;  // strides in elements
  void* out;
  float* lse;
  float scale;  // softmax scale · log2 e
};


template <int DP, int TILES, bool BF16, int ROWS>
__global__ void __launch_bounds__(FwdCfg<DP, TILES, ROWS>::kThreads, FwdCfg<DP, TILES, ROWS>::kCtas)
packed_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, FwdArgs a) {
  using C = FwdCfg<DP, TILES, ROWS>;
  extern __shared__ uint8_t smem_raw[];
  using Smem = FwdSmem<DP, TILES, ROWS>;
  Smem& sm = *reinterpret_cast<Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const PackedShape& ps = a.s;
  let_next_start();
  wait_for_previous();
  const int unit = blockIdx.x / ps.units, head = blockIdx.x - unit * ps.units;
  if (unit >= reinterpret_cast<const int*>(a.plan)[kHdrItems]) return;
  const QItem it = reinterpret_cast<const QItem*>(a.plan + ps.items)[unit];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = ps.few ? ps.group : 1;        // rows of a query in a tile
  const int kv_head = ps.few ? head : head / ps.group;
  const int rows = it.tokens * group;
  // 64-key steps of each tile (a causal first tile ends before the second) and one past the last key that any row sees
  int steps[TILES], see_end = 0;
#pragma unroll
  for (int m = 0; m < TILES; ++m) {
    const int n = TILES == 2 ? min(kPackBlock, it.tokens - m * kPackBlock) : it.tokens;
    int end = 0;
    if (n > 0) end = ps.causal ? min(it.lk, max(0, it.see + m * kPackBlock + n)) : it.lk;
    steps[m] = max(0, min(2 * it.kb1, (end + kHalf - 1) / kHalf) - 2 * it.kb0);
    see_end = max(see_end, end);
  }
  const int all_steps = max(steps[0], steps[TILES - 1]), nkb = (all_steps + 1) >> 1;
  const int dim16 = (ps.dim + 15) & ~15;
  // V blocks that are looked at before they are multiplied: those with keys hidden from some row (weight 0, but 0 · NaN
  // is NaN), and a last one that ends inside a 16-key group of the MMAs
  const int hidden = ps.causal ? min(see_end, max(0, it.see + 1)) : see_end;  // first key that a row does not see
  const int used_last = see_end - (it.kb0 + nkb - 1) * kPackBlock;            // keys of the last block
  const int checked = hidden < see_end ? max(it.kb0, hidden / kPackBlock)
                      : (used_last & 15) && used_last < kPackBlock ? it.kb0 + nkb - 1
                                                                   : it.kb0 + nkb;

  if (tid == 0) {
    mbar_init(&sm.q_full, 1);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&sm.kv_full[i], 1);
      mbar_init(&sm.kv_empty[i], TILES);
    }
    for (int m = 0; m < TILES; ++m) {
      for (int r = 0; r < 2; ++r) {
        mbar_init(&sm.s_full[m][r], 1);
        mbar_init(&sm.p_full[m][r], 128);
        mbar_init(&sm.o_done[m][r], 1);
      }
    }
    for (int i = 0; i < kMaxChecked; ++i) mbar_init(&sm.v_sent[i], 1), mbar_init(&sm.v_ready[i], 1);
    sm.loose = 0;
    mbar_init(&sm.fin, TILES);
    sm.abort = 0;
    sm.sent = 0;
    fence_mbar_init();
  }
  if (warp == TILES * 4) {
    tmem_alloc(&sm.tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  // ── V check (a whole warp): zeroes rows past the last key in its 16-key group, and what is not finite in blocks with
  // hidden keys (rows that see such a value get it back when the output is written) ──
  auto check_v = [&](int kb) -> bool {
    const int g = 2 * (kb - it.kb0) + 1, sv = g % C::kSlots, used = min(kPackBlock, see_end - kb * kPackBlock);
    if (!__all_sync(0xffffffffu, mbar_wait(&sm.kv_full[sv], (g / C::kSlots) & 1, &sm.abort, &g_packed_status, 4)))
      return false;
    auto cell = [&](int row, int c) {
      return reinterpret_cast<uint4*>(sm.kv[sv] + (c >> 3) * kPackBlock * 128 + sw128_off(row, c & 7));
    };
    for (int i = lane; i < ((used + 15) / 16 * 16 - used) * (DP / 8); i += 32)
      *cell(used + i / (DP / 8), i % (DP / 8)) = make_uint4(0, 0, 0, 0);
    if (hidden < see_end) {
      uint32_t any = 0;  // all cells are read without a branch between them; the rare second pass mends
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const uint4* base = reinterpret_cast<const uint4*>(sm.kv[sv] + c * kPackBlock * 128);
        const int cells = used * 8;  // 16-byte cells of the block's rows, in whatever order the swizzle has them
#pragma unroll 8
        for (int i = lane; i < cells; i += 32) {
          const uint4 x = base[i];
          any |= not_finite2<BF16>(x.x) | not_finite2<BF16>(x.y) | not_finite2<BF16>(x.z) | not_finite2<BF16>(x.w);
        }
      }
      bool found = false;
      if (__any_sync(0xffffffffu, any != 0)) {
        for (int i = lane; i < used * (DP / 8); i += 32) {
          uint4* p = cell(i / (DP / 8), i % (DP / 8));
          const uint4 x = *p;
          auto keep = [&](uint32_t w) {
            const uint32_t kept = finite2<BF16>(w);
            found |= kept != w;
            return kept;
          };
          *p = make_uint4(keep(x.x), keep(x.y), keep(x.z), keep(x.w));
        }
      }
      if (found) *(volatile int*)&sm.loose = 1;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.v_ready[kb - checked]);
    return true;
  };

  if (warp == TILES * 4) {
    // ── TMA producer: Q, then K and V blocks alternately through the slot ring.  A unit of one tile has its V blocks
    // checked here (a warp more would cost its softmax registers; what it holds up is at most the last two blocks) ──
    if (nkb > 0) {
      constexpr int NB = DP / 64;
      const uint32_t q_bytes = (uint32_t)(ps.few ? ps.q_tile * group : kPackBlock) * 128 * NB;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sm.q_full, q_bytes * TILES);
        for (int m = 0; m < TILES; ++m)
          for (int b = 0; b < NB; ++b)
            tma_load_3d(sm.q[m] + b * ROWS * 128, &map_q, &sm.q_full, b * 64, ps.few ? head * group : head,
                        it.q0 + m * kPackBlock);
      }
      int issued = 0;
      for (int g = 0; g < 2 * nkb; ++g) {
        const int st = g % C::kSlots, kb = it.kb0 + (g >> 1);
        if (g >= C::kSlots &&
            !__all_sync(0xffffffffu, mbar_wait(&sm.kv_empty[st], (g / C::kSlots - 1) & 1, &sm.abort, &g_packed_status, 1)))
          break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.kv_full[st], C::kSlotBytes);
          for (int b = 0; b < NB; ++b)
            tma_load_3d(sm.kv[st] + b * kPackBlock * 128, (g & 1) ? &map_v : &map_k, &sm.kv_full[st], b * 64, kv_head,
                        it.k0 + kb * kPackBlock);
        }
        ++issued;
        if ((g & 1) && kb >= checked) {
          if constexpr (TILES == 1) {
            if (!check_v(kb)) break;
          } else if (lane == 0) {
            mbar_arrive(&sm.v_sent[kb - checked]);
          }
        }
        if (TILES == 2 && lane == 0) *(volatile int*)&sm.sent = issued;
      }
      // loads issued here land (bounded) before the CTA can exit, also when it was another role that gave up
      for (int g = max(0, issued - C::kSlots); g < issued; ++g) {
        const long long c0 = clock64();
        while (!mbar_try_wait(&sm.kv_full[g % C::kSlots], (g / C::kSlots) & 1) && clock64() - c0 < kSpinCycles) {
        }
      }
      const long long c0 = clock64();
      while (!mbar_try_wait(&sm.q_full, 0) && clock64() - c0 < kSpinCycles) {
      }
    }
    __syncwarp();
  } else if (TILES == 2 && warp == TILES * 5 + 1) {
    // (the slot's barrier is in the phase of a block's load only once the load is sent, which may be as far ahead as the
    // unit is long)
    for (int kb = checked; kb < it.kb0 + nkb; ++kb)
      if (!__all_sync(0xffffffffu,
                      mbar_wait_behind(&sm.v_sent[kb - checked], 0, &sm.abort, &sm.sent, &g_packed_status, 12)) ||
          !check_v(kb))
        break;
    __syncwarp();
  } else if (warp > TILES * 4) {
    // ── MMA issuer of tile m: a converged warp whose values are uniform (the instructions between two MMAs are on
    // the critical path; operands that differ between lanes cost ~60 cycles an MMA), one elected lane issues ──
    const int m = TILES == 2 ? __shfl_sync(0xffffffffu, warp - TILES * 4 - 1, 0) : 0;
    if (nkb > 0) {
      auto uniform = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
      const uint32_t lead = elect_lead(), tm = uniform(tmem);
      const int n = uniform(steps[TILES == 2 ? m : 0]), all = uniform(all_steps), end = uniform(see_end - 2 * it.kb0 * kHalf);
      const uint32_t fmt = BF16 ? AB_BF16 : AB_F16;
      auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, &sm.abort, &g_packed_status, where));
      };
      constexpr int kBlk = (kPackBlock * 128) >> 4;              // 64 dims further, in descriptor units
      constexpr int kQBlk = (ROWS * 128) >> 4;
      constexpr int kHalfRows = (kHalf * 128) >> 4, kSlot = C::kSlotBytes >> 4;
      const uint32_t idesc_o = idesc_f32acc(kPackBlock, dim16, fmt, false, true);
      const uint32_t idesc_s = idesc_f32acc(kPackBlock, kHalf, fmt, false, false);
      const uint64_t dq = sdesc(smem_u32(sm.q[m]), 16, 1024, SW_128B);
      const uint64_t dk0 = sdesc(smem_u32(sm.kv[0]), 16, 1024, SW_128B);
      const uint64_t dv0 = sdesc(smem_u32(sm.kv[0]), kPackBlock * 128, 1024, SW_128B);
      const uint32_t ts = tm + C::kColS + m * 128, to = tm + C::kColO + m * DP;
      // S of step h (64 keys of K block h / 2, in slot st) into buffer h mod 2
      auto issue_s = [&](int h, int st) {
        const int left = end - h * kHalf;  // keys that some row sees, as the MMAs' extent
        const uint32_t idesc =
            left >= kHalf ? idesc_s : idesc_f32acc(kPackBlock, (left + 15) & ~15, fmt, false, false);
        const uint64_t dk = dk0 + (uint64_t)(st * kSlot + (h & 1) * kHalfRows);
        const uint32_t d = ts + (h & 1) * kHalf;
        if (dim16 == DP) {
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) {
            mma_ss_p(d, dq + (uint64_t)((s >> 2) * kQBlk + (s & 3) * 2), dk + (uint64_t)((s >> 2) * kBlk + (s & 3) * 2),
                     idesc, s > 0 ? 1u : 0u, lead);
          }
        } else {
          for (int s = 0; s < dim16 / 16; ++s) {
            mma_ss_p(d, dq + (uint64_t)((s >> 2) * kQBlk + (s & 3) * 2), dk + (uint64_t)((s >> 2) * kBlk + (s & 3) * 2),
                     idesc, s > 0 ? 1u : 0u, lead);
          }
        }
        mma_commit_p(&sm.s_full[m][h & 1], lead);
      };
      const bool fine = n <= kFineSteps;
      // Both tiles' threads wait for every K and V slot and release it, also where their own tile has no step left.
      int sk = 0, sv = 1;          // ring slots of the K block ahead and of this step's V block, and their parities
      uint32_t pk = 0, pv = 0;
      auto ahead = [&](int& slot, uint32_t& par) {
        slot += 2;
        if (slot >= C::kSlots) slot -= C::kSlots, par ^= 1;
      };
      bool ok = wait(&sm.q_full, 0, 2) && wait(&sm.kv_full[0], 0, 3);
      tc_fence_after();
      if (ok) {
        for (int h = 0; h < min(2, n); ++h) issue_s(h, 0);
        mma_commit_p(&sm.kv_empty[0], lead);
        ahead(sk, pk);
      }
      const int last_j = (all - 1) >> 1, in_last = uniform(used_last), check_j = uniform(checked - it.kb0);
      for (int h = 0; ok && h < all; ++h) {
        const int r = h & 1, g = h + 2;  // g: the step whose scores take this one's buffer
        const bool last = (h >> 1) == last_j;
        if (r == 0) {
          if (!(ok = wait(&sm.kv_full[sv], pv, 4))) break;
          if ((h >> 1) >= check_j && !(ok = wait(&sm.v_ready[(h >> 1) - check_j], 0, 11))) break;
        }
        if (h < n) {
          if (!(ok = wait(&sm.p_full[m][r], (h >> 1) & 1, 5))) break;
          tc_fence_after();
          const uint64_t dv = dv0 + (uint64_t)(sv * kSlot + r * kHalfRows);
          const uint32_t tp = ts + r * kHalf;
          const int ks = last ? min(kHalf / 16, (in_last - r * kHalf + 15) >> 4) : kHalf / 16;
          if (ks == kHalf / 16 && !fine) {
#pragma unroll
            for (int s = 0; s < kHalf / 16; ++s)
              mma_ts_p(to, tp + s * 8, dv + (uint64_t)(s * (2048 >> 4)), idesc_o, (h > 0 || s > 0) ? 1u : 0u, lead);
          } else {
            for (int s = 0; s < ks; ++s)
              mma_ts_p(to, tp + s * 8, dv + (uint64_t)(s * (2048 >> 4)), idesc_o, (h > 0 || s > 0) ? 1u : 0u, lead);
            for (int s = 0; fine && s < ks; ++s)
              mma_ts_p(to, tp + 32 + s * 8, dv + (uint64_t)(s * (2048 >> 4)), idesc_o, 1u, lead);
          }
          mma_commit_p(&sm.o_done[m][r], lead);
        }
        if (r == 0 && g < all && !(ok = wait(&sm.kv_full[sk], pk, 6))) break;
        if (g < n) {
          // the next scores overwrite P's columns: P·V has to be done with them
          if (!(ok = wait(&sm.o_done[m][r], (h >> 1) & 1, 7))) break;
          tc_fence_after();
          issue_s(g, sk);
        }
        if (r == 1 || h == all - 1) {
          mma_commit_p(&sm.kv_empty[sv], lead);
          ahead(sv, pv);
        }
        if (g < all && (r == 1 || g == all - 1)) {
          mma_commit_p(&sm.kv_empty[sk], lead);
          ahead(sk, pk);
        }
      }
      mma_commit_p(&sm.fin, lead);  // every MMA issued here completes before the CTA tears down
      const long long c0 = clock64();
      while (!mbar_try_wait(&sm.fin, 0) && clock64() - c0 < kSpinCycles) {
      }
    }
    __syncwarp();
  } else {
    // ── softmax: thread = row of tile m ──
    const int m = TILES == 2 ? warp >> 2 : 0, row = tid - m * 128;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + C::kColS + m * 128, to = tmem + lanes + C::kColO + m * DP;
    const int my_row = m * kPackBlock + row;
    const bool mine = my_row < rows;
    // one past the last key this row sees
    const int see = !mine ? 0 : ps.causal ? min(it.lk, it.see + my_row / group + 1) : it.lk;
    const int all_see = __reduce_min_sync(0xffffffffu, mine ? see : it.lk);  // keys below are hidden from no row here
    const float scale = a.scale;
    float ref = -INFINITY, sum = 0.0f;  // reference in log2 units
    bool ok = true;
    // warps without a row of the unit only keep the barriers going
    const bool idle = (m * kPackBlock + (warp & 3) * 32) >= rows;
    const int n = steps[m];
    // A wait that gives up is passed over, as are the thread's later ones: the loop goes on to its end, so the lanes of a
    // warp never part at its votes and TMEM instructions; nothing is written then.
    auto wait = [&](uint64_t* bar, int parity, int where) {
      ok = ok && mbar_wait(bar, parity, &sm.abort, &g_packed_status, where);
    };
    // Parts of a step's work on its 64 scores u:
    auto fetch = [&](int h, uint32_t (&u)[2][32]) {  // starts reading them
      wait(&sm.s_full[m][h & 1], (h >> 1) & 1, 8);
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld32(ts + (h & 1) * kHalf + c * 32, u[c]);
    };
    auto top_of = [&](int h, uint32_t (&u)[2][32]) -> float {  // has them, hides keys, largest in log2 units
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 2; ++c) reg_fence(u[c]);
      const int limit = see - (2 * it.kb0 + h) * kHalf;  // columns ≥ limit are hidden
      if ((2 * it.kb0 + h + 1) * kHalf > all_see) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= limit) u[c][i] = 0xff800000u;  // −∞
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 32; i += 4)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int x = (c & 1) * 2 + i;
          mx[c] = max3(mx[c], __uint_as_float(u[c >> 1][x]), __uint_as_float(u[c >> 1][x + 1]));
        }
      return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
    };
    auto follow = [&](int h, float top) {  // the reference follows, O is rescaled
      const bool grow = mine && (top > ref + kRescaleAt || ref == -INFINITY);
      if (!__any_sync(0xffffffffu, grow)) return;
      const float next = grow ? fmaxf(ref, top) : ref;  // a row's result does not depend on its warp's other rows
      if (h > 0) {
        const float f = next == -INFINITY ? 1.0f : ex2(ref - next);
        wait(&sm.o_done[m][(h & 1) ^ 1], ((h - 1) >> 1) & 1, 9);
        tc_fence_after();
        for (int c = 0; c < dim16; c += 16) {
          uint32_t o[16];
          tmem_ld16(to + c, o);
          tmem_ld_wait();
          reg_fence(o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st16(to + c, o);
        }
        sum *= f;
      }
      ref = next;
    };
    float part[4];
    auto exps = [&](int h, const uint32_t (&u)[32], int c, auto fine) {  // P of 32 keys
      const float base = ref == -INFINITY ? 0.0f : BF16 ? ref : ref - kF16Shift;
      uint32_t p[16], rest[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p0, p1;
        ffma2(p0, p1, __uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]), scale, scale, -base, -base);
        p0 = ex2(p0);
        p1 = ex2(p1);
        fadd2(part[2 * (i & 1)], part[2 * (i & 1) + 1], p0, p1);
        p[i] = pack2<BF16>(p0, p1);
        if constexpr (decltype(fine)::value) rest[i] = pack2_rest<BF16>(p[i], p0, p1);
      }
      tmem_st16(ts + (h & 1) * kHalf + c * 16, p);
      if constexpr (decltype(fine)::value) tmem_st16(ts + (h & 1) * kHalf + 32 + c * 16, rest);
    };
    auto give = [&](int h) {
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_full[m][h & 1]);
    };
    if (idle) {
      for (int h = 0; h < n; ++h) {
        wait(&sm.s_full[m][h & 1], (h >> 1) & 1, 8);
        mbar_arrive(&sm.p_full[m][h & 1]);
      }
    } else {
      auto steps_of = [&](auto fine) {
        for (int h = 0; h < n; ++h) {
          uint32_t u[2][32];
          fetch(h, u);
          follow(h, top_of(h, u));
          part[0] = part[1] = part[2] = part[3] = 0.0f;
          exps(h, u[0], 0, fine);
          exps(h, u[1], 1, fine);
          give(h);
        }
      };
      if (n <= kFineSteps) steps_of(std::true_type{});
      else steps_of(std::false_type{});
    }
    // ── output ──
    if (n > 0) wait(&sm.o_done[m][(n - 1) & 1], ((n - 1) >> 1) & 1, 10);
    if (__all_sync(0xffffffffu, ok) && !idle) {
      tc_fence_after();
      // a row without a key; one of NaN scores has no maximum either, but its sum is NaN
      const bool none = n <= 0 || (ref == -INFINITY && sum == sum);
      const float inv = 1.0f / sum;
      const float lse = !none ? (ref - (BF16 ? 0.0f : kF16Shift) + log2f(sum)) * kLn2 : -INFINITY;
      const int t = my_row / group, h = ps.few ? head * group + my_row - t * group : head;
      // Values that are not finite were left out of the product: a row that sees one has it in the output whatever its weight.
      const bool loose = n > 0 && checked < it.kb0 + nkb && *(volatile int*)&sm.loose;
      auto add_loose = [&](uint32_t (&o)[16], int c) {
        for (int j = checked * kPackBlock; j < min(see, it.kb1 * kPackBlock); ++j) {
          const uint16_t* vj = a.v + (it.k0 + j) * a.v_row + kv_head * a.v_head + c;
          for (int i = 0; i < 16 && c + i < ps.dim; ++i) {
            const float x = BF16 ? __uint_as_float((uint32_t)vj[i] << 16) : __half2float(__ushort_as_half(vj[i]));
            if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
          }
        }
      };
      if (it.slot < 0) {
        const long long at = (long long)(it.q0 + t) * ps.heads + h;
        uint16_t* out = static_cast<uint16_t*>(a.out) + at * ps.dim;
        for (int c = 0; c < dim16; c += 16) {
          uint32_t o[16];
          if (n > 0) {
            tmem_ld16(to + c, o);
            tmem_ld_wait();
            reg_fence(o);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = none ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
          if (loose && mine) add_loose(o, c);
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack2<BF16>(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
          if (mine) {
            *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
            if (c + 8 < ps.dim) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
          __syncwarp();
        }
        if (mine) a.lse[(long long)h * ps.total_q + it.q0 + t] = lse;
      } else {
        const long long at = ((long long)it.slot * ps.units + head) * ROWS + row;
        float* out = reinterpret_cast<float*>(const_cast<uint8_t*>(a.plan) + ps.part_o) + at * ps.dim;
        for (int c = 0; c < dim16; c += 16) {
          uint32_t o[16];
          if (n > 0) {
            tmem_ld16(to + c, o);
            tmem_ld_wait();
            reg_fence(o);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = none ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
          if (loose && mine) add_loose(o, c);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            if (mine && c + i < ps.dim)
              *reinterpret_cast<uint4*>(out + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          __syncwarp();
        }
        if (mine) reinterpret_cast<float*>(const_cast<uint8_t*>(a.plan) + ps.part_lse)[at] = lse;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == TILES * 4) tmem_dealloc(tmem, C::kTmemCols);

  if constexpr (TILES == 1) {
    if (it.slot < 0) return;
    // ── the last of a tile's parts joins them: O = Σ w_k O_k, w_k = exp(lse_k − lse).  A part whose wait gave up arrives too:
    // this call's result is void (the status says so), the counter is whole for the next ──
    if (tid == 0) {
      __threadfence();
      int* cnt = reinterpret_cast<int*>(const_cast<uint8_t*>(a.plan) + ps.counters) + (long long)it.counter * ps.units + head;
      sm.last = atomicAdd(cnt, 1) == it.parts - 1;
      if (sm.last) *cnt = 0;  // for the next call with this plan
      __threadfence();
    }
    __syncthreads();
    if (!sm.last) return;
    const float* plse = reinterpret_cast<const float*>(a.plan + ps.part_lse);
    const float* po = reinterpret_cast<const float*>(a.plan + ps.part_o);
    const long long base = ((long long)it.slot0 * ps.units + head) * ROWS, step = (long long)ps.units * ROWS;
    for (int r = warp; r < rows; r += C::kThreads / 32) {
      float top = -INFINITY;
      for (int k = lane; k < it.parts; k += 32) top = fmaxf(top, __ldcg(plse + base + k * step + r));
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float ref = top == -INFINITY ? 0.0f : top;
      float total = 0.0f;
      for (int k = lane; k < it.parts; k += 32) total += exp2f((__ldcg(plse + base + k * step + r) - ref) * kLog2e);
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
      const int t = r / group, h = head * group + r - t * group;
      uint16_t* out = static_cast<uint16_t*>(a.out) + ((long long)(it.q0 + t) * ps.heads + h) * ps.dim;
      for (int c = lane * 4; c < ps.dim; c += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < it.parts; ++k) {
          const float w = exp2f((__ldcg(plse + base + k * step + r) - ref) * kLog2e) * inv;
          const float4 f = __ldcg(reinterpret_cast<const float4*>(po + (base + k * step + r) * ps.dim + c));
          acc.x = fmaf(w, f.x, acc.x);
          acc.y = fmaf(w, f.y, acc.y);
          acc.z = fmaf(w, f.z, acc.z);
          acc.w = fmaf(w, f.w, acc.w);
        }
        *reinterpret_cast<uint2*>(out + c) = make_uint2(pack2<BF16>(acc.x, acc.y), pack2<BF16>(acc.z, acc.w));
      }
      if (lane == 0) a.lse[(long long)h * ps.total_q + it.q0 + t] = total > 0.0f || total != total ? ref + logf(total) : -INFINITY;
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

}  // namespace

int packed_map(CUtensorMap* m, const void* base, bool bf16, int rows, int heads, int dim, long long row_stride,
               long long head_stride, int box_heads, int box_rows, const char* what) {
  auto fn = encode_fn();
  if (!fn) return set_error(VA_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled unavailable");
  if (heads == 1) head_stride = dim;
  if (rows <= 1) row_stride = (long long)heads * dim;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || row_stride % 8 || head_stride % 8 || row_stride <= 0 || head_stride <= 0)
    return set_error(VA_ERR_ALIGN, "packed attention: %s needs a 16-byte aligned base and strides of 16 bytes", what);
  const cuuint64_t d[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t s[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t bx[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, es[3] = {1, 1, 1};
  CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(base), d, s, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(VA_ERR_ALIGN, "packed attention: tensor map for %s rejected (CUresult %d)", what, (int)r);
  return VA_OK;
}

namespace {

template <int DP, int TILES, bool BF16, int ROWS>
int launch_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const FwdArgs& a, cudaStream_t st) {
  using C = FwdCfg<DP, TILES, ROWS>;
  auto kernel = packed_attn_kernel<DP, TILES, BF16, ROWS>;
  constexpr int smem = (int)sizeof(FwdSmem<DP, TILES, ROWS>) + 1024;
  static PerDeviceOnce once;
  if (int rc = once.run([&]() -> int {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        return e == cudaSuccess ? VA_OK : set_error(VA_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      }))
    return rc;
  const long long grid = (long long)a.s.max_items * a.s.units;
  VA_CHECK_ARG(grid < (1LL << 31), "packed attention: too many units");
  return launch_behind("packed attention", kernel, (unsigned)grid, C::kThreads, smem, st, mq, mk, mv, a);
}

template <bool BF16>
int packed_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int64_t* strides, int num_seqs,
               int total_q, int total_k, int heads, int kv_heads, int dim, int causal, int training, float scale,
               void* plan, size_t plan_bytes, cudaStream_t st) {
  if (int rc = packed_check(num_seqs, total_q, total_k, heads, kv_heads, dim, training)) return rc;
  VA_CHECK_ARG(scale > 0.0f && scale < INFINITY, "packed attention: the scale must be positive and finite");
  if (total_q == 0) return VA_OK;
  VA_CHECK_ARG(q && out && lse && strides && (total_k == 0 || (k && v)), "packed attention: null pointer");
  FwdArgs a{static_cast<const uint8_t*>(plan),
            packed_shape(num_seqs, total_q, total_k, heads, kv_heads, dim, causal != 0, training != 0),
            static_cast<const uint16_t*>(v), strides[4], strides[5], out, lse, scale * kLog2e};
  if (!plan || plan_bytes < a.s.total)
    return set_error(VA_ERR_WORKSPACE, "packed attention: plan of %zu < %zu bytes", plan_bytes, a.s.total);
  if ((reinterpret_cast<uintptr_t>(plan) & 255) || (reinterpret_cast<uintptr_t>(out) & 15))
    return set_error(VA_ERR_ALIGN, "packed attention: the plan needs 256-byte and the output 16-byte alignment");
  CUtensorMap mq, mk, mv;
  const PackedShape& s = a.s;
  if (int rc = packed_map(&mq, q, BF16, total_q, heads, dim, strides[0], strides[1], s.few ? s.group : 1,
                          s.few ? s.q_tile : kPackBlock, "q"))
    return rc;
  if (total_k > 0) {
    if (int rc = packed_map(&mk, k, BF16, total_k, kv_heads, dim, strides[2], strides[3], 1, kPackBlock, "k")) return rc;
    if (int rc = packed_map(&mv, v, BF16, total_k, kv_heads, dim, strides[4], strides[5], 1, kPackBlock, "v")) return rc;
  } else {
    mk = mv = mq;  // no unit has a key block: never read
  }
  auto go = [&](auto dp) -> int {
    if (!s.few) return launch_fwd<dp, 2, BF16, 128>(mq, mk, mv, a, st);
    return s.tile_rows == 32 ? launch_fwd<dp, 1, BF16, 32>(mq, mk, mv, a, st) : launch_fwd<dp, 1, BF16, 128>(mq, mk, mv, a, st);
  };
  return dim <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace

int packed_status_read(int* out, cudaStream_t st) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_packed_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "device status read: %s", cudaGetErrorString(e));
  return VA_OK;
}

int packed_status_clear(cudaStream_t st) {
  static const int zero = 0;
  cudaError_t e = cudaMemcpyToSymbolAsync(g_packed_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "device status clear: %s", cudaGetErrorString(e));
  return VA_OK;
}

}  // namespace va

using namespace va;

extern "C" {

int va_packed_attention_fwd_bf16(const va_bf16* q, const va_bf16* k, const va_bf16* v, va_bf16* out, float* lse,
                                 const int64_t* strides, int num_seqs, int total_q, int total_k, int num_heads,
                                 int num_kv_heads, int head_dim, int causal, int training, float softmax_scale,
                                 void* plan, size_t plan_bytes, va_stream_t stream) {
  return packed_fwd<true>(q, k, v, out, lse, strides, num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim,
                          causal, training, softmax_scale, plan, plan_bytes, (cudaStream_t)stream);
}

int va_packed_attention_fwd_f16(const void* q, const void* k, const void* v, void* out, float* lse,
                                const int64_t* strides, int num_seqs, int total_q, int total_k, int num_heads,
                                int num_kv_heads, int head_dim, int causal, int training, float softmax_scale,
                                void* plan, size_t plan_bytes, va_stream_t stream) {
  return packed_fwd<false>(q, k, v, out, lse, strides, num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim,
                           causal, training, softmax_scale, plan, plan_bytes, (cudaStream_t)stream);
}

}  // extern "C"
