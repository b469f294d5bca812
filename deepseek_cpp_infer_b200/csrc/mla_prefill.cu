// Prompt attention in expanded form (the per-head attention of
// src/models/deepseek/mla.cpp:86-116 for whole chunks of query rows), sm_100a:
//   s_ij = ([q_nope_i | q_rope_i] . [k_nope_j | k_rope_j]) * scale
//   out_i = sum_j softmax_j(s_ij) v_j,  lse_i = ln sum_j exp(s_ij)
//
// One pass over the keys with a running maximum and sum per query row.  A work
// item is 256 query rows of one (sequence, head) as two tiles of 128, each a
// tcgen05 M = 128: while the tensor core computes S of one tile, the other
// tile's softmax runs.  Per 128 keys and tile
//   S [128 x 128] = Q K^T  (12 K-steps over nope | rope, operands by TMA; the
//                           rope key is one tensor for all heads)
//   P = exp2(S - m) in bf16, written over S in tensor memory
//   O [128 x vd] += P V    (P from tensor memory, V as stored, MN-major)
// TMEM: S0 | S1 | O0 | O1, 4 x 128 columns.  O is rescaled only when a row's
// maximum has grown by 2^8 since its reference was set.
//
// Roles (12 warps): two softmax warpgroups (thread = query row), a TMA warp,
// an MMA warp, and two warps that make masked values harmless: a zero
// probability times an infinite or NaN value would be NaN, so values of rows
// past a sequence's keys are cleared, and in tiles that the causal border
// crosses non-finite values are replaced by zero and added to the outputs of
// the rows that do see them.  Persistent CTAs walk the items, heavy ones
// first within groups of heads whose keys and values stay in L2; an item's
// prologue overlaps the last one's epilogue.
//
// What bounds it.  With equal items (2048 rows, 128 heads, no causal mask) 311 us,
// 1104 TFLOP/s: a step's softmax and hand-overs, which only the other tile's MMAs
// hide (2048 causal rows: the tensor pipe at 38%).  Causal prompts lose more
// to the items' fixed stride: they differ in length, and the same CTAs get the
// long ones of every round, so that with an item counted as its steps and one
// the most loaded SM has 324 of a mean 249 at 4096 rows x 128 heads (710 - 810 us
// by GPU and power, 860 - 970 TFLOP/s), 124 of 104 at 1024 rows behind 3000 keys
// (280 - 330 us), 48 of 31 at 4096 rows x 16 heads (105 us) and 31 of 16 at prompts
// of 2048, 1500, 600 and 100 rows; handed to whichever CTA is free they would
// have 253, 118, 33 and 19.  Long calls at 128 heads also run at 1.6 - 1.75 GHz
// under the 1000 W limit.  32 prompts of 512 rows at 16 heads take 83 - 91 us, 2
// times the time of their bytes: an item is only 1 to 4 steps long, so that its Q
// load, first softmax and output show.  What did not help: an MMA warp for each tile
// (15% slower: the tiles fall into step), two softmax warpgroups a tile, P
// handed over in halves, part of the exponentials as polynomials, the next
// item's first scores ahead of this item's output.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "dsb_internal.h"
#include "dsb_ptx.cuh"
#include "packed.cuh"

namespace dsb {
namespace {

constexpr int kRows = 128;       // query rows per tile, keys per step
constexpr int kThreads = 12 * 32;
constexpr int kTmaWarp = 8, kMmaWarp = 9, kScanWarp = 10;
// Non-finite values that were taken out of an item's bordering tiles, a word per
// column: for +inf, -inf and NaN the first key that holds one, 10 bits each,
// counted from the first bordering step.  (The border crosses at most 255 keys
// behind the first step's common ones: three steps, 384 keys; 1023: none.)
constexpr int kPlusInf = 0, kMinusInf = 10, kNan = 20;  // shifts
constexpr uint32_t kKeyMask = 1023, kNothing = 0x3fffffffu;
constexpr float kLazy = 8.0f;    // log2 headroom before O is rescaled

template <int NOPE, int P, int VD>
struct Shape {
  static constexpr int NN = NOPE / 64;                // 64-column slabs
  static constexpr int NQ = NN + 1;                   // slabs of Q and K: nope, rope
  static constexpr int NV = VD / 64;
  static constexpr int SLAB = kRows * 128;            // bytes
  static constexpr int NS = 8;                        // ring slots
  static constexpr int OFF_RING = 0;
  static constexpr int OFF_Q = NS * SLAB;             // [2 tiles][NQ slabs]
  static constexpr int OFF_BAD = OFF_Q + 2 * NQ * SLAB;  // [3 items]: a word per column, any [2]
  static constexpr int BAD_BYTES = VD * 4 + 8;
  static constexpr int NBAR = 2 * NS + 2 + 8 + 4 * 2 + 1 + 6;
  static constexpr int OFF_BAR = OFF_BAD + 3 * BAD_BYTES;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 32 + 1024;
  static constexpr int ROPE_BYTES = kRows * P * 2;
  static constexpr int K_BYTES = NN * SLAB + ROPE_BYTES;
  static_assert(SMEM_BYTES <= 232448, "shared memory");
  static_assert(OFF_BAR % 8 == 0, "alignment");
  // TMEM columns
  static constexpr uint32_t T_S = 0, T_O = 256;
};

// Ring slots in load order.  A V tile of two slabs is one MMA operand, so its
// slots must follow one another: a single last slot is passed over.
template <int NS>
struct Ring {
  int slot = 0;
  uint32_t used = 0;  // parity of each slot's uses
  __device__ int peek(int n) const { return slot + n > NS ? 0 : slot; }
  __device__ int take(int n) {  // n neighbouring slots
    const int s = peek(n);
    slot = s + n == NS ? 0 : s + n;
    return s;
  }
  __device__ uint32_t phase(int s) const { return (used >> s) & 1u; }
  __device__ void flip(int s) { used ^= 1u << s; }
};

// A work item: 256 query rows of one head of one sequence.
struct Item {
  int b, h, row0;        // first query row within the sequence
  int q0, k0, lq, lk;    // the sequence's rows
  int rows;              // rows of the sequence that are computed (at most max_q)
  int n[2];              // key steps of each tile
  __device__ int steps() const { return max(n[0], n[1]); }
  // keys that all rows of the item see: a step that reaches further is a bordering one
  __device__ int common(bool causal) const { return min(lk, causal ? row0 + 1 + lk - lq : lk); }
  // the first bordering step
  __device__ int border(bool causal) const { return max(0, common(causal)) / kRows; }
  // keys that query row i of the sequence sees
  __device__ int sees(int i, bool causal) const { return causal ? max(0, min(lk, i + 1 + lk - lq)) : lk; }
};

struct Order {
  int pairs;      // B * H
  int blocks;     // 256-row blocks of max_q
  int group;      // heads per group
};

// Item `it`: groups of heads; within a group the last (longest) block of every
// head first.
__device__ __forceinline__ bool get_item(const dsb_mla_prefill_args& a, const Order& o, int it, Item* x, bool* bad) {
  const int per = o.group * o.blocks, g = it / per;
  const int first = g * o.group, heads = min(o.group, o.pairs - first);
  const int r = it - g * per;
  const int blk = o.blocks - 1 - r / heads, pair = first + r % heads;
  x->b = pair / a.H;
  x->h = pair % a.H;
  x->row0 = blk * 2 * kRows;
  x->q0 = a.cu_q[x->b];
  x->k0 = a.cu_k[x->b];
  x->lq = a.cu_q[x->b + 1] - x->q0;
  x->lk = a.cu_k[x->b + 1] - x->k0;
  *bad = x->q0 < 0 || x->k0 < 0 || x->lq < 0 || x->lk < 0 || x->lq > a.Tq - x->q0 || x->lk > a.Tk - x->k0;
  if (*bad) return false;
  x->rows = min(x->lq, a.max_q);
  *bad = x->lq > a.max_q;
  if (x->row0 >= x->rows) return false;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = min(x->row0 + (t + 1) * kRows, x->rows) - 1;  // the tile's last row
    const int keys = x->row0 + t * kRows < x->rows ? x->sees(last, a.causal != 0) : 0;
    x->n[t] = (keys + kRows - 1) / kRows;
  }
  return true;
}

// Stores 32 bf16 columns of 32 consecutive rows, a row per lane.  Lanes of four
// exchange their 16-byte pieces so that a store writes 64 contiguous bytes of
// each of 8 rows, whole sectors (a lane storing its own row's pieces writes
// half sectors of 32 rows: the epilogue of a 256-row item took 15,000 cycles).
// dst: the first column in the first row of this lane's four; n_live: how many
// of the four are wanted (or more).
__device__ __forceinline__ void store_rows(uint32_t (&w)[16], __nv_bfloat16* dst, int64_t ld, int n_live) {
  const int lane = (int)lane_id();
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {  // transpose 4 x 4 pieces
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q & o) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t& lo = w[4 * q + e];
        uint32_t& hi = w[4 * (q | o) + e];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, o);
        if (up) lo = got;
        else hi = got;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (q < n_live)
      *reinterpret_cast<uint4*>(dst + q * ld + (lane & 3) * 8) =
          make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
}

template <int NOPE, int P, int VD>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap map_qn, const __grid_constant__ CUtensorMap map_qr,
                   const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_kr,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ dsb_mla_prefill_args a,
                   const __grid_constant__ Order order, int items, float scale_log2, int* __restrict__ status) {
  using S = Shape<NOPE, P, VD>;
  constexpr int NN = S::NN, NQ = S::NQ, NV = S::NV, NS = S::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);  // [NS] slab(s) landed
  uint64_t* empty = full + NS;                                      // [NS] its last MMA done
  uint64_t* q_full = empty + NS;                                    // Q of an item landed
  uint64_t* q_empty = q_full + 1;                                   // its last QK done
  uint64_t* v_safe = q_empty + 1;                                   // [4] V of a bordering step seen to, in turn
  uint64_t* v_load = v_safe + 4;                                    // [4] its load has been issued
  uint64_t* s_full = v_load + 4;                                    // [2] per tile: S ready
  uint64_t* p_full = s_full + 2;                                    // [2] P written
  uint64_t* pv_done = p_full + 2;                                   // [2] PV done
  uint64_t* o_free = pv_done + 2;                                   // [2] O read
  uint64_t* drain = o_free + 2;                                     // every MMA issued is done
  uint64_t* bad_full = drain + 1;                                   // [3] an item's non-finite values recorded
  uint64_t* bad_free = bad_full + 3;                                // [3] and its outputs written
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + S::OFF_MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile int* no_abort = reinterpret_cast<volatile int*>(misc + 2);  // never raised: for drain waits

  const int warp = uniform((int)warp_id()), lane = (int)lane_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&v_safe[i], 2);
      mbar_init(&v_load[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bad_full[i], 2);
      mbar_init(&bad_free[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(drain, 1);
    *abort = 0;
    *no_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(misc, 512);
    tmem_relinquish();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&map_qn);
    tma_prefetch_desc(&map_qr);
    tma_prefetch_desc(&map_kn);
    tma_prefetch_desc(&map_kr);
    tma_prefetch_desc(&map_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem = (uint32_t)uniform((int)misc[0]);
  const uint32_t smem_base = smem_u32(smem);
  const bool causal = a.causal != 0;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
  };
  bool ok = true;
  // 384 threads were launched with 168 registers each; the softmax warps hold
  // a row's 128 scores: 256 * 192 + 128 * 120 = 384 * 168 (208 + 88 spill in the
  // other roles: 32 prompts of 512 rows, 16 heads, 90.6 us instead of 85.4)
#define DSB_FEW_REGS asm volatile("setmaxnreg.dec.sync.aligned.u32 120;")

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ TMA producer
    DSB_FEW_REGS;
    Ring<NS> ring;
    uint32_t n_item = 0, n_safe = 0;
    uint32_t ever = 0;  // slots used at least once
    auto slab = [&](int s, const CUtensorMap* map, int bytes, int x, int y) {
      if (((ever >> s) & 1u) && !wait(&empty[s], ring.phase(s) ^ 1u)) return false;
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[s], bytes);
        tma_load_2d(smem + S::OFF_RING + s * S::SLAB, map, &full[s], x, y);
      }
      ever |= 1u << s;
      ring.flip(s);
      return true;
    };
    for (int it = blockIdx.x; ok && it < items; it += gridDim.x) {
      Item x;
      bool bad;
      const bool live = get_item(a, order, it, &x, &bad);
      if (bad && lane == 0) atomicCAS(status, 0, kStatusBadInput);
      if (!live || x.steps() == 0) continue;
      if (n_item > 0 && !wait(q_empty, (n_item - 1) & 1u)) { ok = false; break; }
      ++n_item;
      if (elect_one()) {
        const int tiles = (x.n[0] > 0 ? 1 : 0) + (x.n[1] > 0 ? 1 : 0);
        mbar_arrive_expect_tx(q_full, tiles * S::K_BYTES);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (x.n[t] == 0) continue;
          uint8_t* dst = smem + S::OFF_Q + t * NQ * S::SLAB;
          const int y = x.q0 + x.row0 + t * kRows;
          for (int i = 0; i < NN; ++i)
            tma_load_2d(dst + i * S::SLAB, &map_qn, q_full, (int)(x.h * a.hd_q_nope) + 64 * i, y);
          tma_load_2d(dst + NN * S::SLAB, &map_qr, q_full, (int)(x.h * a.hd_q_rope), y);
        }
      }
      const int n = x.steps();
      const int full_keys = x.common(causal);
      for (int s = 0; ok && s < n; ++s) {
        const int y = x.k0 + s * kRows;
        for (int i = 0; ok && i < NN; ++i)
          ok = slab(ring.take(1), &map_kn, S::SLAB, (int)(x.h * a.hd_k_nope) + 64 * i, y);
        if (ok) ok = slab(ring.take(1), &map_kr, S::ROPE_BYTES, 0, y);
        if (!ok) break;
        const int v0 = ring.take(NV);
        for (int i = 0; ok && i < NV; ++i) ok = slab(v0 + i, &map_v, S::SLAB, (int)(x.h * a.hd_v) + 64 * i, y);
        if (ok && (s + 1) * kRows > full_keys) warp_arrive(&v_load[n_safe++ & 3u]);
      }
    }
    if (!ok) raise_abort(abort, status, kStatusTimeout);
    // every copy must land before shared memory is released, also when a
    // consumer has given up
    for (int s = 0; s < NS; ++s)
      if ((ever >> s) & 1u) mbar_wait(&full[s], ring.phase(s) ^ 1u, no_abort);
    if (n_item > 0) mbar_wait(q_full, (n_item - 1) & 1u, no_abort);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------- MMA issuer
    // One elected lane runs the role, its operands in uniform registers (an MMA
    // issued from a lane == 0 branch costs 147 cycles; so 66 at N = 128).
    DSB_FEW_REGS;
    if (elect_one()) {
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort); };
      constexpr uint32_t ID_QK = idesc_bf16_f32(128, 128, 0, 0), ID_PV = idesc_bf16_f32(128, VD, 0, 1);
      const uint64_t d_q = smem_desc(smem_base + S::OFF_Q, 16, 1024, kSwizzle128B);
      const uint64_t d_k = smem_desc(smem_base + S::OFF_RING, 16, 1024, kSwizzle128B);
      const uint64_t d_qr = P == 64 ? d_q : smem_desc(smem_base + S::OFF_Q, 16, 512, kSwizzle64B);
      const uint64_t d_kr = P == 64 ? d_k : smem_desc(smem_base + S::OFF_RING, 16, 512, kSwizzle64B);
      const uint64_t d_v = smem_desc(smem_base + S::OFF_RING, S::SLAB, 1024, kSwizzle128B);
      Ring<NS> ring;
      uint32_t n_item = 0, n_safe = 0;
      uint32_t step_of[2] = {0, 0}, item_of[2] = {0, 0};  // PV steps and items of each tile
      int k_slot[NQ], v_slot = 0;
      // K of the next step has landed
      auto wait_k = [&]() {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          k_slot[i] = ring.take(1);
          if (!wait(&full[k_slot[i]], ring.phase(k_slot[i]))) return false;
          ring.flip(k_slot[i]);
        }
        tc_fence_after();
        return true;
      };
      auto issue_qk = [&](int t) {
        const uint32_t d = tmem + S::T_S + t * 128;
        const uint32_t qo = (uint32_t)(t * NQ * S::SLAB) >> 4;
#pragma unroll
        for (int i = 0; i < NN; ++i)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_bf16_ss(d, d_q + qo + ((i * S::SLAB) >> 4) + ks * 2,
                        d_k + ((uint32_t)(k_slot[i] * S::SLAB) >> 4) + ks * 2, ID_QK, i > 0 || ks > 0 ? 1u : 0u);
#pragma unroll
        for (int ks = 0; ks < P / 16; ++ks)
          mma_bf16_ss(d, d_qr + qo + ((NN * S::SLAB) >> 4) + ks * 2,
                      d_kr + ((uint32_t)(k_slot[NN] * S::SLAB) >> 4) + ks * 2, ID_QK, 1u);
        tc_commit(&s_full[t]);
      };
      auto release_k = [&]() {
#pragma unroll
        for (int i = 0; i < NQ; ++i) tc_commit(&empty[k_slot[i]]);
      };
      int it = blockIdx.x;
      // Of an item this role needs its tiles' steps and the keys that all rows see.
      // Finding them takes 1400 cycles (the lengths, five divisions): it is done
      // for the next item while this one's first softmax runs.
      int n_next[2], keys_next;
      auto find_next = [&] {
        for (; it < items; it += gridDim.x) {
          Item x;
          bool bad;
          if (!get_item(a, order, it, &x, &bad) || x.steps() == 0) continue;
          n_next[0] = x.n[0];
          n_next[1] = x.n[1];
          keys_next = x.common(causal);
          return true;
        }
        return false;
      };
      bool have = find_next();
      while (ok && have) {
        const int n_of[2] = {n_next[0], n_next[1]}, n = max(n_of[0], n_of[1]), full_keys = keys_next;
        ok = wait(q_full, n_item & 1u) && wait_k();
        if (!ok) break;
        ++n_item;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (n_of[t] > 0) issue_qk(t);
        release_k();
        if (n == 1) tc_commit(q_empty);
        it += gridDim.x;
        have = find_next();
        for (int s = 0; ok && s < n; ++s) {
          // V of this step
          v_slot = ring.take(NV);
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            ok = ok && wait(&full[v_slot + i], ring.phase(v_slot + i));
            ring.flip(v_slot + i);
          }
          if (ok && (s + 1) * kRows > full_keys) {  // its masked values have been seen to
            ok = wait(&v_safe[n_safe & 3u], (n_safe >> 2) & 1u);
            ++n_safe;
          }
          const int vs = v_slot;
          const bool more = s + 1 < n;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && s < n_of[t]) {
              if (s == 0 && item_of[t]++ > 0) ok = wait(&o_free[t], (item_of[t] - 2) & 1u);
              ok = ok && wait(&p_full[t], step_of[t] & 1u);
              if (!ok) break;
              ++step_of[t];
              tc_fence_after();
              const uint32_t d = tmem + S::T_O + t * 128, p = tmem + S::T_S + t * 128;
              const uint64_t v = d_v + ((uint32_t)(vs * S::SLAB) >> 4);
#pragma unroll
              for (int ks = 0; ks < kRows / 16; ++ks)
                mma_bf16_ts(d, p + ks * 8, v + ks * (2048 >> 4), ID_PV, s > 0 || ks > 0 ? 1u : 0u);
              tc_commit(&pv_done[t]);
            }
            if (t == 1) {
#pragma unroll
              for (int i = 0; i < NV; ++i) tc_commit(&empty[vs + i]);
            }
            if (ok && more) {
              // the next scores of this tile, while the other tile's softmax runs
              if (t == 0) ok = wait_k();
              if (ok && s + 1 < n_of[t]) issue_qk(t);
              if (ok && t == 1) {
                release_k();
                if (s + 2 == n) tc_commit(q_empty);
              }
            }
          }
        }
      }
      if (!ok) raise_abort(abort, status, kStatusTimeout);
      // every issued MMA must finish before TMEM and shared memory are released
      tc_commit(drain);
      mbar_wait(drain, 0, no_abort);
    }
  } else if (warp >= kScanWarp) {
    // ------------------------------------- masked values (each warp one half)
    DSB_FEW_REGS;
    Ring<NS> ring;
    uint32_t n_safe = 0, n_item = 0;
    const int half = warp - kScanWarp;
    for (int it = blockIdx.x; ok && it < items; it += gridDim.x) {
      Item x;
      bool bad;
      if (!get_item(a, order, it, &x, &bad) || x.steps() == 0) continue;
      const int n = x.steps();
      const int full_keys = x.common(causal), border = x.border(causal);
      uint32_t* word = reinterpret_cast<uint32_t*>(smem + S::OFF_BAD + (n_item % 3) * S::BAD_BYTES);
      uint32_t* any = word + VD;
      const uint32_t turn = n_item % 3, use = n_item / 3;
      ++n_item;
      if (use > 0 && !wait(&bad_free[turn], (use - 1) & 1u)) { ok = false; break; }
      for (int i = half * (VD / 2) + lane; i < (half + 1) * (VD / 2); i += 32) word[i] = kNothing;
      if (lane == 0) any[half] = 0;
      __syncwarp();
      for (int s = 0; ok && s < n; ++s) {
        for (int i = 0; i < NQ; ++i) ring.flip(ring.take(1));
        const int v_slot = ring.take(NV);
        if ((s + 1) * kRows > full_keys) {
          // (only once this load is the barriers' current phase can it be waited for)
          ok = wait(&v_load[n_safe & 3u], (n_safe >> 2) & 1u);
          for (int i = 0; ok && i < NV; ++i) ok = wait(&full[v_slot + i], ring.phase(v_slot + i));
          if (!ok) break;
          const int valid = min(kRows, x.lk - s * kRows);
          // this warp's 64 (VD = 64: 32) value columns: a row's 16-byte chunks
          constexpr int CH = VD / 2 / 8;        // chunks per row and warp
          constexpr int PER = kRows * CH / 32;  // and per lane
          auto chunk_at = [&](int k) {
            const int e = lane + 32 * k, row = e / CH, chunk = half * CH + e % CH, c = chunk % 8;
            return reinterpret_cast<uint4*>(smem + S::OFF_RING + (v_slot + chunk / 8) * S::SLAB + row * 128 +
                                            ((c ^ (row & 7)) * 16));
          };
          // an exponent of all ones carries into the sign bit (two bf16 a word)
          auto non_finite = [](uint32_t w) { return ((w & 0x7fff7fffu) + 0x00800080u) & 0x80008000u; };
          uint32_t hits = 0;
#pragma unroll 8
          for (int k = 0; k < PER; ++k) {
            const uint4 v = *chunk_at(k);
            hits |= non_finite(v.x) | non_finite(v.y) | non_finite(v.z) | non_finite(v.w);
          }
          if (__any_sync(0xffffffffu, hits != 0) || valid < kRows) {
#pragma unroll 1
            for (int k = 0; k < PER; ++k) {
              const int e = lane + 32 * k, row = e / CH, chunk = half * CH + e % CH;
              uint4* at = chunk_at(k);
              if (row >= valid) {
                *at = make_uint4(0, 0, 0, 0);
                continue;
              }
              const uint4 v = *at;
              uint32_t w[4] = {v.x, v.y, v.z, v.w};
              if ((non_finite(w[0]) | non_finite(w[1]) | non_finite(w[2]) | non_finite(w[3])) == 0) continue;
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                const uint32_t value = (w[i / 2] >> (16 * (i & 1))) & 0xffffu;
                if ((value & 0x7f80u) != 0x7f80u) continue;
                const int col = chunk * 8 + i;
                const int kind = (value & 0x7fu) != 0 ? kNan : (value & 0x8000u) != 0 ? kMinusInf : kPlusInf;
                const uint32_t key = (uint32_t)((s - border) * kRows + row);
                uint32_t old = word[col], now;
                do {
                  now = old;
                  const uint32_t first = min((now >> kind) & kKeyMask, key);
                  old = atomicCAS(&word[col], now, (now & ~(kKeyMask << kind)) | (first << kind));
                } while (old != now);
                w[i / 2] &= (i & 1) ? 0x0000ffffu : 0xffff0000u;
              }
              *at = make_uint4(w[0], w[1], w[2], w[3]);
              any[half] = 1;
            }
          }
          fence_proxy_async_shared();
          warp_arrive(&v_safe[n_safe & 3u]);
          ++n_safe;
        }
        for (int i = 0; i < NV; ++i) ring.flip(v_slot + i);
      }
      warp_arrive(&bad_full[turn]);
    }
    if (!ok) raise_abort(abort, status, kStatusTimeout);
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int t = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t ts = tl + S::T_S + t * 128, to = tl + S::T_O + t * 128;
    uint32_t c = 0, n_item = 0;  // steps of this tile; items with keys
    for (int it = blockIdx.x; ok && it < items; it += gridDim.x) {
      Item x;
      bool bad;
      if (!get_item(a, order, it, &x, &bad)) continue;
      const int i = x.row0 + t * kRows + r;  // row within the sequence
      const bool live = i < x.rows;
      const int64_t row = (int64_t)x.q0 + i;
      const int n = t == 0 ? x.n[0] : x.n[1];
      const int sees = x.sees(i, causal);
      float m = -INFINITY, l = 0.0f;  // m in the exp2 domain
      for (int s = 0; s < n; ++s, ++c) {
        if (!wait(&s_full[t], c & 1u)) { ok = false; break; }
        tc_fence_after();
        float v[128];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t u[32];
          tmem_ld32(ts + 32 * k, u);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[32 * k + e] = __uint_as_float(u[e]);
        }
        tmem_ld_wait();
        const int limit = sees - s * kRows;
        if (__any_sync(0xffffffffu, limit < kRows)) {
#pragma unroll
          for (int e = 0; e < 128; ++e) v[e] = e < limit ? v[e] : (scale_log2 >= 0.0f ? -INFINITY : INFINITY);
        }
        float top;
        {
          float q[4] = {v[0], v[1], v[2], v[3]};
          if (scale_log2 >= 0.0f) {
#pragma unroll
            for (int e = 4; e < 124; e += 2) q[(e >> 1) & 3] = max3(q[(e >> 1) & 3], v[e], v[e + 1]);
            q[0] = max3(q[0], v[124], v[125]);
            q[1] = max3(q[1], v[126], v[127]);
            top = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
          } else {
#pragma unroll
            for (int e = 4; e < 124; e += 2) q[(e >> 1) & 3] = min3(q[(e >> 1) & 3], v[e], v[e + 1]);
            q[0] = min3(q[0], v[124], v[125]);
            q[1] = min3(q[1], v[126], v[127]);
            top = fminf(fminf(q[0], q[1]), fminf(q[2], q[3]));
          }
        }
        top = limit > 0 ? top * scale_log2 : -INFINITY;
        float f = 1.0f;
        if (top > m + kLazy || m == -INFINITY) {
          f = fast_exp2(m - top);
          if (m == -INFINITY) f = 0.0f;
          m = top;
        }
        if (s > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
          if (!wait(&pv_done[t], (c - 1) & 1u)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int k = 0; k < VD / 32; ++k) {
            uint32_t o[32];
            tmem_ld32(to + 32 * k, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(to + 32 * k, o);
          }
        }
        l *= f;
        const float mm = m == -INFINITY ? 0.0f : m;  // a row that has seen no key yet
        const uint64_t scale2 = pair(scale_log2, scale_log2), minus_m = pair(-mm, -mm);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float p0, p1;
            unpair(fma2(pair(v[32 * k + 2 * e], v[32 * k + 2 * e + 1]), scale2, minus_m), p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            sum[e & 1] = add2(sum[e & 1], pair(p0, p1));
            w[e] = pack_bf16x2(p0, p1);
          }
          tmem_st16(ts + 16 * k, w);
        }
        {
          float s0, s1;
          unpair(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
        }
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&p_full[t]);
      }
      if (!ok) break;
      // -------------------------------------------------------------- result
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      if (live && a.lse != nullptr)
        a.lse[row * a.H + x.h] = l > 0.0f ? m * 0.6931471805599453f + logf(l) : l == 0.0f ? -INFINITY : l;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + row * a.ld_out + (int64_t)x.h * VD;
      const uint32_t* word = reinterpret_cast<const uint32_t*>(smem + S::OFF_BAD + (n_item % 3) * S::BAD_BYTES);
      const uint32_t* any = word + VD;
      const uint32_t turn = n_item % 3;
      if (x.steps() > 0) {
        if (!wait(&bad_full[turn], (n_item / 3) & 1u)) { ok = false; break; }
        ++n_item;
      }
      if (n == 0) {
        if (live)
          for (int k = 0; k < VD / 8; ++k) reinterpret_cast<uint4*>(dst)[k] = make_uint4(0, 0, 0, 0);
        if (x.steps() > 0) warp_arrive(&bad_free[turn]);
        continue;
      }
      __nv_bfloat16* const first = dst - (lane & 3) * a.ld_out;  // of this lane's four rows
      if (!wait(&pv_done[t], (c - 1) & 1u)) { ok = false; break; }
      tc_fence_after();
      const bool fix = (any[0] | any[1]) != 0;
#pragma unroll 1
      for (int k = 0; k < VD / 32; ++k) {
        uint32_t o[32];
        tmem_ld32(to + 32 * k, o);
        tmem_ld_wait();
        if (fix) {
          const int seen = sees - x.border(causal) * kRows;  // of the recorded keys
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t b = word[32 * k + e];
            if (b != kNothing) {
              auto has = [&](int kind) { return (int)((b >> kind) & kKeyMask) < seen; };
              float add = has(kPlusInf) ? INFINITY : 0.0f;
              add += has(kMinusInf) ? -INFINITY : 0.0f;
              o[e] = __float_as_uint(__uint_as_float(o[e]) + (has(kNan) ? NAN : add));
            }
          }
        }
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[e] = pack_bf16x2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
        store_rows(w, first + 32 * k, a.ld_out, x.rows - (i - (lane & 3)));
      }
      tc_fence_before();
      warp_arrive(&bad_free[turn]);
      warp_arrive(&o_free[t]);
    }
    if (!ok) raise_abort(abort, status, kStatusTimeout);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int NOPE, int P, int VD>
int launch(dsb_ctx* ctx, const dsb_mla_prefill_args& a) {
  using S = Shape<NOPE, P, VD>;
  CUtensorMap m[5];
  const struct {
    const void* p;
    int64_t ld, hd;
    int rows, dim;
  } t[5] = {{a.q_nope, a.ld_q_nope, a.hd_q_nope, a.Tq, NOPE},
            {a.q_rope, a.ld_q_rope, a.hd_q_rope, a.Tq, P},
            {a.k_nope, a.ld_k_nope, a.hd_k_nope, a.Tk, NOPE},
            {a.k_rope, a.ld_k_rope, 0, a.Tk, P},
            {a.v, a.ld_v, a.hd_v, a.Tk, VD}};
  for (int i = 0; i < 5; ++i) {
    const bool rope = i == 1 || i == 3;
    const int64_t heads = i == 3 ? 1 : a.H;
    const int box = rope ? P : 64;
    // no key is loaded where there is none: any valid address will do
    const void* base = i >= 2 && a.Tk == 0 ? a.out : t[i].p;
    if (int rc = make_tmap_2d(ctx, &m[i], base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              (uint64_t)((heads - 1) * t[i].hd + t[i].dim), (uint64_t)std::max(1, t[i].rows),
                              (uint64_t)t[i].ld * 2, (uint32_t)box, kRows,
                              box == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
        rc != DSB_OK)
      return rc;
  }
  Order o;
  o.pairs = a.B * a.H;
  // (one with max_q = 0 too: the lengths are checked)
  o.blocks = std::max(1, (int)(((int64_t)a.max_q + 2 * kRows - 1) / (2 * kRows)));
  // heads per group: two items for every SM, so that a group's keys and
  // values are read from HBM once and from L2 by the other blocks
  o.group = std::min(o.pairs, std::max(1, (2 * ctx->sm_count + o.blocks - 1) / o.blocks));
  const int64_t items = (int64_t)o.pairs * o.blocks;
  if (items >= (int64_t)1 << 30)
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_prefill: %d sequences x %d heads x %d blocks of queries", a.B, a.H,
                o.blocks);
  auto kern = prefill_kernel<NOPE, P, VD>;
  static std::atomic<bool> attr_set[kMaxDevices];
  if (int rc = smem_attr_once(ctx, kern, S::SMEM_BYTES, attr_set); rc != DSB_OK) return rc;
  // a zero scale would make NaN of masked scores; this one makes zeros of all others
  const float scale_log2 = a.softmax_scale == 0.0f ? 1e-37f : a.softmax_scale * 1.4426950408889634f;
  const unsigned grid = (unsigned)std::min<int64_t>(items, ctx->sm_count);
  DSB_CUDA_TRY(ctx, launch_pdl(kern, dim3(grid), kThreads, S::SMEM_BYTES, ctx->stream, m[0], m[1], m[2], m[3], m[4], a,
                               o, (int)items, scale_log2, ctx->d_status));
  ctx->stats.kernel_launches++;
  return DSB_OK;
}

}  // namespace
}  // namespace dsb

extern "C" int dsb_mla_prefill(dsb_ctx* ctx, const dsb_mla_prefill_args* args) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (args == nullptr) return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: null arguments");
  const dsb_mla_prefill_args& a = *args;
  // (an empty tensor may come without memory)
  if (a.cu_q == nullptr || a.cu_k == nullptr ||
      (a.Tq != 0 && (a.q_nope == nullptr || a.q_rope == nullptr || a.out == nullptr)) ||
      (a.Tk != 0 && (a.k_nope == nullptr || a.k_rope == nullptr || a.v == nullptr)))
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: null pointer argument");
  const bool big = a.nope == 128 && a.P == 64 && a.vd == 128, small = a.nope == 64 && a.P == 32 && a.vd == 64;
  if (!big && !small)
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_prefill: (nope, P, vd) = (%d, %d, %d) not supported", a.nope, a.P,
                a.vd);
  if (a.B <= 0 || a.B > 65535 || a.H <= 0 || a.H > 4096 || a.Tq < 0 || a.Tk < 0 || a.Tk >= 1 << 28 || a.max_q < 0 ||
      !std::isfinite(a.softmax_scale))
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: bad arguments B=%d H=%d Tq=%d Tk=%d max_q=%d scale=%g", a.B, a.H,
                a.Tq, a.Tk, a.max_q, a.softmax_scale);
  const int64_t ld[] = {a.ld_q_nope, a.ld_q_rope, a.ld_k_nope, a.ld_k_rope, a.ld_v, a.ld_out};
  const int64_t hd[] = {a.hd_q_nope, a.hd_q_rope, a.hd_k_nope, 0, a.hd_v, a.vd};
  const int dim[] = {a.nope, a.P, a.nope, a.P, a.vd, a.vd};
  for (int i = 0; i < 6; ++i) {
    const int64_t heads = i == 3 ? 1 : a.H;
    if (ld[i] % 8 != 0 || hd[i] % 8 != 0 || hd[i] < 0 || (heads > 1 && hd[i] < dim[i]) ||
        ld[i] < (heads - 1) * hd[i] + dim[i] || ld[i] >= (int64_t)1 << 31)
      return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: tensor %d: token pitch %lld, head pitch %lld", i,
                  (long long)ld[i], (long long)hd[i]);
  }
  if ((reinterpret_cast<uintptr_t>(a.q_nope) | reinterpret_cast<uintptr_t>(a.q_rope) |
       reinterpret_cast<uintptr_t>(a.k_nope) | reinterpret_cast<uintptr_t>(a.k_rope) |
       reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out)) & 15u)
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: pointers must be 16-byte aligned");
  if (a.Tq == 0) return DSB_OK;
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_mla_prefill: cudaSetDevice(%d) failed", ctx->device);
  return big ? launch<128, 64, 128>(ctx, a) : launch<64, 32, 64>(ctx, a);
}
