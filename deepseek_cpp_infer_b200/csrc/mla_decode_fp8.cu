// Absorbed MLA decode attention over the 8-bit paged latent cache, sm_100a.
//
//   s_j = softmax_scale * sigma_j * (q_lat . c8_j + q_rope . kr_j)
//   out = sum_j softmax(s)_j * sigma_j * c8_j
// (c8_j the token's e4m3 latents, kr_j its bf16 rope part, sigma_j its scale).
//
// The cached bytes are tensor-core operands as they are stored; nothing is
// converted.  Tokens are the MMA's M: a tile is 128 tokens (two pages), and
//   S^T [128 tokens x heads] = C8 . Q^T  (+ KR . Qr^T, kind::f16)
//   O^T [R x heads] += C8^T . P          (the same bytes, MN-major)
// so that few heads cost few columns and the tile is read once for both
// products.
//
// Precision.  An e4m3 value has 4 significant bits, a bf16 query 8: q / a (a
// a power of two per head) is split into hi = e4m3(q / a) and lo = e4m3(q / a
// - hi), to 2^-17 of the head's largest value.  hi and lo are
// separate columns of one MMA (N = 2 heads), summed in fp32.  Probabilities
// are split the same way (8 significant bits, like bf16) in units of a moving
// reference per head that keeps what falls below the digits' steps small against
// the sum (see kTileCost), so that thousands of small probabilities behind a large one
// (an attention sink) keep their digits.  O^T accumulates in TMEM in fp32 and is
// rescaled there when the reference moves.
// The token's scale joins its probability: with u = s log2(e) + log2(sigma),
// p' = 2^(u - r) carries sigma, and the softmax sum takes p' / sigma.
//
// Work.  Sequences' tiles in order, cut into one even run per SM (per head
// group of up to 64 heads; both groups of 128 heads walk the same tiles at
// the same time and share them through L2).  The lengths are read on the
// device.  A run's first and last sequences may be shared with its neighbours:
// such segments go to fp32 partials that a second kernel merges.
//
// Roles (11 warps): 8 softmax warps, two warpgroups with half the heads each
// (thread = token for S^T, thread = latent column for O^T), a TMA warp, a warp
// for QK and one for PV.  Shared memory is a ring of 128-token x 128-byte
// slabs (R / 128 of latents and one of rope keys per tile): a slab serves QK
// and, as soon as its block of O^T is done, is free again.
//
// What bounds it.  16 heads (12 slabs): HBM; 64 sequences of 1024 .. 8192
// tokens take 41 us, 4.8 TB/s with all overheads, and a tile's 3100 cycles in
// mid-run are the copy rate.  64 heads (72 KB of query digits leave 8 slabs):
// the chain of a tile, about 5000 cycles against 2840 of MMAs: PV's first block
// frees a slab, the next tile's last slab is loaded into it (1300 - 1900), QK,
// softmax (1900), PV.  128 heads, the same sequences: 132 us, 640 TFLOP/s; 32 of
// 4112 tokens 67 us; 3 of 60000 .. 131072 tokens (344,000 in all) 125 us.  At a
// sequence's end a run takes another 14000 cycles for its output and the next
// query's digits; the runs have equal tiles whatever ends they hold.
// One short sequence takes 11.2 us with the merge, two launches and a tile's
// chain.
// What did not help (all figures of this paragraph: 128 heads, when the kernel
// took 120 - 130 us): O^T accumulated in registers per tile, one warp for QK
// and PV, four softmax warpgroups, 48 heads per CTA (9 slabs, 138 us), a
// reference that lags one tile behind (168 us), partials of four heads a
// float4 (134 us).  At 64 heads the softmax warps use all 168 registers that
// three warps a partition leave: more loads in flight for the query's digits
// spill, and any spill beside 228 KB of shared memory costs 5% or more
// (setmaxnreg with a twelfth warp: 139 us; the query's digits between the
// output's blocks: 123 us).  Whole tiles prefetched into L2 cost more of its
// bandwidth than they save (127 us).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "dsb_internal.h"
#include "dsb_ptx.cuh"
#include "mla_fp8.cuh"
#include "packed.cuh"

namespace dsb {
namespace {

constexpr int kTileTok = 128;       // tokens per tile: MMA M
constexpr int kMaxHeadsPerCta = 64;
constexpr int kMaxSeqs = 65536;     // runs of sequences in the scratch
constexpr int kMaxLen = 1 << 30;    // tokens of a sequence: token and page numbers stay in 32 bits
constexpr int kScaleStages = 4;

template <int R, int P, int HB>
struct Shape {
  static constexpr int NL = R / 128;                 // latent slabs per tile
  static constexpr int NSLAB = NL + 1;               // + rope
  static constexpr int NWG = 2;                      // softmax warpgroups
  static constexpr int SM_WARPS = NWG * 4;
  static constexpr int THREADS = (SM_WARPS + 3) * 32;  // + TMA, QK and PV
  static constexpr int HW = HB / NWG;                // heads per warpgroup
  static constexpr int SLAB = kTileTok * 128;        // bytes
  static constexpr int NS = HB == 16 ? 12 : HB == 32 || NL == 1 ? 10 : 8;  // ring slots: what fits
  static_assert(NS >= NSLAB + 1, "ring");
  static constexpr bool LATE = NS < 2 * NSLAB - 1;  // a tile's last slab waits for the last tile's PV
  static constexpr int Q8_BYTES = 2 * HB * R;        // [slab][hi heads | lo heads][128 B], SW128
  static constexpr int QR_BYTES = HB * P * 2;        // [head][P bf16], SW128 (P = 64) or SW64
  static constexpr int P_BYTES = HB * kTileTok;      // one digit of the probabilities
  static constexpr int OFF_RING = 0;
  static constexpr int OFF_Q8 = OFF_RING + NS * SLAB;
  static constexpr int OFF_QR = OFF_Q8 + Q8_BYTES;
  static constexpr int OFF_P = OFF_QR + QR_BYTES;
  static constexpr int OFF_SC = OFF_P + 2 * P_BYTES;                     // [stages][128] token scales
  static constexpr int OFF_RED = OFF_SC + kScaleStages * kTileTok * 4;   // [2 parity][NWG][4 warps][HW] maxima
  static constexpr int OFF_LRED = OFF_RED + 2 * 4 * HB * 4;              // [NWG][4 warps][HW] sums
  static constexpr int OFF_MT = OFF_LRED + 4 * HB * 4;                   // per warp [HW]: references (or 1 / sums)
  static constexpr int OFF_FH = OFF_MT + 4 * HB * 4;              // [HB] a_h * scale * log2(e)
  static constexpr int NBAR = 2 * NS + 4 + 6 + NWG + 2 * kScaleStages;
  static constexpr int OFF_BAR = (OFF_FH + HB * 4 + 7) / 8 * 8;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;                    // tmem base, abort flags, start, scan
  static constexpr int SMEM_BYTES = OFF_MISC + 128 + 1024;               // + alignment slack
  static_assert(SMEM_BYTES <= 232448, "shared memory");
  static_assert(OFF_Q8 % 1024 == 0 && OFF_QR % 1024 == 0 && OFF_P % 128 == 0 && OFF_SC % 16 == 0, "alignment");
  // TMEM columns: S^T two buffers of [hi | lo], then O^T per latent slab.  Where
  // there is room both digits of the probabilities are columns of one MMA (42
  // cycles up to N = 32, 50 at 64, 66 at 128) and O^T is [hi | lo] too: 16 heads
  // x 777 tokens 11.4 -> 11.1 us, x 64 sequences 41.1 -> 40.3.
  static constexpr int DIG = 4 * HB + 2 * NL * HB <= 512 ? 2 : 1;  // blocks of HB columns per slab
  // In columns of their own the lo digits are held 16-fold (a remainder is at
  // most 16: half a step of 256 .. 448), which moves their floor down as much.
  static constexpr int LO = DIG == 2 ? 16 : 1;
  static constexpr uint32_t T_S = 0, T_O = 4 * HB;
  static constexpr int USED = 4 * HB + NL * DIG * HB;
  static constexpr uint32_t T_COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(USED <= 512, "TMEM");
};

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Two floats as e4m3 digits: hi = e4m3(v), lo = e4m3((v - hi) * LO), through
// fp16 (11 significant bits; the difference is exact).
template <int LO = 1>
__device__ __forceinline__ void split_digits(float a, float b, uint32_t& hi, uint32_t& lo) {
  const uint32_t v = pack_half2(a, b);
  uint16_t h, l;
  uint32_t hf, d;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(v));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hf) : "h"(h));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(hf));
  if constexpr (LO == 16) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(d), "r"(0x4c004c00u));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l) : "r"(d));
  hi = h;
  lo = l;
}

// 1D bulk copy global -> shared, completing on `bar` (addresses and size multiples of 16).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Bring a box into L2 ahead of its load.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y)
               : "memory");
}

// N columns of this thread's TMEM lane; tmem_ld_wait() before their use.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_ld32(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld8(taddr, r);
}

__device__ __forceinline__ bool bad_len(int len, int max_blocks) {
  return len < 0 || len > kMaxLen || len > (int64_t)max_blocks * kPageTok;
}

__device__ __forceinline__ int tiles_of(int len, int max_blocks) {
  return bad_len(len, max_blocks) ? 0 : len / kTileTok + (len % kTileTok != 0 ? 1 : 0);
}

// A run of tiles through the sequences; every role walks its own copy.
struct Walk {
  const int32_t* lens;
  int B, max_blocks;
  int b, tile, ntile, len;
  int len_ahead;  // the next sequence's, read long before it is needed
  __device__ void start(const int32_t* l, int B_, int mb, int b_, int tile_) {
    lens = l;
    B = B_;
    max_blocks = mb;
    b = b_;
    tile = tile_;
    len = lens[b];
    len_ahead = b + 1 < B ? lens[b + 1] : 1;
    ntile = tiles_of(len, max_blocks);
  }
  __device__ void next() {  // only called while tiles are left
    if (++tile < ntile) return;
    tile = 0;
    do {
      ++b;
      len = len_ahead;
      len_ahead = b + 1 < B ? lens[b + 1] : 1;
      ntile = tiles_of(len, max_blocks);
    } while (ntile == 0);
  }
  __device__ int valid() const { return min(kTileTok, len - tile * kTileTok); }  // tokens of this tile
};

// A position in the ring: slot and phase parity.
template <int NS>
struct Cursor {
  int slot = 0;
  uint32_t phase = 0;
  __device__ void step(int k) {
    slot += k;
    if (slot >= NS) {
      slot -= NS;
      phase ^= 1u;
    }
  }
  __device__ Cursor plus(int k) const {
    Cursor c = *this;
    c.step(k);
    return c;
  }
};

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// First tile of run i of n over T tiles.
__device__ __forceinline__ int64_t run_start(int64_t i, int64_t T, int n) { return i * T / n; }
// What the merge has to do for a sequence: its first partial's slot and
// its last run (written by the runs that begin and end it), or one of these.
constexpr int kSeqEmpty = -1, kSeqWhole = -2;

template <int R, int P, int HB>
__global__ void __launch_bounds__(Shape<R, P, HB>::THREADS, 1)
    decode_fp8_kernel(const __grid_constant__ CUtensorMap map_lat, const __grid_constant__ CUtensorMap map_rope,
                      const __nv_bfloat16* __restrict__ q_lat, const __nv_bfloat16* __restrict__ q_rope,
                      const float* __restrict__ scales, int64_t n_blocks, const int32_t* __restrict__ block_table,
                      int max_blocks, const int32_t* __restrict__ seq_lens, int B, int H, int runs, float scale_log2,
                      __nv_bfloat16* __restrict__ out, float* __restrict__ ws_o, float2* __restrict__ ws_ml,
                      int2* __restrict__ seq_runs, int* __restrict__ status) {
  using S = Shape<R, P, HB>;
  constexpr int NL = S::NL, NS = S::NS, HW = S::HW, NSLAB = S::NSLAB, NWG = S::NWG;
  constexpr int kSmWarps = S::SM_WARPS, kThreads = S::THREADS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint64_t* full = bars;                     // [NS] slab landed
  uint64_t* empty = full + NS;               // [NS] slab's last MMA done
  uint64_t* s_full = empty + NS;             // [2] scores of a tile ready
  uint64_t* s_free = s_full + 2;             // [2] scores read
  uint64_t* pv_done = s_free + 2;            // a tile's PV done
  uint64_t* p_full = pv_done + 1;            // probabilities of a tile written
  uint64_t* o_free = p_full + 1;             // O^T of a segment read
  uint64_t* q_ready = o_free + 1;            // query digits of a segment written
  uint64_t* wg_bar = q_ready + 1;            // [NWG] rendezvous of a warpgroup
  uint64_t* sc_full = wg_bar + NWG;           // [stages] token scales landed
  uint64_t* sc_empty = sc_full + kScaleStages;
  uint64_t* drain = sc_empty + kScaleStages;  // [2] every MMA that a warp issued is done
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + S::OFF_MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(misc + 1);
  volatile int* no_abort = reinterpret_cast<volatile int*>(misc + 2);  // never raised: for drain waits
  int* start = reinterpret_cast<int*>(misc + 3);                       // sequence and tile of the run's start
  int* scan = reinterpret_cast<int*>(misc + 8);                        // [20] warp totals, at most

  // warp-uniform for the compiler, so that the MMA and TMA operands stay in
  // uniform registers
  const int warp = __shfl_sync(0xffffffffu, (int)warp_id(), 0), lane = (int)lane_id();
  const int hg = blockIdx.x / runs, run = blockIdx.x % runs;  // head group and run
  constexpr int kTmaWarp = kSmWarps, kQkWarp = kSmWarps + 1, kPvWarp = kSmWarps + 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kSmWarps);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < NWG; ++i) mbar_init(&wg_bar[i], 4);
    mbar_init(pv_done, 1);
    mbar_init(p_full, kSmWarps);
    mbar_init(o_free, kSmWarps);
    mbar_init(q_ready, kSmWarps);
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&sc_empty[i], kSmWarps);
    }
    *abort = 0;
    *no_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(misc, S::T_COLS);
    tmem_relinquish();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&map_lat);
    tma_prefetch_desc(&map_rope);
  }
  pdl_wait();
  pdl_launch_dependents();

  // Tiles before each thread's share of the sequences, and this CTA's run.
  int64_t run0;
  int count;
  {
    const int per = (B + kThreads - 1) / kThreads;
    const int b0 = min(B, (int)threadIdx.x * per), b1 = min(B, b0 + per);
    int mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const int len = seq_lens[b];
      if (blockIdx.x == 0 && bad_len(len, max_blocks)) atomicCAS(status, 0, kStatusBadInput);
      mine += tiles_of(len, max_blocks);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int before = inc - mine, T = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      T += scan[w];
    }
    const int n_run = min(runs, T);  // no empty runs
    run0 = run < n_run ? run_start(run, T, n_run) : 0;
    count = run < n_run ? (int)(run_start(run + 1, T, n_run) - run0) : 0;
    if (count > 0 && run0 >= before && run0 < before + mine) {
      int t = before, b = b0;
#pragma unroll 1
      for (;; ++b) {
        const int n = tiles_of(seq_lens[b], max_blocks);
        if (run0 < t + n) break;
        t += n;
      }
      start[0] = b;
      start[1] = (int)run0 - t;
    }
    if (blockIdx.x == 0) {
#pragma unroll 1
      for (int b = b0; b < b1; ++b)
        if (tiles_of(seq_lens[b], max_blocks) == 0) seq_runs[b] = make_int2(kSeqEmpty, 0);
    }
    __syncthreads();
  }
  const uint32_t tmem = (uint32_t)uniform((int)misc[0]);
  const uint32_t smem_base = smem_u32(smem);
  Walk w;
  if (count > 0) w.start(seq_lens, B, max_blocks, start[0], start[1]);

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ TMA producer
    // Slab order per tile: rope, latents 0 .. NL - 1 (the rope slab is free
    // again after QK, so its slot goes to the next tile's slab first).
    if (count > 0) {
      const uint64_t policy = l2_policy_evict_first();
      int it = 0;   // slabs issued
      Cursor<NS> at_slab;
      int nsc = 0;  // scale stages issued
      int pages = 0, at = 32;  // page ids of the next 16 tiles of the sequence, two lanes a tile
      bool ok = true;
      for (int n = 0; ok && n < count; ++n) {
        if (n > 0) w.next();
        if (at == 32 || w.tile == 0) {
          const int p = w.tile * 2 + lane;
          pages = 0;
          if (p * kPageTok < w.len) {
            pages = block_table[(int64_t)w.b * max_blocks + p];
            if (pages < 0 || pages >= n_blocks) {  // read some page instead, and report it
              pages = 0;
              atomicCAS(status, 0, kStatusBadInput);
            }
          }
          at = 0;
        }
        const int np = w.valid() > kPageTok ? 2 : 1;
        const int page[2] = {__shfl_sync(0xffffffffu, pages, at), __shfl_sync(0xffffffffu, pages, at + 1)};
        at += 2;
        const int sc = n % kScaleStages;
        if (n >= kScaleStages &&
            !__all_sync(0xffffffffu, mbar_wait(&sc_empty[sc], (uint32_t)(n / kScaleStages - 1) & 1u, abort))) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(&sc_full[sc], np * kPageTok * 4);
          for (int p = 0; p < np; ++p)
            bulk_load(smem + S::OFF_SC + (sc * kTileTok + p * kPageTok) * 4, scales + (int64_t)page[p] * kPageTok,
                      kPageTok * 4, &sc_full[sc]);
        }
        ++nsc;
#pragma unroll 1
        for (int k = 0; k < NSLAB; ++k, ++it) {
          const int slot = at_slab.slot;
          const int row = k == 0 ? P * 2 : 128;  // bytes of a slab's row
          const int x = k == 0 ? R : (k - 1) * 128;
          const CUtensorMap* map = k == 0 ? &map_rope : &map_lat;
          if (S::LATE && k == NSLAB - 1 &&  it >= NS && elect_one()) {
            tma_prefetch_2d(map, x, page[0] * kPageTok);
            if (np == 2) tma_prefetch_2d(map, x, page[1] * kPageTok);
          }
          if (it >= NS && !__all_sync(0xffffffffu, mbar_wait(&empty[slot], at_slab.phase ^ 1u, abort))) {
            ok = false;
            break;
          }
          at_slab.step(1);
          uint8_t* dst = smem + S::OFF_RING + slot * S::SLAB;
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[slot], np * kPageTok * row);
            tma_load_2d(dst, map, &full[slot], x, page[0] * kPageTok, policy);
            if (np == 2) tma_load_2d(dst + kPageTok * row, map, &full[slot], x, page[1] * kPageTok, policy);
          }
        }
      }
      if (!ok) raise_abort(abort, status, kStatusTimeout);
      // every copy must land before shared memory is released, also when a
      // consumer has given up
      for (int i = max(0, it - NS); i < it; ++i) mbar_wait(&full[i % NS], (uint32_t)(i / NS) & 1u, no_abort);
      for (int i = max(0, nsc - kScaleStages); i < nsc; ++i)
        mbar_wait(&sc_full[i % kScaleStages], (uint32_t)(i / kScaleStages) & 1u, no_abort);
    }
  } else if (warp == kQkWarp) {
    // ------------------------------------------------------ QK: S^T of each tile
    // One elected lane runs the role.  (Issued from a lane == 0 branch, or by a
    // warp with operands that the compiler does not know to be uniform, an MMA
    // costs 147 cycles whatever its N, measured; elected 42 at N = 32, 50 at
    // 64, 66 at 128: its shared-memory reads.)  QK and PV have a warp each, so
    // that neither waits behind the other's operands.
    if (count > 0 && elect_one()) {
      constexpr uint32_t ID_QK = idesc_e4m3_f32(128, 2 * HB), ID_QR = idesc_bf16_f32(128, HB, 0, 0);
      const uint64_t d_q8 = smem_desc(smem_base + S::OFF_Q8, 16, 1024, kSwizzle128B);
      const uint64_t d_qr = P == 64 ? smem_desc(smem_base + S::OFF_QR, 16, 1024, kSwizzle128B)
                                    : smem_desc(smem_base + S::OFF_QR, 16, 512, kSwizzle64B);
      const uint64_t d_slab = smem_desc(smem_base + S::OFF_RING, 16, 1024, kSwizzle128B);
      const uint64_t d_rope = P == 64 ? d_slab : smem_desc(smem_base + S::OFF_RING, 16, 512, kSwizzle64B);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort); };
      Cursor<NS> at;  // the tile's first slab
      int seg = 0;
      bool ok = true;
#pragma unroll 1
      for (int n = 0; ok && n < count; ++n) {
        if (n > 0) w.next();
        if (n == 0 || w.tile == 0) ok = wait(q_ready, (uint32_t)seg++ & 1u);
        if (ok && n >= 2) ok = wait(&s_free[n & 1], (uint32_t)((n >> 1) - 1) & 1u);
        if (!ok) break;
        const uint32_t d = tmem + S::T_S + (uint32_t)(n & 1) * 2 * HB;
        // latents 0 (its first MMA clears both digits' columns), rope, latents 1 ..
#pragma unroll
        for (int step = 0; step < NSLAB; ++step) {
          const int k = step == 0 ? 1 : step == 1 ? 0 : step;  // slab of the tile, in load order
          const Cursor<NS> c = at.plus(k);
          if (!wait(&full[c.slot], c.phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t off = (uint32_t)(c.slot * S::SLAB) >> 4;
          if (k == 0) {
#pragma unroll
            for (int ks = 0; ks < P / 16; ++ks) mma_bf16_ss(d, d_rope + off + ks * 2, d_qr + ks * 2, ID_QR, 1u);
            tc_commit(&empty[c.slot]);
          } else {
            constexpr uint32_t kSlabQ = 2 * HB * 128 >> 4;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_f8_ss(d, d_slab + off + ks * 2, d_q8 + (k - 1) * kSlabQ + ks * 2, ID_QK, k > 1 || ks > 0 ? 1u : 0u);
          }
          if (step == NSLAB - 1) tc_commit(&s_full[n & 1]);
        }
        at.step(NSLAB);
      }
      if (!ok) raise_abort(abort, status, kStatusTimeout);
      // every issued MMA must finish before TMEM and shared memory are released
      tc_commit(&drain[0]);
      mbar_wait(&drain[0], 0, no_abort);
    }
  } else if (warp == kPvWarp) {
    // --------------------------------------------------- PV: O^T of the segment
    if (count > 0 && elect_one()) {
      constexpr int DIG = S::DIG;
      constexpr uint32_t ID_PV = idesc_e4m3_f32(128, DIG * HB) | (1u << 15) | (1u << 16);  // A and B MN-major
      // P digits, no swizzle: 16 heads x 8 tokens per 128-byte core matrix,
      // token groups 128 bytes apart, head groups 2048 (the lo digits' behind the hi ones')
      const uint64_t d_p = smem_desc(smem_base + S::OFF_P, 128, kTileTok * 16, kSwizzleNone);
      const uint64_t d_slab = smem_desc(smem_base + S::OFF_RING, 16, 1024, kSwizzle128B);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort); };
      Cursor<NS> at;  // the tile's first latent slab
      at.step(1);
      int seg = 0;
      bool ok = true;
#pragma unroll 1
      for (int n = 0; ok && n < count; ++n) {
        if (n > 0) w.next();
        const bool first = n == 0 || w.tile == 0;  // of its segment
        if (first && n > 0) ok = wait(o_free, (uint32_t)seg++ & 1u);
        if (!ok || !wait(p_full, (uint32_t)n & 1u)) { ok = false; break; }
        tc_fence_after();
        int slot[NL];
#pragma unroll
        for (int g = 0; g < NL; ++g) slot[g] = at.plus(g).slot;
#pragma unroll
        for (int g = 0; g < NL; ++g) {
          const uint64_t a = d_slab + ((uint32_t)(slot[g] * S::SLAB) >> 4);
          const uint32_t d = tmem + S::T_O + (uint32_t)(g * DIG * HB);
#pragma unroll
          for (int ks = 0; ks < kTileTok / 32; ++ks) {
            mma_f8_ss(d, a + ks * (4096 >> 4), d_p + ks * (512 >> 4), ID_PV, first && ks == 0 ? 0u : 1u);
            if constexpr (DIG == 1)
              mma_f8_ss(d, a + ks * (4096 >> 4), d_p + (S::P_BYTES >> 4) + ks * (512 >> 4), ID_PV, 1u);
          }
          tc_commit(&empty[slot[g]]);
        }
        tc_commit(pv_done);
        at.step(NSLAB);
      }
      if (!ok) raise_abort(abort, status, kStatusTimeout);
      tc_commit(&drain[1]);
      mbar_wait(&drain[1], 0, no_abort);
    }
  } else if (count > 0) {
    // ------------------------------------------------------- softmax warps
    const int wg = warp >> 2, quarter = warp & 3;
    const int j = quarter * 32 + lane;  // token of the tile; row of an O^T block
    const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
    float* red = reinterpret_cast<float*>(smem + S::OFF_RED);
    float* lred = reinterpret_cast<float*>(smem + S::OFF_LRED);
    float* mt = reinterpret_cast<float*>(smem + S::OFF_MT) + warp * HW;
    float* fh = reinterpret_cast<float*>(smem + S::OFF_FH);
    const int h0 = hg * HB;  // first head of the group
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
    };

    // Query digits of sequence b: a warp per head, 16 (4) latents a lane.  A
    // warpgroup loads its own heads: its warps have all read the old factors
    // (fh) when one of them is past the tile's rendezvous.
    auto load_q = [&](int b) {
      constexpr int CPL = R / 32;               // latents per lane
      constexpr int NQ = HW / 4 < 4 ? HW / 4 : 4;  // heads whose loads are in flight together
#pragma unroll 1
      for (int i0 = 0; i0 < HW / 4; i0 += NQ) {
        uint32_t xs[NQ][CPL / 2];
        uint4 rs[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int h = wg * HW + quarter + 4 * (i0 + q);
          const int64_t row = (int64_t)b * H + h0 + h;
          rs[q] = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < CPL / 2; ++i) xs[q][i] = 0;
          if (h0 + h < H) {
            if constexpr (CPL == 16) {
              const uint4* src = reinterpret_cast<const uint4*>(q_lat + row * R + lane * 16);
              const uint4 u = src[0], v = src[1];
              xs[q][0] = u.x, xs[q][1] = u.y, xs[q][2] = u.z, xs[q][3] = u.w;
              xs[q][4] = v.x, xs[q][5] = v.y, xs[q][6] = v.z, xs[q][7] = v.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(q_lat + row * R + lane * 4);
              xs[q][0] = u.x, xs[q][1] = u.y;
            }
            if (lane < P / 8) rs[q] = *reinterpret_cast<const uint4*>(q_rope + row * P + lane * 8);
          }
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int h = wg * HW + quarter + 4 * (i0 + q);
          const uint32_t (&x)[CPL / 2] = xs[q];
          const uint4 r = rs[q];
          const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
          uint32_t am = 0, rm = 0;  // magnitudes, two bf16 at once: their order is that of the bits
#pragma unroll
          for (int i = 0; i < CPL / 2; ++i) am = max_u16x2(am, x[i] & 0x7fff7fffu);
#pragma unroll
          for (int i = 0; i < 4; ++i) rm = max_u16x2(rm, rr[i] & 0x7fff7fffu);
          const float al = __uint_as_float(max(am & 0xffff0000u, am << 16));
          const float ar = __uint_as_float(max(rm & 0xffff0000u, rm << 16));
          // the latents' scale; a rope part over 64 times larger sets it
          // instead (it is divided by the same factor, in bf16, exactly)
          const float top = redux_max(fmaxf(al, ar * 0.015625f));
          const int e = min(120, max(-100, top > 0.0f ? (int)(__float_as_uint(top) >> 23) - 127 - 7 : 0));
          const float inv = exp2i(-e);
          const uint64_t inv2 = pair(inv, inv);
          uint32_t hi[CPL / 4], lo[CPL / 4];
#pragma unroll
          for (int i = 0; i < CPL / 4; ++i) {
            uint32_t a, b2, c, d;
            float v[4];
            unpair(mul2(pair(bf16lo_to_f32(x[2 * i]), bf16hi_to_f32(x[2 * i])), inv2), v[0], v[1]);
            unpair(mul2(pair(bf16lo_to_f32(x[2 * i + 1]), bf16hi_to_f32(x[2 * i + 1])), inv2), v[2], v[3]);
            split_digits(v[0], v[1], a, b2);
            split_digits(v[2], v[3], c, d);
            hi[i] = a | (c << 16);
            lo[i] = b2 | (d << 16);
          }
          // row h (hi) and HB + h (lo) of each 128-column slab, 16-byte chunk c
          // of a row at c ^ (row & 7)
          const int col = lane * CPL, slab = col / 128, chunk = (col % 128) / 16, in = col % 16;
          uint8_t* q8 = smem + S::OFF_Q8 + slab * 2 * HB * 128 + ((chunk ^ (h & 7)) * 16) + in;
          if constexpr (CPL == 16) {
            *reinterpret_cast<uint4*>(q8 + h * 128) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(q8 + (HB + h) * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
            *reinterpret_cast<uint32_t*>(q8 + h * 128) = hi[0];
            *reinterpret_cast<uint32_t*>(q8 + (HB + h) * 128) = lo[0];
          }
          if (lane < P / 8) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(bf16lo_to_f32(rr[i]) * inv, bf16hi_to_f32(rr[i]) * inv);
            const int c = P == 64 ? (lane ^ (h & 7)) : (lane ^ ((h >> 1) & 3));
            *reinterpret_cast<uint4*>(smem + S::OFF_QR + h * (P * 2) + c * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          // (an infinite query would saturate to a finite one: NaN instead)
          if (lane == 0) fh[h] = (top < INFINITY ? exp2i(e) : NAN) * scale_log2;
        }
      }
      fence_proxy_async_shared();
      warp_arrive(q_ready);
    };

    // Probabilities and sums are in units of 2^r, r a per-head reference (held
    // by lane head % HW).  Digits hold up to 448; a probability's are off by at
    // most 2^-8 of it, or by 2^-10 (2^-14 with lo held 16-fold) where that is
    // more.  A tile's 128 could thus lose 2^-3 (2^-7) together, if they all round
    // the same way, while the sums take them whole.  The segment has to be worth
    // it: of what its probabilities add up to at least (each warp's largest of
    // every tile) a tile takes kTileCost, and `credit` is what is left.  A tile
    // that it does not cover, or whose largest is above 2^kHigh, moves the
    // reference, to make its largest 2^kNew, and the head's columns of O^T are
    // rescaled in TMEM.  So this floor costs a segment at most 2^-3 / 32 = 2^-8
    // (2^-7 / 8 = 2^-10) of the sum of its probabilities, no more than rounding
    // each to bf16.  fp32 has the range for moves in both directions (r never falls
    // more than 2^40 below the largest: what lies further down is out of an fp32
    // sum's reach).  64 sequences of 1024 .. 8192, 128 heads: 132.5 us, a window
    // [2^0, 2^8.75] for every tile's largest 127.5 (peaks could lose a tail of 11%
    // of them), one that holds as much as the credit, [2^5, 2^8.75], 149; kTileCost
    // 16 130.5; kNew 5 133.7, 7 135.3.  (Scores there have a deviation of 1.7.  Of
    // 3.5 and 7: 143 - 146 and 149 - 151 us, by the first window 146 - 148 and 153
    // - 155: its moves do not count what later tiles are worth.  Equal ones: 124.)
    constexpr int DIG = S::DIG;
    constexpr float kNew = DIG == 1 ? 6.0f : 5.0f, kHigh = 8.75f;  // log2
    constexpr float kTileCost = DIG == 1 ? 32.0f : 8.0f;
    float ls[HW];  // softmax sums over this thread's tokens
    float r_ref = 0.0f, r_top = 0.0f, credit = 0.0f;
    if (lane < HW) mt[lane] = 0.0f;
    __syncwarp();
    int meet = 0;  // phase of wg_bar
    bool ok = true, first = true;       // first: the tile begins a segment
    bool shared_front = w.tile != 0;    // the segment's sequence began in an earlier run
    int n_seg = 0, sc = 0;
    uint32_t sc_phase = 0;
    // n = -1: the first query alone
#pragma unroll 1
    for (int n = -1; n < count; ++n) {
      const int b_now = w.b;
      const bool seq_end = n < 0 || w.tile == w.ntile - 1;
      const bool seg_end = seq_end || n + 1 == count;
      if (n >= 0) {
        const int valid = w.valid();
        if (!wait(&sc_full[sc], sc_phase)) { ok = false; break; }
        // a scale of zero (a row never written) counts as a tiny one
        const float sigma =
            j < valid ? fmaxf(reinterpret_cast<const float*>(smem + S::OFF_SC)[sc * kTileTok + j], 0x1p-100f) : 1.0f;
        warp_arrive(&sc_empty[sc]);
        if (++sc == kScaleStages) {
          sc = 0;
          sc_phase ^= 1u;
        }
        const float lsig = __log2f(sigma), isig = __frcp_rn(sigma);
        const uint64_t sigma2 = pair(sigma, sigma), lsig2 = pair(lsig, lsig), isig2 = pair(isig, isig);
        if (!wait(&s_full[n & 1], (uint32_t)(n >> 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        float u[HW];
        {
          constexpr int HC = HW < 16 ? HW : 16;  // heads read at once
          const uint32_t ts = t_lane + S::T_S + (uint32_t)(n & 1) * 2 * HB + wg * HW;
#pragma unroll
          for (int c = 0; c < HW; c += HC) {
            uint32_t s_hi[HC], s_lo[HC];
            tmem_ld(ts + c, s_hi);
            tmem_ld(ts + HB + c, s_lo);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < HC; h += 4) {
              const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(fh + wg * HW + c + h);
              const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(mt + c + h);  // - reference
              auto score = [&](int i, uint64_t f2, uint64_t r2) {
                const uint64_t s2 = add2(pair(__uint_as_float(s_hi[i]), __uint_as_float(s_hi[i + 1])),
                                         pair(__uint_as_float(s_lo[i]), __uint_as_float(s_lo[i + 1])));
                unpair(fma2(mul2(s2, sigma2), f2, add2(lsig2, r2)), u[c + i], u[c + i + 1]);
              };
              score(h, f.x, r.x);
              score(h + 2, f.y, r.y);
            }
          }
          tc_fence_before();
          warp_arrive(&s_free[n & 1]);
          if (valid < kTileTok) {
#pragma unroll
            for (int h = 0; h < HW; ++h) u[h] = j < valid ? u[h] : -INFINITY;
          }
        }
        // the tile's maximum per head (against r): the warp's by reductions that
        // do not wait for one another, then the warpgroup's (lane head % HW)
        const int hl = lane % HW;
        float* red_n = red + ((n & 1) * NWG + wg) * 4 * HW;
#pragma unroll
        for (int h = 0; h < HW; h += 4) {
          const float4 m = make_float4(redux_max(u[h]), redux_max(u[h + 1]), redux_max(u[h + 2]), redux_max(u[h + 3]));
          if (lane == 0) *reinterpret_cast<float4*>(red_n + quarter * HW + h) = m;
        }
        warp_arrive(&wg_bar[wg]);
        if (!wait(&wg_bar[wg], (uint32_t)meet & 1u)) { ok = false; break; }
        ++meet;
        const float t0 = red_n[hl], t1 = red_n[HW + hl], t2 = red_n[2 * HW + hl], t3 = red_n[3 * HW + hl];
        const float t = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
        auto part = [](float v) { return fast_exp2(fminf(v, 100.0f)); };  // (finite: a move scales it down)
        credit = (first ? 0.0f : credit) + ((part(t0) + part(t1)) + (part(t2) + part(t3)));
        r_top = first ? t + r_ref : fmaxf(r_top, t + r_ref);
        // (a bound for falls: r_top may be rounded up by more than t)
        const float want = fmaxf(t, fminf(r_top - 40.0f - r_ref, kNew));
        const bool move = first || !(want <= kHigh && credit >= kTileCost);
        // the previous PV has read P and written O^T
        if (n > 0 && !wait(pv_done, (uint32_t)(n - 1) & 1u)) { ok = false; break; }
        if (uint32_t moved = __ballot_sync(0xffffffffu, move)) {
          // O^T moves with the reference as it is held: next to one of 2^24 and
          // more a step is wider than the window, and the difference to `by` is
          // within the rounding of such scores
          // (-inf: no score yet that weighs anything, so O^T and the sums are zero,
          // and stay it at a fall of any height)
          const float by = move && want != -INFINITY ? want - kNew : 0.0f, r_new = r_ref + by;
          const float f = fast_exp2(fminf(r_ref - r_new, 126.0f));
          r_ref = r_new;
          credit *= f;
          if (!first) tc_fence_after();
#pragma unroll
          for (int c = 0; c < HW; c += 8) {
            if (((moved >> c) & 0xffu) == 0) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) u[c + i] -= __shfl_sync(0xffffffffu, by, c + i);
            if (first) {
#pragma unroll
              for (int i = 0; i < 8; ++i) ls[c + i] = 0.0f;
              continue;
            }
            float fs[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              fs[i] = __shfl_sync(0xffffffffu, f, c + i);
              ls[c + i] *= fs[i];
            }
            constexpr int BLK = DIG == 1 && NL % 2 == 0 ? 2 : 1;  // blocks in flight (more spill)
#pragma unroll 1
            for (int g = 0; g < NL * DIG; g += BLK) {
              const uint32_t at = t_lane + S::T_O + g * HB + wg * HW + c;
              uint32_t o[BLK][8];
#pragma unroll
              for (int k = 0; k < BLK; ++k) tmem_ld8(at + k * HB, o[k]);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < BLK; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[k][i] = __float_as_uint(__uint_as_float(o[k][i]) * fs[i]);
                tmem_st8(at + k * HB, o[k]);
              }
            }
          }
          if (!first) tmem_st_wait();
          __syncwarp();
          if (lane < HW) mt[lane] = -r_ref;
          __syncwarp();
        }
        credit = fmaxf(credit - kTileCost, 0.0f);  // (less: beyond the bound for falls)
        // probabilities, their sums and digits
        uint32_t hi[HW / 4], lo[HW / 4];
#pragma unroll
        for (int h = 0; h < HW; h += 4) {
          u[h + 0] = fast_exp2(u[h + 0]);
          u[h + 1] = fast_exp2(u[h + 1]);
          u[h + 2] = fast_exp2(u[h + 2]);
          u[h + 3] = fast_exp2(u[h + 3]);
          uint32_t a, b2, c, d;
          split_digits<S::LO>(u[h + 0], u[h + 1], a, b2);
          split_digits<S::LO>(u[h + 2], u[h + 3], c, d);
          hi[h / 4] = a | (c << 16);
          lo[h / 4] = b2 | (d << 16);
        }
        {
          uint8_t* dst = smem + S::OFF_P + (wg * HW / 16) * (kTileTok * 16) + j * 16 + (wg * HW) % 16;
          if constexpr (HW >= 16) {
#pragma unroll
            for (int i = 0; i < HW / 16; ++i) {
              *reinterpret_cast<uint4*>(dst + i * (kTileTok * 16)) =
                  make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
              *reinterpret_cast<uint4*>(dst + S::P_BYTES + i * (kTileTok * 16)) =
                  make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
            }
          } else {
            *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(dst + S::P_BYTES) = make_uint2(lo[0], lo[1]);
          }
        }
        if (j >= valid) {
          // whatever lies past the sequence's end must not meet a zero
          // probability as NaN: this warpgroup clears its share of the slabs
          const uint4 z = make_uint4(0, 0, 0, 0);
          for (int g = wg; g < NL; g += NWG) {
            const int slot = (int)(((int64_t)n * NSLAB + 1 + g) % NS);
            uint4* r = reinterpret_cast<uint4*>(smem + S::OFF_RING + slot * S::SLAB + j * 128);
#pragma unroll 1
            for (int i = 0; i < 8; ++i) r[i] = z;
          }
        }
        fence_proxy_async_shared();
        tc_fence_before();
        warp_arrive(p_full);
        first = false;
#pragma unroll
        for (int h = 0; h < HW; h += 2)
          unpair(fma2(pair(u[h], u[h + 1]), isig2, pair(ls[h], ls[h + 1])), ls[h], ls[h + 1]);
        if (n + 1 < count) w.next();
      }
      if (!seg_end) continue;
      if (n + 1 < count) load_q(w.b);  // the old query's last QK is done
      if (n < 0) continue;

      // ------------------------------------------------ the segment's result
      // softmax sums over the warp's tokens (lane head % HW), then the warpgroup's
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        if (o >= HW) {
#pragma unroll
          for (int h = 0; h < HW; ++h) ls[h] += __shfl_xor_sync(0xffffffffu, ls[h], o);
        } else {
          const bool up = (lane & o) != 0;
#pragma unroll
          for (int h = 0; h < o; ++h) {
            const float give = up ? ls[h] : ls[h + o], keep = up ? ls[h + o] : ls[h];
            ls[h] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        }
      }
      if (lane < HW) lred[(wg * 4 + quarter) * HW + lane] = ls[0];
      warp_arrive(&wg_bar[wg]);
      if (!wait(&wg_bar[wg], (uint32_t)meet & 1u)) { ok = false; break; }
      ++meet;
      const int hl = lane % HW;
      const float l = lred[(wg * 4 + 0) * HW + hl] + lred[(wg * 4 + 1) * HW + hl] + lred[(wg * 4 + 2) * HW + hl] +
                      lred[(wg * 4 + 3) * HW + hl];
      const int hb = h0 + wg * HW;  // first head of this warpgroup
      const bool whole = !shared_front && seq_end;
      const int64_t slot = (int64_t)blockIdx.x * 2 + (n_seg > 0 ? 1 : 0);
      if (hg == 0 && threadIdx.x == 0) {
        if (whole) seq_runs[b_now].x = kSeqWhole;
        else if (!shared_front) seq_runs[b_now].x = run * 2 + (n_seg > 0 ? 1 : 0);
        if (!whole && seq_end) seq_runs[b_now].y = run;
      }
      if (lane < HW) {
        mt[lane] = 1.0f / l;
        if (!whole && quarter == 0) ws_ml[slot * HB + wg * HW + lane] = make_float2(l == 0.0f ? -3e38f : r_ref, l);
      }
      __syncwarp();
      if (!wait(pv_done, (uint32_t)n & 1u)) { ok = false; break; }
      tc_fence_after();
#pragma unroll 1
      for (int g = 0; g < NL; ++g) {
        uint32_t o[HW];
        tmem_ld(t_lane + S::T_O + g * S::DIG * HB + wg * HW, o);
        if constexpr (S::DIG == 2) {
          uint32_t lo[HW];
          tmem_ld(t_lane + S::T_O + g * S::DIG * HB + HB + wg * HW, lo);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < HW; ++h)
            o[h] = __float_as_uint(__uint_as_float(o[h]) + __uint_as_float(lo[h]) * (1.0f / S::LO));
        } else {
          tmem_ld_wait();
        }
        if (whole) {
          // four lanes swap so that each stores four latents of one head
          const bool s1 = lane & 1, s2 = lane & 2;
          const int mine = (s1 ? 2 : 0) + (s2 ? 1 : 0);  // of each four heads
          __nv_bfloat16* dst = out + ((int64_t)b_now * H + hb + mine) * R + g * 128 + (j & ~3);
          // (one exchange for all heads, then the other: their latencies overlap)
          uint32_t x[HW / 4], y[HW / 4];
#pragma unroll
          for (int h = 0; h < HW; h += 4) {
            const float4 il = *reinterpret_cast<const float4*>(mt + h);
            x[h / 4] = pack_bf16x2(__uint_as_float(o[h]) * il.x, __uint_as_float(o[h + 1]) * il.y);
            y[h / 4] = pack_bf16x2(__uint_as_float(o[h + 2]) * il.z, __uint_as_float(o[h + 3]) * il.w);
          }
          uint32_t got[HW / 4];
#pragma unroll
          for (int i = 0; i < HW / 4; ++i) got[i] = __shfl_xor_sync(0xffffffffu, s1 ? x[i] : y[i], 1);
#pragma unroll
          for (int i = 0; i < HW / 4; ++i) {  // two heads of latents j & ~1 and j | 1
            const uint32_t a = s1 ? got[i] : x[i], c = s1 ? y[i] : got[i];
            x[i] = __byte_perm(a, c, 0x5410);
            y[i] = __byte_perm(a, c, 0x7632);
          }
#pragma unroll
          for (int i = 0; i < HW / 4; ++i) got[i] = __shfl_xor_sync(0xffffffffu, s2 ? x[i] : y[i], 2);
#pragma unroll
          for (int i = 0; i < HW / 4; ++i)
            if (hb + 4 * i + mine < H)
              *reinterpret_cast<uint2*>(dst + 4 * i * R) = s2 ? make_uint2(got[i], y[i]) : make_uint2(x[i], got[i]);
        } else {
          float* dst = ws_o + (slot * HB + wg * HW) * R + g * 128 + j;
#pragma unroll
          for (int h = 0; h < HW; ++h)
            if (hb + h < H) dst[h * R] = __uint_as_float(o[h]);
        }
      }
      tc_fence_before();
      warp_arrive(o_free);
      __syncwarp();
      if (lane < HW) mt[lane] = 0.0f;
      r_ref = 0.0f;
      __syncwarp();
      first = true;
      shared_front = false;
      ++n_seg;
    }
    if (!ok) raise_abort(abort, status, kStatusTimeout);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, S::T_COLS);
  }
}

// Sequences shared by several runs (their partials: sum_i 2^(m_i - M) O_i /
// sum_i 2^(m_i - M) l_i), and empty ones (zero rows).  Many sequences have few
// partials each (about runs / B): a warp takes 128 V columns of a head and reads
// them in turn.  Few sequences have many: a CTA takes a head, its warps every
// 8th partial.
// Bound by latency for small batches: with V = 1 a CTA (128 threads, 48
// registers, no shared memory) is resident beside a decode CTA before that ends
// (with the decode kernel then, 32 sequences x 16 heads 16.4 us, 64 x 16 40.9;
// whole heads 18.1, 42.6).  Bound by the partials' bytes out of L2 for large ones, where
// so many CTAs cost more (64 x 64 75.1 against 77.4 us, 74 x 128 whole sequences
// 15.5 against 24.0).  Without the merge those four take 12.5, 37.7, 69.8, 13.4.
constexpr int kCombineWarps = 8;
// The border is that of 16 heads (513 .. 768 tokens: 24 sequences 12.5 us by a
// CTA a head, 13.5 by a warp a part; 32 14.7 and 14.9; 48 16.8 and 15.9).  With
// more heads it lies lower: 64 heads, 8 sequences 17.6 and 18.4, 16 19.5 and
// 18.9; 128 heads, 4 17.7 and 18.4, 8 19.6 and 18.7, 24 33.7 and 27.9.
constexpr int kFewFrom = 32;         // sequences
constexpr int kSplitRows = 2048;     // sequences x heads up to which V = 1

__device__ __forceinline__ void store_bf16x4(__nv_bfloat16* dst, const float4& v, float f) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
}

template <int R, int V>
__global__ void __launch_bounds__(V == 1 ? 128 : 256, V == 1 ? 10 : 4)
    combine_few_kernel(const int2* __restrict__ seq_runs, int H, int HB, int runs, const float* __restrict__ ws_o,
                       const float2* __restrict__ ws_ml, __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  static_assert(V == 1 || V * 128 == R, "a warp of 8 takes whole heads");
  constexpr int kPerHead = R / 128 / V, kWarps = V == 1 ? 4 : 8;  // warps
  const int warp = (int)warp_id(), lane = (int)lane_id();
  const int b = blockIdx.x, h = blockIdx.y * (kWarps / kPerHead) + warp / kPerHead;
  const int col = (warp % kPerHead) * 128 * V + lane * 4;
  const int2 mine = seq_runs[b];
  if (mine.x == kSeqWhole || h >= H) return;
  float4 o[V];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 1.0f;
  if (mine.x != kSeqEmpty) {
    // (bounded, because a call that gave up leaves them unwritten)
    const int i0 = max(0, min(mine.x >> 1, runs - 1)), i1 = min(mine.y, runs - 1);
    // partial slots: the last segment of the first run, the first of the others
    const int cta0 = h / HB * runs, hl = h % HB;
    l = 0.0f;
#pragma unroll 4
    for (int i = i0; i <= i1; ++i) {
      const int64_t s = (int64_t)((cta0 + i) * 2 + (i == i0 ? mine.x & 1 : 0)) * HB + hl;
      const float2 ml = ws_ml[s];
      const float mn = fmaxf(m, ml.x), a = fast_exp2(m - mn), c = fast_exp2(ml.x - mn);
      m = mn;
      l = l * a + ml.y * c;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float4 x = *reinterpret_cast<const float4*>(ws_o + s * R + col + v * 128);
        o[v].x = o[v].x * a + x.x * c;
        o[v].y = o[v].y * a + x.y * c;
        o[v].z = o[v].z * a + x.z * c;
        o[v].w = o[v].w * a + x.w * c;
      }
    }
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int v = 0; v < V; ++v) store_bf16x4(out + ((int64_t)b * H + h) * R + col + v * 128, o[v], inv);
}

template <int R>
__global__ void __launch_bounds__(kCombineWarps * 32)
    combine_many_kernel(const int2* __restrict__ seq_runs, int H, int HB, int runs, const float* __restrict__ ws_o,
                        const float2* __restrict__ ws_ml, __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int V = R / 128;  // float4 per lane
  const int warp = (int)warp_id(), lane = (int)lane_id();
  const int b = blockIdx.x, h = blockIdx.y;
  const int2 mine = seq_runs[b];
  if (mine.x == kSeqWhole) return;
  __nv_bfloat16* dst = out + ((int64_t)b * H + h) * R + lane * 4;
  float m = -INFINITY, l = 0.0f;
  float4 o[V];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine.x == kSeqEmpty) {
    if (warp < V) store_bf16x4(dst + warp * 128, o[0], 1.0f);
    return;
  }
  const int i0 = max(0, min(mine.x >> 1, runs - 1)), i1 = min(mine.y, runs - 1);
  const int cta0 = h / HB * runs, hl = h % HB;
#pragma unroll 4
  for (int i = i0 + warp; i <= i1; i += kCombineWarps) {
    const int64_t s = (int64_t)((cta0 + i) * 2 + (i == i0 ? mine.x & 1 : 0)) * HB + hl;
    const float2 ml = ws_ml[s];
    const float mn = fmaxf(m, ml.x), a = fast_exp2(m - mn), c = fast_exp2(ml.x - mn);
    m = mn;
    l = l * a + ml.y * c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float4 x = *reinterpret_cast<const float4*>(ws_o + s * R + v * 128 + lane * 4);
      o[v].x = o[v].x * a + x.x * c;
      o[v].y = o[v].y * a + x.y * c;
      o[v].z = o[v].z * a + x.z * c;
      o[v].w = o[v].w * a + x.w * c;
    }
  }
  __shared__ float sm[kCombineWarps], sl[kCombineWarps];
  __shared__ float4 so[kCombineWarps][R / 4];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) so[warp][v * 32 + lane] = o[v];
  __syncthreads();
  if (warp >= V) return;  // warp v merges columns [128 v, 128 v + 128)
  float top = -INFINITY, den = 0.0f;
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < kCombineWarps; ++i) top = fmaxf(top, sm[i]);
  const int filled = min(kCombineWarps, i1 - i0 + 1);  // warps that had a partial (a NaN one's sm is -inf as well)
  for (int i = 0; i < filled; ++i) {
    const float c = fast_exp2(sm[i] - top);
    const float4 x = so[i][warp * 32 + lane];
    den += sl[i] * c;
    r.x += x.x * c;
    r.y += x.y * c;
    r.z += x.z * c;
    r.w += x.w * c;
  }
  store_bf16x4(dst + warp * 128, r, 1.0f / den);
}

// The scratch: the sequences' runs, then every CTA's two partials.  One size for
// every call (128 KB a partial at 64 heads x 512 columns), so that captured
// calls keep their addresses.
size_t scratch_bytes(int sm) {
  const size_t partials = (size_t)sm * 2 * kMaxHeadsPerCta;
  return kMaxSeqs * sizeof(int2) + partials * (512 * sizeof(float) + sizeof(float2));
}

template <int R, int P, int HB>
int launch(dsb_ctx* ctx, const void* q_lat, const void* q_rope, const void* cache, const float* scales,
           int64_t n_blocks, const int32_t* block_table, int max_blocks, const int32_t* seq_lens, int B, int H,
           float softmax_scale, void* out) {
  using S = Shape<R, P, HB>;
  CUtensorMap map_lat, map_rope;
  const uint64_t rows = (uint64_t)n_blocks * kPageTok, pitch = R + 2 * P;
  int rc = make_tmap_2d(ctx, &map_lat, cache, CU_TENSOR_MAP_DATA_TYPE_UINT8, pitch, rows, pitch, 128, kPageTok,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != DSB_OK) return rc;
  rc = make_tmap_2d(ctx, &map_rope, cache, CU_TENSOR_MAP_DATA_TYPE_UINT8, pitch, rows, pitch, P * 2, kPageTok,
                    P == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc != DSB_OK) return rc;
  const int groups = (H + HB - 1) / HB;
  const int runs = std::max(1, ctx->sm_count / groups);
  auto* seq_runs = static_cast<int2*>(ctx->mla8);
  auto* ws_ml = reinterpret_cast<float2*>(seq_runs + kMaxSeqs);
  auto* ws_o = reinterpret_cast<float*>(ws_ml + (size_t)ctx->sm_count * 2 * kMaxHeadsPerCta);
  auto kern = decode_fp8_kernel<R, P, HB>;
  static std::atomic<bool> attr_set[kMaxDevices];
  if (rc = smem_attr_once(ctx, kern, S::SMEM_BYTES, attr_set); rc != DSB_OK) return rc;
  DSB_CUDA_TRY(ctx, launch_pdl(kern, dim3((unsigned)(groups * runs)), S::THREADS, S::SMEM_BYTES, ctx->stream, map_lat,
                               map_rope, static_cast<const __nv_bfloat16*>(q_lat),
                               static_cast<const __nv_bfloat16*>(q_rope), scales, n_blocks, block_table, max_blocks,
                               seq_lens, B, H, runs, softmax_scale * 1.4426950408889634f,
                               static_cast<__nv_bfloat16*>(out), ws_o, ws_ml, seq_runs, ctx->d_status));
  auto combine = [&](auto kernel, int heads, int threads) {  // heads per CTA
    return launch_pdl(kernel, dim3((unsigned)B, (unsigned)((H + heads - 1) / heads)), threads, 0, ctx->stream, seq_runs,
                      H, HB, runs, ws_o, ws_ml, static_cast<__nv_bfloat16*>(out));
  };
  // a sequence has about runs / B partials
  cudaError_t err = cudaSuccess;
  if (B < kFewFrom) {
    err = combine(combine_many_kernel<R>, 1, kCombineWarps * 32);
  } else if (R == 128 || B * H <= kSplitRows) {
    err = combine(combine_few_kernel<R, 1>, 512 / R, 128);
  } else {
    if constexpr (R == 512) err = combine(combine_few_kernel<R, 4>, 8, 256);
  }
  DSB_CUDA_TRY(ctx, err);
  ctx->stats.kernel_launches += 2;
  ctx->stats.mla_calls++;
  return DSB_OK;
}

}  // namespace
}  // namespace dsb

extern "C" int dsb_mla_decode_fp8(dsb_ctx* ctx, const void* q_lat, const void* q_rope, const void* cache,
                                  const float* scales, int64_t n_blocks, const int32_t* block_table, int max_blocks,
                                  const int32_t* seq_lens, int B, int H, int R, int P, float softmax_scale,
                                  void* out_lat) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (q_lat == nullptr || q_rope == nullptr || cache == nullptr || scales == nullptr || block_table == nullptr ||
      seq_lens == nullptr || out_lat == nullptr)
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: null pointer argument");
  if (!cache_shape_ok(R, P))
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_decode_fp8: (R, P) = (%d, %d) not supported", R, P);
  if (B <= 0 || B > kMaxSeqs || H <= 0 || H > 128 || max_blocks <= 0 || n_blocks <= 0 || n_blocks >= (1 << 25) ||
      (int64_t)B * max_blocks > INT32_MAX || !std::isfinite(softmax_scale))
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: bad arguments B=%d H=%d max_blocks=%d n_blocks=%lld scale=%g", B,
                H, max_blocks, (long long)n_blocks, softmax_scale);
  if ((reinterpret_cast<uintptr_t>(q_lat) | reinterpret_cast<uintptr_t>(q_rope) | reinterpret_cast<uintptr_t>(scales) |
       reinterpret_cast<uintptr_t>(out_lat) | reinterpret_cast<uintptr_t>(cache)) & 15u)
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: pointers must be 16-byte aligned");
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_mla_decode_fp8: cudaSetDevice(%d) failed", ctx->device);
  if (ctx->mla8 == nullptr) {
    const size_t need = scratch_bytes(ctx->sm_count);
    if (int rc = ensure_buffer(ctx, &ctx->mla8, &ctx->mla8_bytes, need, need, "dsb_mla_decode_fp8"); rc != DSB_OK)
      return rc;
  }
  auto run = [&](auto f) {
    return f(ctx, q_lat, q_rope, cache, scales, n_blocks, block_table, max_blocks, seq_lens, B, H, softmax_scale,
             out_lat);
  };
  // the fewest columns of 16, 32 and 64 that hold the heads, or groups of 64: a
  // tile's MMA time grows with them (64 sequences, 16 heads 41 us, 32 50, 64 80,
  // 96 and 128 128 - 132; two groups of 48 took 138 when two of 64 took 130)
  if (R == 512) return H <= 16 ? run(launch<512, 64, 16>) : H <= 32 ? run(launch<512, 64, 32>) : run(launch<512, 64, 64>);
  return H <= 16 ? run(launch<128, 32, 16>) : H <= 32 ? run(launch<128, 32, 32>) : run(launch<128, 32, 64>);
}
