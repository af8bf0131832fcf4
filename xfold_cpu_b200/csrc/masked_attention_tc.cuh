// Masked attention on tcgen05 for bf16 (the mathematics: masked_attention.cuh).
//
// Rows are tiles of nqt = 128 / rep queries with all rep heads of one K/V head (row
// i rep + h), so a TMA box (64 dims, rep heads, nqt queries) fills one 128-row operand and K and V
// are read once for the group, whether the tile is 128 queries of one head or one new
// token of 128 heads.
//
// Forward, per key tile of 64 and row tile ("slot"):
//   S  = Q K^T      tcgen05.mma, f32 in TMEM
//   P  = 2^(s - m)  one row a thread: masks, cap and distance on f32 scores, running maximum m that
//                   moves only when a tile exceeds it by 2^8 (then O and l shrink), row sum l of
//                   the f32 probabilities; P goes back over S as bf16
//   O += P V        tcgen05.mma with P from TMEM
// A slot has two softmax warpgroups with an S buffer each, which take its tiles in turn: while
// one waits for products, the other computes.  They share the rows' m through shared
// memory (a tile's maximum is compared with m once the tile before has moved it) and keep a
// part of l each.  A tile's chain of handoffs is long (about 100 cycles a wait), so
// it is the number of tiles in flight that fills the MUFU and the tensor core: two warpgroups
// and two tiles in flight took 2200 cycles per 2 x 128 x 64 scores at head dim 128.  Measured at
// 8192 causal tokens, 16 heads on 4: 1030 TFLOP/s at head dim 128, 608 at 64 (softmax
// instructions: 56 % of the issue slots), 747 and 460 with P in two parts; one token of eight
// sequences over 30011 keys 157 us, 5.2 TB/s.
// The tensor core takes P no wider than bf16 next to bf16 V.  P rounded once puts an error of
// the size of the result's own rounding on O (2^-9 of the value at most).  Inference over
// many rows takes that.  With what the backward pass needs, and in blocks of one row
// tile, which wait on memory, P goes in two bf16 parts (its rounding and what that took away,
// 2^-17) as two products: D = do . o then carries no error of P into every score gradient.
//
// Every block first lists, with all its threads, the key tiles that its rows see at all, and
// which need masks; the loader, the MMA issuers and the softmax walk the list.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "masked_attention.cuh"

namespace xfb {

constexpr int kMtKeys = 64;       // keys a tile of the forward kernel
// Tiles that a block's list holds: forward 2^17 keys (more are split over blocks), backward 2^19
// keys, or 2^19 rows of a K/V head.
constexpr int kMtMaxTiles = 2048, kMtMaxStream = 8192;

// A list entry: a tile's number and what its visitors have to know.
constexpr uint32_t kMtTile = 0x00FFFFFF;    // number, less the block's first
constexpr uint32_t kMtListed = 0x80000000;  // set in every entry
constexpr uint32_t kMtMasked = 0x01000000;  // some row of the tile does not see some column
constexpr uint32_t kMtPadded = 0x02000000;  // has columns of no document
constexpr uint32_t kMtSlot0 = 0x04000000;   // forward: seen by slot 0, by slot 1
constexpr uint32_t kMtSlot1 = 0x08000000;

// Multipliers (0 or 1) of the head and batch coordinates in a K or V tensor map: a
// broadcast dimension has size 1 there.
struct MtMap {
  int head, batch;
};

// SLOTS row tiles a block; 0: one tile of up to 32 rows, spread (see the kernel).
template <int DP, int SLOTS_>
struct MtForward {
  static constexpr bool kSpread = SLOTS_ == 0;
  static constexpr int SLOTS = kSpread ? 1 : SLOTS_;
  static constexpr int kSBufs = SLOTS == 2 ? 2 : 4;  // S / P buffers a slot
  static constexpr int kQTile = 128 * DP * 2;
  static constexpr int kTile = kMtKeys * DP * 2;
  static constexpr int kStages = DP == 64 ? 6 : SLOTS == 2 ? 4 : 5;  // of K and of V
  // TMEM columns of a slot: S / P buffers, O
  static constexpr int kOCol = kSBufs * kMtKeys;
  static constexpr int kSlotCols = kOCol + DP;
  static constexpr int kKOff = SLOTS * kQTile;
  static constexpr int kVOff = kKOff + kStages * kTile;
  static constexpr int kMarkOff = kVOff + kStages * kTile;
  // lengths of the lists (the block's tiles, each slot's), which come last: as long as the call
  // needs them, for what shared memory does not take is L1 (16 KB more of it: 182 -> 164 us a dq)
  static constexpr int kRowOff = kMarkOff + 16;  // m, l of each half
  static constexpr int kBarOff = kRowOff + SLOTS * 3 * 128 * 4;
  static constexpr int kBars = SLOTS + 4 * kStages + SLOTS * (3 * kSBufs + 2);
  static constexpr int kBytes = kBarOff + kBars * 8 + 16;
  static constexpr int kListOff = kBytes;
  static constexpr int launch_bytes(int64_t tiles) {
    return kListOff + (1 + SLOTS) * static_cast<int>(tiles) * 4 + 1024;
  }
  static constexpr int kMostBytes = launch_bytes(kMtMaxTiles);
  static constexpr int kSoftmaxThreads = SLOTS * 256;
  static constexpr int kThreads = kSoftmaxThreads + 128;
  static constexpr int kControl = SLOTS * 8;  // first control warp: loader, S issuers, P V issuer
  // registers a thread: 640 threads start with 96; 512 * 104 + 128 * 64 = 640 * 96
  static constexpr int kRegsSoftmax = 104, kRegsOther = 64;
  static_assert(kMostBytes <= 232448, "shared memory exceeds 227 KB");
};

// Loads a tile of ROWS keys: DP / 64 boxes of 64 dims.
template <int DP, int ROWS>
__device__ __forceinline__ void mt_load_keys(uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                                             int key0, int g, int b) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + c * ROWS * 128, map, bar, c * 64, key0, g, b);
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3), "r"(c4)
      : "memory");
}

// Issue by a whole warp: every lane walks the loop and the waits, one elected lane (always the
// same for a full mask, as a commit demands) issues.  So the descriptors stay warp-uniform and
// need no move per instruction: a lane of its own took 130 cycles a product to issue.
__device__ __forceinline__ void mt_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mt_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mt_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar))
      : "memory");
}

// K-major operand: k-step of 16 dims (chunks of 64 dims are `chunk` bytes apart).
__device__ __forceinline__ uint64_t mt_k_desc(uint32_t addr, int step, uint32_t chunk) {
  return sw128_desc(addr + (step >> 2) * chunk + (step & 3) * 32, 16, 1024);
}
// The same tile as the MN-major operand of a product over its rows: 16 rows a step.
__device__ __forceinline__ uint64_t mt_mn_desc(uint32_t addr, int step, uint32_t chunk) {
  return sw128_desc(addr + step * 2048, chunk, 1024);
}

// Zeros the rows `used`.. of `count` operand tiles of ROWS rows (whole 128-byte rows, so no
// swizzle matters), which no TMA box covers when rep does not divide ROWS.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void mt_zero_tail_rows(uint8_t* tiles, int count, int used) {
  if (used == ROWS) return;
  const int per = (ROWS - used) * 8;  // 16-byte pieces of a 64-dim chunk
  for (int x = threadIdx.x; x < count * (DP / 64) * per; x += THREADS)
    *reinterpret_cast<uint4*>(tiles + (x / per) * (ROWS * 128) + used * 128 + (x % per) * 16) =
        make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
}
// Zeros one row of a tile.
template <int DP, int ROWS>
__device__ __forceinline__ void mt_zero_row(uint8_t* tile, int row) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      reinterpret_cast<uint4*>(tile + c * (ROWS * 128) + row * 128)[e] = make_uint4(0u, 0u, 0u, 0u);
}

// After a wait that gave up: time for the loads in flight to land before the block exits.
__device__ __forceinline__ void mt_drain(volatile int* abort_flag) {
  if (!*abort_flag) return;
  const uint64_t start = global_ns();
  while (global_ns() - start < 1000000ull) __nanosleep(1000);
}

// Packs the marked tiles' entries into `list` and returns their number: one warp, `entry(t)`
// gives an entry of tile t or 0.
template <class Entry>
__device__ __forceinline__ int mt_compact(uint32_t* list, int tiles, Entry entry) {
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const uint32_t e = t0 + lane < tiles ? entry(t0 + lane) : 0u;
    const uint32_t marked = __ballot_sync(0xffffffffu, e != 0);
    if (e != 0) list[count + __popc(marked & ((1u << lane) - 1))] = e;
    count += __popc(marked);
  }
  return count;
}

// The capped score in log2 units: cap tanh(x / cap) = cap - 2 cap r with r = 1 / (1 + e^(2 x / cap))
// of the part mt_cap_part(2 x / cap log2(e)); `c` = cap log2(e).  A masked x of -inf stays -inf:
// x + 3e38 is far above any score otherwise.
__device__ __forceinline__ float mt_cap_part(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2_approx(z)));
  return r;
}
__device__ __forceinline__ float mt_capped(float x, float r, float c) {
  return fminf(fmaf(-2.f * c, r, c), x + 3e38f);
}

// What turns products into scores, fixed at compile time: a cap, a distance.  Scores are in
// log2 units; without either they stay raw products and the exponent's FMA scales them.
template <bool CAP, bool SLOPES>
struct MtScore {
  static constexpr bool kRaw = !CAP && !SLOPES;
  // A distance alone is added as if all keys came before the query, in packed arithmetic: keys
  // after it are put right in TMEM by the pass that masks.
  static constexpr bool kOneSided = SLOPES && !CAP;
  // of a row's products with a tile's keys, in place; `offset` = the row's position less the first key
  template <int N>
  static __device__ __forceinline__ void apply(const MaskedArgs& a, float (&s)[N], float slope2,
                                               float offset) {
    if constexpr (CAP) {
      const float k = a.scale * a.inv_cap * (2.f * kLog2e);
      const float c = a.cap * kLog2e;
#pragma unroll
      for (int j = 0; j < N; ++j) s[j] = mt_capped(s[j], mt_cap_part(s[j] * k), c);
      if constexpr (SLOPES) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          s[j] = fmaf(-slope2, fabsf(offset - static_cast<float>(j)), s[j]);
      }
    } else if constexpr (SLOPES) {
      // -slope (offset - j): four pairs of columns at a time step on by 8 slope
      const float k = a.scale * kLog2e;
      const float2 k2 = make_float2(k, k), step = make_float2(8.f * slope2, 8.f * slope2);
      float2* s2 = reinterpret_cast<float2*>(s);
      float2 t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        t[e] = make_float2(-slope2 * (offset - static_cast<float>(2 * e)),
                           -slope2 * (offset - static_cast<float>(2 * e + 1)));
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        s2[j] = fma2(s2[j], k2, t[j & 3]);
        t[j & 3] = add2(t[j & 3], step);
      }
    }
  }
};

// Masks of a row and COLS columns, in TMEM: the scores a row does not see become -inf before the
// common code loads them (and `dp` 0, where there is one).  Done there and not in registers,
// so that tiles without masks keep one straight path from load to store: a branch that
// changes 64 registers cost every tile as many moves.  `hidden(j, out)` fills the flags of
// columns j..j+3.  With AFTER, the score of a key `ahead` > 0 places after the query, which the
// common code takes as before it, loses 2 slope ahead (in products: `twice` = 2 slope / scale).
template <bool DPART, int COLS, bool AFTER, class Hidden>
__device__ __forceinline__ void mt_mask_tmem(uint32_t s_row, uint32_t dp_row, float twice,
                                             float ahead0, Hidden hidden) {
#pragma unroll 1
  for (int c = 0; c < COLS; c += 16) {
    float v[16], w[16];
    tmem_ld16(s_row + c, v);
    if (DPART) tmem_ld16(dp_row + c, w);
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      bool off[4];
      hidden(c + j, off);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (AFTER) v[j + e] = fmaf(-twice, fmaxf(ahead0 + static_cast<float>(c + j + e), 0.f), v[j + e]);
        if (off[e]) v[j + e] = -INFINITY;
        if (DPART && off[e]) w[j + e] = 0.f;
      }
    }
    tmem_st16_from(s_row + c, v);
    if (DPART) tmem_st16_from(dp_row + c, w);
  }
  tmem_wait_st();
}

// What rounding a pair to the bf16 pair `high` took away, as a bf16 pair.
__device__ __forceinline__ uint32_t mt_low_part(float2 v, uint32_t high) {
  const float2 hi = make_float2(__uint_as_float(high << 16), __uint_as_float(high & 0xFFFF0000u));
  const float2 lo = fma2(hi, make_float2(-1.f, -1.f), v);
  return pack_bf16x2(lo.x, lo.y);
}

// Stores a warp's eight words of P at its columns w * 8.. of 32, zeros at the others.
__device__ __forceinline__ void mt_st_spread(uint32_t taddr, const uint32_t* v, int w) {
  uint32_t all[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) all[e] = (e >> 3) == w ? v[e & 7] : 0u;
  tmem_st32_u(taddr, all);
}

// SLOTS_ = 0 is for a few rows (up to 32, a new token's heads) over many keys: one thread a row
// would leave all the softmax of a tile to one warp.  The rows are loaded four times, into
// the lanes of each warp; warp w takes columns 16 w.. of a tile, leaves zeros for the others, and
// the four partial O, m and l are joined at the end as key splits are.
template <int DP, int SLOTS_, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(MtForward<DP, SLOTS_>::kThreads, 1)
    mt_forward_kernel(const __grid_constant__ CUtensorMap tmQ,
                      const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const MtMap mk, const MtMap mv,
                      const __grid_constant__ MaskedArgs a) {
  using L = MtForward<DP, SLOTS_>;
  constexpr int SLOTS = L::SLOTS, NB = L::kSBufs;
  constexpr bool kSpread = L::kSpread;
  constexpr int NS = L::kStages;
  constexpr uint32_t kIdescS = idesc_bf16(128, kMtKeys, false, false);
  constexpr uint32_t kIdescO = idesc_bf16(128, DP, false, true);
  constexpr uint32_t kSlotCols = L::kSlotCols;
  constexpr uint32_t kTmemCols = SLOTS * kSlotCols <= 256 ? 256 : 512;
  static_assert(SLOTS * kSlotCols <= 512, "TMEM has 512 columns");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::kKOff;
  uint8_t* sV = smem + L::kVOff;
  const int per = (a.k_tiles + a.splits - 1) / a.splits;  // key tiles of a split
  uint32_t* all_tiles = reinterpret_cast<uint32_t*>(smem + L::kListOff);
  uint32_t* slot_tiles = all_tiles + per;  // [SLOTS][per]
  int* counts = reinterpret_cast<int*>(smem + L::kMarkOff);  // all, each slot's
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_full = q_full + SLOTS;
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* s_full = v_empty + NS;          // [SLOTS][NB], as tile m of a slot has buffer m % NB
  uint64_t* p_full = s_full + SLOTS * NB;   // [SLOTS][NB]
  uint64_t* pv_done = p_full + SLOTS * NB;  // [SLOTS][NB]
  uint64_t* m_full = pv_done + SLOTS * NB;  // [SLOTS][2] the rows' m includes the half's last tile
  float* row_m = reinterpret_cast<float*>(smem + L::kRowOff);  // [SLOTS][128]
  float* row_l = row_m + SLOTS * 128;                          // [SLOTS][2][128]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(m_full + SLOTS * 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---- this block's rows and keys
  const int nqt = (kSpread ? 32 : 128) / a.rep;
  int item = blockIdx.x;
  const int split = item % a.splits;
  item /= a.splits;
  const int g = item % a.G;
  item /= a.G;
  const int b = item % a.B;
  const int pairs = (a.q_tiles + SLOTS - 1) / SLOTS;
  const int pair = pairs - 1 - item / a.B;  // causal rows with the most keys come first
  const int prefix = ma_prefix(a, b);
  const int tile0 = split * per;
  const int tiles = max(0, min(a.k_tiles - tile0, per));
  const bool docs = a.qdoc != nullptr;
  const bool two_parts = SLOTS == 1 || a.lse != nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&q_full[s], 1);
      for (int i = NB * s; i < NB * s + NB; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 128);
        mbar_init(&pv_done[i], 1);
      }
      for (int i = 2 * s; i < 2 * s + 2; ++i) mbar_init(&m_full[i], 128);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], SLOTS);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == L::kControl) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // rows past the box's rep * nqt are zeros
  if constexpr (kSpread) {
    for (int w = 0; w < 4 * (DP / 64); ++w)
      mt_zero_tail_rows<64, 32, L::kThreads>(sQ + w * 4096, 1, a.rep * nqt);
  } else {
    mt_zero_tail_rows<DP, 128, L::kThreads>(sQ, SLOTS, a.rep * nqt);
  }
  // ---- lists: warp 0 the block's, warps 1.. the slots'
  if (warp <= SLOTS) {
    int4 qr[SLOTS];
    int lim_lo[SLOTS], lim_hi[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int i0 = (pair * SLOTS + s) * nqt;
      const int i1 = min(i0 + nqt, a.nq) - 1;
      lim_lo[s] = i0 < a.nq ? ma_limit(a, i0, prefix) : 0;
      lim_hi[s] = i0 < a.nq ? ma_limit(a, i1, prefix) : 0;
      qr[s] = make_int4(0, 0, 0, 0);
      if (docs && i0 < a.nq) qr[s] = ma_join_ranges(a.qrange + b * a.qrange_sb, i0 / 64, i1 / 64);
    }
    const auto slot_entry = [&](int s, int t) -> uint32_t {
      const int key0 = (tile0 + t) * kMtKeys;
      if (key0 >= lim_hi[s]) return 0u;
      bool masked = key0 + kMtKeys > lim_lo[s];
      // a distance alone: keys after the slot's first query are put right with the masks
      if (MtScore<CAP, SLOPES>::kOneSided)
        masked = masked || key0 + kMtKeys > (pair * SLOTS + s) * nqt + a.off;
      uint32_t pad = 0u;
      if (docs) {
        const int4 kr = a.krange[b * a.krange_sb + tile0 + t];
        if (!ma_ranges_meet(qr[s], kr)) return 0u;
        // one and the same document on both sides needs no masks
        masked = masked || qr[s].z || kr.z || qr[s].x != qr[s].y || kr.x != kr.y;
        pad = kr.z ? kMtPadded : 0u;
      }
      return kMtListed | t | (masked ? kMtMasked : 0u) | pad;
    };
    int count;
    if (warp == 0) {
      count = mt_compact(all_tiles, tiles, [&](int t) -> uint32_t {
        const uint32_t e0 = slot_entry(0, t), e1 = SLOTS > 1 ? slot_entry(SLOTS - 1, t) : 0u;
        return e0 | e1 | (e0 ? kMtSlot0 : 0u) | (e1 ? kMtSlot1 : 0u);
      });
    } else {
      count = mt_compact(slot_tiles + (warp - 1) * per, tiles,
                         [&](int t) -> uint32_t { return slot_entry(SLOTS > 1 ? warp - 1 : 0, t); });
    }
    if (lane == 0) counts[warp] = count;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= L::kControl) {
    if constexpr (SLOTS == 2)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRegsOther));
    if (warp == L::kControl && lane == 0) {
      // ------------------------------------------------ TMA loader
      for (int s = 0; s < SLOTS; ++s) {
        constexpr int kCopies = kSpread ? 4 : 1;
        mbar_arrive_expect_tx(&q_full[s], kCopies * (DP / 64) * 128 * a.rep * nqt);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
          for (int w = 0; w < kCopies; ++w)
            tma_load_5d(sQ + s * L::kQTile + c * 16384 + w * 4096, &tmQ, &q_full[s], c * 64, 0,
                        (pair * SLOTS + s) * nqt, g, b);
      }
      const int count = counts[0];
      int st = 0;
      uint32_t ph = 1;
      for (int n = 0; n < count; ++n) {
        const uint32_t entry = all_tiles[n];
        const int key0 = (tile0 + (entry & kMtTile)) * kMtKeys;
        // The softmax warps wait for V of a padded tile, but not for every tile's, so their wait
        // could pass on the phase of the stage's last tile.  K, and with it S, of a padded tile
        // comes after that tile's V has been used.
        if ((entry & kMtPadded) && !mbar_wait(&v_empty[st], ph, kErrWaitProducer, abort_flag)) break;
        if (!mbar_wait(&k_empty[st], ph, kErrWaitProducer, abort_flag)) break;
        mbar_arrive_expect_tx(&k_full[st], L::kTile);
        mt_load_keys<DP, kMtKeys>(sK + st * L::kTile, &tmK, &k_full[st], key0, g * mk.head, b * mk.batch);
        if (!mbar_wait(&v_empty[st], ph, kErrWaitProducer, abort_flag)) break;
        mbar_arrive_expect_tx(&v_full[st], L::kTile);
        mt_load_keys<DP, kMtKeys>(sV + st * L::kTile, &tmV, &v_full[st], key0, g * mv.head, b * mv.batch);
        if (++st == NS) st = 0, ph ^= 1;
      }
    } else if (warp > L::kControl && warp <= L::kControl + SLOTS) {
      // ------------------------------------------------ issuer of a slot's S
      const int s = warp - L::kControl - 1;
      const uint32_t q_addr = smem_u32(sQ + s * L::kQTile);
      const uint32_t slot_tmem = tmem_base + s * kSlotCols;
      const int count = counts[0];
      int m = 0;  // tiles of the slot
      int st = 0;
      uint32_t ph = 0;
      bool ok = mbar_wait(&q_full[s], 0, kErrWaitMma, abort_flag);
      for (int n = 0; ok && n < count; ++n) {
        ok = mbar_wait(&k_full[st], ph, kErrWaitMma, abort_flag);
        if (!ok) break;
        const int here = st;
        if (++st == NS) st = 0, ph ^= 1;
        if (SLOTS > 1 && !(all_tiles[n] & (s == 0 ? kMtSlot0 : kMtSlot1))) {
          if (lane == 0) mbar_arrive(&k_empty[here]);
          continue;
        }
        const int buf = m % NB;
        // the product that read this buffer's last P
        if (m >= NB)
          ok = mbar_wait(&pv_done[NB * s + buf], (m / NB - 1) & 1, kErrWaitMma, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(sK + here * L::kTile);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          mt_mma(slot_tmem + buf * kMtKeys, mt_k_desc(q_addr, k, 16384),
                 mt_k_desc(k_addr, k, kMtKeys * 128), kIdescS, k > 0 ? 1u : 0u);
        mt_commit(&s_full[NB * s + buf]);
        mt_commit(&k_empty[here]);
        ++m;
      }
    } else if (warp == L::kControl + SLOTS + 1) {
      // ------------------------------------------------ issuer of O += P V
      const int count = counts[0];
      int m[SLOTS] = {};
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int n = 0; ok && n < count; ++n) {
        const uint32_t entry = all_tiles[n];
        ok = mbar_wait(&v_full[st], ph, kErrWaitMma, abort_flag);
        const uint32_t v_addr = smem_u32(sV + st * L::kTile);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
          if (!ok || (SLOTS > 1 && !(entry & (s == 0 ? kMtSlot0 : kMtSlot1)))) continue;
          const int buf = m[s] % NB;
          ok = mbar_wait(&p_full[NB * s + buf], (m[s] / NB) & 1, kErrWaitMma, abort_flag);
          if (!ok) continue;
          tc_fence_after();
          const uint32_t o_tmem = tmem_base + s * kSlotCols + L::kOCol;
          const uint32_t p_tmem = tmem_base + s * kSlotCols + buf * kMtKeys;
#pragma unroll
          for (int k = 0; k < kMtKeys / 16; ++k)
            mt_mma_ts(o_tmem, p_tmem + 8 * k, mt_mn_desc(v_addr, k, kMtKeys * 128), kIdescO,
                      m[s] > 0 || k > 0 ? 1u : 0u);
          if (two_parts) {
#pragma unroll
            for (int k = 0; k < kMtKeys / 16; ++k)
              mt_mma_ts(o_tmem, p_tmem + kMtKeys / 2 + 8 * k,
                        mt_mn_desc(v_addr, k, kMtKeys * 128), kIdescO, 1u);
          }
          mt_commit(&pv_done[NB * s + buf]);
          ++m[s];
        }
        mt_commit(&v_empty[st]);
        if (++st == NS) st = 0, ph ^= 1;
      }
    }
  } else {
    if constexpr (SLOTS == 2)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRegsSoftmax));
    // ------------------------------------------------ softmax warps, one row a thread
    const int s = warp >> 3, half = (warp >> 2) & 1;
    const int row = threadIdx.x & 127;
    const uint32_t t_row = tmem_base + s * kSlotCols + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_row = t_row + L::kOCol;
    // the thread's row of q, and its columns of a tile
    const int q_row = kSpread ? row & 31 : row;
    constexpr int kCols = kSpread ? 16 : kMtKeys;
    const int col0 = kSpread ? (warp & 3) * kCols : 0;
    const int i = (pair * SLOTS + s) * nqt + q_row / a.rep;
    const int h = g * a.rep + q_row % a.rep;
    const bool live = q_row < nqt * a.rep && i < a.nq;
    const bool warp_live = __any_sync(0xffffffffu, live);  // a warp without rows only keeps time
    const int limit = live ? ma_limit(a, i, prefix) : 0;
    int doc = docs && live ? a.qdoc[b * a.qdoc_sb + i] : -1;
    if (doc < 0) doc = -2;  // padding does not see padding
    const float slope2 = live && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
    using Score = MtScore<CAP, SLOPES>;
    const float twice = Score::kOneSided ? 2.f * slope2 / (a.scale * kLog2e) : 0.f;
    const float unit = Score::kRaw ? a.scale * kLog2e : 1.f;  // raw scores need a scale > 0
    const uint32_t* list = slot_tiles + s * per;
    const int count = counts[1 + s];
    float m_ref = -INFINITY, l = 0.f;  // l belongs to the m_ref of this half's last tile
    bool ok = true;
    for (int m = half; m < count; m += 2) {
      const uint32_t entry = list[m];
      const int buf = m % NB;
      const uint32_t s_row = t_row + buf * kMtKeys;
      const int key0 = (tile0 + (entry & kMtTile)) * kMtKeys + col0;
      ok = mbar_wait(&s_full[NB * s + buf], (m / NB) & 1, kErrWaitSoftmax, abort_flag);
      if (!ok) break;
      tc_fence_after();
      float x[kCols];
      float mt = -INFINITY;
      if (warp_live) {
        if (entry & kMtMasked) {
          const int32_t* kdoc = docs ? a.kdoc + b * a.kdoc_sb + key0 : nullptr;
          const float ahead0 = static_cast<float>(key0 - i - a.off);
          mt_mask_tmem<false, kCols, Score::kOneSided>(s_row + col0, 0u, twice, ahead0, [&](int j, bool (&off)[4]) {
            int4 id = make_int4(doc, doc, doc, doc);
            if (docs) id = *reinterpret_cast<const int4*>(kdoc + j);
            off[0] = key0 + j >= limit || id.x != doc;
            off[1] = key0 + j + 1 >= limit || id.y != doc;
            off[2] = key0 + j + 2 >= limit || id.z != doc;
            off[3] = key0 + j + 3 >= limit || id.w != doc;
          });
        }
        if constexpr (kSpread) {
          tmem_ld16(s_row + col0, x);
        } else {
          tmem_ld32_to(s_row, x);
          tmem_ld32_to(s_row + 32, x + 32);
          tmem_wait_ld();
        }
        Score::apply(a, x, slope2, static_cast<float>(i + a.off - key0));
        if constexpr (kSpread) {
          float top[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = max_nan(max3_nan(x[4 * e], x[4 * e + 1], x[4 * e + 2]), x[4 * e + 3]);
          mt = max_nan(max3_nan(top[0], top[1], top[2]), top[3]) * unit;
        } else {
          mt = tile_max64(x) * unit;
        }
      }
      // ---- the rows' m, as the other half left it, and what this tile makes of it
      float m_last = m_ref;
      if (m > 0) {
        ok = mbar_wait(&m_full[2 * s + 1 - half], ((m - 1) >> 1) & 1, kErrWaitSoftmax, abort_flag);
        if (!ok) break;
        m_last = row_m[s * 128 + row];
      }
      const bool grow = !(mt <= m_last + 8.f);
      const float m_new = grow ? mt : m_last;
      row_m[s * 128 + row] = m_new;
      mbar_arrive(&m_full[2 * s + half]);
      if (warp_live) {
      if (m > 0 && __any_sync(0xffffffffu, grow)) {
        ok = mbar_wait(&pv_done[NB * s + (m - 1) % NB], ((m - 1) / NB) & 1, kErrWaitSoftmax,
                       abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float shrink = grow ? ex2_approx(m_last - m_new) : 1.f;  // 0 when m_last = -inf
#pragma unroll 1
        for (int c = 0; c < DP / 16; ++c) {
          float o[16];
          tmem_ld16(o_row + c * 16, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= shrink;
          tmem_st16_from(o_row + c * 16, o);
        }
        tmem_wait_st();
      }
      // ---- probabilities and their sum
      const float base = m_new == -INFINITY ? 0.f : m_new;
      // this half's l catches up with m (an m of -inf leaves l = 0)
      l *= m_new == m_ref ? 1.f : ex2_approx(m_ref - base);
      m_ref = m_new;
      const float2 unit2 = make_float2(unit, unit), neg = make_float2(-base, -base);
      float2* x2 = reinterpret_cast<float2*>(x);
      float2 sum[2] = {};
      uint32_t pk[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        float2 p = fma2(x2[j], unit2, neg);
        p.x = ex2_approx(p.x);
        p.y = ex2_approx(p.y);
        sum[j & 1] = add2(sum[j & 1], p);
        pk[j] = pack_bf16x2(p.x, p.y);
        x2[j] = p;
      }
      const float2 both = add2(sum[0], sum[1]);
      l += both.x + both.y;
      if constexpr (kSpread) {
        mt_st_spread(s_row, pk, warp & 3);
      } else {
        tmem_st32_u(s_row, pk);
      }
      if (two_parts) {
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) {
          pk[j] = mt_low_part(x2[j], pk[j]);
        }
        if constexpr (kSpread) {
          mt_st_spread(s_row + kMtKeys / 2, pk, warp & 3);
        } else {
          tmem_st32_u(s_row + kMtKeys / 2, pk);
        }
      }
      tmem_wait_st();
      }
      // ---- V rows of keys in no document become zeros, whatever their memory holds
      if (entry & kMtPadded) {
        int n = m;  // the tile's place among the block's: its stage
        while ((all_tiles[n] & kMtTile) != (entry & kMtTile)) ++n;
        ok = mbar_wait(&v_full[n % NS], (n / NS) & 1, kErrWaitSoftmax, abort_flag);
        if (!ok) break;
        if (row < kMtKeys && a.kdoc[b * a.kdoc_sb + key0 - col0 + row] < 0)
          mt_zero_row<DP, kMtKeys>(sV + (n % NS) * L::kTile, row);
        fence_async_smem();
      }
      tc_fence_before();
      mbar_arrive(&p_full[NB * s + buf]);
    }
    const int m = count - 1;
    // ---- results: the halves' l on the last m, then half of the columns each
    // Both halves are done with the rows' m.  The half that did not take the last tile has not
    // seen its buffer's last phase, which the other half's scores came after: it waits behind it.
    tc_fence_before();
    named_barrier(1 + s, 256);
    tc_fence_after();
    if (m >= 0 && ok) {
      ok = mbar_wait(&pv_done[NB * s + m % NB], (m / NB) & 1, kErrWaitSoftmax, abort_flag);
      tc_fence_after();
    }
    if (m >= 0) {
      const float m_end = row_m[s * 128 + row];
      l *= m_end == m_ref || m_end == -INFINITY ? 1.f : ex2_approx(m_ref - m_end);
      m_ref = m_end;
    } else {
      row_m[s * 128 + row] = -INFINITY;  // no tile has set it
    }
    row_l[(2 * s + half) * 128 + row] = l;
    named_barrier(1 + s, 256);
    l += row_l[(2 * s + 1 - half) * 128 + row];
    float join = 1.f;  // of this lane's O and l, when four lanes have a row
    if constexpr (kSpread) {
      named_barrier(1 + s, 256);
      row_l[half * 128 + row] = l;
      named_barrier(1 + s, 256);
      const float* m4 = row_m + q_row;
      const float top = max_nan(max3_nan(m4[0], m4[32], m4[64]), m4[96]);
      const float base = top == -INFINITY ? 0.f : top;
      join = ex2_approx(m_ref - base);
      l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) l = fmaf(row_l[half * 128 + 32 * w + q_row], ex2_approx(m4[32 * w] - base), l);
      m_ref = top;
    }
    const int64_t index = (static_cast<int64_t>(b) * a.H + h) * a.nq + i;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int64_t part = split * (static_cast<int64_t>(a.B) * a.H * a.nq) + index;
    if (live && ok && half == 0 && row == q_row) {
      const float lse = l == 0.f ? -INFINITY : (m_ref + __log2f(l)) * 0.6931471805599453f;
      if (a.splits > 1) {
        a.part_lse[part] = lse;
      } else if (a.lse != nullptr) {
        a.lse[index] = lse;
      }
    }
    if constexpr (kSpread) {
      // the lanes' O side by side in the room of K and V, whose last reader is done
      constexpr int kPitch = DP + 4;
      float* all_o = reinterpret_cast<float*>(sK);
      if (ok) {
#pragma unroll
        for (int c = half * DP / 64; c < (half + 1) * DP / 64; ++c) {
          float o[32];
          if (m >= 0) {
            tmem_ld32_to(o_row + c * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (m >= 0 && inv != 0.f && join != 0.f)
              v = make_float4(o[e] * join * inv, o[e + 1] * join * inv, o[e + 2] * join * inv,
                              o[e + 3] * join * inv);
            *reinterpret_cast<float4*>(all_o + row * kPitch + c * 32 + e) = v;
          }
        }
      }
      named_barrier(1 + s, 256);
      for (int at = threadIdx.x; ok && at < nqt * a.rep * (DP / 4); at += 256) {
        const int r = at / (DP / 4), c = (at - r * (DP / 4)) * 4;
        const int qi = pair * nqt + r / a.rep, qh = g * a.rep + r % a.rep;
        if (c >= a.d || qi >= a.nq) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(all_o + (32 * w + r) * kPitch + c);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int64_t to_row = (static_cast<int64_t>(b) * a.H + qh) * a.nq + qi;
        if (a.splits > 1) {
          *reinterpret_cast<float4*>(
              a.part_o + (split * (static_cast<int64_t>(a.B) * a.H * a.nq) + to_row) * a.d + c) = v;
          continue;
        }
        const uint32_t w0 = pack_bf16x2(v.x, v.y), w1 = pack_bf16x2(v.z, v.w);
        *reinterpret_cast<uint2*>(ma_at<__nv_bfloat16>(a.out, b, qh, qi) + c) = make_uint2(w0, w1);
        if (a.low != nullptr)
          *reinterpret_cast<uint2*>(a.low + to_row * a.d + c) = make_uint2(
              pack_bf16x2(v.x - __uint_as_float(w0 << 16), v.y - __uint_as_float(w0 & 0xFFFF0000u)),
              pack_bf16x2(v.z - __uint_as_float(w1 << 16), v.w - __uint_as_float(w1 & 0xFFFF0000u)));
      }
    }
#pragma unroll
    for (int c = half * DP / 64; !kSpread && c < (half + 1) * DP / 64; ++c) {
      float o[32];
      if (m >= 0) {
        tmem_ld32_to(o_row + c * 32, o);
        tmem_wait_ld();
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = m >= 0 && inv != 0.f ? o[e] * inv : 0.f;
      if (!live || !ok) continue;
      if (a.splits > 1) {
        float* to = a.part_o + part * a.d + c * 32;
#pragma unroll
        for (int e = 0; e < 32; e += 4)  // d is a multiple of 8
          if (c * 32 + e < a.d)
            *reinterpret_cast<float4*>(to + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        continue;
      }
      __nv_bfloat16* to = ma_at<__nv_bfloat16>(a.out, b, h, i) + c * 32;
      __nv_bfloat16* low = a.low == nullptr ? nullptr : a.low + index * a.d + c * 32;
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        if (c * 32 + e >= a.d) continue;
        uint32_t w[4], r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float u = o[e + 2 * q], v = o[e + 2 * q + 1];
          w[q] = pack_bf16x2(u, v);
          r[q] = pack_bf16x2(u - __uint_as_float(w[q] << 16),
                             v - __uint_as_float(w[q] & 0xFFFF0000u));
        }
        *reinterpret_cast<uint4*>(to + e) = make_uint4(w[0], w[1], w[2], w[3]);
        if (low != nullptr) *reinterpret_cast<uint4*>(low + e) = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  }

  mt_drain(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == L::kControl) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------- backward
//
// One kernel body makes dq (KV = false) and dk, dv (KV = true).  A block keeps two 128-row
// operands X0, X1 in shared memory and streams tiles of 64 rows Y0, Y1 past them:
//            X0   X1    Y0   Y1     S = X0 Y0^T        dP = X1 Y1^T      results
//   dq       q    do    k    v      rows x keys                          dq += dX Y0
//   dk, dv   k    v     q    do     keys x rows (S^T)  (dP^T)            dk += dX^T Y0, dv += P^T Y1
// so P and dX always are the left operand of the next product and go to it through TMEM.  Two
// pairs of warpgroups take tiles in turn, a warpgroup of a pair half of the columns each (half
// the columns halve the longest link of the chain from a tile's products to its P and dX); one
// issuer warp feeds them (front), another adds up the results (back).  S and dP are free for
// the next tile as soon as the pair has them in registers, and P and dX have two buffers of
// their own.
// The dq kernel runs first and also makes D_i = do_i . o_i for both, as the diagonal of O dO^T:
// the same product as dP, so a row that sees one key alone (o = v) has dP - D = 0 but for what the
// saved residual of o holds (2^-22 of it).
// A tile is 64 wide so that S, dP, two P and dX and two 128-column sums fit the 512 columns.
// Measured at 8192 causal tokens, 16 heads on 4: dq 1000 TFLOP/s at head dim 128 and 660 at 64 (three
// products), dk and dv 1130 and 640 (four); bound by the handoffs between a tile's products
// and its P and dX, with the tensor pipe 47 to 59 % busy at 128 and 30 to 32 % at 64.

constexpr int kMtStream = 64;  // streamed rows a tile

// Stores 16 consecutive TMEM columns of this thread's lane from raw words.
__device__ __forceinline__ void mt_st16(uint32_t taddr, const uint32_t* v) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// What a column (a row of q) of a dk, dv tile needs; one set a stage.
struct MtColumns {
  float neg_lse2[kMtStream];  // log2 units; -inf for a row that sees no key
  float neg_delta[kMtStream];
  float slope2[kMtStream];
  float pos[kMtStream];
  int limit[kMtStream];
  int doc[kMtStream];
  uint32_t dead[2];        // rows that see no key, a bit each
  uint32_t unused[2];
};

template <int DP>
struct MtBackward {
  static constexpr int kX = 128 * DP * 2;
  static constexpr int kY = kMtStream * DP * 2;
  static constexpr int kStages = 3;
  static constexpr int kYOff = 2 * kX;
  static constexpr int kColOff = kYOff + kStages * 2 * kY;
  static constexpr int kBarOff = kColOff + kStages * int(sizeof(MtColumns));
  static constexpr int kBars = 1 + 3 * kStages + 8 + 1 + 2;
  static_assert(2 * kY == kX, "o takes one stage's room");
  static_assert(kStages * sizeof(MtColumns) >= 4 * 128 * 4, "the parts of D take the columns' room");
  static constexpr int kBytes = kBarOff + kBars * 8 + 16;
  static constexpr int kListOff = kBytes;  // the list, as long as the call needs it
  static constexpr int launch_bytes(int64_t tiles) {
    return kListOff + static_cast<int>(tiles) * 4 + 1024;
  }
  static constexpr int kMostBytes = launch_bytes(kMtMaxStream);
  static constexpr int kControl = 16;  // first control warp: loader, front, back, columns
  static constexpr int kThreads = 640;
  // as in the forward kernel: 512 * 104 + 128 * 64 = 640 * 96
  static constexpr int kRegsMath = 104, kRegsOther = 64;
  static_assert(kMostBytes <= 232448, "shared memory exceeds 227 KB");
};

// With TWO, P and dX go in two bf16 parts, as P does in the forward pass, and take both buffers: for
// short sequences, where a block has a few tiles and waits on its start and end, so that the
// further products are free.  The error of dq, dk and dv is then that of a result rounded once;
// in one part it is sqrt(2) times that, whatever the length of rows and documents (1.41 to 1.42
// measured with documents of 2 to 4096 tokens).  Two parts in every block of few tiles, chosen in
// the kernel, took 3 to 5 % more on packed rows and 3 % where no block is short.
template <int DP, bool KV, bool CAP, bool SLOPES, bool TWO>
__global__ void __launch_bounds__(MtBackward<DP>::kThreads, 1)
    mt_backward_kernel(const __grid_constant__ CUtensorMap tmX0,
                       const __grid_constant__ CUtensorMap tmX1,
                       const __grid_constant__ CUtensorMap tmY0,
                       const __grid_constant__ CUtensorMap tmY1,
                       const __grid_constant__ CUtensorMap tmO, const MtMap mk, const MtMap mv,
                       const __grid_constant__ MaskedArgs a) {
  using L = MtBackward<DP>;
  constexpr int NS = L::kStages;
  constexpr uint32_t kIdescS = idesc_bf16(128, kMtStream, false, false);
  constexpr uint32_t kIdescG = idesc_bf16(128, DP, false, true);
  // TMEM columns: S and dP (one buffer where two sums of 128 leave no more), two of P and dX,
  // the sums
  constexpr int NB = KV && DP == 128 ? 1 : 2;
  constexpr uint32_t kDpCol = kMtStream, kGCol = NB * 2 * kMtStream;
  constexpr uint32_t kSum0 = kGCol + 2 * kMtStream, kSum1 = kSum0 + DP;
  static_assert((KV ? kSum1 : kSum0) + (KV ? DP : 128) <= 512, "TMEM has 512 columns");
  constexpr uint32_t kTmemCols = 512;
  // !KV: o waits in the last stage for its product with do, which goes to the columns of the sums
  constexpr int kOStage = NS - 1;
  constexpr uint32_t kIdescD = idesc_bf16(128, 128, false, false);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sX0 = smem;
  uint8_t* sX1 = smem + L::kX;
  uint8_t* sY = smem + L::kYOff;  // stage: Y0, Y1
  MtColumns* columns = reinterpret_cast<MtColumns*>(smem + L::kColOff);
  uint32_t* list = reinterpret_cast<uint32_t*>(smem + L::kListOff);
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* y_full = x_full + 1;
  uint64_t* y_empty = y_full + NS;
  uint64_t* col_full = y_empty + NS;
  // of each pair's tiles:
  uint64_t* s_full = col_full + NS;  // [2] S and dP are in TMEM
  uint64_t* s_free = s_full + 2;     // [2] they are in registers
  uint64_t* g_full = s_free + 2;     // [2] P and dX are in TMEM
  uint64_t* g_free = g_full + 2;     // [2] their products are done
  uint64_t* all_done = g_free + 2;
  uint64_t* d_done = all_done + 1;   // !KV: O dO^T is made, its shared memory free
  uint64_t* d_read = d_done + 1;     // !KV: every thread has its D
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_read + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* list_count = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---- the block's X rows, and the tiles of Y rows
  const int nqx = 128 / a.rep;         // queries of a 128-row tile
  const int nqy = kMtStream / a.rep;   // queries of a streamed tile
  int item = blockIdx.x;
  const int g = item % a.G;
  item /= a.G;
  const int b = item % a.B;
  item /= a.B;
  const int prefix = ma_prefix(a, b);
  const bool docs = a.qdoc != nullptr;
  // KV: key tiles in order (the first are seen by most rows); rows: the last first
  const int x_tile = KV ? item : a.q_tiles - 1 - item;
  const int key0_x = x_tile * 128;     // KV
  const int i0_x = x_tile * nqx;       // !KV
  const int i1_x = min(i0_x + nqx, a.nq) - 1;
  const int y_tiles = KV ? (a.nq + nqy - 1) / nqy : (a.nk + kMtStream - 1) / kMtStream;
  // the causal mask cuts the tiles at one end: the first query that sees key0_x, or the last
  // key that query i1_x sees
  const int first = KV && a.causal && key0_x >= prefix ? max(0, key0_x - a.off) / nqy : 0;
  const int last = KV ? y_tiles
                      : min(y_tiles, (max(0, ma_limit(a, i1_x, prefix)) + kMtStream - 1) / kMtStream);
  const int tiles = max(0, last - first);

  if (threadIdx.x == 0) {
    mbar_init(x_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&y_full[i], 1);
      mbar_init(&y_empty[i], 1);
      mbar_init(&col_full[i], 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 256);
      mbar_init(&g_full[i], 256);
      mbar_init(&g_free[i], 1);
    }
    mbar_init(all_done, 1);
    mbar_init(d_done, 1);
    mbar_init(d_read, 512);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == L::kControl) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // rows past the boxes' rep * queries are zeros
  if constexpr (KV) {
    mt_zero_tail_rows<DP, kMtStream, L::kThreads>(sY, NS * 2, nqy * a.rep);
  } else {
    mt_zero_tail_rows<DP, 128, L::kThreads>(sX0, 2, nqx * a.rep);
    mt_zero_tail_rows<DP, 128, L::kThreads>(sY + kOStage * 2 * L::kY, 1, nqx * a.rep);
  }
  // ---- the list
  if (warp == 0) {
    int4 xr = make_int4(0, 0, 0, 0);
    if (docs) {
      xr = KV ? ma_join_ranges(a.krange + b * a.krange_sb, 2 * x_tile, 2 * x_tile + 1)
              : ma_join_ranges(a.qrange + b * a.qrange_sb, i0_x / 64, i1_x / 64);
    }
    const int count = mt_compact(list, tiles, [&](int t) -> uint32_t {
      const int i_lo = KV ? (first + t) * nqy : i0_x;
      const int i_hi = KV ? min(i_lo + nqy, a.nq) - 1 : i1_x;
      const int key_lo = KV ? key0_x : (first + t) * kMtStream;
      const int key_hi = key_lo + (KV ? 128 : kMtStream);
      if (key_lo >= ma_limit(a, i_hi, prefix)) return 0u;
      bool masked = key_hi > ma_limit(a, i_lo, prefix);
      uint32_t pad = 0u;
      if (docs) {
        const int4 yr = KV ? ma_join_ranges(a.qrange + b * a.qrange_sb, i_lo / 64, i_hi / 64)
                           : a.krange[b * a.krange_sb + first + t];
        if (!ma_ranges_meet(xr, yr)) return 0u;
        masked = masked || xr.z || yr.z || xr.x != xr.y || yr.x != yr.y;
        pad = yr.z ? kMtPadded : 0u;
      }
      return kMtListed | t | (masked ? kMtMasked : 0u) | pad;
    });
    if (lane == 0) *list_count = count;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int count = *list_count;
  const uint32_t x0_addr = smem_u32(sX0), x1_addr = smem_u32(sX1), y_addr = smem_u32(sY);

  if (warp >= L::kControl) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRegsOther));
    if (warp == L::kControl && lane == 0) {
      // ------------------------------------------------ TMA loader
      if constexpr (KV) {
        mbar_arrive_expect_tx(x_full, 2 * L::kX);
        mt_load_keys<DP, 128>(sX0, &tmX0, x_full, key0_x, g * mk.head, b * mk.batch);
        mt_load_keys<DP, 128>(sX1, &tmX1, x_full, key0_x, g * mv.head, b * mv.batch);
      } else {
        mbar_arrive_expect_tx(x_full, 3 * (DP / 64) * 128 * a.rep * nqx);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          tma_load_5d(sX0 + c * 16384, &tmX0, x_full, c * 64, 0, i0_x, g, b);
          tma_load_5d(sX1 + c * 16384, &tmX1, x_full, c * 64, 0, i0_x, g, b);
          tma_load_5d(sY + kOStage * 2 * L::kY + c * 16384, &tmO, x_full, c * 64, 0, i0_x, g, b);
        }
      }
      for (int n = 0; n < count; ++n) {
        const int t = list[n] & kMtTile;
        const int st = n % NS;
        if (!mbar_wait(&y_empty[st], ((n / NS) & 1) ^ 1, kErrWaitProducer, abort_flag)) break;
        if (!KV && n == kOStage && !mbar_wait(d_done, 0, kErrWaitProducer, abort_flag)) break;
        uint8_t* y0 = sY + st * 2 * L::kY;
        uint8_t* y1 = y0 + L::kY;
        if constexpr (KV) {
          mbar_arrive_expect_tx(&y_full[st], 2 * (DP / 64) * 128 * a.rep * nqy);
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_5d(y0 + c * 8192, &tmY0, &y_full[st], c * 64, 0, (first + t) * nqy, g, b);
            tma_load_5d(y1 + c * 8192, &tmY1, &y_full[st], c * 64, 0, (first + t) * nqy, g, b);
          }
        } else {
          mbar_arrive_expect_tx(&y_full[st], 2 * L::kY);
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_4d(y0 + c * 8192, &tmY0, &y_full[st], c * 64, (first + t) * kMtStream,
                        g * mk.head, b * mk.batch);
            tma_load_4d(y1 + c * 8192, &tmY1, &y_full[st], c * 64, (first + t) * kMtStream,
                        g * mv.head, b * mv.batch);
          }
        }
      }
    } else if (warp == L::kControl + 1) {
      // ------------------------------------------------ front: S and dP
      if (mbar_wait(x_full, 0, kErrWaitMma, abort_flag)) {
        if constexpr (!KV) {
          tc_fence_after();
          const uint32_t o_addr = y_addr + kOStage * 2 * L::kY;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            mt_mma(tmem_base + kSum0, mt_k_desc(o_addr, k, 16384), mt_k_desc(x1_addr, k, 16384),
                      kIdescD, k > 0 ? 1u : 0u);
          mt_commit(d_done);
        }
        for (int n = 0; n < count; ++n) {
          const int st = n % NS;
          const uint32_t s_tmem = tmem_base + (n % NB) * 2 * kMtStream;
          if (!mbar_wait(&y_full[st], (n / NS) & 1, kErrWaitMma, abort_flag)) break;
          // the buffer's last tile, n - NB
          if (n >= NB && !mbar_wait(&s_free[(n - NB) & 1], ((n - NB) >> 1) & 1, kErrWaitMma, abort_flag))
            break;
          tc_fence_after();
          const uint32_t y0 = y_addr + st * 2 * L::kY, y1 = y0 + L::kY;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            mt_mma(s_tmem, mt_k_desc(x0_addr, k, 16384),
                      mt_k_desc(y0, k, 8192), kIdescS, k > 0 ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            mt_mma(s_tmem + kDpCol, mt_k_desc(x1_addr, k, 16384),
                      mt_k_desc(y1, k, 8192), kIdescS, k > 0 ? 1u : 0u);
          mt_commit(&s_full[n & 1]);
        }
      }
    } else if (warp == L::kControl + 2) {
      // ------------------------------------------------ back: the sums
      const bool ready = KV || mbar_wait(d_read, 0, kErrWaitMma, abort_flag);
      for (int n = 0; ready && n < count; ++n) {
        const int st = n % NS, buf = n & 1;
        if (!mbar_wait(&g_full[buf], (n >> 1) & 1, kErrWaitMma, abort_flag)) break;
        tc_fence_after();
        const uint32_t y0 = y_addr + st * 2 * L::kY, y1 = y0 + L::kY;
        const uint32_t p = tmem_base + kGCol + (TWO ? 0 : buf) * kMtStream;
        const uint32_t dx = p + kMtStream / 2;
        if constexpr (KV) {
#pragma unroll
          for (int k = 0; k < kMtStream / 16; ++k)
            mt_mma_ts(tmem_base + kSum1, p + 8 * k, mt_mn_desc(y1, k, 8192), kIdescG,
                         n > 0 || k > 0 ? 1u : 0u);
        }
#pragma unroll
        for (int k = 0; k < kMtStream / 16; ++k)
          mt_mma_ts(tmem_base + kSum0, dx + 8 * k, mt_mn_desc(y0, k, 8192), kIdescG,
                       n > 0 || k > 0 ? 1u : 0u);
        if constexpr (TWO) {
#pragma unroll
          for (int k = 0; k < kMtStream / 16; ++k) {
            if (KV)
              mt_mma_ts(tmem_base + kSum1, p + kMtStream + 8 * k, mt_mn_desc(y1, k, 8192), kIdescG, 1u);
            mt_mma_ts(tmem_base + kSum0, dx + kMtStream + 8 * k, mt_mn_desc(y0, k, 8192), kIdescG, 1u);
          }
        }
        mt_commit(&g_free[buf]);
        mt_commit(&y_empty[st]);
      }
      if (count > 0) mt_commit(all_done);
    } else if (warp == L::kControl + 3 && KV) {
      // ------------------------------------------------ what the columns need
      // A tile's numbers are loaded before the wait for its stage, so that the loads' latency
      // is spent beside it.
      float lse[2], del[2], slope[2];
      int head[2], shift[2], doc[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = 32 * e + lane;
        shift[e] = c / a.rep;
        head[e] = g * a.rep + c % a.rep;
        slope[e] = SLOPES ? a.slopes[head[e]] * kLog2e : 0.f;
      }
      const auto fetch = [&](int n) {
        const int i0 = (first + (list[n] & kMtTile)) * nqy;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = i0 + shift[e];
          const bool live = shift[e] < nqy && i < a.nq;
          const int64_t index = (static_cast<int64_t>(b) * a.H + head[e]) * a.nq + i;
          lse[e] = live ? a.lse[index] : -INFINITY;
          del[e] = live ? a.delta[index] : 0.f;
          doc[e] = docs && live ? a.qdoc[b * a.qdoc_sb + i] : -1;
        }
      };
      if (count > 0) fetch(0);
      for (int n = 0; n < count; ++n) {
        const int i0 = (first + (list[n] & kMtTile)) * nqy;
        const int st = n % NS;
        if (!mbar_wait(&y_empty[st], ((n / NS) & 1) ^ 1, kErrWaitProducer, abort_flag)) break;
        MtColumns& col = columns[st];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 32 * e + lane;
          const int i = i0 + shift[e];
          const bool dead = lse[e] == -INFINITY;
          col.neg_lse2[c] = dead ? -INFINITY : -lse[e] * kLog2e;
          col.neg_delta[c] = dead ? 0.f : -del[e];
          col.slope2[c] = slope[e];
          col.pos[c] = static_cast<float>(i + a.off);
          col.limit[c] = dead ? 0 : ma_limit(a, i, prefix);
          col.doc[c] = doc[e] < 0 ? -2 : doc[e];  // padding does not see padding
          const uint32_t bits = __ballot_sync(0xffffffffu, dead && shift[e] < nqy);
          if (lane == 0) col.dead[e] = bits;
        }
        mbar_arrive(&col_full[st]);
        if (n + 1 < count) fetch(n + 1);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRegsMath));
    // ------------------------------------------------ P and dX: one X row a thread
    const int wg = warp >> 3, half = (warp >> 2) & 1;  // tiles wg, wg + 2, ...; columns half * 32...
    const int row = threadIdx.x & 127;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float unit = a.scale * kLog2e;
    const float2 unit2 = make_float2(unit, unit);
    // the row's own numbers: a key (KV) or a row of q
    const int key = key0_x + row;
    const int i = i0_x + row / a.rep;
    const int h = g * a.rep + row % a.rep;
    const bool live = KV ? key < a.nk : row < nqx * a.rep && i < a.nq;
    const int64_t index = (static_cast<int64_t>(b) * a.H + h) * a.nq + i;
    float lse2 = 0.f, delta = 0.f, slope2 = 0.f;
    const float own_pos = static_cast<float>(KV ? key : i + a.off);
    int limit = 0, doc = -1;
    bool dead = false;
    if constexpr (KV) {
      if (docs) doc = a.kdoc[b * a.kdoc_sb + key];
    } else {
      const float lse = live ? a.lse[index] : -INFINITY;
      dead = lse == -INFINITY;
      lse2 = dead ? INFINITY : lse * kLog2e;
      slope2 = live && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
      limit = dead ? 0 : ma_limit(a, i, prefix);
      if (docs && live) doc = a.qdoc[b * a.qdoc_sb + i];
      if (doc < 0) doc = -2;
    }
    bool ok = true;
    if constexpr (!KV) {
      // D: the row's own column of O dO^T, and the part of o that its rounding took away
      ok = mbar_wait(d_done, 0, kErrWaitSoftmax, abort_flag);
      tc_fence_after();
      float own[32];
      tmem_ld32_to(t_row + kSum0 + (warp & 3) * 32, own);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (e == lane) delta = own[e];
      tc_fence_before();
      mbar_arrive(d_read);
      // a quarter of the columns a warpgroup, all its loads in flight at once
      float rest = 0.f;
      if (live) {
        const uint4* low = reinterpret_cast<const uint4*>(a.low + index * a.d);
        const uint4* dout = reinterpret_cast<const uint4*>(ma_at<__nv_bfloat16>(a.dout, b, h, i));
        uint4 lw[DP / 32], dw[DP / 32];
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) {
          const int c = (warp >> 2) * (DP / 32) + e;
          const bool in = c * 8 < a.d;
          lw[e] = in ? low[c] : make_uint4(0u, 0u, 0u, 0u);
          dw[e] = in ? dout[c] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) {
          float u[8], v[8];
          unpack8_bf16(lw[e], u);
          unpack8_bf16(dw[e], v);
#pragma unroll
          for (int q = 0; q < 8; ++q) rest = fmaf(u[q], v[q], rest);
        }
      }
      float* rests = reinterpret_cast<float*>(columns);  // [4][128]; dq has no columns
      rests[(warp >> 2) * 128 + row] = rest;
      named_barrier(1, 512);
      delta += (rests[row] + rests[128 + row]) + (rests[256 + row] + rests[384 + row]);
      if (dead) delta = 0.f;
      if (warp < 4 && live) a.delta[index] = delta;
    }
    for (int n = wg; n < count; n += 2) {
      const uint32_t entry = list[n];
      const int t = entry & kMtTile;
      const int st = n % NS;
      const int key0 = (first + t) * kMtStream + 32 * half;  // !KV
      const int32_t* kdoc = !KV && docs ? a.kdoc + b * a.kdoc_sb + key0 : nullptr;
      const MtColumns& col = columns[st];
      if (KV) ok = mbar_wait(&col_full[st], (n / NS) & 1, kErrWaitSoftmax, abort_flag);
      ok = ok && mbar_wait(&s_full[wg], (n >> 1) & 1, kErrWaitSoftmax, abort_flag);
      if (!ok) break;
      tc_fence_after();
      constexpr int kCols = kMtStream / 2;
      float s[kCols], dp[kCols];
      const int col0 = 32 * half;
      const uint32_t s_row = t_row + (n % NB) * 2 * kMtStream + col0;
      const uint32_t dp_row = s_row + kDpCol;
      const uint32_t p_row = t_row + kGCol + (TWO ? 0 : wg) * kMtStream + 16 * half;
      // ---- p and dx are 0 where the row does not see the column, whatever it holds
      bool masks = (entry & kMtMasked) || dead;
      if (KV) masks = masks || (col.dead[0] | col.dead[1]) != 0;
      if (__any_sync(0xffffffffu, masks)) {
        mt_mask_tmem<true, kCols, false>(s_row, dp_row, 0.f, 0.f, [&](int j, bool (&off)[4]) {
          int4 lim = make_int4(limit, limit - 1, limit - 2, limit - 3), id = make_int4(doc, doc, doc, doc);
          if constexpr (KV) {
            lim = *reinterpret_cast<const int4*>(&col.limit[col0 + j]);
            if (docs) id = *reinterpret_cast<const int4*>(&col.doc[col0 + j]);
          } else {
            if (docs) id = *reinterpret_cast<const int4*>(kdoc + j);
          }
          const int at = KV ? key : key0 + j;
          off[0] = at >= lim.x || id.x != doc;
          off[1] = at >= lim.y || id.y != doc;
          off[2] = at >= lim.z || id.z != doc;
          off[3] = at >= lim.w || id.w != doc;
        });
      }
      tmem_ld32_to(s_row, s);
      tmem_ld32_to(dp_row, dp);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&s_free[wg]);
      // ---- s <- log2 p, dp <- (dp - D) (1 - tanh^2)
      float2* s2 = reinterpret_cast<float2*>(s);
      float2* dp2 = reinterpret_cast<float2*>(dp);
      const float2 own_lse = make_float2(-lse2, -lse2), own_delta = make_float2(-delta, -delta);
#pragma unroll
      for (int j = 0; j < kCols / 2; j += 2) {
        float2 l2[2] = {own_lse, own_lse}, d2[2] = {own_delta, own_delta};
        if constexpr (KV) {
          const float4 lw = *reinterpret_cast<const float4*>(&col.neg_lse2[col0 + 2 * j]);
          const float4 dw = *reinterpret_cast<const float4*>(&col.neg_delta[col0 + 2 * j]);
          l2[0] = make_float2(lw.x, lw.y), l2[1] = make_float2(lw.z, lw.w);
          d2[0] = make_float2(dw.x, dw.y), d2[1] = make_float2(dw.z, dw.w);
        }
        float sl[4], dist[4];
        if constexpr (SLOPES) {
          if constexpr (KV) {
            const float4 sw = *reinterpret_cast<const float4*>(&col.slope2[col0 + 2 * j]);
            const float4 pw = *reinterpret_cast<const float4*>(&col.pos[col0 + 2 * j]);
            sl[0] = sw.x, sl[1] = sw.y, sl[2] = sw.z, sl[3] = sw.w;
            dist[0] = pw.x - own_pos, dist[1] = pw.y - own_pos, dist[2] = pw.z - own_pos,
            dist[3] = pw.w - own_pos;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sl[e] = slope2;
              dist[e] = (own_pos - static_cast<float>(key0)) - static_cast<float>(2 * j + e);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float2 d = add2(dp2[j + e], d2[e]);
          float2 z;
          if constexpr (CAP) {
            // with r as in mt_capped: tanh = 1 - 2 r, 1 - tanh^2 = 4 r (1 - r)
            const float k = 2.f * unit * a.inv_cap, c = a.cap * kLog2e;
            const float2 r = make_float2(mt_cap_part(s2[j + e].x * k), mt_cap_part(s2[j + e].y * k));
            const float2 bend = fma2(mul2(r, make_float2(-4.f, -4.f)), r,
                                     mul2(r, make_float2(4.f, 4.f)));
            d = mul2(d, bend);
            z = add2(make_float2(mt_capped(s2[j + e].x, r.x, c), mt_capped(s2[j + e].y, r.y, c)), l2[e]);
          } else {
            z = fma2(s2[j + e], unit2, l2[e]);
          }
          if constexpr (SLOPES) {
            z.x = fmaf(-sl[2 * e], fabsf(dist[2 * e]), z.x);
            z.y = fmaf(-sl[2 * e + 1], fabsf(dist[2 * e + 1]), z.y);
          }
          s2[j + e] = z;
          dp2[j + e] = d;
        }
      }
      uint32_t pk[kCols / 2], dk[kCols / 2];
      uint32_t pk_low[TWO ? kCols / 2 : 1], dk_low[TWO ? kCols / 2 : 1];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        const float2 p = make_float2(ex2_approx(s2[j].x), ex2_approx(s2[j].y));
        const float2 x = mul2(p, dp2[j]);
        pk[j] = pack_bf16x2(p.x, p.y);
        dk[j] = pack_bf16x2(x.x, x.y);
        if constexpr (TWO) {
          pk_low[j] = mt_low_part(p, pk[j]);
          dk_low[j] = mt_low_part(x, dk[j]);
        }
      }
      // the products that read what the columns held: those of the pair's last tile, or of the last
      constexpr int kBack = TWO ? 1 : 2;
      if (n >= kBack) {
        ok = mbar_wait(&g_free[(n - kBack) & 1], ((n - kBack) >> 1) & 1, kErrWaitSoftmax, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      if constexpr (KV) mt_st16(p_row, pk);
      mt_st16(p_row + kMtStream / 2, dk);
      if constexpr (TWO) {
        if constexpr (KV) mt_st16(p_row + kMtStream, pk_low);
        mt_st16(p_row + kMtStream + kMtStream / 2, dk_low);
      }
      tmem_wait_st();
      // ---- streamed rows that no row may see become zeros, whatever their memory holds: a
      // zero of P or dX would not hide a NaN there from the products
      bool wrote = false;
      uint8_t* y0 = sY + st * 2 * L::kY;
      if constexpr (KV) {
        const int r = row & 63;
        if (half == 0 && ((col.dead[r >> 5] >> (r & 31)) & 1u)) {
          mt_zero_row<DP, kMtStream>(row < 64 ? y0 : y0 + L::kY, r);
          wrote = true;
        }
      } else {
        // (this warpgroup's 32 keys; kdoc starts there)
        if ((entry & kMtPadded) && row < kCols && kdoc[row] < 0) {
          mt_zero_row<DP, kMtStream>(y0, col0 + row);
          wrote = true;
        }
      }
      if (wrote) fence_async_smem();
      tc_fence_before();
      mbar_arrive(&g_full[wg]);
    }
    // ---- results: dq 32 columns a warpgroup; dk by the first pair, dv by the second
    const bool any = count > 0;
    if (any && ok) {
      ok = mbar_wait(all_done, 0, kErrWaitSoftmax, abort_flag);
      tc_fence_after();
    }
    const uint32_t sum = t_row + (!KV || wg == 0 ? kSum0 : kSum1);
    const float factor = !KV || wg == 0 ? a.scale : 1.f;
    const MaTensor& dst = KV ? (wg == 0 ? a.dk : a.dv) : a.dq;
    __nv_bfloat16* to = live ? (KV ? ma_at<__nv_bfloat16>(dst, b, g, key)
                                   : ma_at<__nv_bfloat16>(dst, b, h, i))
                             : nullptr;
#pragma unroll 1
    for (int c = KV ? half : 2 * wg + half; c < DP / 32; c += KV ? 2 : 4) {
      float o[32];
      if (any) {
        tmem_ld32_to(sum + c * 32, o);
        tmem_wait_ld();
      }
      if (!live || !ok) continue;
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        if (c * 32 + e >= a.d) continue;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          w[q] = any ? pack_bf16x2(o[e + 2 * q] * factor, o[e + 2 * q + 1] * factor) : 0u;
        *reinterpret_cast<uint4*>(to + c * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }

  mt_drain(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == L::kControl) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace xfb
