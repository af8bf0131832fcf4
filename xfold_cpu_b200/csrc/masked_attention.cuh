// Masked attention with its backward pass: arguments, masks and the CUDA-core kernels.
//
//   x_ij = scale q_i . k_j                    query i stands at position i + nk - nq
//   s_ij = cap tanh(x_ij / cap) - slope_h |i + nk - nq - j|      (cap 0: s = x - ...)
//   j is visible to i when it is not past i (causal), or lies in the batch row's prefix,
//     and belongs to the same document (ids equal and not negative)
//   p_ij = softmax over the visible j,  o_i = sum_j p_ij v_j,  lse_i = log sum_j exp s_ij
//   a row that sees no key: o = 0, lse = -inf, gradients 0
//
//   backward  D_i = do_i . o_i,  dp_ij = do_i . v_j
//             dx_ij = p_ij (dp_ij - D_i) (1 - tanh^2(x_ij / cap))
//             dv_j = sum_i p_ij do_i,  dk_j = scale sum_i dx_ij q_i,  dq_i = scale sum_j dx_ij k_j
//
// The `rep` query heads that share a K/V head are one set of rows: row r of (b, g) is
// query r / rep of head g rep + r % rep.  So K and V are read once for the group, a
// single new token still fills rep rows of a tile, and dk, dv sum over the group's
// heads inside one block, without atomics: the results do not depend on scheduling.
//
// Two kernels make the gradients: one block owns keys and adds up dk, dv over the rows;
// one owns rows and adds up dq over the keys.  That computes s and dp twice (7
// products in place of 5) and needs neither atomics nor an order between blocks.
//
// This file: the CUDA-core kernels (f32 inputs, and what the tensor-core
// kernels do not take), the document ranges, D and the joining of key splits.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "layer_norm_train.cuh"  // ln_float, ln_round

namespace xfb {

// One [B][heads][n][d] tensor: strides in elements, the head dim contiguous.
struct MaTensor {
  void* p;
  int64_t sb, sh, sn;
};

struct MaskedArgs {
  MaTensor q, k, v, out, dout, dq, dk, dv;
  float* lse;            // [B][H][nq], or null
  __nv_bfloat16* low;    // [B][H][nq][d]: what rounding took from bf16 `out`, or null
  float* delta;          // [B][H][nq]: D
  const float* slopes;   // [H], or null
  const int32_t* prefix; // [B], or null
  // documents, padded with -1 to whole 128-token tiles, or null; batch strides (0: shared)
  const int32_t* qdoc;
  const int32_t* kdoc;
  int64_t qdoc_sb, kdoc_sb;
  const int4* qrange;    // {lowest, highest id >= 0, any token of none, 0} of each 64 tokens
  const int4* krange;
  int64_t qrange_sb, krange_sb;
  int B, H, G, rep, nq, nk, d, off;
  int causal;
  float scale, cap, inv_cap;
  int q_tiles, k_tiles, splits;
  float* part_o;         // [splits][B * H * nq][d], when splits > 1
  float* part_lse;       // [splits][B * H * nq]
  int vec4;              // rows of every tensor can be read four values at a time
};

// ---------------------------------------------------------------- masks

// Keys below this index are not hidden from query i by the causal and prefix masks.
__device__ __forceinline__ int ma_limit(const MaskedArgs& a, int i, int prefix) {
  return a.causal ? min(a.nk, max(i + a.off + 1, prefix)) : a.nk;
}
__device__ __forceinline__ int ma_prefix(const MaskedArgs& a, int b) {
  return a.prefix != nullptr ? a.prefix[b] : 0;
}

// Ids of the 64-token ranges first..last joined.
__device__ __forceinline__ int4 ma_join_ranges(const int4* r, int first, int last) {
  int4 j = r[first];
  for (int t = first + 1; t <= last; ++t) {
    const int4 n = r[t];
    j.x = min(j.x, n.x);
    j.y = max(j.y, n.y);
    j.z |= n.z;
  }
  return j;
}
__device__ __forceinline__ bool ma_ranges_meet(int4 q, int4 k) {
  return max(q.x, k.x) <= min(q.y, k.y);
}

// Padded copy of the document ids and the ids' range of each 64 tokens; one warp a
// range, grid (ranges / 8, batch rows, q or k).
struct MaDocs {
  const int32_t* in[2];
  int64_t in_sb[2];
  int n[2];
  int32_t* out[2];
  int64_t out_sb[2];
  int4* range[2];
  int64_t range_sb[2];
};
__global__ void __launch_bounds__(256) ma_documents_kernel(MaDocs a) {
  const int w = blockIdx.z, b = blockIdx.y, lane = threadIdx.x & 31;
  const int range = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int start = range * 64;
  if (start >= a.out_sb[w]) return;  // the longer of q and k sets the grid
  int lo = INT_MAX, hi = -1, pad = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = start + 32 * e + lane;
    int id = i < a.n[w] ? a.in[w][b * a.in_sb[w] + i] : -1;
    if (id < 0) {
      id = -1;
      pad |= i < a.n[w];  // past the end there is nothing to hide: no row, a key no limit lets in
    } else {
      lo = min(lo, id);
      hi = max(hi, id);
    }
    a.out[w][b * a.out_sb[w] + i] = id;
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  pad = __any_sync(0xffffffffu, pad);
  if (lane == 0) a.range[w][b * a.range_sb[w] + range] = make_int4(lo, hi, pad, 0);
}

// 64-bit ids made 32-bit ones: a document's number is the place of its first token among the
// row's keys and then its queries, so equal ids keep equal numbers, other ids other ones, and
// the numbers of documents in order are in order, as the ranges want them.  A hash table of at
// least twice as many entries as tokens holds (id, first place); only the first token of a
// run of equal ids enters it, and the least place is the same whatever order they come in.
struct MaIds {
  const int64_t* q;
  const int64_t* k;
  int64_t q_sb, k_sb;
  int nq, nk;
  int32_t* q_out;             // [B][nq]
  int32_t* k_out;             // [B][nk]
  unsigned long long* ids;    // [B][2^bits], all ones: empty (no id, ids are not negative)
  uint32_t* first;            // [B][2^bits], all ones at the start
  int bits;
};
__device__ __forceinline__ int64_t ma_id(const MaIds& a, int b, int64_t at) {
  return at < a.nk ? a.k[b * a.k_sb + at] : a.q[b * a.q_sb + at - a.nk];
}
// The entry of an id: its own, or the first empty one on its way, which ENTER claims.
template <bool ENTER>
__device__ __forceinline__ int64_t ma_id_entry(const MaIds& a, int b, int64_t id) {
  const int64_t size = int64_t(1) << a.bits;
  unsigned long long* ids = a.ids + b * size;
  const auto key = static_cast<unsigned long long>(id);
  // the product's high bits spread neighbouring ids (the multiplier is 2^64 over the golden ratio)
  int64_t e = static_cast<int64_t>((key * 0x9E3779B97F4A7C15ull) >> (64 - a.bits));
  for (int64_t tries = 0; tries < size; ++tries, e = (e + 1) & (size - 1)) {
    const unsigned long long there = ENTER ? atomicCAS(ids + e, ~0ull, key) : ids[e];
    if (there == key || (ENTER && there == ~0ull)) break;
  }
  return b * size + e;
}
__global__ void __launch_bounds__(256) ma_ids_enter_kernel(MaIds a) {
  const int b = blockIdx.y;
  const int64_t n = int64_t(a.nk) + a.nq;
  for (int64_t at = blockIdx.x * 256 + threadIdx.x; at < n; at += gridDim.x * 256) {
    const int64_t id = ma_id(a, b, at);
    if (id < 0 || (at > 0 && at != a.nk && ma_id(a, b, at - 1) == id)) continue;
    atomicMin(a.first + ma_id_entry<true>(a, b, id), static_cast<uint32_t>(at));
  }
}
__global__ void __launch_bounds__(256) ma_ids_number_kernel(MaIds a) {
  const int b = blockIdx.y;
  const int64_t n = int64_t(a.nk) + a.nq;
  for (int64_t at = blockIdx.x * 256 + threadIdx.x; at < n; at += gridDim.x * 256) {
    const int64_t id = ma_id(a, b, at);
    const int32_t number = id < 0 ? -1 : static_cast<int32_t>(a.first[ma_id_entry<false>(a, b, id)]);
    if (at < a.nk) {
      a.k_out[static_cast<int64_t>(b) * a.nk + at] = number;
    } else {
      a.q_out[static_cast<int64_t>(b) * a.nq + at - a.nk] = number;
    }
  }
}

// ---------------------------------------------------------------- rows

struct MaRow {
  int h, i;
};
__device__ __forceinline__ MaRow ma_row(const MaskedArgs& a, int g, int r) {
  const int i = r / a.rep;
  return {g * a.rep + (r - i * a.rep), i};
}
__device__ __forceinline__ int64_t ma_row_index(const MaskedArgs& a, int b, MaRow r) {
  return (static_cast<int64_t>(b) * a.H + r.h) * a.nq + r.i;
}
template <typename T>
__device__ __forceinline__ T* ma_at(const MaTensor& t, int b, int h, int i) {
  return static_cast<T*>(t.p) + b * t.sb + h * t.sh + static_cast<int64_t>(i) * t.sn;
}

// ---------------------------------------------------------------- CUDA-core tiles
//
// 256 threads as 16 x 16 (ty, tx) multiply 64 x 64 tiles: a thread owns rows ty + 16 e and
// columns tx + 16 f.  Tiles are row-major in shared memory with a pitch of DP + 4 floats,
// so that the 16-byte reads of eight neighbouring threads cover all banks.  A product step reads
// 12 shared-memory wavefronts for 64 FMA a warp, near the ratio of the two rates.  f32, 2 x 1024
// causal tokens, 8 heads of 128: forward 25 TFLOP/s, backward 18, of 72; short rows are bound
// by one block an SM of 8 warps (FMA pipe 33 % at 777 tokens of 8 heads of 32).

constexpr int kMaTile = 64;
constexpr int kMaP = kMaTile + 4;

// 64 rows of d values (zeros up to DP, and for rows whose pointer is null) on their way to
// shared memory: fetch() reads them into registers, put() writes them there.  The kernels fetch
// a tile while they work on the one before, so its latency is not waited for.
template <typename T, int DP>
struct MaRows {
  static constexpr int C = DP / 4, kPer = DP / 16, kStep = 256 / C;
  float4 v[kPer];
  static __device__ __forceinline__ int row(int k) { return threadIdx.x / C + k * kStep; }
  template <typename RowPtr>
  __device__ __forceinline__ void fetch(int d, int vec4, RowPtr row_ptr) {
    const int c = (threadIdx.x % C) * 4;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const T* p = row_ptr(row(k));
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (p != nullptr && c < d) {
        if (vec4) {
          const LnVec<T, 4> w = *reinterpret_cast<const LnVec<T, 4>*>(p + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = ln_float(w.v[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < d) x[e] = ln_float(p[c + e]);
        }
      }
      v[k] = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  __device__ __forceinline__ void put(float* dst) const {
    const int c = (threadIdx.x % C) * 4;
#pragma unroll
    for (int k = 0; k < kPer; ++k) *reinterpret_cast<float4*>(dst + row(k) * (DP + 4) + c) = v[k];
  }
};
template <typename T, int DP, typename RowPtr>
__device__ __forceinline__ void ma_load_rows(float* dst, int d, int vec4, RowPtr row_ptr) {
  MaRows<T, DP> rows;
  rows.fetch(d, vec4, row_ptr);
  rows.put(dst);
}

// acc[e][f] = A[ty + 16 e] . B[tx + 16 f] over the first d4 * 4 values.
template <int DP>
__device__ __forceinline__ void ma_tile_dot(const float* A, const float* B, int d4,
                                            float (&acc)[4][4]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[e][f] = 0.f;
#pragma unroll 4
  for (int c = 0; c < d4; ++c) {
    float4 x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = *reinterpret_cast<const float4*>(A + (ty + 16 * e) * (DP + 4) + 4 * c);
      y[e] = *reinterpret_cast<const float4*>(B + (tx + 16 * e) * (DP + 4) + 4 * c);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        acc[e][f] = fmaf(x[e].x, y[f].x, acc[e][f]);
        acc[e][f] = fmaf(x[e].y, y[f].y, acc[e][f]);
        acc[e][f] = fmaf(x[e].z, y[f].z, acc[e][f]);
        acc[e][f] = fmaf(x[e].w, y[f].w, acc[e][f]);
      }
  }
}

// Column u of a thread's DP / 16 columns.
template <int DP>
__device__ __forceinline__ int ma_col(int u) {
  const int tx = threadIdx.x & 15;
  if constexpr (DP == 32) return tx * 2 + u;
  return (u >> 2) * 64 + tx * 4 + (u & 3);
}

// o[e][u] += sum_j P[ty + 16 e][j] V[j][col(u)] over the tile's 64 j.
template <int DP>
__device__ __forceinline__ void ma_tile_add(const float* P, const float* V,
                                            float (&o)[4][DP / 16]) {
  const int ty = threadIdx.x >> 4;
#pragma unroll 4
  for (int j = 0; j < kMaTile; j += 4) {
    float4 p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      p[e] = *reinterpret_cast<const float4*>(P + (ty + 16 * e) * kMaP + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const float* row = V + (j + jj) * (DP + 4);
      float v[DP / 16];
      if constexpr (DP == 32) {
        const float2 w = *reinterpret_cast<const float2*>(row + ma_col<DP>(0));
        v[0] = w.x;
        v[1] = w.y;
      } else {
#pragma unroll
        for (int u = 0; u < DP / 16; u += 4) {
          const float4 w = *reinterpret_cast<const float4*>(row + ma_col<DP>(u));
          v[u] = w.x;
          v[u + 1] = w.y;
          v[u + 2] = w.z;
          v[u + 3] = w.w;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pe = jj == 0 ? p[e].x : jj == 1 ? p[e].y : jj == 2 ? p[e].z : p[e].w;
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) o[e][u] = fmaf(pe, v[u], o[e][u]);
      }
    }
  }
}

// Score of a raw product; with BEND, `bend` receives its derivative 1 - tanh^2(x / cap), as
// 4 e / (1 + e)^2 with e = exp(-2 |x / cap|): 1 - t^2 of a rounded t near 1 has few digits left.
template <bool BEND>
__device__ __forceinline__ float ma_score(const MaskedArgs& a, float dot, float slope, int pos,
                                          int key, float& bend) {
  float s = dot * a.scale;
  bend = 1.f;
  if (a.cap > 0.f) {
    const float y = s * a.inv_cap;
    s = a.cap * tanhf(y);
    if (BEND) {
      const float e = expf(-2.f * fabsf(y));
      bend = 4.f * e / ((1.f + e) * (1.f + e));
    }
  }
  return s - slope * fabsf(static_cast<float>(pos - key));
}

// What a thread has to know about one of its rows.
struct MaRowInfo {
  int limit, doc, pos;
  float slope;
};
__device__ __forceinline__ MaRowInfo ma_row_info(const MaskedArgs& a, int b, MaRow r, bool live,
                                                 int prefix) {
  MaRowInfo w;
  w.limit = live ? ma_limit(a, r.i, prefix) : 0;
  w.doc = live && a.qdoc != nullptr ? a.qdoc[b * a.qdoc_sb + r.i] : -1;
  if (w.doc < 0) w.doc = -2;  // padding does not see padding
  w.pos = r.i + a.off;
  w.slope = live && a.slopes != nullptr ? a.slopes[r.h] : 0.f;
  return w;
}

template <int DP>
struct MaForwardSmem {
  static constexpr int kRows = kMaTile * (DP + 4);
  static constexpr int kBytes = (3 * kRows + kMaTile * kMaP) * 4 + kMaTile * 4;
};

// One block: 64 rows of (b, g) over the keys of one split.
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1) ma_forward_kernel(const __grid_constant__ MaskedArgs a) {
  extern __shared__ float ma_smem[];
  float* sQ = ma_smem;
  float* sK = sQ + MaForwardSmem<DP>::kRows;
  float* sV = sK + MaForwardSmem<DP>::kRows;
  float* sP = sV + MaForwardSmem<DP>::kRows;
  int* sDoc = reinterpret_cast<int*>(sP + kMaTile * kMaP);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int item = blockIdx.x;
  const int split = item % a.splits;
  item /= a.splits;
  const int g = item % a.G;
  item /= a.G;
  const int b = item % a.B;
  const int qt = a.q_tiles - 1 - item / a.B;  // causal rows with the most keys come first
  const int rows = a.nq * a.rep;
  const int r0 = qt * kMaTile;
  const int last_i = (min(r0 + kMaTile, rows) - 1) / a.rep;
  const int prefix = ma_prefix(a, b);
  const int d4 = (a.d + 3) / 4;
  const bool docs = a.qdoc != nullptr;

  ma_load_rows<T, DP>(sQ, a.d, a.vec4, [&](int r) -> const T* {
    if (r0 + r >= rows) return nullptr;
    const MaRow w = ma_row(a, g, r0 + r);
    return ma_at<const T>(a.q, b, w.h, w.i);
  });
  MaRowInfo info[4];
  float m[4], l[4], o[4][DP / 16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = r0 + ty + 16 * e;
    info[e] = ma_row_info(a, b, ma_row(a, g, r), r < rows, prefix);
    m[e] = -INFINITY;
    l[e] = 0.f;
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) o[e][u] = 0.f;
  }
  const int per = (a.k_tiles + a.splits - 1) / a.splits;
  const int limit = ma_limit(a, last_i, prefix);
  const int t1 = min(min(a.k_tiles, (split + 1) * per), (limit + kMaTile - 1) / kMaTile);
  int4 qr = make_int4(0, 0, 0, 0);
  if (docs) qr = ma_join_ranges(a.qrange + b * a.qrange_sb, (r0 / a.rep) / 64, last_i / 64);

  const auto next_tile = [&](int t) {
    while (t < t1 && docs && !ma_ranges_meet(qr, a.krange[b * a.krange_sb + t])) ++t;
    return t;
  };
  MaRows<T, DP> k_rows, v_rows;
  // K and V of keys in no document read as zeros, whatever their memory holds
  const auto fetch = [&](int t) {
    const int key0 = t * kMaTile;
    const int* kdoc = docs ? a.kdoc + b * a.kdoc_sb + key0 : nullptr;
    const auto key_row = [&](const MaTensor& x, int r) -> const T* {
      if (key0 + r >= a.nk || (docs && kdoc[r] < 0)) return nullptr;
      return ma_at<const T>(x, b, g, key0 + r);
    };
    k_rows.fetch(a.d, a.vec4, [&](int r) { return key_row(a.k, r); });
    v_rows.fetch(a.d, a.vec4, [&](int r) { return key_row(a.v, r); });
  };
  int t = next_tile(split * per);
  if (t < t1) fetch(t);
  for (int after; t < t1; t = after) {
    const int key0 = t * kMaTile;
    __syncthreads();  // the last tile is consumed
    k_rows.put(sK);
    v_rows.put(sV);
    if (docs && threadIdx.x < kMaTile) sDoc[threadIdx.x] = a.kdoc[b * a.kdoc_sb + key0 + threadIdx.x];
    __syncthreads();
    after = next_tile(t + 1);
    if (after < t1) fetch(after);
    float s[4][4];
    ma_tile_dot<DP>(sQ, sK, d4, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float top = -INFINITY;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int key = key0 + tx + 16 * f;
        const bool seen = key < info[e].limit && (!docs || sDoc[tx + 16 * f] == info[e].doc);
        float bend;
        s[e][f] = seen ? ma_score<false>(a, s[e][f], info[e].slope, info[e].pos, key, bend) : -INFINITY;
        top = fmaxf(top, s[e][f]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float m_new = fmaxf(m[e], top);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float shrink = expf(m[e] - base);
      float sum = 0.f;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const float p = expf(s[e][f] - base);
        sP[(ty + 16 * e) * kMaP + tx + 16 * f] = p;
        sum += p;
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[e] = fmaf(l[e], shrink, sum);
      m[e] = m_new;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) o[e][u] *= shrink;
    }
    __syncthreads();
    ma_tile_add<DP>(sP, sV, o);
  }

#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = r0 + ty + 16 * e;
    if (r >= rows) continue;
    const MaRow w = ma_row(a, g, r);
    const int64_t index = ma_row_index(a, b, w);
    const float inv = l[e] > 0.f || l[e] != l[e] ? 1.f / l[e] : 0.f;  // a NaN score stays NaN
    const float lse = l[e] == 0.f ? -INFINITY : m[e] + logf(l[e]);
    if (a.splits > 1) {
      const int64_t at = split * (static_cast<int64_t>(a.B) * a.H * a.nq) + index;
      if (tx == 0) a.part_lse[at] = lse;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u)
        if (ma_col<DP>(u) < a.d) a.part_o[at * a.d + ma_col<DP>(u)] = o[e][u] * inv;
      continue;
    }
    if (tx == 0 && a.lse != nullptr) a.lse[index] = lse;
    T* out = ma_at<T>(a.out, b, w.h, w.i);
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) {
      const int c = ma_col<DP>(u);
      if (c >= a.d) continue;
      const float v = o[e][u] * inv;
      out[c] = ln_round<T>(v);
      if (a.low != nullptr) a.low[index * a.d + c] = __float2bfloat16_rn(v - ln_float(out[c]));
    }
  }
}

// Joins the splits of a row: out = sum_s exp(lse_s - lse) out_s.  A block of 4 warps a row: every
// thread weighs the splits (one each, so at most 128), then thread c % 32 of warp c / 32 adds
// up column c; the loads of eight splits are in flight at once.
constexpr int kMaMaxSplits = 128;
template <typename T>
__global__ void __launch_bounds__(128) ma_join_kernel(const __grid_constant__ MaskedArgs a) {
  __shared__ float weight[kMaMaxSplits];
  __shared__ float top_of[4], sum_of[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t total = static_cast<int64_t>(a.B) * a.H * a.nq;
  const int64_t index = blockIdx.x;
  const float lse = static_cast<int>(threadIdx.x) < a.splits
                        ? a.part_lse[threadIdx.x * total + index]
                        : -INFINITY;
  float top = lse;  // a NaN is passed over here and comes back in the weights' sum
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if (lane == 0) top_of[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
  const float base = top == -INFINITY ? 0.f : top;
  const float w = expf(lse - base);
  weight[threadIdx.x] = w;
  float sum = w;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if (lane == 0) sum_of[warp] = sum;
  __syncthreads();
  sum = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int i = static_cast<int>(index % a.nq);
  const int64_t bh = index / a.nq;
  const int h = static_cast<int>(bh % a.H), b = static_cast<int>(bh / a.H);
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[index] = sum == 0.f ? -INFINITY : top + logf(sum);
  const int c = threadIdx.x;
  if (c >= a.d) return;
  float v = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s)  // a split that saw no key has weight 0 and zeros
    v = fmaf(weight[s], a.part_o[(s * total + index) * a.d + c], v);
  v *= inv;
  T* out = ma_at<T>(a.out, b, h, i);
  out[c] = ln_round<T>(v);
  if (a.low != nullptr) a.low[index * a.d + c] = __float2bfloat16_rn(v - ln_float(out[c]));
}

// D_i = do_i . o_i with o taken back to more than bf16 by `low`: rounded to bf16 alone it
// would put an error of 2^-9 |o| |do| on every score gradient of the row.  One thread a row
// adds the terms in the order in which ma_tile_dot adds those of do . v, so a row that sees one
// key alone (o = v) has do . v - D = 0 exactly.
template <typename T>
__global__ void __launch_bounds__(128) ma_delta_kernel(const __grid_constant__ MaskedArgs a) {
  const int64_t total = static_cast<int64_t>(a.B) * a.H * a.nq;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (index >= total) return;
  const int i = static_cast<int>(index % a.nq);
  const int64_t bh = index / a.nq;
  const int h = static_cast<int>(bh % a.H), b = static_cast<int>(bh / a.H);
  const T* o = ma_at<const T>(a.out, b, h, i);
  const T* dout = ma_at<const T>(a.dout, b, h, i);
  float sum = 0.f, rest = 0.f;
#pragma unroll 8
  for (int c = 0; c < a.d; ++c) {
    const float g = ln_float(dout[c]);
    sum = fmaf(ln_float(o[c]), g, sum);
    if (a.low != nullptr) rest = fmaf(ln_float(a.low[index * a.d + c]), g, rest);
  }
  // a row that sees no key has no gradient, whatever its do holds
  a.delta[index] = a.lse[index] == -INFINITY ? 0.f : sum + rest;
}

template <int DP>
struct MaBackwardSmem {
  static constexpr int kRows = kMaTile * (DP + 4);
  static constexpr int kBytes = (4 * kRows + 2 * kMaTile * kMaP) * 4 + kMaTile * 6 * 4;
};

// One block: dk, dv of 64 keys of (b, g), over all rows that may see them.  Tiles are
// transposed (rows = keys, columns = rows of q), so p and dx are the left operands.
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP == 32 ? 2 : 1) ma_backward_kv_kernel(const __grid_constant__ MaskedArgs a) {
  extern __shared__ float ma_smem[];
  constexpr int R = MaBackwardSmem<DP>::kRows;
  float* sK = ma_smem;
  float* sV = sK + R;
  float* sQ = sV + R;
  float* sO = sQ + R;
  float* sP = sO + R;
  float* sD = sP + kMaTile * kMaP;
  float* sLse = sD + kMaTile * kMaP;
  float* sDelta = sLse + kMaTile;
  float* sSlope = sDelta + kMaTile;
  int* sLimit = reinterpret_cast<int*>(sSlope + kMaTile);
  int* sDoc = sLimit + kMaTile;
  int* sPos = sDoc + kMaTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int item = blockIdx.x;
  const int g = item % a.G;
  item /= a.G;
  const int b = item % a.B;
  const int kt = item / a.B;  // causal keys with the most rows come first
  const int key0 = kt * kMaTile;
  const int rows = a.nq * a.rep;
  const int prefix = ma_prefix(a, b);
  const int d4 = (a.d + 3) / 4;
  const bool docs = a.qdoc != nullptr;
  const int* kdoc = docs ? a.kdoc + b * a.kdoc_sb + key0 : nullptr;
  const auto key_row = [&](const MaTensor& x, int r) -> const T* {
    return key0 + r < a.nk && !(docs && kdoc[r] < 0) ? ma_at<const T>(x, b, g, key0 + r) : nullptr;
  };
  ma_load_rows<T, DP>(sK, a.d, a.vec4, [&](int r) { return key_row(a.k, r); });
  ma_load_rows<T, DP>(sV, a.d, a.vec4, [&](int r) { return key_row(a.v, r); });
  int doc[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) doc[e] = docs ? kdoc[ty + 16 * e] : -1;
  float dk[4][DP / 16], dv[4][DP / 16];
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) dk[e][u] = dv[e][u] = 0.f;
  // the first query that sees the tile's first key
  const int first = !a.causal || key0 < prefix ? 0 : max(0, key0 - a.off);
  int4 kr = make_int4(0, 0, 0, 0);
  if (docs) kr = a.krange[b * a.krange_sb + kt];
  const auto next_tile = [&](int qt) {
    while (docs && qt < a.q_tiles) {
      const int last_i = (min((qt + 1) * kMaTile, rows) - 1) / a.rep;
      if (ma_ranges_meet(ma_join_ranges(a.qrange + b * a.qrange_sb, (qt * kMaTile / a.rep) / 64,
                                        last_i / 64), kr))
        break;
      ++qt;
    }
    return qt;
  };
  MaRows<T, DP> q_rows, o_rows;
  float row_lse[MaRows<T, DP>::kPer];  // of the fetched rows
  float lse_next = 0.f, delta_next = 0.f;
  MaRowInfo info_next{};
  const auto fetch = [&](int qt) {
    const int r0 = qt * kMaTile;
    const auto q_row = [&](const MaTensor& x, int r) -> const T* {
      if (r0 + r >= rows) return nullptr;
      const MaRow w = ma_row(a, g, r0 + r);
      return ma_at<const T>(x, b, w.h, w.i);
    };
    q_rows.fetch(a.d, a.vec4, [&](int r) { return q_row(a.q, r); });
    o_rows.fetch(a.d, a.vec4, [&](int r) { return q_row(a.dout, r); });
#pragma unroll
    for (int k = 0; k < MaRows<T, DP>::kPer; ++k) {
      const int r = r0 + MaRows<T, DP>::row(k);
      row_lse[k] = r < rows ? a.lse[ma_row_index(a, b, ma_row(a, g, r))] : -INFINITY;
    }
    if (threadIdx.x < kMaTile) {
      const int r = r0 + threadIdx.x;
      const bool live = r < rows;
      const MaRow w = ma_row(a, g, r);
      info_next = ma_row_info(a, b, w, live, prefix);
      lse_next = live ? a.lse[ma_row_index(a, b, w)] : -INFINITY;
      delta_next = live ? a.delta[ma_row_index(a, b, w)] : 0.f;
    }
  };
  int qt = next_tile(static_cast<int>(static_cast<int64_t>(first) * a.rep / kMaTile));
  if (qt < a.q_tiles) fetch(qt);
  for (int after; qt < a.q_tiles; qt = after) {
    __syncthreads();  // the last tile is consumed
    // q and do of rows that see no key become zeros, whatever their memory holds
#pragma unroll
    for (int k = 0; k < MaRows<T, DP>::kPer; ++k)
      if (row_lse[k] == -INFINITY) q_rows.v[k] = o_rows.v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    q_rows.put(sQ);
    o_rows.put(sO);
    if (threadIdx.x < kMaTile) {
      sLse[threadIdx.x] = lse_next;
      sDelta[threadIdx.x] = delta_next;
      sSlope[threadIdx.x] = info_next.slope;
      sLimit[threadIdx.x] = lse_next == -INFINITY ? 0 : info_next.limit;
      sDoc[threadIdx.x] = info_next.doc;
      sPos[threadIdx.x] = info_next.pos;
    }
    __syncthreads();
    after = next_tile(qt + 1);
    if (after < a.q_tiles) fetch(after);
    float s[4][4], dp[4][4];
    ma_tile_dot<DP>(sK, sQ, d4, s);
    ma_tile_dot<DP>(sV, sO, d4, dp);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int c = tx + 16 * f;
      const float lse = sLse[c], delta = sDelta[c], slope = sSlope[c];
      const int limit = sLimit[c], pos = sPos[c], qdoc = sDoc[c];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + ty + 16 * e;
        float p = 0.f, dx = 0.f;
        if (key < limit && (!docs || doc[e] == qdoc)) {
          float bend;
          p = expf(ma_score<true>(a, s[e][f], slope, pos, key, bend) - lse);
          dx = p * (dp[e][f] - delta) * bend;
        }
        sP[(ty + 16 * e) * kMaP + c] = p;
        sD[(ty + 16 * e) * kMaP + c] = dx;
      }
    }
    __syncthreads();
    ma_tile_add<DP>(sP, sO, dv);
    ma_tile_add<DP>(sD, sQ, dk);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int key = key0 + ty + 16 * e;
    if (key >= a.nk) continue;
    T* ok = ma_at<T>(a.dk, b, g, key);
    T* ov = ma_at<T>(a.dv, b, g, key);
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) {
      const int c = ma_col<DP>(u);
      if (c < a.d) {
        ok[c] = ln_round<T>(dk[e][u] * a.scale);
        ov[c] = ln_round<T>(dv[e][u]);
      }
    }
  }
}

// One block: dq of 64 rows of (b, g), over all keys that they see.
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP == 32 ? 2 : 1) ma_backward_q_kernel(const __grid_constant__ MaskedArgs a) {
  extern __shared__ float ma_smem[];
  constexpr int R = MaBackwardSmem<DP>::kRows;
  float* sQ = ma_smem;
  float* sO = sQ + R;
  float* sK = sO + R;
  float* sV = sK + R;
  float* sD = sV + R;
  int* sDoc = reinterpret_cast<int*>(sD + kMaTile * kMaP);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int item = blockIdx.x;
  const int g = item % a.G;
  item /= a.G;
  const int b = item % a.B;
  const int qt = a.q_tiles - 1 - item / a.B;
  const int rows = a.nq * a.rep;
  const int r0 = qt * kMaTile;
  const int last_i = (min(r0 + kMaTile, rows) - 1) / a.rep;
  const int prefix = ma_prefix(a, b);
  const int d4 = (a.d + 3) / 4;
  const bool docs = a.qdoc != nullptr;
  const auto q_row = [&](const MaTensor& x, int r) -> const T* {
    if (r0 + r >= rows) return nullptr;
    const MaRow w = ma_row(a, g, r0 + r);
    return ma_at<const T>(x, b, w.h, w.i);
  };
  ma_load_rows<T, DP>(sQ, a.d, a.vec4, [&](int r) { return q_row(a.q, r); });
  ma_load_rows<T, DP>(sO, a.d, a.vec4, [&](int r) { return q_row(a.dout, r); });
  MaRowInfo info[4];
  float lse[4], delta[4], dq[4][DP / 16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = r0 + ty + 16 * e;
    const MaRow w = ma_row(a, g, r);
    info[e] = ma_row_info(a, b, w, r < rows, prefix);
    lse[e] = r < rows ? a.lse[ma_row_index(a, b, w)] : -INFINITY;
    delta[e] = r < rows ? a.delta[ma_row_index(a, b, w)] : 0.f;
    if (lse[e] == -INFINITY) info[e].limit = 0;
#pragma unroll
    for (int u = 0; u < DP / 16; ++u) dq[e][u] = 0.f;
  }
  const int limit = ma_limit(a, last_i, prefix);
  const int t1 = min(a.k_tiles, (limit + kMaTile - 1) / kMaTile);
  int4 qr = make_int4(0, 0, 0, 0);
  if (docs) qr = ma_join_ranges(a.qrange + b * a.qrange_sb, (r0 / a.rep) / 64, last_i / 64);
  const auto next_tile = [&](int t) {
    while (t < t1 && docs && !ma_ranges_meet(qr, a.krange[b * a.krange_sb + t])) ++t;
    return t;
  };
  MaRows<T, DP> k_rows, v_rows;
  const auto fetch = [&](int t) {
    const int key0 = t * kMaTile;
    const int* kdoc = docs ? a.kdoc + b * a.kdoc_sb + key0 : nullptr;
    const auto key_row = [&](const MaTensor& x, int r) -> const T* {
      if (key0 + r >= a.nk || (docs && kdoc[r] < 0)) return nullptr;
      return ma_at<const T>(x, b, g, key0 + r);
    };
    k_rows.fetch(a.d, a.vec4, [&](int r) { return key_row(a.k, r); });
    v_rows.fetch(a.d, a.vec4, [&](int r) { return key_row(a.v, r); });
  };
  int t = next_tile(0);
  if (t < t1) fetch(t);
  for (int after; t < t1; t = after) {
    const int key0 = t * kMaTile;
    __syncthreads();
    k_rows.put(sK);
    v_rows.put(sV);
    if (docs && threadIdx.x < kMaTile) sDoc[threadIdx.x] = a.kdoc[b * a.kdoc_sb + key0 + threadIdx.x];
    __syncthreads();
    after = next_tile(t + 1);
    if (after < t1) fetch(after);
    float s[4][4], dp[4][4];
    ma_tile_dot<DP>(sQ, sK, d4, s);
    ma_tile_dot<DP>(sO, sV, d4, dp);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int c = tx + 16 * f, key = key0 + c;
        float dx = 0.f;
        if (key < info[e].limit && (!docs || sDoc[c] == info[e].doc)) {
          float bend;
          const float p =
              expf(ma_score<true>(a, s[e][f], info[e].slope, info[e].pos, key, bend) - lse[e]);
          dx = p * (dp[e][f] - delta[e]) * bend;
        }
        sD[(ty + 16 * e) * kMaP + c] = dx;
      }
    __syncthreads();
    ma_tile_add<DP>(sD, sK, dq);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = r0 + ty + 16 * e;
    if (r >= rows) continue;
    const MaRow w = ma_row(a, g, r);
    T* out = ma_at<T>(a.dq, b, w.h, w.i);
#pragma unroll
    for (int u = 0; u < DP / 16; ++u)
      if (ma_col<DP>(u) < a.d) out[ma_col<DP>(u)] = ln_round<T>(dq[e][u] * a.scale);
  }
}

}  // namespace xfb
