// Entry points of the training operators (masked attention, rotary positions, LayerNorm with its
// gradients).  Included at the end of capi.cu, whose helpers (fail, XFB_TRY, Carver, tensor
// maps) it uses.
#pragma once

namespace {

// No C++ exception leaves a C entry point: what the body throws (std::bad_alloc
// from an error message) becomes an error code.
template <class Body>
int guarded(Body body) {
  try {
    return body();
  } catch (...) {
    return XFB_ERR_CUDA;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int sm_count_or_default() {
  int sms = 148;
  int dev;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    if (sm_count(&sms) != XFB_OK) sms = 148;
  } else {
    cudaGetLastError();
  }
  return sms;
}

// ---------------------------------------------------------------- LayerNorm

bool row_aligned(const void* p, int64_t ld, int vec, int size) {
  return p == nullptr || (ld % vec == 0 && reinterpret_cast<uintptr_t>(p) % (vec * size) == 0);
}

// The most blocks of the backward pass: each leaves one partial of dw and db, so there are fewer
// where rows are wide (2^21 values of partials, 8 MB), and eight an SM at most.
int64_t ln_most_blocks(int64_t cols) {
  const int64_t sms = sm_count_or_default();
  return std::max(sms, std::min(sms * 8, (int64_t(1) << 21) / cols));
}

// Blocks that the GPU runs at once, found out once for a kernel.
template <class Kernel>
int resident_blocks(Kernel kernel, int threads, std::atomic<int>& known) {
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess ||
        per_sm < 1) {
      cudaGetLastError();
      per_sm = 1;
    }
    known.store(per_sm, std::memory_order_relaxed);
  }
  return per_sm * sm_count_or_default();
}

// `count` receives the backward pass's number of blocks, that is of partials.
template <typename T, int VEC, int TPR, int NV>
int ln_launch_shape(bool backward, const xfb::LnTrainArgs& a, int* count, cudaStream_t st) {
  using S = xfb::LnShape<TPR>;
  static std::atomic<int> known[2];
  const int64_t want = ceil_div(a.rows, S::kGroups);
  if (backward) {
    auto kernel = xfb::ln_train_backward_kernel<T, VEC, TPR, NV>;
    const int64_t at_once = resident_blocks(kernel, S::kBlock, known[1]);
    *count = static_cast<int>(std::min({want, at_once, ln_most_blocks(a.cols)}));
    kernel<<<*count, S::kBlock, 0, st>>>(a);
  } else {
    auto kernel = xfb::ln_train_forward_kernel<T, VEC, TPR, NV>;
    const int64_t at_once = resident_blocks(kernel, S::kBlock, known[0]);
    kernel<<<static_cast<unsigned>(std::min(want, at_once)), S::kBlock, 0, st>>>(a);
  }
  XFB_LAUNCHED();
  return XFB_OK;
}

// Row shapes by the vectors of a row.  A thread takes up to four vectors of it forward, and
// backward, where it adds two sums a column, up to 16 values: enough loads in flight, few
// shuffles a value, and registers for several blocks an SM.  Rows of up to 32 threads
// need no block barrier.  (1 M rows of 128 bf16: one vector a thread and 16 threads a row
// 210 and 197 us, this 98 and 166; 32768 rows of 4096 in another shape, weights read again
// for each row: 282 and 420 us.)
template <typename T, int VEC>
int ln_launch(bool backward, const xfb::LnTrainArgs& a, int* count, cudaStream_t st) {
  const int64_t n = a.cols / VEC;
  if (VEC == 8 && backward) {
    if (n <= 4) return ln_launch_shape<T, VEC, 2, 2>(backward, a, count, st);
    if (n <= 8) return ln_launch_shape<T, VEC, 4, 2>(backward, a, count, st);
    if (n <= 16) return ln_launch_shape<T, VEC, 8, 2>(backward, a, count, st);
    if (n <= 32) return ln_launch_shape<T, VEC, 16, 2>(backward, a, count, st);
    if (n <= 64) return ln_launch_shape<T, VEC, 32, 2>(backward, a, count, st);
    if (n <= 128) return ln_launch_shape<T, VEC, 64, 2>(backward, a, count, st);
    if (n <= 256) return ln_launch_shape<T, VEC, 128, 2>(backward, a, count, st);
    if (n <= 512) return ln_launch_shape<T, VEC, 256, 2>(backward, a, count, st);
    if (n <= 1024) return ln_launch_shape<T, VEC, 512, 2>(backward, a, count, st);
  } else {
    if (n <= 8) return ln_launch_shape<T, VEC, 2, 4>(backward, a, count, st);
    if (n <= 16) return ln_launch_shape<T, VEC, 4, 4>(backward, a, count, st);
    if (n <= 32) return ln_launch_shape<T, VEC, 8, 4>(backward, a, count, st);
    if (n <= 64) return ln_launch_shape<T, VEC, 16, 4>(backward, a, count, st);
    if (n <= 128) return ln_launch_shape<T, VEC, 32, 4>(backward, a, count, st);
    if (n <= 256) return ln_launch_shape<T, VEC, 64, 4>(backward, a, count, st);
    if (n <= 512) return ln_launch_shape<T, VEC, 128, 4>(backward, a, count, st);
    if (n <= 1024) return ln_launch_shape<T, VEC, 256, 4>(backward, a, count, st);
  }
  if (n <= 2048) return ln_launch_shape<T, VEC, 512, 4>(backward, a, count, st);
  return ln_launch_shape<T, VEC, 512, 8>(backward, a, count, st);
}
constexpr int64_t kLnMostVectors = 4096;  // a row of more takes the kernels that read it again

// Values per load: 16 bytes where width, strides and bases allow it, else 8, else one.
template <typename T>
int ln_vector(const xfb::LnTrainArgs& a) {
  constexpr int kWide = 16 / sizeof(T);
  for (int vec = kWide; vec > 1; vec /= 2) {
    if (vec != kWide && vec != 4) continue;
    if (a.cols % vec == 0 && row_aligned(a.x, a.ldx, vec, sizeof(T)) &&
        row_aligned(a.y, a.ldy, vec, sizeof(T)) && row_aligned(a.dy, a.lddy, vec, sizeof(T)) &&
        row_aligned(a.dx, a.lddx, vec, sizeof(T)) && aligned16(a.w) && aligned16(a.b))
      return vec;
  }
  return 1;
}

template <typename T>
int ln_dispatch(bool backward, const xfb::LnTrainArgs& a, int vec, int* count, cudaStream_t st) {
  if (vec == 8) {
    if constexpr (sizeof(T) == 2) return ln_launch<T, 8>(backward, a, count, st);
  }
  if (vec == 4) return ln_launch<T, 4>(backward, a, count, st);
  return ln_launch<T, 1>(backward, a, count, st);
}

template <typename T>
int ln_forward(const xfb::LnTrainArgs& a, cudaStream_t st) {
  const int vec = ln_vector<T>(a);
  if (a.cols / vec > kLnMostVectors) {
    const int64_t most = int64_t(sm_count_or_default()) * 4;
    xfb::ln_wide_forward_kernel<T><<<static_cast<unsigned>(std::min(a.rows, most)), 512, 0, st>>>(a);
    XFB_LAUNCHED();
    return XFB_OK;
  }
  int count = 0;
  return ln_dispatch<T>(false, a, vec, &count, st);
}

template <typename T>
int ln_backward(xfb::LnTrainArgs a, float* dw, float* db, cudaStream_t st) {
  const int vec = ln_vector<T>(a);
  int count = 0;
  if (a.cols / vec > kLnMostVectors) {
    if (a.dx != nullptr) {
      const int64_t most = int64_t(sm_count_or_default()) * 4;
      xfb::ln_wide_backward_kernel<T>
          <<<static_cast<unsigned>(std::min(a.rows, most)), 512, 0, st>>>(a);
      XFB_LAUNCHED();
    }
    if (a.partial == nullptr) return XFB_OK;
    count = static_cast<int>(std::min<int64_t>(a.rows, 32));
    const dim3 grid(static_cast<unsigned>(ceil_div(a.cols, 256)), count);
    xfb::ln_columns_kernel<T><<<grid, 256, 0, st>>>(a);
    XFB_LAUNCHED();
  } else {
    XFB_TRY(ln_dispatch<T>(true, a, vec, &count, st));
    if (a.partial == nullptr) return XFB_OK;
  }
  xfb::ln_reduce_kernel<<<static_cast<unsigned>(ceil_div(2ll * a.cols, 32)), 1024, 0, st>>>(
      a.partial, count, a.cols, dw, db);
  XFB_LAUNCHED();
  return XFB_OK;
}

// Rows that are only read may overlap (one row seen many times has stride 0).
int check_ln(int dtype, int64_t rows, int64_t cols, int64_t ldx) {
  XFB_REQUIRE(dtype == XFB_F32 || dtype == XFB_BF16, "LayerNorm data must be f32 or bf16");
  XFB_REQUIRE(rows >= 0, "rows must be non-negative");
  XFB_REQUIRE(cols >= 1 && cols <= (1 << 24), "LayerNorm width must be in [1, 2^24]");
  XFB_REQUIRE(ldx >= 0 || rows <= 1, "LayerNorm row stride is negative");
  return XFB_OK;
}

}  // namespace

extern "C" {

XFB_API int xfb_layer_norm_forward(const void* x, int dtype, int64_t rows, int64_t cols,
                                   int64_t ldx, const float* weight, const float* bias,
                                   double eps, void* y, int64_t ldy, float* mean, float* rstd,
                                   void* stream) {
  return guarded([&]() -> int {
    XFB_TRY(check_ln(dtype, rows, cols, ldx));
    XFB_REQUIRE(ldy >= cols || rows <= 1, "LayerNorm row stride is shorter than a row");
    XFB_REQUIRE(std::isfinite(eps) && eps >= 0, "LayerNorm eps must be finite and non-negative");
    XFB_REQUIRE((mean == nullptr) == (rstd == nullptr), "mean and rstd go together");
    if (rows == 0) return XFB_OK;
    XFB_REQUIRE(x != nullptr && y != nullptr, "LayerNorm needs x and y");
    xfb::LnTrainArgs a{};
    a.x = x;
    a.rows = rows;
    a.cols = static_cast<int>(cols);
    a.ldx = ldx;
    a.w = weight;
    a.b = bias;
    a.eps = static_cast<float>(eps);
    a.y = y;
    a.ldy = ldy;
    a.mean = mean;
    a.rstd = rstd;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == XFB_F32 ? ln_forward<float>(a, st) : ln_forward<bf16>(a, st);
  });
}

XFB_API int64_t xfb_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return std::min(rows, ln_most_blocks(cols)) * 2 * cols * 4;
}

XFB_API int xfb_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                    int dtype, int64_t rows, int64_t cols, const float* weight,
                                    const float* mean, const float* rstd, void* dx, int64_t lddx,
                                    float* dweight, float* dbias, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    XFB_TRY(check_ln(dtype, rows, cols, ldx));
    XFB_REQUIRE(lddy >= 0 || rows <= 1, "LayerNorm row stride is negative");
    XFB_REQUIRE(dx == nullptr || lddx >= cols || rows <= 1,
                "LayerNorm row stride is shorter than a row");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
      if (dweight) XFB_CUDA(cudaMemsetAsync(dweight, 0, cols * 4, st));
      if (dbias) XFB_CUDA(cudaMemsetAsync(dbias, 0, cols * 4, st));
      return XFB_OK;
    }
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (!sums && dx == nullptr) return XFB_OK;
    XFB_REQUIRE(dy && x && mean && rstd, "the LayerNorm gradient needs dy, x, mean and rstd");
    Carver cv{static_cast<uint8_t*>(workspace), 0, workspace_bytes};
    xfb::LnTrainArgs a{};
    if (sums) {
      a.partial = cv.take<float>(std::min(rows, ln_most_blocks(cols)) * 2 * cols);
      XFB_TRY(check_workspace(cv, workspace, workspace_bytes));
    }
    a.x = x;
    a.rows = rows;
    a.cols = static_cast<int>(cols);
    a.ldx = ldx;
    a.w = weight;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.dy = dy;
    a.lddy = lddy;
    a.dx = dx;
    a.lddx = lddx;
    return dtype == XFB_F32 ? ln_backward<float>(a, dweight, dbias, st)
                            : ln_backward<bf16>(a, dweight, dbias, st);
  });
}

}  // extern "C"

// ---------------------------------------------------------------- rotary positions

namespace {

bool rotary_fits(const xfb_rotary_args& a, int vec, int size) {
  const int64_t unit = a.interleaved ? a.rotated : a.rotated / 2;
  if (unit % vec != 0 || a.d % vec != 0 || a.rotated % vec != 0) return false;
  const int64_t strides[] = {a.q_sb,  a.q_sh,  a.q_sn,  a.k_sb,  a.k_sh,  a.k_sn,
                             a.qo_sb, a.qo_sh, a.qo_sn, a.ko_sb, a.ko_sh, a.ko_sn};
  for (const int64_t s : strides)
    if (s % vec != 0) return false;
  const void* bases[] = {a.q, a.k, a.q_out, a.k_out};
  for (const void* p : bases)
    if (reinterpret_cast<uintptr_t>(p) % (vec * size) != 0) return false;
  return true;
}

template <typename T, int VEC, bool INTERLEAVED>
int rotary_launch(xfb::RotaryArgs r, cudaStream_t st) {
  constexpr int W = INTERLEAVED && VEC == 1 ? 2 : VEC;
  const int64_t per_token = (INTERLEAVED ? r.rotated / W : r.rotated / 2 / VEC) +
                            (r.d - r.rotated + VEC - 1) / VEC;
  const int64_t threads = r.B * r.n * per_token;
  if (threads == 0) return XFB_OK;
  const int64_t blocks = ceil_div(threads, 256);
  const int64_t sms = sm_count_or_default();
  // Heads are shared out until there are 16 blocks an SM; a thread serves eight heads or more
  // once the tokens alone fill the GPU, which leaves the sines and cosines 1/8 of the work.
  const int heads = r.H + r.G;
  const int64_t share =
      std::max<int64_t>(1, std::min<int64_t>(heads, ceil_div(sms * 16, blocks)));
  r.head_step = static_cast<int>(std::max<int64_t>(share, heads / 8));
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20)), r.head_step);
  xfb::rotary_kernel<T, VEC, INTERLEAVED><<<grid, 256, 0, st>>>(r);
  XFB_LAUNCHED();
  return XFB_OK;
}

template <typename T, int VEC>
int rotary_layout(bool interleaved, const xfb::RotaryArgs& r, cudaStream_t st) {
  return interleaved ? rotary_launch<T, VEC, true>(r, st) : rotary_launch<T, VEC, false>(r, st);
}

}  // namespace

extern "C" {

XFB_API int xfb_rotary(const xfb_rotary_args* args, void* stream) {
  return guarded([&]() -> int {
    XFB_REQUIRE(args != nullptr, "rotary needs its arguments");
    const xfb_rotary_args& a = *args;
    XFB_REQUIRE(a.dtype == XFB_F32 || a.dtype == XFB_BF16, "rotary data must be f32 or bf16");
    XFB_REQUIRE(a.batch >= 0 && a.heads >= 0 && a.kv_heads >= 0 && a.n >= 0,
                "rotary sizes must be non-negative");
    XFB_REQUIRE(a.heads + a.kv_heads <= 65535, "rotary takes at most 65535 heads");
    XFB_REQUIRE(a.d >= 1 && a.d <= 65536, "rotary head dimension must be in [1, 65536]");
    XFB_REQUIRE(a.rotated >= 0 && a.rotated <= a.d && a.rotated % 2 == 0,
                "rotated dims must be even and at most the head dimension");
    XFB_REQUIRE(std::isfinite(static_cast<float>(a.magnitude)),
                "rotary magnitude must be finite in f32");
    if (a.batch == 0 || a.n == 0 || a.heads + a.kv_heads == 0) return XFB_OK;
    XFB_REQUIRE(a.heads == 0 || (a.q != nullptr && a.q_out != nullptr), "rotary needs q");
    XFB_REQUIRE(a.kv_heads == 0 || (a.k != nullptr && a.k_out != nullptr), "rotary needs k");
    XFB_REQUIRE(a.rotated == 0 || a.frequencies != nullptr, "rotary needs frequencies");
    xfb::RotaryArgs r{};
    r.q = {a.q, a.q_sb, a.q_sh, a.q_sn, a.q_out, a.qo_sb, a.qo_sh, a.qo_sn};
    r.k = {a.k, a.k_sb, a.k_sh, a.k_sn, a.k_out, a.ko_sb, a.ko_sh, a.ko_sn};
    r.H = static_cast<int>(a.heads);
    r.G = static_cast<int>(a.kv_heads);
    r.B = a.batch;
    r.n = a.n;
    r.d = static_cast<int>(a.d);
    r.rotated = static_cast<int>(a.rotated);
    r.freq = a.frequencies;
    r.positions = a.positions;
    r.positions_64 = a.positions_64;
    r.pos_sb = a.positions_sb;
    r.offset = a.offset;
    r.magnitude = static_cast<float>(a.magnitude);
    r.inverse = a.inverse;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool il = a.interleaved != 0;
    // the widest load of up to 16 bytes that every row and part of a head allows
    if (a.dtype == XFB_F32) {
      if (rotary_fits(a, 4, 4)) return rotary_layout<float, 4>(il, r, st);
      if (rotary_fits(a, 2, 4)) return rotary_layout<float, 2>(il, r, st);
      return rotary_layout<float, 1>(il, r, st);
    }
    if (rotary_fits(a, 8, 2)) return rotary_layout<bf16, 8>(il, r, st);
    if (rotary_fits(a, 4, 2)) return rotary_layout<bf16, 4>(il, r, st);
    if (rotary_fits(a, 2, 2)) return rotary_layout<bf16, 2>(il, r, st);
    return rotary_layout<bf16, 1>(il, r, st);
  });
}

}  // extern "C"

// ---------------------------------------------------------------- masked attention

namespace {

// One [B][heads][n][d] operand of the tensor-core kernels: 16-byte rows for TMA and vector
// stores.  `shared` allows a broadcast head or batch dimension (stride 0).
bool ma_tma_ok(const void* p, int64_t sb, int64_t sh, int64_t sn, int64_t B, int64_t heads,
               int64_t n, bool shared) {
  const auto stride_ok = [](int64_t s, int64_t size, bool zero) {
    return size <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)) || (zero && s == 0);
  };
  return aligned16(p) && stride_ok(sb, B, shared) && stride_ok(sh, heads, shared) &&
         stride_ok(sn, n, false);
}

// How a call is cut up, and its scratch.
struct MaPlan {
  bool tensor = false;  // the tcgen05 kernels take it
  int slots = 1;        // row tiles a block (tcgen05 forward)
  bool spread = false;  // one tile of up to 32 rows, each in four lanes
  int splits = 1;
  int q_tiles = 0, k_tiles = 0;
  int64_t blocks = 0;  // of the forward kernel, or of the one that makes dq
  // byte offsets into the workspace
  int64_t qdoc = 0, kdoc = 0, qrange = 0, krange = 0, part_o = 0, part_lse = 0, delta = 0;
  int64_t bytes = 0;
};

// Key splits of `items` blocks' worth of rows: the count with the least waves x (tiles a
// block + what a block costs besides, about `fixed` tiles), and no more than one split per
// `least` tiles, below which joining costs more than it saves.
int ma_splits(int64_t items, int64_t k_tiles, int64_t at_once, int fixed, int least) {
  if (items <= 0 || k_tiles <= 0) return 1;
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int64_t s = 1; s <= std::max<int64_t>(1, k_tiles / least) && s <= xfb::kMaMaxSplits; ++s) {
    const int64_t per = ceil_div(k_tiles, s);
    if (ceil_div(k_tiles, per) != s) continue;  // a split would start past the last tile
    const int64_t cost = ceil_div(items * s, at_once) * (per + fixed) * 16 + s;
    if (cost < best_cost) {
      best_cost = cost;
      best = static_cast<int>(s);
    }
    if (items * s > 8 * at_once) break;
  }
  return best;
}

// They also take the cap as cap - 2 cap r, which is off by 2^-23 cap: up to here that is 1e-4 of a
// score's unit, well under the rounding of P.
constexpr double kMaMostCap = 1024.0;

// The tcgen05 kernels take a positive scale (maxima are taken of raw products, masks are raw
// products of -inf) and bf16 whose rows TMA can address (16-byte strides and bases, head dims
// in eights) and up to 128 query heads a K/V head (64 in the backward pass, whose tiles have 64
// rows); everything else runs on the CUDA cores.
bool ma_tensor(const xfb_masked_attention_args& a, bool backward) {
  if (a.dtype != XFB_BF16 || a.d % 8 != 0 || a.nk == 0 || a.nq == 0 ||
      !(static_cast<float>(a.scale) > 0.f) || a.softcap > kMaMostCap)
    return false;
  const int64_t rep = a.heads / a.kv_heads;
  if (rep < 1 || rep > (backward ? 64 : 128)) return false;
  return ma_tma_ok(a.q, a.q_sb, a.q_sh, a.q_sn, a.batch, a.heads, a.nq, false) &&
         ma_tma_ok(a.k, a.k_sb, a.k_sh, a.k_sn, a.batch, a.kv_heads, a.nk, true) &&
         ma_tma_ok(a.v, a.v_sb, a.v_sh, a.v_sn, a.batch, a.kv_heads, a.nk, true) &&
         ma_tma_ok(a.out, a.out_sb, a.out_sh, a.out_sn, a.batch, a.heads, a.nq, false) &&
         aligned16(a.out_low) &&
         (!backward ||
          (ma_tma_ok(a.dout, a.dout_sb, a.dout_sh, a.dout_sn, a.batch, a.heads, a.nq, false) &&
           ma_tma_ok(a.dq, a.dq_sb, a.dq_sh, a.dq_sn, a.batch, a.heads, a.nq, false) &&
           ma_tma_ok(a.dk, a.dk_sb, a.dk_sh, a.dk_sn, a.batch, a.kv_heads, a.nk, false) &&
           ma_tma_ok(a.dv, a.dv_sb, a.dv_sh, a.dv_sn, a.batch, a.kv_heads, a.nk, false)));
}

MaPlan ma_plan(const xfb_masked_attention_args& a, bool backward) {
  MaPlan p;
  const int64_t rep = a.heads / a.kv_heads;
  const int64_t rows = a.nq * rep;
  const int64_t sms = sm_count_or_default();
  p.tensor = ma_tensor(a, backward);
  int64_t items;
  if (p.tensor) {
    p.q_tiles = static_cast<int>(ceil_div(a.nq, 128 / rep));
    p.k_tiles = static_cast<int>(ceil_div(a.nk, xfb::kMtKeys));
    // Two row tiles a block let one tile's softmax run under the other's products; with fewer
    // than two tiles an SM that would leave SMs empty, so a block takes one, and
    // splits the keys where even that does not fill the GPU.
    p.slots = !backward && a.batch * a.kv_heads * p.q_tiles >= 2 * sms &&
                      p.k_tiles <= xfb::kMtMaxTiles
                  ? 2
                  : 1;
    items = a.batch * a.kv_heads * ceil_div(p.q_tiles, p.slots);
    p.spread = !backward && p.slots == 1 && rows <= 32;
    if (p.slots == 1 && !backward) {
      p.splits = ma_splits(items, p.k_tiles, sms, 8, 4);
      // a block's list holds so many tiles
      const int64_t least = ceil_div(p.k_tiles, xfb::kMtMaxTiles);
      if (least > xfb::kMaMaxSplits) p.tensor = false;
      if (p.splits < least) p.splits = static_cast<int>(ceil_div(p.k_tiles, ceil_div(p.k_tiles, least)));
    }
    // the backward pass has no splits: its lists hold tiles of 64 keys, and of 64 rows
    if (backward && std::max(ceil_div(a.nk, xfb::kMtStream),
                             ceil_div(a.nq, xfb::kMtStream / std::min<int64_t>(rep, 64))) >
                        xfb::kMtMaxStream)
      p.tensor = false;
  }
  if (!p.tensor) {
    p.slots = 1;
    p.splits = 1;
    p.q_tiles = static_cast<int>(ceil_div(rows, xfb::kMaTile));
    p.k_tiles = static_cast<int>(ceil_div(a.nk, xfb::kMaTile));
    items = a.batch * a.kv_heads * p.q_tiles;
    if (!backward && items > 0) p.splits = ma_splits(items, p.k_tiles, sms * 2, 2, 4);
  }
  p.blocks = items * p.splits;
  int64_t at = 0;
  const auto take = [&at](int64_t bytes) {
    const int64_t here = round_up(at, 256);
    at = here + bytes;
    return here;
  };
  if (a.q_documents != nullptr) {
    const int64_t nqp = round_up(a.nq, 128), nkp = round_up(a.nk, 128);
    p.qdoc = take(a.batch * nqp * 4);
    p.kdoc = take(a.batch * nkp * 4);
    p.qrange = take(a.batch * (nqp / 64) * 16);
    p.krange = take(a.batch * (nkp / 64) * 16);
  }
  const int64_t all_rows = a.batch * a.heads * a.nq;
  if (p.splits > 1) {
    p.part_o = take(p.splits * all_rows * a.d * 4);
    p.part_lse = take(p.splits * all_rows * 4);
  }
  if (backward) p.delta = take(all_rows * 4);
  p.bytes = at;
  return p;
}

int ma_check(const xfb_masked_attention_args* args) {
  XFB_REQUIRE(args != nullptr, "masked attention needs its arguments");
  const xfb_masked_attention_args& a = *args;
  XFB_REQUIRE(a.dtype == XFB_F32 || a.dtype == XFB_BF16, "attention data must be f32 or bf16");
  XFB_REQUIRE(a.batch >= 0 && a.heads >= 0 && a.nq >= 0 && a.nk >= 0,
              "attention sizes must be non-negative");
  XFB_REQUIRE(a.kv_heads >= 1 && a.heads % a.kv_heads == 0,
              "query heads must be a multiple of K/V heads");
  XFB_REQUIRE(a.d >= 1 && a.d <= 128, "attention head dimension must be in [1, 128]");
  XFB_REQUIRE(a.batch <= 65535, "attention batch must be at most 65535");
  XFB_REQUIRE(a.heads <= (1 << 20) && a.nk < (1 << 30) &&
                  a.nq * std::max<int64_t>(a.heads / a.kv_heads, 1) < (1 << 30),
              "attention is too long");
  XFB_REQUIRE(std::isfinite(static_cast<float>(a.scale)), "attention scale must be finite in f32");
  XFB_REQUIRE(std::isfinite(a.softcap) && a.softcap >= 0,
              "attention softcap must be finite and non-negative (0 = none)");
  XFB_REQUIRE(a.prefix == nullptr || a.causal, "a prefix needs causal attention");
  XFB_REQUIRE((a.q_documents == nullptr) == (a.k_documents == nullptr),
              "documents are given for queries and keys, or for neither");
  XFB_REQUIRE(a.out_low == nullptr || a.dtype == XFB_BF16, "out_low goes with bf16 data");
  return XFB_OK;
}

bool ma_vec4(const void* p, int64_t sb, int64_t sh, int64_t sn, int size) {
  return p == nullptr || (sb % 4 == 0 && sh % 4 == 0 && sn % 4 == 0 &&
                          reinterpret_cast<uintptr_t>(p) % (4 * size) == 0);
}

// Device arguments of a call; `ws` has ma_plan's bytes.
xfb::MaskedArgs ma_args(const xfb_masked_attention_args& a, const MaPlan& p, uint8_t* ws,
                        bool backward) {
  xfb::MaskedArgs m{};
  // (the stride of a dimension of size one is never used, and may be one that no tensor map takes)
  const auto tensor = [&a](const void* ptr, int64_t sb, int64_t sh, int64_t sn, int64_t heads,
                           int64_t n) {
    return xfb::MaTensor{const_cast<void*>(ptr), a.batch > 1 ? sb : 0, heads > 1 ? sh : 0,
                         n > 1 ? sn : 0};
  };
  m.q = tensor(a.q, a.q_sb, a.q_sh, a.q_sn, a.heads, a.nq);
  m.k = tensor(a.k, a.k_sb, a.k_sh, a.k_sn, a.kv_heads, a.nk);
  m.v = tensor(a.v, a.v_sb, a.v_sh, a.v_sn, a.kv_heads, a.nk);
  m.out = tensor(a.out, a.out_sb, a.out_sh, a.out_sn, a.heads, a.nq);
  m.lse = a.lse;
  m.low = static_cast<bf16*>(a.out_low);
  m.slopes = a.slopes;
  m.prefix = a.prefix;
  m.B = static_cast<int>(a.batch);
  m.H = static_cast<int>(a.heads);
  m.G = static_cast<int>(a.kv_heads);
  m.rep = static_cast<int>(a.heads / a.kv_heads);
  m.nq = static_cast<int>(a.nq);
  m.nk = static_cast<int>(a.nk);
  m.d = static_cast<int>(a.d);
  m.off = m.nk - m.nq;
  m.causal = a.causal != 0;
  m.scale = static_cast<float>(a.scale);
  // A cap is held where it and its inverse are normal f32 numbers: below 1e-30 all scores are one
  // to f32, and above 2^100 no score (2^88 in f32, without an infinity in a product) is bent.
  const double cap = a.softcap > 0x1p100 ? 0.0 : a.softcap > 0 ? std::max(a.softcap, 1e-30) : 0.0;
  m.cap = static_cast<float>(cap);
  m.inv_cap = cap > 0 ? static_cast<float>(1.0 / cap) : 0.f;
  m.q_tiles = p.q_tiles;
  m.k_tiles = p.k_tiles;
  m.splits = p.splits;
  if (a.q_documents != nullptr) {
    const int64_t nqp = round_up(a.nq, 128), nkp = round_up(a.nk, 128);
    m.qdoc = reinterpret_cast<const int32_t*>(ws + p.qdoc);
    m.kdoc = reinterpret_cast<const int32_t*>(ws + p.kdoc);
    m.qrange = reinterpret_cast<const int4*>(ws + p.qrange);
    m.krange = reinterpret_cast<const int4*>(ws + p.krange);
    m.qdoc_sb = nqp;
    m.kdoc_sb = nkp;
    m.qrange_sb = nqp / 64;
    m.krange_sb = nkp / 64;
  }
  if (p.splits > 1) {
    m.part_o = reinterpret_cast<float*>(ws + p.part_o);
    m.part_lse = reinterpret_cast<float*>(ws + p.part_lse);
  }
  const int size = a.dtype == XFB_F32 ? 4 : 2;
  m.vec4 = a.d % 4 == 0 && ma_vec4(a.q, a.q_sb, a.q_sh, a.q_sn, size) &&
           ma_vec4(a.k, a.k_sb, a.k_sh, a.k_sn, size) && ma_vec4(a.v, a.v_sb, a.v_sh, a.v_sn, size);
  if (backward) {
    m.dout = tensor(a.dout, a.dout_sb, a.dout_sh, a.dout_sn, a.heads, a.nq);
    m.dq = tensor(a.dq, a.dq_sb, a.dq_sh, a.dq_sn, a.heads, a.nq);
    m.dk = tensor(a.dk, a.dk_sb, a.dk_sh, a.dk_sn, a.kv_heads, a.nk);
    m.dv = tensor(a.dv, a.dv_sb, a.dv_sh, a.dv_sn, a.kv_heads, a.nk);
    m.delta = reinterpret_cast<float*>(ws + p.delta);
    m.vec4 = m.vec4 && ma_vec4(a.dout, a.dout_sb, a.dout_sh, a.dout_sn, size);
  }
  return m;
}

int ma_documents(const xfb_masked_attention_args& a, const MaPlan& p, uint8_t* ws,
                 cudaStream_t st) {
  if (a.q_documents == nullptr) return XFB_OK;
  const int64_t nqp = round_up(a.nq, 128), nkp = round_up(a.nk, 128);
  xfb::MaDocs d{};
  d.in[0] = a.q_documents;
  d.in[1] = a.k_documents;
  d.in_sb[0] = a.q_documents_sb;
  d.in_sb[1] = a.k_documents_sb;
  d.n[0] = static_cast<int>(a.nq);
  d.n[1] = static_cast<int>(a.nk);
  d.out[0] = reinterpret_cast<int32_t*>(ws + p.qdoc);
  d.out[1] = reinterpret_cast<int32_t*>(ws + p.kdoc);
  d.out_sb[0] = nqp;
  d.out_sb[1] = nkp;
  d.range[0] = reinterpret_cast<int4*>(ws + p.qrange);
  d.range[1] = reinterpret_cast<int4*>(ws + p.krange);
  d.range_sb[0] = nqp / 64;
  d.range_sb[1] = nkp / 64;
  const int64_t ranges = std::max(nqp, nkp) / 64;
  if (ranges == 0) return XFB_OK;
  const dim3 grid(static_cast<unsigned>(ceil_div(ranges, 8)), static_cast<unsigned>(a.batch), 2);
  xfb::ma_documents_kernel<<<grid, 256, 0, st>>>(d);
  XFB_LAUNCHED();
  return XFB_OK;
}

// Runs f with the padded head dim of the CUDA-core kernels.
template <class F>
int ma_with_dim(int64_t d, F f) {
  if (d <= 32) return f(std::integral_constant<int, 32>());
  if (d <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

// Tensor maps of K or V: boxes of 64 dims x 128 keys; a broadcast head or batch
// dimension has size 1 and the coordinate 0.
int mt_key_map(CUtensorMap* map, xfb::MtMap* mul, const xfb::MaTensor& t, const xfb::MaskedArgs& m,
               int rows) {
  mul->head = t.sh == 0 ? 0 : 1;
  mul->batch = t.sb == 0 ? 0 : 1;
  const uint64_t dims[4] = {uint64_t(m.d), uint64_t(m.nk), uint64_t(mul->head ? m.G : 1),
                            uint64_t(mul->batch ? m.B : 1)};
  const uint64_t strides[3] = {uint64_t(t.sn) * 2, uint64_t(t.sh) * 2, uint64_t(t.sb) * 2};
  const uint32_t box[4] = {64, uint32_t(rows), 1, 1};
  return make_map_nd(map, false, 4, t.p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Tensor map of a row tensor: boxes of 64 dims x rep heads x `queries` queries.
int mt_row_map(CUtensorMap* map, const xfb::MaTensor& t, const xfb::MaskedArgs& m, int queries) {
  const uint64_t dims[5] = {uint64_t(m.d), uint64_t(m.rep), uint64_t(m.nq), uint64_t(m.G),
                            uint64_t(m.B)};
  const uint64_t strides[4] = {uint64_t(t.sh) * 2, uint64_t(t.sn) * 2, uint64_t(t.sh) * m.rep * 2,
                               uint64_t(t.sb) * 2};
  const uint32_t box[5] = {64, uint32_t(m.rep), uint32_t(queries), 1, 1};
  return make_map_nd(map, false, 5, t.p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Runs f with the score variant of the call: raw products, a cap, a distance, or both.
template <class F>
int mt_with_score(const xfb::MaskedArgs& m, F f) {
  using Yes = std::true_type;
  using No = std::false_type;
  const bool slopes = m.slopes != nullptr;
  if (m.cap > 0.f) return slopes ? f(Yes(), Yes()) : f(Yes(), No());
  return slopes ? f(No(), Yes()) : f(No(), No());
}

template <int DP, int SLOTS>
int mt_forward_launch(const xfb::MaskedArgs& m, const MaPlan& p, cudaStream_t st) {
  using L = xfb::MtForward<DP, SLOTS>;
  CUtensorMap tq, tk, tv;
  xfb::MtMap mk, mv;
  XFB_TRY(mt_row_map(&tq, m.q, m, (L::kSpread ? 32 : 128) / m.rep));
  XFB_TRY(mt_key_map(&tk, &mk, m.k, m, xfb::kMtKeys));
  XFB_TRY(mt_key_map(&tv, &mv, m.v, m, xfb::kMtKeys));
  return mt_with_score(m, [&](auto cap, auto slopes) -> int {
    auto kernel =
        xfb::mt_forward_kernel<DP, SLOTS, decltype(cap)::value, decltype(slopes)::value>;
    XFB_TRY(set_smem(kernel, L::kMostBytes));
    const int bytes = L::launch_bytes(ceil_div(m.k_tiles, m.splits));
    kernel<<<static_cast<unsigned>(p.blocks), L::kThreads, bytes, st>>>(tq, tk, tv, mk,
                                                                                mv, m);
    XFB_LAUNCHED();
    return XFB_OK;
  });
}

int mt_forward(const xfb::MaskedArgs& m, const MaPlan& p, cudaStream_t st) {
  if (m.d <= 64) {
    if (p.spread) return mt_forward_launch<64, 0>(m, p, st);
    return p.slots == 2 ? mt_forward_launch<64, 2>(m, p, st) : mt_forward_launch<64, 1>(m, p, st);
  }
  if (p.spread) return mt_forward_launch<128, 0>(m, p, st);
  return p.slots == 2 ? mt_forward_launch<128, 2>(m, p, st) : mt_forward_launch<128, 1>(m, p, st);
}

template <typename T>
int ma_forward(const xfb::MaskedArgs& m, const MaPlan& p, cudaStream_t st) {
  if (p.tensor) {
    XFB_TRY(mt_forward(m, p, st));
  } else XFB_TRY(ma_with_dim(m.d, [&](auto dim) -> int {
    constexpr int DP = decltype(dim)::value;
    auto kernel = xfb::ma_forward_kernel<T, DP>;
    XFB_TRY(set_smem(kernel, xfb::MaForwardSmem<DP>::kBytes));
    kernel<<<static_cast<unsigned>(p.blocks), 256, xfb::MaForwardSmem<DP>::kBytes, st>>>(m);
    XFB_LAUNCHED();
    return XFB_OK;
  }));
  if (p.splits > 1) {
    const int64_t rows = int64_t(m.B) * m.H * m.nq;
    xfb::ma_join_kernel<T><<<static_cast<unsigned>(rows), 128, 0, st>>>(m);
    XFB_LAUNCHED();
  }
  return XFB_OK;
}

// In calls of up to this many queries and keys the backward pass takes P and dX in two parts (eight tiles of 64;
// 2 x 8 heads of 64: 13.8 us in one part and 14.1 in two at 64 tokens, 25.8 and 28.7 at 512).
constexpr int kMtTwoParts = 512;

template <int DP, bool TWO>
int mt_backward_launch(const xfb::MaskedArgs& m, cudaStream_t st) {
  using L = xfb::MtBackward<DP>;
  CUtensorMap q128, q64, o128, o64, out128, k128, k64, v128, v64;
  xfb::MtMap mk, mv;
  XFB_TRY(mt_row_map(&q128, m.q, m, 128 / m.rep));
  XFB_TRY(mt_row_map(&o128, m.dout, m, 128 / m.rep));
  XFB_TRY(mt_row_map(&out128, m.out, m, 128 / m.rep));
  XFB_TRY(mt_row_map(&q64, m.q, m, xfb::kMtStream / m.rep));
  XFB_TRY(mt_row_map(&o64, m.dout, m, xfb::kMtStream / m.rep));
  XFB_TRY(mt_key_map(&k128, &mk, m.k, m, 128));
  XFB_TRY(mt_key_map(&v128, &mv, m.v, m, 128));
  XFB_TRY(mt_key_map(&k64, &mk, m.k, m, xfb::kMtStream));
  XFB_TRY(mt_key_map(&v64, &mv, m.v, m, xfb::kMtStream));
  const unsigned heads = static_cast<unsigned>(m.B) * m.G;
  return mt_with_score(m, [&](auto cap, auto slopes) -> int {
    constexpr bool kCap = decltype(cap)::value, kSlopes = decltype(slopes)::value;
    auto dq = xfb::mt_backward_kernel<DP, false, kCap, kSlopes, TWO>;
    XFB_TRY(set_smem(dq, L::kMostBytes));
    const int key_list = L::launch_bytes(ceil_div(m.nk, xfb::kMtStream));
    dq<<<heads * m.q_tiles, L::kThreads, key_list, st>>>(q128, o128, k64, v64, out128, mk,
                                                               mv, m);
    XFB_LAUNCHED();
    auto kv = xfb::mt_backward_kernel<DP, true, kCap, kSlopes, TWO>;
    XFB_TRY(set_smem(kv, L::kMostBytes));
    const int row_list = L::launch_bytes(ceil_div(m.nq, xfb::kMtStream / m.rep));
    const unsigned key_tiles = static_cast<unsigned>(ceil_div(m.nk, 128));
    kv<<<heads * key_tiles, L::kThreads, row_list, st>>>(k128, v128, q64, o64, out128, mk,
                                                               mv, m);
    XFB_LAUNCHED();
    return XFB_OK;
  });
}

template <typename T>
int ma_backward(const xfb::MaskedArgs& m, const MaPlan& p, cudaStream_t st) {
  const int64_t rows = int64_t(m.B) * m.H * m.nq;
  if (p.tensor) {
    const bool two = m.nq <= kMtTwoParts && m.nk <= kMtTwoParts;
    if (m.d <= 64) return two ? mt_backward_launch<64, true>(m, st) : mt_backward_launch<64, false>(m, st);
    return two ? mt_backward_launch<128, true>(m, st) : mt_backward_launch<128, false>(m, st);
  }
  xfb::ma_delta_kernel<T><<<static_cast<unsigned>(ceil_div(rows, 128)), 128, 0, st>>>(m);
  XFB_LAUNCHED();
  return ma_with_dim(m.d, [&](auto dim) -> int {
    constexpr int DP = decltype(dim)::value;
    constexpr int kBytes = xfb::MaBackwardSmem<DP>::kBytes;
    auto kv = xfb::ma_backward_kv_kernel<T, DP>;
    XFB_TRY(set_smem(kv, kBytes));
    kv<<<static_cast<unsigned>(int64_t(m.B) * m.G * m.k_tiles), 256, kBytes, st>>>(m);
    XFB_LAUNCHED();
    auto dq = xfb::ma_backward_q_kernel<T, DP>;
    XFB_TRY(set_smem(dq, kBytes));
    dq<<<static_cast<unsigned>(p.blocks), 256, kBytes, st>>>(m);
    XFB_LAUNCHED();
    return XFB_OK;
  });
}

// log2 of the entries of a hash table of n ids: at least twice as many.
int ma_id_bits(int64_t n) {
  int bits = 1;
  while ((int64_t(1) << bits) < 2 * n) ++bits;
  return bits;
}

// Sets a strided [B][heads][n][d] tensor to zero.
template <typename T>
__global__ void ma_zero_kernel(xfb::MaTensor t, int64_t heads, int64_t n, int64_t d, int64_t total) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t row = i / d, bh = row / n;
    static_cast<T*>(t.p)[(bh / heads) * t.sb + (bh % heads) * t.sh + (row - bh * n) * t.sn +
                         (i - row * d)] = xfb::ln_round<T>(0.f);
  }
}
int ma_zero(const xfb::MaTensor& t, int dtype, int64_t B, int64_t heads, int64_t n, int64_t d,
            cudaStream_t st) {
  const int64_t total = B * heads * n * d;
  if (total == 0) return XFB_OK;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(ceil_div(total, 256), 4096));
  if (dtype == XFB_F32) {
    ma_zero_kernel<float><<<blocks, 256, 0, st>>>(t, heads, n, d, total);
  } else {
    ma_zero_kernel<bf16><<<blocks, 256, 0, st>>>(t, heads, n, d, total);
  }
  XFB_LAUNCHED();
  return XFB_OK;
}

}  // namespace

extern "C" {

XFB_API int64_t xfb_number_documents_workspace(int64_t batch, int64_t nq, int64_t nk) {
  if (batch <= 0 || nq < 0 || nk < 0 || nq >= (1 << 30) || nk >= (1 << 30) || batch > 65535) return 0;
  return (batch << ma_id_bits(nq + nk)) * 12;
}

XFB_API int xfb_number_documents(const int64_t* q_ids, int64_t q_sb, int64_t nq,
                                 const int64_t* k_ids, int64_t k_sb, int64_t nk, int64_t batch,
                                 int32_t* q_out, int32_t* k_out, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    XFB_REQUIRE(batch >= 0 && nq >= 0 && nk >= 0, "document sizes must be non-negative");
    XFB_REQUIRE(batch <= 65535 && nq < (1 << 30) && nk < (1 << 30), "documents are too many");
    if (batch == 0 || nq + nk == 0) return XFB_OK;
    XFB_REQUIRE(nq == 0 || (q_ids != nullptr && q_out != nullptr), "documents need query ids");
    XFB_REQUIRE(nk == 0 || (k_ids != nullptr && k_out != nullptr), "documents need key ids");
    xfb::MaIds a{q_ids, k_ids, q_sb, k_sb, static_cast<int>(nq), static_cast<int>(nk), q_out, k_out};
    a.bits = ma_id_bits(nq + nk);
    const int64_t entries = batch << a.bits;
    Carver cv{static_cast<uint8_t*>(workspace), entries * 12, workspace_bytes};
    XFB_TRY(check_workspace(cv, workspace, workspace_bytes));
    a.ids = static_cast<unsigned long long*>(workspace);
    a.first = reinterpret_cast<uint32_t*>(a.ids + entries);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    XFB_CUDA(cudaMemsetAsync(workspace, 0xFF, entries * 12, st));
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(nq + nk, 256), 4096)),
                    static_cast<unsigned>(batch));
    xfb::ma_ids_enter_kernel<<<grid, 256, 0, st>>>(a);
    XFB_LAUNCHED();
    xfb::ma_ids_number_kernel<<<grid, 256, 0, st>>>(a);
    XFB_LAUNCHED();
    return XFB_OK;
  });
}

XFB_API int64_t xfb_masked_attention_workspace(const xfb_masked_attention_args* args,
                                               int backward) {
  int64_t bytes = 0;
  guarded([&]() -> int {
    XFB_TRY(ma_check(args));
    bytes = ma_plan(*args, backward != 0).bytes;
    return XFB_OK;
  });
  return bytes;
}

XFB_API int xfb_masked_attention(const xfb_masked_attention_args* args, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    XFB_TRY(ma_check(args));
    const xfb_masked_attention_args& a = *args;
    if (a.batch == 0 || a.heads == 0 || a.nq == 0) return XFB_OK;
    XFB_REQUIRE(a.q != nullptr && a.out != nullptr, "masked attention needs q and out");
    XFB_REQUIRE(a.nk == 0 || (a.k != nullptr && a.v != nullptr), "masked attention needs k and v");
    const MaPlan p = ma_plan(a, false);
    XFB_REQUIRE(p.blocks <= INT32_MAX, "attention has too many tiles");
    Carver cv{static_cast<uint8_t*>(workspace), p.bytes, workspace_bytes};
    XFB_TRY(check_workspace(cv, workspace, workspace_bytes));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    XFB_TRY(ma_documents(a, p, ws, st));
    const xfb::MaskedArgs m = ma_args(a, p, ws, false);
    return a.dtype == XFB_F32 ? ma_forward<float>(m, p, st) : ma_forward<bf16>(m, p, st);
  });
}

XFB_API int xfb_masked_attention_backward(const xfb_masked_attention_args* args, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    XFB_TRY(ma_check(args));
    const xfb_masked_attention_args& a = *args;
    if (a.batch == 0) return XFB_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const MaPlan p = ma_plan(a, true);
    const xfb::MaskedArgs m = ma_args(a, p, ws, true);
    if (a.heads == 0 || a.nq == 0 || a.nk == 0) {  // what there is of gradients is zero
      if (a.dq) XFB_TRY(ma_zero(m.dq, a.dtype, a.batch, a.heads, a.nq, a.d, st));
      if (a.dk) XFB_TRY(ma_zero(m.dk, a.dtype, a.batch, a.kv_heads, a.nk, a.d, st));
      if (a.dv) XFB_TRY(ma_zero(m.dv, a.dtype, a.batch, a.kv_heads, a.nk, a.d, st));
      return XFB_OK;
    }
    XFB_REQUIRE(a.q && a.k && a.v && a.out && a.lse && a.dout && a.dq && a.dk && a.dv,
                "the attention gradient needs q, k, v, out, lse, dout, dq, dk and dv");
    XFB_REQUIRE(a.dtype == XFB_F32 || a.out_low != nullptr,
                "the bf16 attention gradient needs out_low");
    XFB_REQUIRE(p.blocks <= INT32_MAX && a.batch * a.kv_heads * p.k_tiles <= INT32_MAX,
                "attention has too many tiles");
    Carver cv{ws, p.bytes, workspace_bytes};
    XFB_TRY(check_workspace(cv, workspace, workspace_bytes));
    XFB_TRY(ma_documents(a, p, ws, st));
    return a.dtype == XFB_F32 ? ma_backward<float>(m, p, st) : ma_backward<bf16>(m, p, st);
  });
}

}  // extern "C"
