// qrb200 -- C ABI of the layer operators: the root-mean-square norm (qrb_norm.cuh) and the matrix
// product with its epilogue (qrb_linear.cuh).  Every entry point checks its arguments before it
// touches the GPU, enqueues on the caller's stream and returns a QRB200_* status.
#include "../../include/qrb200_layer.h"
#include "qrb_host.h"
#include "qrb_linear.cuh"
#include "qrb_linear_pair.cuh"
#include "qrb_norm.cuh"

#include <algorithm>
#include <atomic>
#include <mutex>
#include <utility>

namespace qrb {
namespace {

constexpr int kSMs = 148;

bool float_type(int32_t t) { return t == QRB200_F32 || t == QRB200_BF16 || t == QRB200_F16; }
int esize(int32_t t) { return t == QRB200_F32 ? 4 : (t == QRB200_E4M3 ? 1 : 2); }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Rows of this base and stride (elements) all start on 16 bytes.
bool rows_on16(const void* p, int64_t ld, int es) { return on16(p) && (ld * es & 15) == 0; }

// Launches one kernel (see qrb_pdl.cuh) and counts it.
template <typename... P, typename... A>
int launch_as(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, unsigned cluster, bool early, A&&... args) {
  const cudaError_t e = launch_kernel(kernel, grid, block, smem, st, cluster, early, std::forward<A>(args)...);
  count_launches(1);
  if (note(e) == cudaSuccess) return QRB200_OK;
  cudaGetLastError();  // not left for a later call to find
  return QRB200_ERR_CUDA;
}
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  return launch_as(kernel, grid, block, smem, st, 0, true, std::forward<A>(args)...);
}

// Lets a kernel use `bytes` of dynamic shared memory, once per context (`ready`: each device's context
// that it is done for).
using Ready = std::atomic<unsigned long long>[128];
int raise_smem(const void* kernel, int bytes, Ready& ready) {
  int dev = 0;
  unsigned long long ctx = 0;
  if (note(current_ctx(&dev, &ctx)) != cudaSuccess) return QRB200_ERR_CUDA;
  if (ready[dev].load(std::memory_order_relaxed) == ctx) return QRB200_OK;
  if (note(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) != cudaSuccess)
    return QRB200_ERR_CUDA;
  ready[dev].store(ctx, std::memory_order_relaxed);
  return QRB200_OK;
}

// A workspace may start anywhere: its first byte on 16 is where it is used from, so the sizes that
// the queries report hold 15 bytes more than the buffers in it (TMA and 16-byte stores need the
// alignment, and what is planned for aligned buffers would not fit the copies of others).
size_t workspace_size(size_t need) { return need ? need + 15 : 0; }

// Device memory for one call: the caller's, or our own when there is none, freed in stream order.
struct Scratch {
  void* p = nullptr;
  cudaStream_t st;
  bool own = false;
  explicit Scratch(cudaStream_t s) : st(s) {}
  int get(void* given, size_t given_bytes, size_t need) {
    if (!need) return QRB200_OK;
    if (given) {
      const size_t skip = -reinterpret_cast<uintptr_t>(given) & 15;
      if (given_bytes < need || given_bytes - need < skip) return QRB200_ERR_WORKSPACE;
      p = static_cast<char*>(given) + skip;
      return QRB200_OK;
    }
    if (note(cudaMallocAsync(&p, need, st)) != cudaSuccess) return QRB200_ERR_CUDA;
    own = true;
    return QRB200_OK;
  }
  ~Scratch() { if (own) cudaFreeAsync(p, st); }
};

// ------------------------------------------------------------------ norm
// Threads of a row, groups of 8 elements a thread, rows a block.  Up to 1024 elements a warp or a part
// of one takes the row (128 threads a block).  Longer rows of 16-bit vectors: with enough rows to fill the
// GPU, 4 groups a thread (more bytes in flight, fewer barriers); with few rows, one.  float32
// groups take twice the registers: 2 at most.  Rows of single elements: 32, 256 or 512 threads.
struct Shape { int nt, vpt, rows; };
Shape single_shape(int dim, int most_256) {  // most_256: longest row that 256 threads take
  const int nt = dim <= 1024 ? 32 : (dim <= most_256 ? 256 : 512);
  int vpt = 1;
  while (nt * vpt * 8 < dim) vpt *= 2;
  return {nt, vpt, nt == 32 ? 4 : 1};
}
Shape norm_shape(int64_t rows, int dim, bool wide, bool vec) {
  const int vecs = (dim + 7) / 8;
  if (!vec) return single_shape(dim, 8192);
  if (dim <= 1024 && rows > kSMs) {
    int vpt = vecs <= 32 ? 1 : (vecs <= 64 || wide ? 2 : 4), nt = 4;
    while (nt * vpt < vecs) nt *= 2;
    if (nt <= 32) return {nt, vpt, 128 / nt};
    return {nt, vpt, 1};
  }
  const int most = wide ? 2 : 4;
  int vpt = 1;
  if (rows > 2 * kSMs) vpt = vecs <= 128 ? 1 : (vecs <= 256 ? 2 : most);
  while ((vecs + vpt - 1) / vpt > norm::max_threads(vpt)) vpt *= 2;
  const int nt = std::max(32, ((vecs + vpt - 1) / vpt + 31) / 32 * 32);
  return {nt, vpt, 1};
}

template <typename TX, typename TH, bool RES, bool Q8, bool NORM>
int launch_fwd(const norm::FwdArgs& a, bool vec, cudaStream_t st) {
  constexpr bool wide = sizeof(TX) == 4 || sizeof(TH) == 4;
  if (a.dim > norm::kRegDim) {
    return launch(norm::fwd_long_kernel<TX, TH, Q8, NORM>, (unsigned)a.rows, norm::kMaxThreads, 0, st, a);
  }
  const Shape s = norm_shape(a.rows, a.dim, wide, vec);
  const dim3 block(s.nt, s.rows);
  const unsigned grid = (unsigned)((a.rows + s.rows - 1) / s.rows);
#define QRB_FWD(V, NT) launch(norm::fwd_kernel<TX, TH, RES, Q8, NORM, V, NT>, grid, block, 0, st, a)
  if (vec) {
    if (s.vpt == 1) return QRB_FWD(1, 0);
    if (s.vpt == 2 || wide) return QRB_FWD(2, 0);
    if constexpr (!wide) return QRB_FWD(4, 0);
  }
  if (s.nt == 32) return s.vpt == 1 ? QRB_FWD(1, 32) : s.vpt == 2 ? QRB_FWD(2, 32) : QRB_FWD(4, 32);
  if (s.nt == 256) return s.vpt == 1 ? QRB_FWD(1, 256) : s.vpt == 2 ? QRB_FWD(2, 256) : QRB_FWD(4, 256);
  return QRB_FWD(4, 512);
#undef QRB_FWD
}

template <typename TX>
int launch_norm(const norm::FwdArgs& a, bool q8, bool stream_f32, bool vec, cudaStream_t st) {
  if (!a.res) return q8 ? launch_fwd<TX, TX, false, true, true>(a, vec, st) : launch_fwd<TX, TX, false, false, true>(a, vec, st);
  if (stream_f32) return q8 ? launch_fwd<TX, float, true, true, true>(a, vec, st) : launch_fwd<TX, float, true, false, true>(a, vec, st);
  return q8 ? launch_fwd<TX, TX, true, true, true>(a, vec, st) : launch_fwd<TX, TX, true, false, true>(a, vec, st);
}

// Rows of no elements have a scale all the same.
int scales_of_empty_rows(float* scale, int64_t rows, void* stream) {
  if (!rows || !scale) return QRB200_OK;
  if (rows >= ((int64_t)1 << 31)) return QRB200_ERR_INVALID_ARG;
  const norm::FwdArgs a{nullptr, 0, nullptr, 0, nullptr, 0, nullptr, scale, nullptr, rows, 0, 0.f};
  return launch_fwd<float, float, false, true, false>(a, true, static_cast<cudaStream_t>(stream));
}

// Shape, rows of look-ahead and grid of the backward kernel; parts = rows of partial weight gradients
// it writes, one a block.  A block walks over its rows, so the grid is what the GPU holds at once: 128
// registers a thread (64 for rows of single elements up to 4096, which have no look-ahead and need
// the warps), and shared memory for `depth` rows.  As many groups a thread as registers
// allow: the two reductions of a row cost the same for few elements as for many.
constexpr int kBwdRing = 220 * 1024;  // shared memory of a block at most
struct BwdPlan { Shape s; int depth; size_t smem; int64_t grid, parts; };
BwdPlan bwd_plan(int64_t rows, int dim, int es, int hs, bool vec) {
  BwdPlan p{};
  if (dim > norm::kRegDim) {
    p.s = {norm::kMaxThreads, 0, 1};
    p.grid = p.parts = std::min<int64_t>(rows, 2 * kSMs);
    return p;
  }
  if (!vec) {
    p.s = single_shape(dim, 4096);
  } else {
    const int vecs = (dim + 7) / 8;
    const int vpt = vecs <= 32 ? 1 : (vecs <= 64 ? 2 : 4);
    int nt = 4;
    while (nt < 32 && nt * vpt < vecs) nt *= 2;
    if (nt * vpt < vecs) nt = ((vecs + vpt - 1) / vpt + 31) / 32 * 32;
    p.s = {nt, vpt, nt <= 32 ? 128 / nt : 1};
  }
  const int threads = p.s.nt * p.s.rows;
  const size_t row = (size_t)threads * p.s.vpt * 8 * (es + 2 * hs);
  p.depth = 2 * row <= (size_t)kBwdRing ? 2 : 1;
  // the ring also holds the sums of a block's rows at the end
  p.smem = std::max(vec ? p.depth * row : 0, p.s.rows > 1 ? (size_t)p.s.rows * dim * 4 : 0);
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>((!vec && threads <= 256 ? 1024 : 512) / threads, 225 * 1024 / (int64_t)(p.smem + 1536)));
  p.grid = p.parts = std::min<int64_t>((rows + p.s.rows - 1) / p.s.rows, kSMs * per_sm);
  return p;
}

template <typename TX, typename TH, typename TW, int VPT, int NT>
int launch_bwd_as(const norm::BwdArgs& a, const BwdPlan& p, cudaStream_t st) {
  auto kernel = norm::bwd_kernel<TX, TH, TW, VPT, NT>;
  static Ready ready;
  if (const int rc = raise_smem(reinterpret_cast<const void*>(kernel), kBwdRing, ready)) return rc;
  return launch(kernel, (unsigned)p.grid, dim3(p.s.nt, p.s.rows), p.smem, st, a, p.depth);
}
template <typename TX, typename TH, typename TW>
int launch_bwd_w(const norm::BwdArgs& a, bool vec, const BwdPlan& p, cudaStream_t st) {
#define QRB_BWD(V, NT) launch_bwd_as<TX, TH, TW, V, NT>(a, p, st)
  if (vec) return p.s.vpt == 1 ? QRB_BWD(1, 0) : p.s.vpt == 2 ? QRB_BWD(2, 0) : QRB_BWD(4, 0);
  if (p.s.nt == 32) return p.s.vpt == 1 ? QRB_BWD(1, 32) : p.s.vpt == 2 ? QRB_BWD(2, 32) : QRB_BWD(4, 32);
  if (p.s.nt == 256) return p.s.vpt == 1 ? QRB_BWD(1, 256) : QRB_BWD(2, 256);
  return p.s.vpt == 2 ? QRB_BWD(2, 512) : QRB_BWD(4, 512);
#undef QRB_BWD
}
template <typename TX, typename TH>
int launch_bwd(const norm::BwdArgs& a, bool vec, const BwdPlan& p, cudaStream_t st) {
  if (a.dim > norm::kRegDim) {
    return launch(norm::bwd_long_kernel<TX, TH>, (unsigned)p.grid, norm::kMaxThreads, 0, st, a);
  }
  if constexpr (sizeof(TX) == 2) {
    if (a.w && a.w_f32) return launch_bwd_w<TX, TH, float>(a, vec, p, st);
  }
  return launch_bwd_w<TX, TH, TX>(a, vec, p, st);
}

template <typename T>
int launch_colsum(const float* part, int64_t parts, int64_t cols, void* out, cudaStream_t st) {
  // Not early: its blocks of 1024 threads would take their places while the blocks whose sums it adds
  // still work (forward and backward of 16384 x 4096: 182 us, 207 with an early start).
  return launch_as(norm::colsum_kernel<T>, (unsigned)((cols + 31) / 32), dim3(32, 32), 0, st, 0, false, part, parts, cols,
                   static_cast<T*>(out));
}
int colsum(const float* part, int64_t parts, int64_t cols, void* out, int32_t dtype, cudaStream_t st) {
  if (dtype == QRB200_F32) return launch_colsum<float>(part, parts, cols, out, st);
  if (dtype == QRB200_BF16) return launch_colsum<__nv_bfloat16>(part, parts, cols, out, st);
  return launch_colsum<__half>(part, parts, cols, out, st);
}

// ------------------------------------------------------------------ linear
// An operand seen as rows x k: k-major (rows contiguous along k) or row-major.
struct Operand {
  const void* p;
  int64_t ld;      // elements between the stored rows
  bool row_major;
  int64_t stored_rows(int64_t rows, int64_t k) const { return row_major ? k : rows; }
  int64_t stored_cols(int64_t rows, int64_t k) const { return row_major ? rows : k; }
};
int64_t padded_cols(int64_t cols, int es) { return (cols * es + 15) / 16 * 16 / es; }
bool addressable(const Operand& o, int es) { return rows_on16(o.p, o.ld, es); }
size_t aligned_copy_bytes(const Operand& o, int64_t rows, int64_t k, int es) {
  if (addressable(o, es)) return 0;
  const size_t b = (size_t)o.stored_rows(rows, k) * padded_cols(o.stored_cols(rows, k), es) * es;
  return (b + 255) & ~size_t(255);
}
// Points operands whose rows TMA cannot address to copies in `buf`, all made by one launch.
struct Aligner {
  lin::AlignJobs jobs{};
  int count = 0, es;
  int64_t most = 0;  // 16-byte pieces of the largest
  char* buf;
  void want(Operand& o, int64_t rows, int64_t k) {
    const size_t bytes = aligned_copy_bytes(o, rows, k, es);
    if (!bytes) return;
    const int64_t sr = o.stored_rows(rows, k), sc = o.stored_cols(rows, k), ldd = padded_cols(sc, es);
    jobs.job[count++] = {o.p, o.ld, sc, sr, buf, ldd};
    most = std::max(most, sr * ldd * es / 16);
    o.p = buf;
    o.ld = ldd;
    buf += bytes;
  }
  int run(cudaStream_t st) const {
    if (!count) return QRB200_OK;
    const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, kSMs * 8), (unsigned)count);
    return es == 2 ? launch(lin::align_rows_kernel<uint16_t>, grid, 256, 0, st, jobs)
                   : launch(lin::align_rows_kernel<uint8_t>, grid, 256, 0, st, jobs);
  }
};

bool encode_operand(CUtensorMap* map, const Operand& o, int64_t rows, int64_t k, int32_t dtype, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const int es = esize(dtype);
  const CUtensorMapDataType t = dtype == QRB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                              : dtype == QRB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const cuuint64_t dims[2] = {(cuuint64_t)o.stored_cols(rows, k), (cuuint64_t)o.stored_rows(rows, k)};
  const cuuint64_t strides[1] = {(cuuint64_t)o.ld * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)(o.row_major ? 64 : box_rows)};
  const cuuint32_t one[2] = {1, 1};
  return fn(map, t, 2, const_cast<void*>(o.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Out, int ES, int T, bool SLOPE, int RINGS>
int launch_tile_as(const lin::Maps& maps, const lin::Args& a, cudaStream_t st) {
  auto kernel = lin::tile_kernel<Out, ES, T, SLOPE, RINGS>;
  using C = lin::TileCfg<T, RINGS>;
  static Ready ready;
  if (const int rc = raise_smem(reinterpret_cast<const void*>(kernel), C::SMEM, ready)) return rc;
  const dim3 grid((unsigned)a.splits, (unsigned)((a.n + 127) / 128), (unsigned)((a.m + T - 1) / T));
  return launch_as(kernel, grid, lin::kTileThreads, C::SMEM, st, (unsigned)a.splits, true, maps, a);
}
template <typename Out, int ES, int T, bool SLOPE>
int launch_tile(const lin::Maps& maps, const lin::Args& a, cudaStream_t st) {
  const int64_t ctas = (int64_t)a.splits * ((a.n + 127) / 128) * ((a.m + T - 1) / T);
  return ctas <= kSMs ? launch_tile_as<Out, ES, T, SLOPE, 1>(maps, a, st) : launch_tile_as<Out, ES, T, SLOPE, 2>(maps, a, st);
}

template <typename Out, int ES, bool SLOPE>
int launch_tile_t(int T, const lin::Maps& maps, const lin::Args& a, cudaStream_t st) {
  switch (T) {
    case 16: return launch_tile<Out, ES, 16, SLOPE>(maps, a, st);
    case 32: return launch_tile<Out, ES, 32, SLOPE>(maps, a, st);
    case 64: return launch_tile<Out, ES, 64, SLOPE>(maps, a, st);
    case 128: return launch_tile<Out, ES, 128, SLOPE>(maps, a, st);
    default: return QRB200_ERR_INVALID_ARG;  // the maps' boxes are made for T
  }
}

// A map over rows of 16-bit results (or a residual), in blocks of 32 rows x 64 columns.
bool encode_result(CUtensorMap* map, const void* p, int64_t ld, int64_t m, int64_t n) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)m};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, 32}, one[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Out, int ES, int TN, bool SLOPE>
int launch_pair(const Operand& P, const Operand& Q, int64_t m, int64_t n, int64_t k, int32_t dtype,
                const lin::Epilogue& e, cudaStream_t st) {
  auto kernel = lin::pair_kernel<Out, ES, TN, SLOPE>;
  using C = lin::PairCfg<TN>;
  static Ready ready;
  if (const int rc = raise_smem(reinterpret_cast<const void*>(kernel), C::SMEM, ready)) return rc;
  lin::PairMaps maps{};
  lin::PairArgs a{};
  a.m = (int)m; a.n = (int)n; a.k = (int)k;
  a.p_row = P.row_major; a.q_row = Q.row_major;
  a.idesc = lin::idesc(dtype == QRB200_BF16 ? 1 : 0, a.p_row, a.q_row, lin::kPairM, TN);
  a.tiles_i = (int)((m + lin::kPairM - 1) / lin::kPairM);
  a.tiles_j = (int)((n + TN - 1) / TN);
  a.group = 8;
  a.e = e;
  a.tma_out = rows_on16(e.out, e.ldo, 2);
  a.tma_res = e.res && rows_on16(e.res, e.ldr, 2) && e.ldr > 0;
  a.tma_slope = e.slope && rows_on16(e.slope, n, 2);
  bool good = encode_operand(&maps.p, P, m, k, dtype, 128) && encode_operand(&maps.q, Q, n, k, dtype, TN / 2);
  if (good && a.tma_out) good = encode_result(&maps.out, e.out, e.ldo, m, n);
  if (good && a.tma_res) good = encode_result(&maps.res, e.res, e.ldr, m, n);
  if (good && a.tma_slope) good = encode_result(&maps.slope, e.slope, n, m, n);
  if (!good) {
    note(cudaErrorInvalidValue);
    return QRB200_ERR_CUDA;
  }
  const int64_t tiles = (int64_t)a.tiles_i * a.tiles_j;
  const unsigned grid = 2 * (unsigned)std::min<int64_t>(tiles, kSMs / 2);
  return launch(kernel, grid, lin::kPairThreads, C::SMEM, st, maps, a);
}

template <int TN>
int product_pair(const Operand& P, const Operand& Q, int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t out_dtype,
                 const lin::Epilogue& e, cudaStream_t st) {
  const bool bf = out_dtype == QRB200_BF16;
  if (dtype == QRB200_E4M3)
    return bf ? launch_pair<__nv_bfloat16, 1, TN, false>(P, Q, m, n, k, dtype, e, st)
              : launch_pair<__half, 1, TN, false>(P, Q, m, n, k, dtype, e, st);
  if (e.slope)
    return bf ? launch_pair<__nv_bfloat16, 2, TN, true>(P, Q, m, n, k, dtype, e, st)
              : launch_pair<__half, 2, TN, true>(P, Q, m, n, k, dtype, e, st);
  return bf ? launch_pair<__nv_bfloat16, 2, TN, false>(P, Q, m, n, k, dtype, e, st)
            : launch_pair<__half, 2, TN, false>(P, Q, m, n, k, dtype, e, st);
}

// A few tokens, W's features in rows: token_kernel.  Up to 2 tokens always; 3 and 4, which make it
// bound by its instructions, where W is small enough for the call's own cost to matter (4 tokens,
// 4096 x 4096: 11.8 us against 10.6 with tiles; 1 token 8.8 against 10.5; 512 x 512: 2.4 against 4.4).
// Features: two a warp from 8192 on (8192 x 8192: 24.0 us against 28.9 with one), one below that
// (4096 x 4096: 8.8 against 9.3), and one a block, its k shared by 8 warps, where k is long for the
// number of features (512 x 16384: 5.5 us against 21.9; 4096 x 16384: 23.8 against 25.9).
bool few_tokens(int64_t m, int64_t n, int64_t k) { return m <= 2 || (m <= 4 && n * k <= 1 << 22); }
template <typename Out, typename In, int M, bool VEC>
int launch_token(const lin::TokenArgs& a, cudaStream_t st) {
  if (a.n >= 8192) return launch(lin::token_kernel<Out, In, M, 2, 1, VEC>, (a.n + 7) / 8, 128, 0, st, a);
  if ((int64_t)a.k * sizeof(In) >= 4 * (int64_t)a.n) return launch(lin::token_kernel<Out, In, M, 1, 8, VEC>, a.n, 256, 0, st, a);
  return launch(lin::token_kernel<Out, In, M, 1, 1, VEC>, (a.n + 3) / 4, 128, 0, st, a);
}
template <typename Out, typename In>
int product_token(const lin::TokenArgs& a, cudaStream_t st) {
  const bool vec = a.k % (16 / sizeof(In)) == 0 && rows_on16(a.w, a.n > 1 ? a.ldw : 0, sizeof(In)) &&
                   rows_on16(a.x, a.m > 1 ? a.ldx : 0, sizeof(In));
  if (a.m == 1) return vec ? launch_token<Out, In, 1, true>(a, st) : launch_token<Out, In, 1, false>(a, st);
  if (a.m == 2) return vec ? launch_token<Out, In, 2, true>(a, st) : launch_token<Out, In, 2, false>(a, st);
  return vec ? launch_token<Out, In, 4, true>(a, st) : launch_token<Out, In, 4, false>(a, st);
}

// Which kernel and tile: the least of their times by a model of them, in microseconds, that fits
// what a sweep over 30 sizes measured (16 x 4096 x 4096 to 2048^3 and 8192 x 256 x 1024, each at 3 to 7
// choices) and picks the fastest or one within 7% of it on all of them, the fastest on 26.  Every kernel moves its operands at the rate
// at which an SM can fetch them, so a CTA's time is its blocks of 128 bytes of k times a cost a block.
//   pair kernel, 256 x 256: 8 + 0.33 a block and wave over 74 pairs; 256 x 128: 7.3 + 0.31
//   (2048^3: 18.6, measured 19.2; 512 x 4096 x 4096 in 256 x 128: 27.1, measured 27.3)
//   tile kernel, 128 x T: 7.3 + T / 128 + 0.21 to 0.28 a block with one CTA an SM, 0.30 to 0.44 with
//   two, and 0.6 to 1.6 for a cluster's exchange (128 x 4096 x 4096 over clusters of 4: 14.0, measured 12.9);
//   clusters of 8 that fill more than 64 SMs do not all find 8 free ones side by side: 6
struct Choice { bool pair; int tile, splits; };
Choice choose(int64_t m, int64_t n, int64_t k, int es, bool p_row) {
  const int64_t nkb = (k * es + 127) / 128, tj = (n + 127) / 128;
  Choice best{false, 128, 1};
  double least = 1e30;
  auto offer = [&](const Choice& c, double t) {
    if (t < least) {
      least = t;
      best = c;
    }
  };
  const struct { int tile; double alone, shared; } kinds[] = {{16, 0.21, 0.30}, {32, 0.21, 0.32}, {64, 0.22, 0.36}, {128, 0.28, 0.44}};
  const struct { int splits; double exchange; } clusters[] = {{1, 0.0}, {2, 0.6}, {4, 1.2}, {8, 1.6}};
  for (const auto& kind : kinds) {
    const int T = kind.tile;
    // no tile that a narrower one would hold, none that m takes more than two of (128: any number);
    // operands contiguous along their rows come 64 rows at a time
    if ((p_row && T < 64) || (T < 128 && m > 2 * T) || (T > (p_row ? 64 : 16) && m <= T / 2)) continue;
    const int64_t tiles = tj * ((m + T - 1) / T);
    for (const auto& cl : clusters) {
      if (cl.splits > 1 && nkb / cl.splits < 2) break;
      const int64_t ctas = tiles * cl.splits, part = (nkb + cl.splits - 1) / cl.splits, waves = (ctas + 2 * kSMs - 1) / (2 * kSMs);
      const double body = ctas <= kSMs ? part * kind.alone : waves * part * kind.shared * (waves > 1 ? 1.25 : 1.0);
      const double exchange = cl.splits == 8 && ctas > 64 ? 6.0 : cl.exchange;
      offer({false, T, cl.splits}, 7.3 + T / 128.0 + exchange + body);
    }
  }
  if (m > 128 && k > 0)
    for (const int tn : {128, 256}) {
      const int64_t tiles = ((m + 255) / 256) * ((n + tn - 1) / tn), waves = (tiles + kSMs / 2 - 1) / (kSMs / 2);
      offer({true, tn, 1}, tn == 256 ? 8.0 + waves * nkb * 0.33 : 7.3 + waves * nkb * 0.31);
    }
  return best;
}

// D = epilogue(P Q^T); P is m x k, Q is n x k, both addressable by TMA.
int product(const Operand& P, const Operand& Q, int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t out_dtype,
            const lin::Epilogue& e, cudaStream_t st) {
  const Choice choice = choose(m, n, k, esize(dtype), P.row_major);
  if (choice.pair)
    return choice.tile == 256 ? product_pair<256>(P, Q, m, n, k, dtype, out_dtype, e, st)
                              : product_pair<128>(P, Q, m, n, k, dtype, out_dtype, e, st);
  lin::Args a{};
  a.m = (int)m; a.n = (int)n; a.k = (int)k;
  a.e = e;
  a.es = esize(dtype);
  a.p_row = P.row_major; a.q_row = Q.row_major;
  auto on8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; };
  a.vec = on8(e.out) && e.ldo % 4 == 0 && (!e.bias || on8(e.bias)) &&
          (!e.res || (on8(e.res) && e.ldr % 4 == 0)) && (!e.slope || (on8(e.slope) && n % 4 == 0));
  const int T = choice.tile, nkb = (int)((k * a.es + 127) / 128);
  a.splits = choice.splits;
  a.part = (nkb + a.splits - 1) / a.splits;
  a.idesc = lin::idesc(dtype == QRB200_BF16 ? 1 : 0, a.q_row, a.p_row, lin::kTileQ, T);
  lin::Maps maps{};
  if (k > 0 && !(encode_operand(&maps.p, P, m, k, dtype, T) && encode_operand(&maps.q, Q, n, k, dtype, lin::kTileQ))) {
    note(cudaErrorInvalidValue);
    return QRB200_ERR_CUDA;
  }
  const bool bf = out_dtype == QRB200_BF16;
  if (a.es == 1)
    return bf ? launch_tile_t<__nv_bfloat16, 1, false>(T, maps, a, st) : launch_tile_t<__half, 1, false>(T, maps, a, st);
  if (e.slope)
    return bf ? launch_tile_t<__nv_bfloat16, 2, true>(T, maps, a, st) : launch_tile_t<__half, 2, true>(T, maps, a, st);
  return bf ? launch_tile_t<__nv_bfloat16, 2, false>(T, maps, a, st) : launch_tile_t<__half, 2, false>(T, maps, a, st);
}

constexpr int64_t kMostRows = 128 * 65535;  // of x, and of the weight
// Kernels walk along k with int indices that run past it: tiles by less than a block of 128, token_kernel
// by less than a turn of all its warps, 32768 elements of 8 bits.
constexpr int64_t kMostColumns = ((int64_t)1 << 31) - 65537;
bool sizes_ok(int64_t m, int64_t n, int64_t k) {
  // a grid's y and z have 16 bits, and an index into one operand's rows 31
  return m >= 0 && n >= 0 && k >= 0 && m <= kMostRows && n <= kMostRows && k <= kMostColumns;
}

// Blocks of dz_kernel along m, each of which leaves one part of the bias' sum: 8 blocks an SM.
int64_t dz_parts(int64_t m, int64_t n) {
  const int64_t strips = (n + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>((m + 7) / 8, std::max<int64_t>(1, 8 * kSMs / strips)));
}

template <typename T>
int launch_dz(const void* dy, int64_t lddy, const uint16_t* slope, void* dz, int64_t lddz, float* part, int64_t m,
              int64_t n, int64_t parts, cudaStream_t st) {
  const bool vec = n % 8 == 0 && rows_on16(dy, lddy, 2) && (!slope || on16(slope)) && (!dz || on16(dz));
  const dim3 grid((unsigned)((n + 255) / 256), (unsigned)parts);
  return launch(vec ? lin::dz_kernel<T, true> : lin::dz_kernel<T, false>, grid, 256, 0, st, static_cast<const T*>(dy), lddy,
                slope, static_cast<T*>(dz), lddz, part, m, n);
}

struct BackwardPlan {
  size_t dz, part, copies, total;
  int64_t parts, lddz;
};
// Buffers of the backward pass: dz (when it is not dy itself), the bias sum's parts, and copies of
// the operands TMA cannot address.
BackwardPlan backward_plan(const void* dy, int64_t lddy, bool slope, const Operand& x, const Operand& w, bool dx,
                           bool dw, bool db, int64_t m, int64_t n, int64_t k) {
  BackwardPlan p{};
  auto up = [](size_t b) { return (b + 255) & ~size_t(255); };
  const bool products = dx || dw;
  p.parts = dz_parts(m, n);
  p.lddz = padded_cols(n, 2);
  p.dz = slope && products ? up((size_t)m * p.lddz * 2) : 0;
  p.part = db ? up((size_t)p.parts * n * 4) : 0;
  if (products && !slope) p.copies += aligned_copy_bytes(Operand{dy, lddy, false}, m, n, 2);
  if (dx) p.copies += aligned_copy_bytes(Operand{w.p, w.ld, !w.row_major}, k, n, 2);
  if (dw) p.copies += aligned_copy_bytes(Operand{x.p, x.ld, true}, k, m, 2);
  p.total = p.dz + p.part + p.copies;
  return p;
}

}  // namespace
}  // namespace qrb

using namespace qrb;

extern "C" {

int qrb200_rms_norm(const void* x, int64_t ldx, const void* weight, int32_t weight_dtype, const void* residual,
                    int64_t ldr, int32_t stream_dtype, void* y, float* scale, void* h, int64_t rows, int64_t dim,
                    float eps, int32_t dtype, int32_t out_dtype, void* stream) {
  const bool q8 = out_dtype == QRB200_E4M3;
  if (!float_type(dtype) || !(q8 || out_dtype == dtype) || rows < 0 || dim < 0 || !(eps >= 0.f))
    return QRB200_ERR_INVALID_ARG;
  if (weight && !(weight_dtype == dtype || weight_dtype == QRB200_F32)) return QRB200_ERR_INVALID_ARG;
  if (residual && !(stream_dtype == dtype || stream_dtype == QRB200_F32)) return QRB200_ERR_INVALID_ARG;
  if (rows == 0 || dim == 0) return q8 ? scales_of_empty_rows(scale, rows, stream) : QRB200_OK;
  if (!x || !y || (q8 && !scale) || (residual && !h)) return QRB200_ERR_INVALID_ARG;
  if (rows >= ((int64_t)1 << 31) || dim >= ((int64_t)1 << 30) || ldx < 0 || (residual && ldr < 0))
    return QRB200_ERR_INVALID_ARG;
  const int es = esize(dtype), rs = residual ? esize(stream_dtype) : es;
  norm::FwdArgs a{x, ldx, residual, ldr, weight, weight && weight_dtype == QRB200_F32, y, scale, h, rows, (int)dim, eps};
  const bool vec = dim % 8 == 0 && rows_on16(x, ldx, es) && on16(y) &&
                   (!residual || (rows_on16(residual, ldr, rs) && on16(h))) && (!weight || on16(weight));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = residual && stream_dtype == QRB200_F32 && dtype != QRB200_F32;
  if (dtype == QRB200_F32) return launch_norm<float>(a, q8, wide, vec, st);
  if (dtype == QRB200_BF16) return launch_norm<__nv_bfloat16>(a, q8, wide, vec, st);
  return launch_norm<__half>(a, q8, wide, vec, st);
}

int qrb200_quantize_rows(const void* x, int64_t ldx, void* q, float* scale, int64_t rows, int64_t dim, int32_t dtype,
                         void* stream) {
  if (!float_type(dtype) || rows < 0 || dim < 0) return QRB200_ERR_INVALID_ARG;
  if (rows == 0 || dim == 0) return scales_of_empty_rows(scale, rows, stream);
  if (!x || !q || !scale || rows >= ((int64_t)1 << 31) || dim >= ((int64_t)1 << 30) || ldx < 0)
    return QRB200_ERR_INVALID_ARG;
  norm::FwdArgs a{x, ldx, nullptr, 0, nullptr, 0, q, scale, nullptr, rows, (int)dim, 0.f};
  const bool vec = dim % 8 == 0 && rows_on16(x, ldx, esize(dtype)) && on16(q);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == QRB200_F32) return launch_fwd<float, float, false, true, false>(a, vec, st);
  if (dtype == QRB200_BF16) return launch_fwd<__nv_bfloat16, __nv_bfloat16, false, true, false>(a, vec, st);
  return launch_fwd<__half, __half, false, true, false>(a, vec, st);
}

int qrb200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t dim, int32_t dtype, int32_t stream_dtype,
                                             size_t* bytes) {
  if (!bytes || !float_type(dtype) || !(stream_dtype == dtype || stream_dtype == QRB200_F32) || rows < 0 || dim < 0 || rows >= ((int64_t)1 << 31) || dim >= ((int64_t)1 << 30))
    return QRB200_ERR_INVALID_ARG;
  size_t need = 0;
  if (rows && dim)  // aligned or not
    for (const bool vec : {false, true})
      need = std::max(need, (size_t)bwd_plan(rows, (int)dim, esize(dtype), esize(stream_dtype), vec).parts * dim * sizeof(float));
  *bytes = workspace_size(need);
  return QRB200_OK;
}

int qrb200_rms_norm_backward(const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* dh, int64_t lddh,
                             const void* weight, int32_t weight_dtype, void* dx, void* dresidual, void* dweight,
                             int64_t rows, int64_t dim, float eps, int32_t dtype, int32_t stream_dtype,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (!float_type(dtype) || !(stream_dtype == dtype || stream_dtype == QRB200_F32) || rows < 0 || dim < 0 ||
      !(eps >= 0.f))
    return QRB200_ERR_INVALID_ARG;
  if (weight && !(weight_dtype == dtype || weight_dtype == QRB200_F32)) return QRB200_ERR_INVALID_ARG;
  if (dweight && !weight) return QRB200_ERR_INVALID_ARG;
  if (dim == 0) return QRB200_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (!dweight) return QRB200_OK;
    return note(cudaMemsetAsync(dweight, 0, (size_t)dim * esize(weight_dtype), st)) == cudaSuccess ? QRB200_OK
                                                                                                 : QRB200_ERR_CUDA;
  }
  if (!dy || !h || rows >= ((int64_t)1 << 31) || dim >= ((int64_t)1 << 30) || lddy < 0 || ldh < 0 || (dh && lddh < 0))
    return QRB200_ERR_INVALID_ARG;
  const int es = esize(dtype), rs = esize(stream_dtype);
  const bool vec = dim % 8 == 0 && rows_on16(dy, lddy, es) && rows_on16(h, ldh, rs) &&
                   (!dh || rows_on16(dh, lddh, rs)) && (!dx || on16(dx)) && (!dresidual || on16(dresidual)) &&
                   (!weight || on16(weight));
  const BwdPlan plan = bwd_plan(rows, (int)dim, es, rs, vec);
  Scratch ws(st);
  int rc = ws.get(workspace, workspace_bytes, dweight ? (size_t)plan.parts * dim * sizeof(float) : 0);
  if (rc != QRB200_OK) return rc;
  norm::BwdArgs a{dy, lddy, h, ldh, dh, lddh, weight, weight && weight_dtype == QRB200_F32, dx, dresidual,
                  static_cast<float*>(ws.p), rows, (int)dim, eps};
  const bool wide = stream_dtype == QRB200_F32 && dtype != QRB200_F32;
  if (dtype == QRB200_F32) rc = launch_bwd<float, float>(a, vec, plan, st);
  else if (dtype == QRB200_BF16)
    rc = wide ? launch_bwd<__nv_bfloat16, float>(a, vec, plan, st)
              : launch_bwd<__nv_bfloat16, __nv_bfloat16>(a, vec, plan, st);
  else
    rc = wide ? launch_bwd<__half, float>(a, vec, plan, st)
              : launch_bwd<__half, __half>(a, vec, plan, st);
  if (rc == QRB200_OK && dweight) rc = colsum(a.part, plan.parts, dim, dweight, weight_dtype, st);
  return rc;
}

int qrb200_linear_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t w_transposed,
                                  int64_t m, int64_t n, int64_t k, int32_t dtype, size_t* bytes) {
  if (!bytes || !(dtype == QRB200_BF16 || dtype == QRB200_F16 || dtype == QRB200_E4M3) || !sizes_ok(m, n, k) ||
      (dtype == QRB200_E4M3 && w_transposed))
    return QRB200_ERR_INVALID_ARG;
  const int es = esize(dtype);
  *bytes = m && n && k ? workspace_size(aligned_copy_bytes(Operand{x, ldx, false}, m, k, es) +
                                        aligned_copy_bytes(Operand{w, ldw, w_transposed != 0}, n, k, es))
                       : 0;
  return QRB200_OK;
}

int qrb200_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t w_transposed, const float* x_scale,
                  const float* w_scale, const void* bias, const void* residual, int64_t ldr, void* y, int64_t ldy,
                  uint16_t* slope, int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t out_dtype,
                  int32_t activation, void* workspace, size_t workspace_bytes, void* stream) {
  const bool q8 = dtype == QRB200_E4M3;
  if (!(dtype == QRB200_BF16 || dtype == QRB200_F16 || q8) || !sizes_ok(m, n, k)) return QRB200_ERR_INVALID_ARG;
  if (q8 ? !(out_dtype == QRB200_BF16 || out_dtype == QRB200_F16) : out_dtype != dtype) return QRB200_ERR_INVALID_ARG;
  if (activation < 0 || activation >= lin::ACT_COUNT || (q8 ? w_transposed || slope : x_scale || w_scale)) return QRB200_ERR_INVALID_ARG;
  if (m == 0 || n == 0) return QRB200_OK;
  if (!y || (k > 0 && (!x || !w))) return QRB200_ERR_INVALID_ARG;
  if (ldy < n || (residual && ldr < 0) || (k > 0 && (ldx < k || ldw < (w_transposed ? n : k))))
    return QRB200_ERR_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int es = esize(dtype);
  Operand X{x, ldx, false}, W{w, ldw, w_transposed != 0};
  lin::Epilogue e{x_scale, w_scale, bias, residual, ldr, y, ldy, slope, activation};
  if (few_tokens(m, n, k) && !w_transposed && !slope && k > 0) {
    const lin::TokenArgs t{x, ldx, w, ldw, (int)m, (int)n, (int)k, e};
    if (q8) return out_dtype == QRB200_BF16 ? product_token<__nv_bfloat16, __nv_fp8_e4m3>(t, st) : product_token<__half, __nv_fp8_e4m3>(t, st);
    return dtype == QRB200_BF16 ? product_token<__nv_bfloat16, __nv_bfloat16>(t, st) : product_token<__half, __half>(t, st);
  }
  Scratch ws(st);
  int rc = ws.get(workspace, workspace_bytes,
                  k ? aligned_copy_bytes(X, m, k, es) + aligned_copy_bytes(W, n, k, es) : 0);
  if (rc == QRB200_OK && k) {
    Aligner align{{}, 0, es, 0, static_cast<char*>(ws.p)};
    align.want(X, m, k);
    align.want(W, n, k);
    rc = align.run(st);
  }
  if (rc != QRB200_OK) return rc;
  return product(X, W, m, n, k, dtype, out_dtype, e, st);
}

int qrb200_linear_backward_workspace_bytes(const void* dy, int64_t lddy, int32_t has_slope, const void* x, int64_t ldx,
                                           const void* w, int64_t ldw, int32_t w_transposed, int32_t want_dx,
                                           int32_t want_dw, int32_t want_dbias, int64_t m, int64_t n, int64_t k,
                                           size_t* bytes) {
  if (!bytes || !sizes_ok(m, n, k) || !sizes_ok(k, m, n)) return QRB200_ERR_INVALID_ARG;
  *bytes = m && n ? workspace_size(backward_plan(dy, lddy, has_slope != 0, Operand{x, ldx, false}, Operand{w, ldw, w_transposed != 0},
                                                 want_dx && k, want_dw && k, want_dbias, m, n, k)
                                       .total)
                  : 0;
  return QRB200_OK;
}

int qrb200_linear_backward(const void* dy, int64_t lddy, const uint16_t* slope, const void* x, int64_t ldx,
                           const void* w, int64_t ldw, int32_t w_transposed, void* dx, void* dw, void* dbias,
                           int64_t m, int64_t n, int64_t k, int32_t dtype, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (!(dtype == QRB200_BF16 || dtype == QRB200_F16) || !sizes_ok(m, n, k) || !sizes_ok(k, m, n))
    return QRB200_ERR_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (m == 0 || n == 0) {  // sums over nothing
    cudaError_t e = cudaSuccess;
    if (dx && m * k) e = cudaMemsetAsync(dx, 0, (size_t)m * k * 2, st);
    if (e == cudaSuccess && dw && n * k) e = cudaMemsetAsync(dw, 0, (size_t)n * k * 2, st);
    if (e == cudaSuccess && dbias && n) e = cudaMemsetAsync(dbias, 0, (size_t)n * 2, st);
    return note(e) == cudaSuccess ? QRB200_OK : QRB200_ERR_CUDA;
  }
  if (k == 0) dx = dw = nullptr;
  if (!dx && !dw && !dbias) return QRB200_OK;
  if (!dy || lddy < n || (dx && (!w || ldw < (w_transposed ? n : k))) || (dw && (!x || ldx < k)))
    return QRB200_ERR_INVALID_ARG;
  const Operand X{x, ldx, false}, W{w, ldw, w_transposed != 0};
  const BackwardPlan p = backward_plan(dy, lddy, slope != nullptr, X, W, dx, dw, dbias, m, n, k);
  Scratch ws(st);
  int rc = ws.get(workspace, workspace_bytes, p.total);
  if (rc != QRB200_OK) return rc;
  char* buf = static_cast<char*>(ws.p);
  void* dz = p.dz ? buf : nullptr;
  buf += p.dz;
  float* part = p.part ? reinterpret_cast<float*>(buf) : nullptr;
  buf += p.part;
  if (dz || part) {
    rc = dtype == QRB200_BF16 ? launch_dz<__nv_bfloat16>(dy, lddy, slope, dz, p.lddz, part, m, n, p.parts, st)
                              : launch_dz<__half>(dy, lddy, slope, dz, p.lddz, part, m, n, p.parts, st);
    if (rc == QRB200_OK && dbias) rc = colsum(part, p.parts, n, dbias, dtype, st);
    if (rc != QRB200_OK) return rc;
  }
  if (!dx && !dw) return QRB200_OK;
  Operand G = dz ? Operand{dz, p.lddz, false} : Operand{dy, lddy, false};
  Operand Wt{w, ldw, !W.row_major}, Xt{x, ldx, true};
  Aligner align{{}, 0, 2, 0, buf};
  align.want(G, m, n);
  if (dx) align.want(Wt, k, n);
  if (dw) align.want(Xt, k, m);
  rc = align.run(st);
  if (rc == QRB200_OK && dx) {  // dx_ik = sum_j dz_ij W_jk
    lin::Epilogue e{nullptr, nullptr, nullptr, nullptr, 0, dx, k, nullptr, lin::ACT_NONE};
    rc = product(G, Wt, m, k, n, dtype, dtype, e, st);
  }
  if (rc == QRB200_OK && dw) {  // dW_jk = sum_i dz_ij x_ik
    lin::Epilogue e{nullptr, nullptr, nullptr, nullptr, 0, dw, k, nullptr, lin::ACT_NONE};
    rc = product(Operand{G.p, G.ld, true}, Xt, n, k, m, dtype, dtype, e, st);
  }
  return rc;
}

int qrb200_layer_status(int32_t* timed_out) {
  if (!timed_out) return QRB200_ERR_INVALID_ARG;
  static std::mutex one;  // calls share g_taken
  const std::lock_guard<std::mutex> lock(one);
  int v = 0;
  // all streams: a copy on the default one does not wait for those made without its blocking
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) {
    lin::take_timeout<<<1, 1>>>();
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, lin::g_taken, sizeof(v));
  *timed_out = v;
  return note(e) == cudaSuccess ? QRB200_OK : QRB200_ERR_CUDA;
}

}  // extern "C"
