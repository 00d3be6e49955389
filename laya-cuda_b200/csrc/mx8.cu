// Entry points of the MX8 operators (see include/laya_b200.h): checks of arguments and launches.
#include <algorithm>
#include <cmath>
#include <exception>

#include "host.cuh"
#include "mx8.cuh"
#include "mx8_gemm.cuh"

using namespace laya;

namespace {

void check_shape(int rows, int cols) {
  if (rows < 0 || cols < 1) fail(LAYA_ERR_INVALID, "bad shape %d x %d: rows may be 0, columns may not", rows, cols);
}

void check_rows(const char* what, const void* p, int64_t ld, int cols, int dtype) {
  if (!p) fail(LAYA_ERR_INVALID, "%s is null", what);
  if (ld < cols) fail(LAYA_ERR_INVALID, "%s: row stride %lld is less than %d columns", what, (long long)ld, cols);
  if (reinterpret_cast<uintptr_t>(p) % dtype_size(dtype)) fail(LAYA_ERR_INVALID, "%s is not aligned to its elements", what);
}

void check_mx8(const char* what, const void* q, int64_t ld, const void* scales, int cols) {
  if (!q || !scales) fail(LAYA_ERR_INVALID, "%s: null values or scales", what);
  if (ld % 16 || ld < cols) fail(LAYA_ERR_INVALID, "%s: row stride %lld is not a multiple of 16 of at least %d", what, (long long)ld, cols);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(scales)) & 15)
    fail(LAYA_ERR_INVALID, "%s: values and scales must be 16-byte aligned", what);
}

void check_vector(const char* what, const float* p) {
  if (p && (reinterpret_cast<uintptr_t>(p) & 15)) fail(LAYA_ERR_INVALID, "%s must be 16-byte aligned", what);
}

// E4M3 values [rows][cols], row stride ld bytes; box {128 columns, box_rows}, 128-byte swizzle.
CUtensorMap value_map(const MxOperand& m, int rows, int cols, int box_rows) {
  CUtensorMap map;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)m.ld};
  cuuint32_t box[2] = {kMxBK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(m.q), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(LAYA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return map;
}

// Scale tiles [row tiles][column tiles][512 bytes]; box {512 bytes, 1, box_tiles}.  Row tiles past the last read as zeros
// (scale 2^-127).
CUtensorMap scale_map(const MxOperand& m, int rows, int cols, int box_tiles) {
  CUtensorMap map;
  const cuuint64_t col_tiles = mx_col_tiles(cols), row_tiles = ((cuuint64_t)rows + kMxTileRows - 1) / kMxTileRows;
  cuuint64_t dims[3] = {kMxTileBytes / 4, col_tiles, row_tiles};
  cuuint64_t strides[2] = {kMxTileBytes, col_tiles * kMxTileBytes};
  cuuint32_t box[3] = {kMxTileBytes / 4, 1, (cuuint32_t)box_tiles};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<uint8_t*>(m.scales), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(LAYA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return map;
}

MxMaps linear_maps(const MxLinearArgs& a, int x_box, int w_box, int w_tiles) {
  MxMaps m{};
  m.x = value_map(a.x, a.M, a.K, x_box);
  m.xs = scale_map(a.x, a.M, a.K, 1);
  m.w = value_map(a.w, a.N, a.K, w_box);
  m.ws = scale_map(a.w, a.N, a.K, w_tiles);
  if (a.gate.q) {
    m.g = value_map(a.gate, a.N, a.K, w_box);
    m.gs = scale_map(a.gate, a.N, a.K, w_tiles);
  }
  return m;
}

template <typename K>
void launch_cluster(K kern, dim3 grid, int threads, int smem, dim3 cluster, cudaStream_t st, const MxMaps& m, const MxLinearArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster.x;
  attr[0].val.clusterDim.y = cluster.y;
  attr[0].val.clusterDim.z = cluster.z;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  CK(cudaLaunchKernelEx(&cfg, kern, m, a));
}

template <int BN, bool kGated, int kRes>
void launch_pair_res(const MxLinearArgs& a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  using Cfg = MxPairCfg<BN>;
  auto kern = mx8_linear_pair_kernel<BN, kGated, kRes>;
  allow_smem(kern, Cfg::kSmemBytes, dev, done);
  const MxMaps m = linear_maps(a, 128, BN / 2, kGated ? 1 : Cfg::kWeightTiles);
  const int out_cols = kGated ? BN / 2 : BN;
  const int64_t tiles = (((int64_t)a.M + 255) / 256) * ((a.N + out_cols - 1) / out_cols);
  if (tiles > INT32_MAX / 2) fail(LAYA_ERR_INVALID, "result of %d x %d is too large", a.M, a.N);
  const int pairs = (int)std::min<int64_t>(tiles, sm_count(dev) / 2);
  launch_cluster(kern, dim3(2 * pairs), kMxThreadsPair, Cfg::kSmemBytes, dim3(2, 1, 1), st, m, a);
}

template <int BN, bool kGated>
void launch_pair(const MxLinearArgs& a, int dev, cudaStream_t st) {
  const bool wide = a.residual_wide && a.N % 32 == 0, full = a.residual_type == LAYA_DTYPE_F32;
  if (!a.residual) launch_pair_res<BN, kGated, MX_RES_NONE>(a, dev, st);
  else if (wide && full) launch_pair_res<BN, kGated, MX_RES_FULL>(a, dev, st);
  else if (wide) launch_pair_res<BN, kGated, MX_RES_HALF>(a, dev, st);
  else if (full) launch_pair_res<BN, kGated, MX_RES_ANY_FULL>(a, dev, st);
  else launch_pair_res<BN, kGated, MX_RES_ANY_HALF>(a, dev, st);
}

// Launch shape of the few-row kernel: 128-feature tiles by BN-row tiles, and K split over the 1 to 4 CTAs for
// which this estimate is the shortest: a k-tile takes a CTA 0.17 us (gated 0.27), and a cluster's exchange up to 1.1
// us, in proportion to the CTAs in flight; clusters of more than two that would fill more than 7/8 of the SMs do
// not all fit at once.  Measured, unsplit / 2 / 4 CTAs: 1 x 4096 x 4096 9.1 / 6.3 / 5.4 us, 16 x 2048 x 2048 5.9 / 4.9 / 4.3, 300 x
// 768 x 768 4.6 / 5.1 / 5.0, 1024 x 8192 x 128 12.1 / 9.0 / 6.9, 1024 x 1024 x 1024 (128 tiles) 4.9 / 6.9 / 12.6.
struct FewGrid {
  int tiles, row_tiles, split;
};
FewGrid few_grid(const MxLinearArgs& a, int bn, int sms) {
  FewGrid g{(a.N + 127) / 128, (a.M + bn - 1) / bn, 1};
  const int k_tiles = mx_col_tiles(a.K);
  const double per_k_tile = a.gate.q ? 0.27 : 0.17;
  double best = k_tiles * per_k_tile;
  for (int split = 2; split <= std::min(kMxMaxSplit, k_tiles); ++split) {
    const double ctas = (double)g.tiles * g.row_tiles * split;
    if (split == 2 ? ctas > sms : 8 * ctas > 7 * sms) break;
    const double t = (k_tiles + split - 1) / split * per_k_tile + 1.1 * ctas / 128;
    if (t < best) { best = t; g.split = split; }
  }
  return g;
}

template <int BN, bool kGated>
void launch_few(const MxLinearArgs& a, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  using Cfg = MxFewCfg<BN, kGated>;
  auto kern = mx8_linear_few_kernel<BN, kGated>;
  allow_smem(kern, Cfg::kSmemBytes, dev, done);
  const MxMaps m = linear_maps(a, BN, 128, 1);
  const FewGrid g = few_grid(a, BN, sm_count(dev));
  launch_cluster(kern, dim3(g.tiles, g.row_tiles, g.split), kMxThreadsFew, Cfg::kSmemBytes, dim3(1, 1, g.split), st, m, a);
}

// Which kernel, and which tile.
//
// The few-row kernel up to 64 rows, and beyond wherever its 128 x 64 tiles fit the SMs at once, unless they
// nearly fill them and K is long (the tiles' operands then come from L2 too slowly): 128 x 4096 x 4096 takes
// 7.8 us against 10.0 for the pair kernel's 256 x 128 tiles, 1024 x 1024 x 1024 4.9 against 5.8, 511 x 776 x 2304 with a
// GELU 6.9 against 9.5, 192 x 4096 x 4096 (96 tiles) 9.3 against 9.9, but 256 x 4096 x 4096 (128) 11.1 against
// 9.7.  Gated, only where K is split: 128 x 4096 x 2 x 4096 14.3 against 16.4, unsplit 256 x 2048 x 2 x 4096
// 11.5 against 10.8.
//
// Otherwise CTA pairs: the tile for which this estimate is the shorter.  A wave of tiles takes the longer of
// its MMAs' and its epilogue's time (microseconds, fitted to 256 .. 3000 rows with 768 .. 4096 columns and
// to 16384 x 64 x 4096: 512 x 4096 x 4096 10.8 with 256 x 128 tiles against 15.6, 1024 rows 17.3 against 17.0,
// 16384 x 1024 x 4096 63.8 against 58.5).
template <bool kGated>
void launch_linear(const MxLinearArgs& a, int dev, cudaStream_t st) {
  if (a.M <= 16) return launch_few<16, kGated>(a, dev, st);
  if (a.M <= 32) return launch_few<32, kGated>(a, dev, st);
  const int sms = sm_count(dev), k_tiles = mx_col_tiles(a.K);
  const FewGrid few = few_grid(a, 64, sms);
  const bool fits = (int64_t)few.tiles * few.row_tiles <= sms;
  const bool slow = few.split == 1 && (kGated || (4LL * few.tiles * few.row_tiles > 3 * sms && k_tiles > 16));
  if (a.M <= 64 || (fits && !slow)) return launch_few<64, kGated>(a, dev, st);
  if constexpr (!kGated) {
    auto estimate = [&](int bn, double per_k_tile, double epilogue, double once) {
      const double tiles = (double)((a.M + 255) / 256) * ((a.N + bn - 1) / bn);
      return once + std::ceil(tiles / (sms / 2)) * std::max(k_tiles * per_k_tile, epilogue);
    };
    if (estimate(128, 0.17, 1.25, 4.8) < estimate(256, 0.28, 2.45, 5.8)) return launch_pair<128, false>(a, dev, st);
  }
  launch_pair<256, kGated>(a, dev, st);
}

// Blocks of a conversion: one pass each up to 32 per SM, several beyond.  Blocks that follow one another through the
// matrix read and write HBM in order; 8 per SM that stride over it took 35.0 us where these take 32.0 (16384 x
// 4096 to bf16; to fp32 61.9 and 51.9, 9216 x 4096 fp32 to MX8 30.3 and 28.3), and two pieces in flight per thread
// made no difference then.
int pieces_grid(int64_t pieces, int per_block, int sms) {
  return (int)std::min<int64_t>((pieces + per_block - 1) / per_block, 32LL * sms);
}

template <typename T, typename R, int CH, bool kVec, bool kShort>
void launch_norm_rows(RmsNormArgs a, int sms, cudaStream_t st) {
  auto kern = rms_norm_mx8_kernel<T, R, CH, kVec, kShort>;
  const int need = (a.cols + 32 * kMxPiece * CH - 1) / (32 * kMxPiece * CH);
  int log = 0;
  while ((1 << log) < need) ++log;
  a.warps = 1 << log;
  a.lanes = a.cols > 8 * kMxPiece ? 16 : 8;
  const int warps = std::max(a.warps, 8), per_block = warps / a.warps * (kShort ? 32 / a.lanes : 1);
  int64_t blocks = ((int64_t)a.rows + per_block - 1) / per_block;
  if (blocks > sms) {
    static std::atomic<int> resident[8];  // by log, 0: not asked yet
    int n = resident[log].load(std::memory_order_relaxed);
    if (!n) {
      CK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, warps * 32, 0));
      n = std::max(n, 1);
      resident[log].store(n, std::memory_order_relaxed);
    }
    blocks = std::min<int64_t>(blocks, (int64_t)n * sms);
  }
  launch_k(kern, dim3((int)blocks), dim3(warps * 32), 0, st, a);
}

template <typename T, typename R>
void launch_norm(const RmsNormArgs& a, int sms, cudaStream_t st) {
  const bool vec = rows_vectored(static_cast<const T*>(a.x), a.ldx, a.cols) &&
                   (!a.residual || rows_vectored(static_cast<const R*>(a.residual), a.ldr, a.cols)) &&
                   (!a.sum_out || rows_vectored(static_cast<const R*>(a.sum_out), a.lds, a.cols));
  constexpr int kCols = 16 * 32 * kMxPiece;  // 16 warps of one piece per thread
  const bool few_cols = a.cols <= 16 * kMxPiece;
  if (vec && few_cols) launch_norm_rows<T, R, 1, true, true>(a, sms, st);
  else if (vec && a.cols <= kCols) launch_norm_rows<T, R, 1, true, false>(a, sms, st);
  else if (vec && a.cols <= 2 * kCols) launch_norm_rows<T, R, 2, true, false>(a, sms, st);
  else if (few_cols) launch_norm_rows<T, R, 1, false, true>(a, sms, st);
  else if (a.cols <= kCols) launch_norm_rows<T, R, 1, false, false>(a, sms, st);
  else if (a.cols <= 2 * kCols) launch_norm_rows<T, R, 2, false, false>(a, sms, st);
  else launch_k(rms_norm_mx8_long_kernel<T, R>, dim3(std::min(a.rows, 8 * sms)), dim3(kMxThreads), 0, st, a);
}

}  // namespace

extern "C" {

int64_t laya_mx8_scale_bytes(int rows, int cols) {
  if (rows < 0 || cols < 1) return -1;
  return ((int64_t)rows + kMxTileRows - 1) / kMxTileRows * (((int64_t)cols + kMxTileCols - 1) / kMxTileCols) * kMxTileBytes;
}

int laya_op_mx8_quantize(const laya_mx8_convert* p, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  const int rows = p->rows, cols = p->cols;
  check_shape(rows, cols);
  dtype_size(p->dtype);
  if (!rows) return LAYA_OK;
  check_rows("x", p->data, p->ld, cols, p->dtype);
  check_mx8("out", p->values, p->ldv, p->scales, cols);
  const int64_t groups = (int64_t)rows * mx_col_tiles(cols);
  if (groups > INT32_MAX) fail(LAYA_ERR_INVALID, "%d x %d values are too many for one call", rows, cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(current_device(st));
  with_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T* x = static_cast<const T*>(p->data);
    auto go = [&](auto kern) {
      launch_k(kern, dim3(pieces_grid(groups, kMxThreads / 8, sms)), dim3(kMxThreads), 0, st, x, p->ld, rows, cols,
               FastDiv((uint32_t)mx_col_tiles(cols)),
               static_cast<uint8_t*>(p->values), p->ldv, static_cast<uint8_t*>(p->scales));
    };
    if (rows_vectored(x, p->ld, cols)) go(mx8_quantize_kernel<T, true>);
    else go(mx8_quantize_kernel<T, false>);
  });
  OP_API_END
}

int laya_op_mx8_dequantize(const laya_mx8_convert* p, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  const int rows = p->rows, cols = p->cols;
  check_shape(rows, cols);
  dtype_size(p->dtype);
  if (!rows) return LAYA_OK;
  check_mx8("x", p->values, p->ldv, p->scales, cols);
  check_rows("out", p->data, p->ld, cols, p->dtype);
  const uint32_t per_row = ((uint32_t)cols + kMxPiece - 1) / kMxPiece;
  const int64_t pieces = (int64_t)rows * per_row;
  if (pieces > INT32_MAX) fail(LAYA_ERR_INVALID, "%d x %d values are too many for one call", rows, cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(current_device(st));
  with_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    T* out = static_cast<T*>(p->data);
    auto go = [&](auto kern) {
      launch_k(kern, dim3(pieces_grid(pieces, kMxThreads, sms)), dim3(kMxThreads), 0, st,
               static_cast<const uint8_t*>(p->values), p->ldv, static_cast<const uint8_t*>(p->scales), rows, cols, FastDiv(per_row), out,
               p->ld);
    };
    // Rows without 32-byte alignment, 16 bits: in runs from 200 columns, where a warp covers three rows at most.  Back
    // to 16384 x 4095 bf16 39 us, 56 us by elements; 65536 x 201 11.6 and 13.0, but 65536 x 133 9.2 and 8.7, 200000 x
    // 15 5.9 and 4.0, and 77 x 1000, all latency, 1.7 and 1.6.  fp32 by elements, 128 bytes per instruction: 78 us against 96 in runs (16384 x 4095).
    if (rows_vectored(out, p->ld, cols)) go(mx8_dequantize_kernel<T, MxStore::kVectors>);
    else if constexpr (sizeof(T) == 2) {
      if (cols >= 200) go(mx8_dequantize_kernel<T, MxStore::kRuns>);
      else go(mx8_dequantize_kernel<T, MxStore::kElements>);
    } else go(mx8_dequantize_kernel<T, MxStore::kElements>);
  });
  OP_API_END
}

int laya_op_rms_norm_mx8(const laya_rms_norm_mx8* p, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  const int rows = p->rows, cols = p->cols;
  check_shape(rows, cols);
  dtype_size(p->dtype);
  dtype_size(p->residual_dtype);
  if (!(p->eps >= 0.f)) fail(LAYA_ERR_INVALID, "eps must be at least 0");
  if (!rows) return LAYA_OK;
  check_rows("x", p->x, p->ldx, cols, p->dtype);
  if (p->residual) check_rows("residual", p->residual, p->ldr, cols, p->residual_dtype);
  if (p->sum_out) check_rows("sum_out", p->sum_out, p->lds, cols, p->residual_dtype);
  if (!p->weight) fail(LAYA_ERR_INVALID, "weight is null");
  check_vector("weight", p->weight);
  check_mx8("out", p->values, p->ldv, p->scales, cols);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(current_device(st));
  RmsNormArgs a{};
  a.x = p->x; a.ldx = p->ldx; a.residual = p->residual; a.ldr = p->ldr; a.sum_out = p->sum_out; a.lds = p->lds;
  a.weight = p->weight; a.eps = p->eps; a.rows = rows; a.cols = cols;
  a.q = static_cast<uint8_t*>(p->values); a.ldq = p->ldv; a.scales = static_cast<uint8_t*>(p->scales);
  with_type(p->dtype, [&](auto* t) {
    with_type(p->residual_dtype, [&](auto* r) {
      launch_norm<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(r)>>(a, sms, st);
    });
  });
  OP_API_END
}

int laya_op_mx8_linear(const laya_mx8_linear* p, int* err, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  const int M = p->rows, N = p->features, K = p->cols;
  check_shape(M, N);
  if (K < 1) fail(LAYA_ERR_INVALID, "bad depth %d", K);
  // A tile's rows and columns are counted in 32 bits past the result's last ones.
  constexpr int kMost = INT32_MAX - 255;
  if (M > kMost || N > kMost) fail(LAYA_ERR_INVALID, "result of %d x %d: rows and features may be at most %d", M, N, kMost);
  if (p->activation < LAYA_ACT_NONE || p->activation > LAYA_ACT_SILU) fail(LAYA_ERR_INVALID, "unknown activation %d", p->activation);
  if (p->out_dtype != LAYA_DTYPE_MX8) dtype_size(p->out_dtype);
  if (p->residual) dtype_size(p->residual_dtype);
  const bool gated = p->gate != nullptr;
  if (p->gate_bias && !gated) fail(LAYA_ERR_INVALID, "gate_bias without a gate");
  if (!M) return LAYA_OK;
  check_mx8("x", p->x, p->ldx, p->x_scales, K);
  check_mx8("w", p->w, p->ldw, p->w_scales, K);
  if (gated) check_mx8("gate", p->gate, p->ldg, p->gate_scales, K);
  check_vector("bias", p->bias);
  check_vector("gate_bias", p->gate_bias);
  if (p->residual) check_rows("residual", p->residual, p->ldr, N, p->residual_dtype);
  if (p->out_dtype == LAYA_DTYPE_MX8) check_mx8("out", p->out, p->ldo, p->out_scales, N);
  else check_rows("out", p->out, p->ldo, N, p->out_dtype);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int dev = current_device(st);
  auto vec4 = [](const void* q, int64_t ld, size_t size) {
    return (reinterpret_cast<uintptr_t>(q) % (4 * size)) == 0 && ld % 4 == 0;
  };
  MxLinearArgs a{};
  a.M = M; a.N = N; a.K = K;
  a.x = {static_cast<const uint8_t*>(p->x), p->ldx, static_cast<const uint8_t*>(p->x_scales)};
  a.w = {static_cast<const uint8_t*>(p->w), p->ldw, static_cast<const uint8_t*>(p->w_scales)};
  a.gate = {static_cast<const uint8_t*>(p->gate), p->ldg, static_cast<const uint8_t*>(p->gate_scales)};
  a.bias = p->bias; a.gate_bias = p->gate_bias; a.act = p->activation;
  a.residual = p->residual; a.ldr = p->ldr; a.residual_type = p->residual_dtype;
  auto wide = [](const void* q, int64_t ld, size_t size) {
    return reinterpret_cast<uintptr_t>(q) % 32 == 0 && ld * (int64_t)size % 32 == 0;
  };
  if (p->residual) {
    a.residual_vec = vec4(p->residual, p->ldr, dtype_size(p->residual_dtype));
    a.residual_wide = wide(p->residual, p->ldr, dtype_size(p->residual_dtype));
  }
  a.out = p->out; a.ldo = p->ldo; a.out_type = p->out_dtype; a.out_scales = static_cast<uint8_t*>(p->out_scales);
  a.out_vec = p->out_dtype == LAYA_DTYPE_MX8 || vec4(p->out, p->ldo, dtype_size(p->out_dtype));
  a.out_wide = wide(p->out, p->ldo, p->out_dtype == LAYA_DTYPE_MX8 ? 1 : dtype_size(p->out_dtype));
  a.err = err;
  a.wait_ns = wait_ns();
  if (gated) launch_linear<true>(a, dev, st);
  else launch_linear<false>(a, dev, st);
  OP_API_END
}

}  // extern "C"
