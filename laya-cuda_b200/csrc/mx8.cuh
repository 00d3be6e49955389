// MX8 matrices: E4M3 values with one power-of-two scale (E8M0) per 32 consecutive values of a row,
// and the row kernels that write and read them.
//
// A block's scale is 2^e, e = floor(log2 a) - 8, plus one where a / 2^floor(log2 a) > 1.75, with a
// the block's largest magnitude: the smallest power of two under which no value passes 448 (1.75 x
// 2^8, E4M3's largest), so no value saturates.  Both steps are exact integer arithmetic on a's
// fp32 bits.  e is raised to -127 where it is lower (a below about 2^-119; such values keep fewer
// than E4M3's bits).  A block that holds an infinity or a NaN has the scale byte 255 (E8M0's NaN) and
// NaN values: it reads back as NaN.
//
// Values: [rows][ld] bytes, ld a multiple of 16; columns from `cols` to the next multiple of 16 are
// written as zeros.  Scales: tiles of 128 rows x 4 blocks (128 columns), 512 bytes each, tile
// (row / 128, block / 4) row-major; in a tile the scale of (row, block) is byte
// (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4, the order in which tcgen05.cp moves a tile into
// tensor memory (lane row % 32, column (row % 128) / 32, one byte per block).  Scale bytes of
// blocks past the last column (inside a tile) are 0; those of rows past the last are never written.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace laya {

constexpr int kMxBlock = 32;
constexpr int kMxTileRows = 128;
constexpr int kMxTileCols = 128;
constexpr int kMxTileBytes = 512;

__host__ __device__ inline int mx_col_tiles(int cols) { return (cols + kMxTileCols - 1) / kMxTileCols; }

__host__ __device__ inline size_t mx_scale_tile(int row, int col_tile, int col_tiles) {
  return ((size_t)(row / kMxTileRows) * col_tiles + col_tile) * kMxTileBytes;
}
// Offset of the four scale bytes of `row` in its tile.
__host__ __device__ inline int mx_scale_row(int row) { return (row & 31) * 16 + ((row >> 5) & 3) * 4; }

// Scale byte of a block whose largest magnitude has the fp32 bits `amax` (sign cleared; infinities
// and NaNs compare above every finite value, so one integer maximum finds them too).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  if (amax >= 0x7F800000u) return 255u;
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 0);
}
// 2^-e of a finite scale byte (bytes are at most 247, so this is a normal fp32).
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^e of a scale byte: 2^-127 is a subnormal fp32, 255 a NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Four values over their block's scale, rounded to nearest even E4M3 (v[0] in the low byte).
__device__ __forceinline__ uint32_t mx_pack4(const float* v, uint32_t byte) {
  if (byte == 255u) return 0x7F7F7F7Fu;
  const float inv = mx_inverse(byte);
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * inv), "f"(v[0] * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * inv), "f"(v[2] * inv));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Four E4M3 values as fp32 (exact: every E4M3 value is an fp16 value).
__device__ __forceinline__ void mx_unpack4(uint32_t q, float* v) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)(q & 0xFFFFu)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(q >> 16)));
  const float2 a = unpack2_f32(lo, (__half*)nullptr), b = unpack2_f32(hi, (__half*)nullptr);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }

// ---------------------------------------------------------------------------------------------
// Eight consecutive elements of a row, `n` of them valid (the others read as zeros).  `vec`: the
// pointer is aligned for whole-vector access and all eight elements are valid.
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2_f32(w[i], (T*)nullptr);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

// Whether rows at `p` with a stride of `ld` elements can be read eight elements at a time.
template <typename T>
__host__ __device__ inline bool rows_aligned(const T* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0;
}

// Writes eight values of columns col .. col + 7 (a multiple of 8) as MX8.  Four neighbouring
// threads hold a block and 16 a scale tile's 128 columns; all 32 threads of the warp call this
// together, with zeros in columns past the last.
__device__ __forceinline__ void mx_store8(const float (&v)[8], int row, int col, int cols, int col_tiles, bool live,
                                          uint8_t* q, int64_t ldq, uint8_t* scales) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, abs_bits(v[i]));
  a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
  const uint32_t byte = mx_scale_byte(a);
  const int lane = threadIdx.x & 31;
  uint32_t word = byte << (8 * ((lane >> 2) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (!live) return;
  if (col < ((cols + 15) & ~15))
    *reinterpret_cast<uint2*>(q + (size_t)row * ldq + col) = make_uint2(mx_pack4(v, byte), mx_pack4(v + 4, byte));
  if ((lane & 15) == 0 && col / kMxTileCols < col_tiles)
    *reinterpret_cast<uint32_t*>(scales + mx_scale_tile(row, col / kMxTileCols, col_tiles) + mx_scale_row(row)) = word;
}

// ---------------------------------------------------------------------------------------------
// x [rows][cols] -> MX8.  16 threads take 128 columns of a row.
// ---------------------------------------------------------------------------------------------
constexpr int kMxThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kMxThreads) mx8_quantize_kernel(const T* x, int64_t ldx, int rows, int cols, uint8_t* q,
                                                                  int64_t ldq, uint8_t* scales) {
  pdl_wait();
  const int col_tiles = mx_col_tiles(cols);
  const int64_t groups = (int64_t)rows * col_tiles;
  const bool aligned = rows_aligned(x, ldx);
  const int64_t step = (int64_t)gridDim.x * (kMxThreads / 16);
  // The loop bound is the warp's first group, so that its 32 threads stay together.
  for (int64_t g0 = (int64_t)blockIdx.x * (kMxThreads / 16) + (threadIdx.x >> 5) * 2; g0 < groups; g0 += step) {
    const int64_t g = g0 + ((threadIdx.x >> 4) & 1);
    const bool live = g < groups;
    const int row = live ? (int)(g / col_tiles) : 0;
    const int col = live ? (int)(g - (int64_t)row * col_tiles) * kMxTileCols + (threadIdx.x & 15) * 8 : 0;
    const int n = live ? min(8, cols - col) : 0;
    float v[8];
    load8(x + (size_t)row * ldx + col, n, aligned && n == 8, v);
    mx_store8(v, row, col, cols, col_tiles, live, q, ldq, scales);
  }
}

// MX8 -> out [rows][cols].  A thread takes 8 columns.
template <typename T>
__global__ void __launch_bounds__(kMxThreads) mx8_dequantize_kernel(const uint8_t* q, int64_t ldq, const uint8_t* scales,
                                                                    int rows, int cols, T* out, int64_t ldo) {
  pdl_wait();
  const int col_tiles = mx_col_tiles(cols);
  const int per_row = (cols + 7) / 8;
  const int64_t pieces = (int64_t)rows * per_row;
  const bool aligned = rows_aligned(out, ldo);
  for (int64_t i = (int64_t)blockIdx.x * kMxThreads + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * kMxThreads) {
    const int row = (int)(i / per_row), col = (int)(i - (int64_t)row * per_row) * 8;
    const uint2 w = *reinterpret_cast<const uint2*>(q + (size_t)row * ldq + col);
    const float s = mx_scale(scales[mx_scale_tile(row, col / kMxTileCols, col_tiles) + mx_scale_row(row) +
                                    ((col / kMxBlock) & 3)]);
    float v[8];
    mx_unpack4(w.x, v);
    mx_unpack4(w.y, v + 4);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= s;
    const int n = min(8, cols - col);
    store8(out + (size_t)row * ldo + col, n, aligned && n == 8, v);
  }
}

// ---------------------------------------------------------------------------------------------
// h = x + residual; sum_out = h; y = h * rsqrt(mean(h^2) + eps) * weight, written as MX8.  The row
// is summed and squared in fp32 and y is formed from the unrounded h.  One block takes one row
// at a time.
// ---------------------------------------------------------------------------------------------
struct RmsNormArgs {
  const void* x; int64_t ldx;
  const void* residual; int64_t ldr;  // or nullptr
  void* sum_out; int64_t lds;         // of the residual's type, or nullptr
  const float* weight;
  float eps;
  int rows, cols;
  uint8_t* q; int64_t ldq;
  uint8_t* scales;
};

template <typename T, typename R>
__global__ void __launch_bounds__(kMxThreads) rms_norm_mx8_kernel(const RmsNormArgs a) {
  pdl_wait();
  __shared__ float part[kMxThreads / 32];
  const int col_tiles = mx_col_tiles(a.cols);
  const int span = col_tiles * kMxTileCols;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
    const R* r = a.residual ? static_cast<const R*>(a.residual) + (size_t)row * a.ldr : nullptr;
    R* s = a.sum_out ? static_cast<R*>(a.sum_out) + (size_t)row * a.lds : nullptr;
    const bool ax = rows_aligned(x, a.ldx), ar = rows_aligned(r, a.ldr), as = rows_aligned(s, a.lds);
    float sq = 0.f;
    auto load = [&](int col, float (&h)[8]) {
      const int n = max(0, min(8, a.cols - col));
      float t[8];
      load8(x + col, n, ax && n == 8, h);
      if (r) {
        load8(r + col, n, ar && n == 8, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += t[i];
      }
      return n;
    };
    for (int col = threadIdx.x * 8; col < a.cols; col += kMxThreads * 8) {
      float h[8];
      load(col, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) sq += h[i] * h[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sq;
    __syncthreads();
    sq = 0.f;
#pragma unroll
    for (int w = 0; w < kMxThreads / 32; ++w) sq += part[w];
    const float inv = rsqrtf(sq / (float)a.cols + a.eps);
    for (int col0 = (threadIdx.x & ~31) * 8; col0 < span; col0 += kMxThreads * 8) {  // whole warps
      const int col = col0 + (threadIdx.x & 31) * 8;
      float h[8];
      const int n = load(col, h);
      if (s) store8(s + col, n, as && n == 8, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = i < n ? h[i] * inv * a.weight[col + i] : 0.f;
      mx_store8(h, row, col, a.cols, col_tiles, true, a.q, a.ldq, a.scales);
    }
    __syncthreads();
  }
}

}  // namespace laya
