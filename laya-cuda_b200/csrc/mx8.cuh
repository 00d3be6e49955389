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

// cols at least 1 and up to 2^31 - 1 (the sum of cols and a tile would wrap).
__host__ __device__ inline int mx_col_tiles(int cols) { return (cols - 1) / kMxTileCols + 1; }

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
// 2^-e of a scale byte (finite ones are at most 247, so this is a normal fp32); NaN for 255.
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : (254u - byte) << 23);
}
// 2^e of a scale byte: 2^-127 is a subnormal fp32, 255 a NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}

// Four values times their block's inverse scale, rounded to nearest even E4M3 (v[0] in the low byte;
// a NaN becomes 0x7F).
__device__ __forceinline__ uint32_t mx_pack4(const float* v, float inverse) {
  const float2 f = make_float2(inverse, inverse);
  const float2 a = mul2(make_float2(v[0], v[1]), f), b = mul2(make_float2(v[2], v[3]), f);
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// max(a, |b|, |c|) that keeps a NaN.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
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
// A piece: sixteen consecutive columns of a row, half a block, held by one thread.  Eight columns a
// thread made the conversions instruction-bound (155 instructions per thread for 8 columns, 52 us
// for 16384 x 4096 bf16 to MX8); sixteen share the addresses and shuffles.
//
// kVec: rows of whole 32-byte vectors (`rows_vectored`), read and written as such; a thread's bf16
// piece is one of them.  (Two 16-byte stores per thread instead fill half sectors: 48 us where this
// took 35 for 16384 x 4096 back to bf16.)  Otherwise rows of any length and alignment: a piece is read
// as the aligned 16-byte granules that hold it, shifted into place, and written through shared memory:
// element by element so that neighbouring lanes write neighbouring elements (`store_any`), or in
// sectors put together from two lanes' pieces (`store_run`).
// ---------------------------------------------------------------------------------------------
constexpr int kMxPiece = 16;

template <typename T>
struct Raw {
  uint32_t w[4 * sizeof(T)];
};

template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p, bool live) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(r.w) / 32; ++i) {
    uint32_t* w = r.w + 8 * i;
    if (live) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(reinterpret_cast<const char*>(p) + 32 * i));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = 0;
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&v)[kMxPiece]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kMxPiece; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kMxPiece / 2; ++i) {
      const float2 f = unpack2_f32(r.w[i], (T*)nullptr);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw<T> pack(const float (&v)[kMxPiece]) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kMxPiece; ++i) r.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kMxPiece / 2; ++i) r.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  }
  return r;
}

// Sixteen elements to 32-byte aligned p.
template <typename T>
__device__ __forceinline__ void store_raw(void* p, const Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(r.w) / 32; ++i) {
    const uint32_t* w = r.w + 8 * i;
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<char*>(p) + 32 * i),
                 "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  }
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, bool live, const float (&v)[kMxPiece]) {
  const Raw<T> r = pack<T>(v);
  if (live) store_raw(p, r);
}

// Sixteen elements out of the 16-byte granules that hold them, the first at byte `shift` of 16.
template <typename T>
__device__ __forceinline__ Raw<T> shift_granules(uint32_t (&w)[4 * (sizeof(T) + 1)], uint32_t shift) {
  constexpr int kWords = 4 * (sizeof(T) + 1);
#pragma unroll
  for (int i = 0; i + 2 < kWords; ++i) w[i] = shift & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i + 1 < kWords - 2; ++i) w[i] = shift & 4 ? w[i + 1] : w[i];
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)(4 * sizeof(T)); ++i)
    r.w[i] = sizeof(T) == 2 && (shift & 2) ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  return r;
}

// The first n of sixteen elements at p, zeros for the others.  Only granules that hold an element
// asked for are read.
template <typename T>
__device__ __forceinline__ void load_any(const T* p, int n, float (&v)[kMxPiece]) {
  n = max(0, min(n, kMxPiece));
  constexpr int kGranules = (int)sizeof(T) + 1;
  const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15;
  const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - shift);
  const int end = n ? (int)shift + n * (int)sizeof(T) : 0;
  uint32_t w[4 * kGranules];
#pragma unroll
  for (int i = 0; i < kGranules; ++i) {
    uint4 g = make_uint4(0, 0, 0, 0);
    if (16 * i < end) g = base[i];
    w[4 * i] = g.x; w[4 * i + 1] = g.y; w[4 * i + 2] = g.z; w[4 * i + 3] = g.w;
  }
  unpack(shift_granules<T>(w, shift), v);
#pragma unroll
  for (int i = 0; i < kMxPiece; ++i) v[i] = i < n ? v[i] : 0.f;
}

// The lanes' sixteen elements to `stage`, 512 elements of shared memory of the warp's own, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void stage_pieces(T* stage, const float (&v)[kMxPiece]) {
  const Raw<T> r = pack<T>(v);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i)
    reinterpret_cast<uint4*>(stage + (threadIdx.x & 31) * kMxPiece)[i] =
        make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  __syncwarp();
}

// The first n of each lane's sixteen elements to its p; the warp calls this together.
template <typename T>
__device__ __forceinline__ void store_any(T* stage, T* p, int n, const float (&v)[kMxPiece]) {
  const int lane = threadIdx.x & 31;
  stage_pieces(stage, v);
#pragma unroll
  for (int j = 0; j < kMxPiece; ++j) {
    const int from = 2 * j + (lane >> 4), at = lane & 15;
    T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
    const int many = __shfl_sync(0xffffffffu, n, from);
    if (at < many) to[at] = stage[32 * j + lane];
  }
}

// The same for 16-bit types where most lanes' pieces follow one another: a lane whose p follows the piece of the
// lane before writes the whole 32-byte sector that holds its first element, the end of that piece and the start of
// its own.  What is in no lane's sector (the ends of rows and of the warp's run) goes an element at a time, two
// lanes' pieces per instruction.
template <typename T>
__device__ __forceinline__ void store_run(T* stage, T* p, int n, const float (&v)[kMxPiece]) {
  static_assert(sizeof(T) == 2, "a piece is a sector");
  const int lane = threadIdx.x & 31;
  stage_pieces(stage, v);
  n = max(0, min(n, kMxPiece));
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const int over = (int)(at & 31);   // bytes of the sector before p
  const int head = (32 - over) / 2;  // elements of this piece in the sector
  const uintptr_t before = __shfl_up_sync(0xffffffffu, (unsigned long long)(n == kMxPiece ? at : 0), 1);
  const bool follows = lane > 0 && before != 0 && before + 32 == at && n >= head;
  const bool whole = follows || (over == 0 && n == kMxPiece);
  const bool followed = __shfl_down_sync(0xffffffffu, (int)follows, 1) && lane < 31;
  if (whole) {
    const int from = lane * 32 - over;  // of the warp's bytes in `stage`
    const uint32_t shift = (uint32_t)from & 15;
    const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(stage) + (from - (int)shift));
    uint32_t w[12];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      uint4 g = make_uint4(0, 0, 0, 0);
      if (i < 2 || shift) g = base[i];
      w[4 * i] = g.x; w[4 * i + 1] = g.y; w[4 * i + 2] = g.z; w[4 * i + 3] = g.w;
    }
    store_raw(reinterpret_cast<char*>(p) - over, shift_granules<T>(w, shift));
  }
  // Bit i: element i is in no lane's sector.
  const uint32_t rest = ((1u << n) - 1) & ((whole ? 0 : (1u << head) - 1) | (followed ? 0 : ~0u << head));
  uint32_t lanes = __ballot_sync(0xffffffffu, rest != 0);
  while (lanes) {
    const int first = __ffs(lanes) - 1;
    lanes &= lanes - 1;
    const int second = lanes ? __ffs(lanes) - 1 : first;
    lanes &= lanes - 1;
    const int of = lane < kMxPiece ? first : second, i = lane & (kMxPiece - 1);
    const uint32_t bits = __shfl_sync(0xffffffffu, rest, of);
    T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, (unsigned long long)at, of));
    if (bits >> i & 1) to[i] = stage[of * kMxPiece + i];
  }
}

template <typename T>
inline bool rows_vectored(const T* p, int64_t ld, int cols) {
  return reinterpret_cast<uintptr_t>(p) % 32 == 0 && ld * (int64_t)sizeof(T) % 32 == 0 && cols % kMxPiece == 0;
}

// Writes a piece as MX8.  Two neighbouring threads hold a block and eight a scale tile's 128 columns;
// all 32 threads of the warp call this together, with zeros in columns past the last.  `col` may be past the last
// column, and past 2^31 with it.
__device__ __forceinline__ void mx_store_piece(const float (&v)[kMxPiece], int row, uint32_t col, int cols, int col_tiles, bool live,
                                               uint8_t* q, int64_t ldq, uint8_t* scales) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kMxPiece; i += 2) most = max_abs3(most, v[i], v[i + 1]);
  uint32_t a = __float_as_uint(most);
  a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
  const uint32_t byte = mx_scale_byte(a);
  const int lane = threadIdx.x & 31;
  uint32_t word = byte << (4 * (lane & 6));
  word |= __shfl_xor_sync(0xffffffffu, word, 2);
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  const uint32_t col_tile = col / kMxTileCols;
  if (!live || col_tile >= (uint32_t)col_tiles) return;
  if (col < (uint32_t)cols) {
    const float inverse = mx_inverse(byte);
    *reinterpret_cast<uint4*>(q + (size_t)row * ldq + col) =
        make_uint4(mx_pack4(v, inverse), mx_pack4(v + 4, inverse), mx_pack4(v + 8, inverse), mx_pack4(v + 12, inverse));
  }
  if ((lane & 7) == 0)
    *reinterpret_cast<uint32_t*>(scales + mx_scale_tile(row, (int)col_tile, col_tiles) + mx_scale_row(row)) = word;
}

// ---------------------------------------------------------------------------------------------
// x [rows][cols] -> MX8.  Eight threads take 128 columns of a row (a group).  HBM-bound: x is read and the
// values and scales written once, 16384 x 4096 bf16 in 32.5 us (6.3 TB/s) and 9216 x 4096 fp32 in 28.3 (6.7; a
// copy's rate is 6.5); a small call is its launch (768 values: 1.2 us).  Rows without 32-byte alignment: 16384 x
// 4095 bf16 in 40 us, three granule loads a piece instead of one vector, fp32 in 54 (16384 x 4096: 52 for its bytes).
// ---------------------------------------------------------------------------------------------
constexpr int kMxThreads = 256;

template <typename T, bool kVec>
__global__ void __launch_bounds__(kMxThreads) mx8_quantize_kernel(const T* x, int64_t ldx, int rows, int cols, FastDiv col_tiles,
                                                                  uint8_t* q, int64_t ldq, uint8_t* scales) {
  pdl_wait();
  const uint32_t groups = (uint32_t)rows * col_tiles.d;  // below 2^31
  const uint32_t step = gridDim.x * (kMxThreads / 8);
  // The loop bound is the warp's first group, so that its 32 threads stay together.
  for (uint32_t g0 = blockIdx.x * (kMxThreads / 8) + (threadIdx.x >> 5) * 4; g0 < groups; g0 += step) {
    const uint32_t g = g0 + ((threadIdx.x >> 3) & 3);
    const bool live = g < groups;
    const int row = live ? (int)col_tiles.div(g) : 0;
    const int col = live ? (int)(g - (uint32_t)row * col_tiles.d) * kMxTileCols + (threadIdx.x & 7) * kMxPiece : 0;
    const T* p = x + (size_t)row * ldx + col;
    float v[kMxPiece];
    if constexpr (kVec) unpack(load_raw(p, live && col < cols), v);
    else load_any(p, live ? cols - col : 0, v);
    mx_store_piece(v, row, col, cols, (int)col_tiles.d, live, q, ldq, scales);
  }
}

// MX8 -> out [rows][cols], a piece per thread.  HBM-bound, two thirds of it writes: 16384 x 4096 to bf16 in
// 32.0 us (6.4 TB/s), to fp32 in 51.9 (6.5).
enum class MxStore { kVectors, kElements, kRuns };

template <typename T, MxStore kStore>
__global__ void __launch_bounds__(kMxThreads) mx8_dequantize_kernel(const uint8_t* q, int64_t ldq, const uint8_t* scales,
                                                                    int rows, int cols, FastDiv per_row, T* out, int64_t ldo) {
  pdl_wait();
  const int col_tiles = mx_col_tiles(cols);
  const uint32_t pieces = (uint32_t)rows * per_row.d;  // below 2^31
  const uint32_t step = gridDim.x * kMxThreads;
  constexpr bool kStaged = kStore != MxStore::kVectors;
  __shared__ __align__(16) T stage[kStaged ? kMxThreads / 32 : 1][kStaged ? 32 * kMxPiece : 8];
  // The loop bound is the warp's first piece, so that its 32 threads stay together.
  for (uint32_t w0 = blockIdx.x * kMxThreads + (threadIdx.x & ~31u); w0 < pieces; w0 += step) {
    const bool live = w0 + (threadIdx.x & 31) < pieces;
    const uint32_t i = min(w0 + (threadIdx.x & 31), pieces - 1);  // past the end: the last piece again, not stored
    const int row = (int)per_row.div(i), col = (int)(i - (uint32_t)row * per_row.d) * kMxPiece;
    const uint4 w = *reinterpret_cast<const uint4*>(q + (size_t)row * ldq + col);
    const float s = mx_scale(scales[mx_scale_tile(row, col / kMxTileCols, col_tiles) + mx_scale_row(row) + ((col / kMxBlock) & 3)]);
    float v[kMxPiece];
    mx_unpack4(w.x, v);
    mx_unpack4(w.y, v + 4);
    mx_unpack4(w.z, v + 8);
    mx_unpack4(w.w, v + 12);
#pragma unroll
    for (int k = 0; k < kMxPiece; k += 2) {
      const float2 t = mul2(make_float2(v[k], v[k + 1]), make_float2(s, s));
      v[k] = t.x;
      v[k + 1] = t.y;
    }
    T* p = out + (size_t)row * ldo + col;
    if constexpr (kStore == MxStore::kVectors) store_vec(p, live, v);
    else if constexpr (kStore == MxStore::kRuns) store_run(stage[threadIdx.x >> 5], p, live ? cols - col : 0, v);
    else store_any(stage[threadIdx.x >> 5], p, live ? cols - col : 0, v);
  }
}

// ---------------------------------------------------------------------------------------------
// h = x + residual; sum_out = h; y = h * rsqrt(mean(h^2) + eps) * weight, written as MX8.  The row
// is summed and squared in fp32 and y is formed from the unrounded h.
//
// HBM-bound: x and the residual are read once and h, the values and the scales written once.  `warps`
// warps (for short rows, 8 or 16 lanes) hold a row in registers, CH pieces per thread, and a block of at least 256 threads
// walks over rows with the weight in registers too; the next row's loads are issued before this
// row's sum of squares is exchanged, so that a block always has a row in flight.  16384 x 4096 bf16 with the
// residual in 73-75 us (6.3-6.5 TB/s, 97-99% of a copy's rate; reading the row twice and eight columns per
// thread took 168); 16384 x 768 bf16 onto fp32 23.6 us (5.9 TB/s); 4096 values 2.3 us.
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
  int warps;                          // per row, a power of two
  int lanes;                          // per short row: 8 or 16
};

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sum over each `lanes` neighbouring lanes, a power of two.
__device__ __forceinline__ float lanes_total(float v, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// kShort: rows of up to 256 columns, held by 8 or 16 lanes each (16384 x 128 bf16: 3.9 us, with a warp each 8.0).
template <typename T, typename R, int CH, bool kVec, bool kShort>
__global__ void __launch_bounds__(512) rms_norm_mx8_kernel(const RmsNormArgs a) {
  pdl_wait();
  __shared__ float part[2][16];
  __shared__ __align__(16) R stage[kVec ? 1 : 16][kVec ? 8 : 32 * kMxPiece];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lanes = kShort ? a.lanes : 32, per_warp = 32 / lanes;
  const int per_block = (int)(blockDim.x >> 5) / a.warps * per_warp;  // rows of a block
  const int team = warp / a.warps, within = warp - team * a.warps;
  const int sub = team * per_warp + lane / lanes, place = lane & (lanes - 1);
  const int col_tiles = mx_col_tiles(a.cols);
  const T* x = static_cast<const T*>(a.x);
  const R* r = static_cast<const R*>(a.residual);
  R* sum = static_cast<R*>(a.sum_out);
  int col[CH];
  float w[CH][kMxPiece];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    col[c] = ((c * a.warps + within) * 32 + place) * kMxPiece;
    load_any(a.weight + col[c], a.cols - col[c], w[c]);
  }
  Raw<T> rx[kVec ? CH : 1];
  Raw<R> rr[kVec ? CH : 1];
  const uint32_t rows = (uint32_t)a.rows;  // rows step past 2^31
  auto fetch = [&](uint32_t row) {
    if constexpr (kVec) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const bool in = row < rows && col[c] < a.cols;
        rx[c] = load_raw(x + (size_t)row * a.ldx + col[c], in);
        rr[c] = load_raw(r + (size_t)row * a.ldr + col[c], in && r);
      }
    }
  };
  const uint32_t step = gridDim.x * per_block;
  int turn = 0;
  uint32_t row = blockIdx.x * per_block + sub;
  fetch(row);
  for (uint32_t row0 = blockIdx.x * per_block; row0 < rows; row0 += step, row += step, turn ^= 1) {
    const bool live = row < rows;
    float h[CH][kMxPiece];
    float2 sq2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float t[kMxPiece];
      if constexpr (kVec) {
        unpack(rx[c], h[c]);
        unpack(rr[c], t);
      } else {
        const int n = live ? a.cols - col[c] : 0;
        load_any(x + (size_t)row * a.ldx + col[c], n, h[c]);
        load_any(r + (size_t)row * a.ldr + col[c], r ? n : 0, t);
      }
#pragma unroll
      for (int i = 0; i < kMxPiece; i += 2) {
        const float2 f = add2(make_float2(h[c][i], h[c][i + 1]), make_float2(t[i], t[i + 1]));
        sq2 = fma2(f, f, sq2);
        h[c][i] = f.x;
        h[c][i + 1] = f.y;
      }
    }
    fetch(row + step);
    if (sum) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        R* p = sum + (size_t)row * a.lds + col[c];
        if constexpr (kVec) store_vec(p, live && col[c] < a.cols, h[c]);
        else store_any(stage[warp], p, live ? a.cols - col[c] : 0, h[c]);
      }
    }
    float sq = kShort ? lanes_total(sq2.x + sq2.y, lanes) : warp_total(sq2.x + sq2.y);
    if (!kShort && a.warps > 1) {
      // Two sets of sums, taken in turn: a warp may be one row ahead of the others here.
      if (lane == 0) part[turn][warp] = sq;
      __syncthreads();
      sq = warp_total(lane < a.warps ? part[turn][team * a.warps + lane] : 0.f);
    }
    const float inv = rsqrtf(sq / (float)a.cols + a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (col[c] - lane * kMxPiece >= a.cols) break;  // the whole warp is past the row
#pragma unroll
      for (int i = 0; i < kMxPiece; i += 2) {
        const float2 f = mul2(mul2(make_float2(h[c][i], h[c][i + 1]), make_float2(inv, inv)), make_float2(w[c][i], w[c][i + 1]));
        // A NaN stays out of the columns past the last.
        h[c][i] = col[c] + (kVec ? 0 : i) < a.cols ? f.x : 0.f;
        h[c][i + 1] = col[c] + (kVec ? 0 : i + 1) < a.cols ? f.y : 0.f;
      }
      mx_store_piece(h[c], (int)row, col[c], a.cols, col_tiles, live, a.q, a.ldq, a.scales);
    }
  }
}

// Rows too long for the registers of 16 warps: one block takes one row at a time and reads it twice
// (1024 x 40000 bf16 with the residual: 159 us, against 80 for 4096 x 16384 in registers).
template <typename T, typename R>
__global__ void __launch_bounds__(kMxThreads) rms_norm_mx8_long_kernel(const RmsNormArgs a) {
  pdl_wait();
  __shared__ float part[kMxThreads / 32];
  __shared__ __align__(16) R stage[kMxThreads / 32][32 * kMxPiece];
  const int col_tiles = mx_col_tiles(a.cols);
  for (uint32_t row = blockIdx.x; row < (uint32_t)a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
    const R* r = a.residual ? static_cast<const R*>(a.residual) + (size_t)row * a.ldr : nullptr;
    R* s = a.sum_out ? static_cast<R*>(a.sum_out) + (size_t)row * a.lds : nullptr;
    const uint32_t cols = (uint32_t)a.cols;  // columns step past 2^31
    auto load = [&](uint32_t col, float (&h)[kMxPiece]) {
      const int n = (int)(cols - col);
      load_any(x + col, n, h);
      if (r) {
        float t[kMxPiece];
        load_any(r + col, n, t);
#pragma unroll
        for (int i = 0; i < kMxPiece; ++i) h[i] += t[i];
      }
    };
    float sq = 0.f;
    for (uint32_t col = threadIdx.x * kMxPiece; col < cols; col += kMxThreads * kMxPiece) {
      float h[kMxPiece];
      load(col, h);
#pragma unroll
      for (int i = 0; i < kMxPiece; ++i) sq = fmaf(h[i], h[i], sq);
    }
    sq = warp_total(sq);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sq;
    __syncthreads();
    sq = 0.f;
#pragma unroll
    for (int w = 0; w < kMxThreads / 32; ++w) sq += part[w];
    const float inv = rsqrtf(sq / (float)a.cols + a.eps);
    for (uint32_t col0 = (threadIdx.x & ~31) * kMxPiece; col0 < cols; col0 += kMxThreads * kMxPiece) {  // whole warps
      const uint32_t col = col0 + (threadIdx.x & 31) * kMxPiece;
      const int n = (int)(cols - col);
      float h[kMxPiece];
      load(col, h);
      if (s) {
        if constexpr (sizeof(R) == 2) store_run(stage[threadIdx.x >> 5], s + col, n, h);
        else store_any(stage[threadIdx.x >> 5], s + col, n, h);
      }
#pragma unroll
      for (int i = 0; i < kMxPiece; ++i) h[i] = i < n ? h[i] * inv * a.weight[col + i] : 0.f;
      mx_store_piece(h, (int)row, col, a.cols, col_tiles, true, a.q, a.ldq, a.scales);
    }
    __syncthreads();
  }
}

}  // namespace laya
