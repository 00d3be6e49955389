// Product of MX8 matrices with the layer's epilogue:
//
//   y = act(X W^T + bias) + residual                        or, gated,
//   y = act(X G^T + gate_bias) * (X W^T + bias) + residual
//
// X [M][K], W and G [N][K] in MX8; y in 16 or 32 bits, or MX8 for the next product.
#pragma once
#include "mx8.cuh"

namespace laya {

enum MxAct : int { MX_ACT_NONE = 0, MX_ACT_RELU = 1, MX_ACT_GELU = 2, MX_ACT_SILU = 3 };
enum MxType : int { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 2, MX_MX8 = 3 };  // as LAYA_DTYPE_*

struct MxOperand {
  const uint8_t* q;
  int64_t ld;
  const uint8_t* scales;
};

struct MxLinearArgs {
  int M, N, K;
  MxOperand x, w, gate;       // gate.q null: not gated
  const float* bias;          // [N] or nullptr
  const float* gate_bias;     // [N] or nullptr
  int act;
  const void* residual;       // [M][N] or nullptr
  int64_t ldr;
  int residual_type;
  void* out;                  // [M][N], or MX8 values
  int64_t ldo;
  int out_type;
  uint8_t* out_scales;        // MX8 output
  int residual_vec, out_vec;  // four columns at a time may be read / written as one vector
  int* err;
  unsigned long long wait_ns;
};

__device__ __forceinline__ float mx_activate(float v, int act) {
  switch (act) {
    case MX_ACT_RELU: return fmaxf(v, 0.f);
    case MX_ACT_GELU: return gelu_erf(v);
    // v / (1 + exp(-v)): exp overflows to infinity for v far below zero, and the quotient to -0.
    case MX_ACT_SILU: return v * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * v));
    default: return v;
  }
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, bool vec, float* v) {
  if (vec && n == 4) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      const float2 f = unpack2_f32(a.x, (T*)nullptr), g = unpack2_f32(a.y, (T*)nullptr);
      v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int n, bool vec, const float* v) {
  if (vec && n == 4) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

// The epilogue of four accumulators of one row, columns col .. col + 3 (col a multiple of 4).
// Eight neighbouring threads hold 32 consecutive columns of one row from a multiple of 32 on, and the warp calls
// this together (an MX8 block's scale is found by shuffles).  Rows and columns outside the
// result are computed as zeros and not written.  The result is rounded once, here.
template <bool kGated>
__device__ __forceinline__ void mx_finish4(const MxLinearArgs& a, int row, int col, const float* acc, const float* gate) {
  const bool live = row < a.M;
  const int n = live ? max(0, min(4, a.N - col)) : 0;
  float v[4], t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = acc[i];
  if (a.bias) {
    load4(a.bias + col, n, true, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += t[i];
  }
  if (kGated) {
    float g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = gate[i];
    if (a.gate_bias) {
      load4(a.gate_bias + col, n, true, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] += t[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= mx_activate(g[i], a.act);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mx_activate(v[i], a.act);
  }
  if (a.residual) {
    const size_t at = (size_t)row * a.ldr + col;
    if (a.residual_type == MX_BF16) load4(static_cast<const __nv_bfloat16*>(a.residual) + at, n, a.residual_vec, t);
    else if (a.residual_type == MX_F16) load4(static_cast<const __half*>(a.residual) + at, n, a.residual_vec, t);
    else load4(static_cast<const float*>(a.residual) + at, n, a.residual_vec, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += t[i];
  }
  const size_t at = (size_t)row * a.ldo + col;
  if (a.out_type == MX_MX8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? v[i] : 0.f;
    uint32_t m = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
    const uint32_t byte = mx_scale_byte(m);
    if (live && col < ((a.N + 15) & ~15)) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + at) = mx_pack4(v, byte);
    const int col_tiles = mx_col_tiles(a.N), col_tile = col / kMxTileCols;
    if (live && (threadIdx.x & 7) == 0 && col_tile < col_tiles)
      a.out_scales[mx_scale_tile(row, col_tile, col_tiles) + mx_scale_row(row) + ((col / kMxBlock) & 3)] = (uint8_t)byte;
  } else if (a.out_type == MX_BF16) {
    store4(static_cast<__nv_bfloat16*>(a.out) + at, n, a.out_vec, v);
  } else if (a.out_type == MX_F16) {
    store4(static_cast<__half*>(a.out) + at, n, a.out_vec, v);
  } else {
    store4(static_cast<float*>(a.out) + at, n, a.out_vec, v);
  }
}

// ---------------------------------------------------------------------------------------------
// Product on the fp32 pipe: 64 x 64 tiles, one block of 32 columns of K at a time through shared
// memory, 4 x 4 sums per thread.
// ---------------------------------------------------------------------------------------------
constexpr int kMxSimpleTile = 64;

__device__ __forceinline__ void mx_stage(const MxOperand& m, int row0, int rows, int k, int K, float (*s)[kMxSimpleTile + 4]) {
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8, row = row0 + r;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (row < rows && k + c < K) {
    const uint2 q = *reinterpret_cast<const uint2*>(m.q + (size_t)row * m.ld + k + c);
    const float f = mx_scale(m.scales[mx_scale_tile(row, k / kMxTileCols, mx_col_tiles(K)) + mx_scale_row(row) + ((k / kMxBlock) & 3)]);
    mx_unpack4(q.x, v);
    mx_unpack4(q.y, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + c + i < K ? v[i] * f : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[c + i][r] = v[i];
}

template <bool kGated>
__global__ void __launch_bounds__(256) mx8_linear_simple_kernel(const MxLinearArgs a) {
  pdl_wait();
  __shared__ float sx[kMxBlock][kMxSimpleTile + 4], sw[kMxBlock][kMxSimpleTile + 4], sg[kGated ? kMxBlock : 1][kMxSimpleTile + 4];
  const int m0 = blockIdx.y * kMxSimpleTile, n0 = blockIdx.x * kMxSimpleTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {}, gate[4][4] = {};
  for (int k = 0; k < a.K; k += kMxBlock) {
    mx_stage(a.x, m0, a.M, k, a.K, sx);
    mx_stage(a.w, n0, a.N, k, a.K, sw);
    if (kGated) mx_stage(a.gate, n0, a.N, k, a.K, sg);
    __syncthreads();
#pragma unroll 8
    for (int i = 0; i < kMxBlock; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[r][c] = fmaf(sx[i][ty * 4 + r], sw[i][tx * 4 + c], acc[r][c]);
          if (kGated) gate[r][c] = fmaf(sx[i][ty * 4 + r], sg[i][tx * 4 + c], gate[r][c]);
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) mx_finish4<kGated>(a, m0 + ty * 4 + r, n0 + tx * 4, acc[r], gate[r]);
}

}  // namespace laya
