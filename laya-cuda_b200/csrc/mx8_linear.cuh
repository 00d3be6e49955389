// The MX8 linear layer's arguments and epilogue (the products are in mx8_gemm.cuh):
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
  int residual_vec, out_vec;    // four columns at a time may be read / written as one vector
  int residual_wide, out_wide;  // and 32 bytes at a time, from columns that are multiples of 32 on
  int* err;
  unsigned long long wait_ns;
};

// v / (1 + exp(-v)): the exponential overflows to infinity for v far below zero, the quotient to -0.
__device__ __forceinline__ float mx_silu(float v) { return v * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * v)); }
// x Phi(x) with a small relative error on both sides of zero, as the fp32 results need it (the encoder's gelu_erf2 keeps an
// absolute one for 16-bit results: it takes 1 - (1 - q) for negative x, which cancels).  With a = |x|,
//   q = Phi(-a) = exp(-a^2 / 2) t P(t),  t = 1 / (1 + p a),  and  x Phi(x) = x q for x <= 0, x (1 - q) for x > 0.
// P: the degree-7 polynomial of least relative error (1.0e-7) for 0 <= a <= 14.5, fitted for this function.  With the roundings
// and the special functions' errors the result is within (25 + 1.5 x^2) 2^-24 of itself, the second term from the
// exponent's rounding; below x = -13.2 the exponential is 0.  16384 x 64 x 4096 in bf16, all epilogue, takes 69 us
// (gelu_erf2 64.5), 4096 x 768 x 3072 in f16 20.0 (19.6), 511 x 776 x 2304 7.0 with either.
__device__ __forceinline__ float2 mx_gelu2(float2 x) {
  auto twice = [](float c) { return make_float2(c, c); };
  const float2 d = fma2(make_float2(fabsf(x.x), fabsf(x.y)), twice(0.305f), twice(1.0f));
  const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  float2 h = fma2(twice(0.03663905f), t, twice(-0.15274677f));
  h = fma2(h, t, twice(0.18531595f));
  h = fma2(h, t, twice(-0.037621517f));
  h = fma2(h, t, twice(0.12084079f));
  h = fma2(h, t, twice(0.10347359f));
  h = fma2(h, t, twice(0.1224587f));
  h = fma2(h, t, twice(0.12164024f));
  const float2 w = mul2(mul2(x, twice(-0.72134752044448170f)), x);  // -x^2 / 2 in powers of two
  const float2 q = mul2(mul2(h, t), make_float2(ex2_approx(w.x), ex2_approx(w.y)));
  const float2 r = fma2(q, twice(-1.0f), twice(1.0f));
  return mul2(x, make_float2(x.x > 0.f ? r.x : q.x, x.y > 0.f ? r.y : q.y));
}
// max(v, 0) that keeps a NaN.
__device__ __forceinline__ float mx_relu(float v) { return v < 0.f ? 0.f : v; }

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

// ---------------------------------------------------------------------------------------------
// Epilogue of R rows by four columns per thread (few rows): the thread's rows row0, row0 + step, ..., columns
// col .. col + 3 (col a multiple of 4).  Eight neighbouring threads hold 32 consecutive columns
// of a row from a multiple of 32 on, and the warp calls these functions together (an MX8 block's scale is
// found by shuffles).  Rows from `end` on (at most M) and columns outside the result are not read or
// written.
//
// MxInputs is what the epilogue reads beside the products.  It is fetched apart from its use, so
// that a caller can have other loads in flight with these.  `whole`: every element of the warp's chunk is
// inside the result and may be accessed four columns at a time (the same in all lanes).
template <int R>
struct MxInputs {
  float bias[4], gate_bias[4];
  uint4 res[R];  // four residual values: fp32, or 16-bit pairs in x and y when `packed`
  bool whole, packed;
};

template <bool kGated, int R>
__device__ __forceinline__ void mx_fetch(const MxLinearArgs& a, int row0, int step, int end, int col, bool whole, MxInputs<R>& in) {
  const int n = max(0, min(4, a.N - col));
  in.whole = whole && a.out_vec && (!a.residual || a.residual_vec);
  if (a.bias) load4(a.bias + col, n, true, in.bias);
  if (kGated && a.gate_bias) load4(a.gate_bias + col, n, true, in.gate_bias);
  if (!a.residual) return;
  in.packed = in.whole && a.residual_type != MX_F32;
  if (in.packed) {
    const uint16_t* p = static_cast<const uint16_t*>(a.residual) + (size_t)row0 * a.ldr + col;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const uint2 w = *reinterpret_cast<const uint2*>(p + (size_t)(k * step) * a.ldr);
      in.res[k].x = w.x;
      in.res[k].y = w.y;
    }
  } else if (in.whole) {
    const float* p = static_cast<const float*>(a.residual) + (size_t)row0 * a.ldr + col;
#pragma unroll
    for (int k = 0; k < R; ++k) in.res[k] = *reinterpret_cast<const uint4*>(p + (size_t)(k * step) * a.ldr);
  } else {
    auto read = [&](auto* p) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int row = row0 + k * step;
        float t[4];
        load4(p + (size_t)row * a.ldr + col, row < end ? n : 0, a.residual_vec, t);
        in.res[k] = make_uint4(__float_as_uint(t[0]), __float_as_uint(t[1]), __float_as_uint(t[2]), __float_as_uint(t[3]));
      }
    };
    if (a.residual_type == MX_BF16) read(static_cast<const __nv_bfloat16*>(a.residual));
    else if (a.residual_type == MX_F16) read(static_cast<const __half*>(a.residual));
    else read(static_cast<const float*>(a.residual));
  }
}

// acc: the products with W, gate: those with G.  Everything is fp32 and rounded once, to the
// output's type.
template <bool kGated, int R>
__device__ __forceinline__ void mx_finish(const MxLinearArgs& a, int row0, int step, int end, int col,
                                          float (&acc)[R][4], float (&gate)[R][4], const MxInputs<R>& in) {
  const int n = max(0, min(4, a.N - col));
  if (a.bias) {
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[k][i] += in.bias[i];
  }
  if (kGated && a.gate_bias) {
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) gate[k][i] += in.gate_bias[i];
  }
  float(&on)[R][4] = kGated ? gate : acc;
  auto apply = [&](auto f) {
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float2 y = f(make_float2(on[k][i], on[k][i + 1]));
        on[k][i] = y.x;
        on[k][i + 1] = y.y;
      }
  };
  if (a.act == MX_ACT_GELU) apply([](float2 v) { return mx_gelu2(v); });
  else if (a.act == MX_ACT_SILU) apply([](float2 v) { return make_float2(mx_silu(v.x), mx_silu(v.y)); });
  else if (a.act == MX_ACT_RELU) apply([](float2 v) { return make_float2(mx_relu(v.x), mx_relu(v.y)); });
  if (kGated) {
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[k][i] *= gate[k][i];
  }
  if (a.residual) {
    auto add = [&](auto* type) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float2 lo = unpack2_f32(in.res[k].x, type), hi = unpack2_f32(in.res[k].y, type);
        acc[k][0] += lo.x; acc[k][1] += lo.y; acc[k][2] += hi.x; acc[k][3] += hi.y;
      }
    };
    if (in.packed && a.residual_type == MX_BF16) add((__nv_bfloat16*)nullptr);
    else if (in.packed) add((__half*)nullptr);
    else {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        acc[k][0] += __uint_as_float(in.res[k].x);
        acc[k][1] += __uint_as_float(in.res[k].y);
        acc[k][2] += __uint_as_float(in.res[k].z);
        acc[k][3] += __uint_as_float(in.res[k].w);
      }
    }
  }
  if (a.out_type != MX_MX8) {
    auto write = [&](auto* p) {
      p += (size_t)row0 * a.ldo + col;
      if (in.whole) {
#pragma unroll
        for (int k = 0; k < R; ++k) store4(p + (size_t)(k * step) * a.ldo, 4, true, acc[k]);
      } else {
#pragma unroll
        for (int k = 0; k < R; ++k)
          if (row0 + k * step < end) store4(p + (size_t)(k * step) * a.ldo, n, a.out_vec, acc[k]);
      }
    };
    if (a.out_type == MX_BF16) write(static_cast<__nv_bfloat16*>(a.out));
    else if (a.out_type == MX_F16) write(static_cast<__half*>(a.out));
    else write(static_cast<float*>(a.out));
  } else {
    const int col_tiles = mx_col_tiles(a.N), col_tile = col / kMxTileCols;
    const bool in_values = col < ((a.N + 15) & ~15), in_scales = (threadIdx.x & 7) == 0 && col_tile < col_tiles;
    uint8_t* q = static_cast<uint8_t*>(a.out) + (size_t)row0 * a.ldo + col;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int row = row0 + k * step;
      if (n < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[k][i] = i < n ? acc[k][i] : 0.f;
      }
      uint32_t m = __float_as_uint(max_abs3(max_abs3(0.f, acc[k][0], acc[k][1]), acc[k][2], acc[k][3]));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
      const uint32_t byte = mx_scale_byte(m);
      if (row < end) {
        if (in_values) *reinterpret_cast<uint32_t*>(q + (size_t)(k * step) * a.ldo) = mx_pack4(acc[k], mx_inverse(byte));
        if (in_scales)
          a.out_scales[mx_scale_tile(row, col_tile, col_tiles) + mx_scale_row(row) + ((col / kMxBlock) & 3)] = (uint8_t)byte;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Epilogue of 32 columns of one row per thread (many rows): the lane's accumulator row as tensor memory
// gives it, columns c0 .. c0 + 31, c0 a multiple of 32.  An MX8 block is one thread's, and 32-byte accesses
// fill whole sectors without a transpose.  With K = 64, where the epilogue is all there is, 16384 x 4096 results
// take 36 us in bf16 (of which 21 to write them), 33 in MX8 (11), 69 in bf16 with a GELU (its two special-
// function operations per result are 2.2 us of a tile's 4.9) and 72 in bf16 with a bf16 residual (41 for the
// bytes): launches in a row over three sets of buffers.  On one set, where the choice was made, 34, 26, 56 (with the
// encoder's shorter GELU) and 71; four columns of eight rows per thread, through shared memory, 39, 112, 79 and 75.
// ---------------------------------------------------------------------------------------------

// How a kernel reads the residual.  The common forms are kernels of their own: a load behind a test (of
// the type, the alignment, the row) is waited for where the paths join again, and not where it is used
// (16384 x 64 x 4096 + bf16: 2,200 cycles a tile before the accumulator was even looked at).
enum MxResidual : int {
  MX_RES_NONE = 0,
  MX_RES_HALF = 1,  // 16-bit rows of whole aligned 32-byte vectors, N a multiple of 32
  MX_RES_FULL = 2,  // 32-bit rows, the same
  MX_RES_ANY_HALF = 3,  // 16-bit rows of any alignment and length
  MX_RES_ANY_FULL = 4   // 32-bit rows, the same
};
__host__ __device__ constexpr int mx_res_size(int res) { return res == MX_RES_HALF || res == MX_RES_ANY_HALF ? 2 : 4; }

// 32 residual values of a row as loaded: whole vectors, or, for rows of any alignment, the aligned 16-byte granules that
// hold them, `shift` bytes into the first.  Fetched apart from their use, so that the loads are in flight while
// the accumulator is waited for.
template <int kRes>
struct MxResidualRow {
  uint32_t w[kRes == MX_RES_NONE ? 1 : kRes == MX_RES_HALF ? 16 : kRes == MX_RES_FULL ? 32 : kRes == MX_RES_ANY_HALF ? 20 : 36];
  uint32_t shift;
};

template <int kRes>
__device__ __forceinline__ void mx_fetch_row(const MxLinearArgs& a, int row, int c0, MxResidualRow<kRes>& in) {
  if constexpr (kRes == MX_RES_HALF || kRes == MX_RES_FULL) {
    // Lanes and chunks outside the result read its last row or chunk again.
    constexpr int kSize = mx_res_size(kRes);
    const size_t at = (size_t)min(row, a.M - 1) * a.ldr + min(c0, a.N - 32);
    const char* p = static_cast<const char*>(a.residual) + at * kSize;
#pragma unroll
    for (int i = 0; i < kSize; ++i) {
      uint32_t* w = in.w + 8 * i;
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p + 32 * i));
    }
  } else if constexpr (kRes != MX_RES_NONE) {
    // Only granules with an element of the result are read: past the row's last one, that one again.
    constexpr int kSize = mx_res_size(kRes);
    const char* first = static_cast<const char*>(a.residual) + (size_t)min(row, a.M - 1) * a.ldr * kSize;
    const uintptr_t at = reinterpret_cast<uintptr_t>(first) + (size_t)min(c0, a.N - 1) * kSize;
    const uintptr_t last = (reinterpret_cast<uintptr_t>(first) + (size_t)(a.N - 1) * kSize) & ~(uintptr_t)15;
    in.shift = (uint32_t)at & 15;
#pragma unroll
    for (int i = 0; i < 2 * kSize + 1; ++i) {
      uintptr_t p = (at & ~(uintptr_t)15) + 16 * i;
      p = p < last ? p : last;
      uint32_t* w = in.w + 4 * i;
      asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
    }
  }
}

// Where element (row r, column c) of a warp's 32 x 32 fp32 block lies in its 4 KB of shared memory: rows of 128
// bytes, 16-byte pieces swizzled by row, so that neither a row per lane nor a column per lane meets in a bank.
__device__ __forceinline__ float* mx_stage_at(uint8_t* stage, int r, int c) {
  return reinterpret_cast<float*>(stage + r * 128 + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4);
}

// Adds `bias` (the same 32 values for all lanes) to v: a whole chunk's loads in flight together.
__device__ __forceinline__ void mx_add_bias(const float* bias, int c0, int N, float (&v)[32]) {
  if (c0 + 32 <= N) {
    float4 t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = reinterpret_cast<const float4*>(bias + c0)[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[4 * j] += t[j].x; v[4 * j + 1] += t[j].y; v[4 * j + 2] += t[j].z; v[4 * j + 3] += t[j].w;
    }
  } else {
    // The lane's own column's value, handed round.
    const int lane = threadIdx.x & 31;
    const float mine = bias[min(c0 + lane, N - 1)];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, mine, i);
  }
}

template <typename T>
__device__ __forceinline__ void mx_store_row(T* p, const float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float t[kMxPiece];
#pragma unroll
    for (int k = 0; k < kMxPiece; ++k) t[k] = v[16 * i + k];
    store_vec(p + 16 * i, true, t);
  }
}

// v: the products with W, g: those with G.  Everything is fp32 and rounded once, to the output's
// type.  Returns the block's scale byte (MX8; the caller writes it with its neighbours').  `stage`: the warp's 4 KB.
template <bool kGated, int kRes>
__device__ __forceinline__ uint32_t mx_finish_row(const MxLinearArgs& a, int row, int c0, float (&v)[32], float (&g)[32],
                                                  const MxResidualRow<kRes>& in, uint8_t* stage) {
  if (a.bias) mx_add_bias(a.bias, c0, a.N, v);
  if (kGated && a.gate_bias) mx_add_bias(a.gate_bias, c0, a.N, g);
  float(&on)[32] = kGated ? g : v;
  auto apply = [&](auto f) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float2 y = f(make_float2(on[i], on[i + 1]));
      on[i] = y.x;
      on[i + 1] = y.y;
    }
  };
  if (a.act == MX_ACT_GELU) apply([](float2 x) { return mx_gelu2(x); });
  else if (a.act == MX_ACT_SILU) apply([](float2 x) { return make_float2(mx_silu(x.x), mx_silu(x.y)); });
  else if (a.act == MX_ACT_RELU) apply([](float2 x) { return make_float2(mx_relu(x.x), mx_relu(x.y)); });
  if (kGated) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float2 y = mul2(make_float2(v[i], v[i + 1]), make_float2(g[i], g[i + 1]));
      v[i] = y.x;
      v[i + 1] = y.y;
    }
  }
  if constexpr (kRes == MX_RES_HALF) {
    auto add = [&](auto* type) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 r = add2(make_float2(v[2 * i], v[2 * i + 1]), unpack2_f32(in.w[i], type));
        v[2 * i] = r.x;
        v[2 * i + 1] = r.y;
      }
    };
    if (a.residual_type == MX_BF16) add((__nv_bfloat16*)nullptr);
    else add((__half*)nullptr);
  } else if constexpr (kRes == MX_RES_FULL) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(in.w[i]);
  } else if constexpr (kRes != MX_RES_NONE) {
    constexpr int kWords = 8 * mx_res_size(kRes);
    uint32_t w[kWords + 4];
#pragma unroll
    for (int i = 0; i < kWords + 4; ++i) w[i] = in.w[i];
#pragma unroll
    for (int i = 0; i < kWords + 2; ++i) w[i] = in.shift & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < kWords + 1; ++i) w[i] = in.shift & 4 ? w[i + 1] : w[i];
    if constexpr (kRes == MX_RES_ANY_FULL) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = in.shift & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
      auto add = [&](auto* type) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 r = unpack2_f32(w[i], type);
          v[2 * i] += r.x;
          v[2 * i + 1] += r.y;
        }
      };
      if (a.residual_type == MX_BF16) add((__nv_bfloat16*)nullptr);
      else add((__half*)nullptr);
    }
  }
  const bool live = row < a.M;
  const size_t at = (size_t)row * a.ldo + c0;
  if (a.out_type == MX_MX8) {
    if (c0 + 32 > a.N) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = c0 + i < a.N ? v[i] : 0.f;
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) most = max_abs3(most, v[i], v[i + 1]);
    const uint32_t byte = mx_scale_byte(__float_as_uint(most));
    const float inverse = mx_inverse(byte);
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = mx_pack4(v + 4 * i, inverse);
    uint8_t* p = static_cast<uint8_t*>(a.out) + at;
    if (a.out_wide && c0 + 16 < a.N) {
      if (live)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]),
                     "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7])
                     : "memory");
    } else {
      if (live && c0 < a.N) reinterpret_cast<uint4*>(p)[0] = make_uint4(q[0], q[1], q[2], q[3]);
      if (live && c0 + 16 < a.N) reinterpret_cast<uint4*>(p)[1] = make_uint4(q[4], q[5], q[6], q[7]);
    }
    return byte;
  }
  if (a.out_wide && a.out_type != MX_F32 && c0 + 32 <= a.N) {
    if (live) {
      if (a.out_type == MX_BF16) mx_store_row(static_cast<__nv_bfloat16*>(a.out) + at, v);
      else mx_store_row(static_cast<__half*>(a.out) + at, v);
    }
    return 0;
  }
  // fp32 rows (a thread's 128 bytes in four stores, 16384 x 64 x 4096 + fp32: 131 us, this way 117; over three sets of buffers 105) and rows
  // that are not made of aligned 32-byte vectors: through shared memory, so that eight lanes write 32
  // neighbouring columns of a row, or, where four columns are no vector, the warp writes one row after the other.
  const int lane = threadIdx.x & 31, row0 = row - lane;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(mx_stage_at(stage, lane, 4 * j)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  auto write = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    if (a.out_vec) {
      const int col = c0 + 4 * (lane & 7), n = max(0, min(4, a.N - col));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = 4 * k + (lane >> 3);
        const float4 t = *reinterpret_cast<const float4*>(mx_stage_at(stage, r, 4 * (lane & 7)));
        const float f[4] = {t.x, t.y, t.z, t.w};
        if (row0 + r < a.M) store4(p + (size_t)(row0 + r) * a.ldo + col, n, true, f);
      }
    } else if (c0 + lane < a.N) {
      T* to = p + (size_t)row0 * a.ldo + c0 + lane;
      const int rows = min(32, a.M - row0);
#pragma unroll 8
      for (int r = 0; r < rows; ++r, to += a.ldo) *to = from_f32<T>(*mx_stage_at(stage, r, lane));
    }
  };
  if (a.out_type == MX_BF16) write(static_cast<__nv_bfloat16*>(a.out));
  else if (a.out_type == MX_F16) write(static_cast<__half*>(a.out));
  else write(static_cast<float*>(a.out));
  return 0;
}

}  // namespace laya
