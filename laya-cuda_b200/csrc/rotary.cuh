// Rotary positions: pairs of a head's values turned by position * f_k.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace laya {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMostPairs = 256;

struct RotaryPart {
  const void* x;
  void* out;
  int64_t x_token, x_head, out_token, out_head;
  int heads;
  int copy;  // values past the turned ones are copied (not in place)
};
struct RotaryArgs {
  RotaryPart part[2];
  const void* positions;
  int positions_64, tokens, dim, pairs;
  float sine_sign, magnitude;
  double turns[kRotaryMostPairs];  // f_k / 2 pi
};

template <typename T> __device__ __forceinline__ float rotary_in(T x) { return to_f32(x); }
template <> __device__ __forceinline__ float rotary_in<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T rotary_out(float x) { return from_f32<T>(x); }
template <> __device__ __forceinline__ float rotary_out<float>(float x) { return x; }

// One block per token: the angles' cosines and sines into shared memory, then the heads.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float2 turn[kRotaryMostPairs];
  pdl_wait();
  for (int token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const double position = a.positions_64 ? (double)static_cast<const int64_t*>(a.positions)[token]
                                           : (double)static_cast<const int*>(a.positions)[token];
    for (int k = threadIdx.x; k < a.pairs; k += kRotaryThreads) {
      const double t = position * a.turns[k];
      float s, c;
      sincospif((float)(2.0 * (t - rint(t))), &s, &c);
      turn[k] = make_float2(c * a.magnitude, s * a.magnitude * a.sine_sign);
    }
    __syncthreads();
    for (int p = 0; p < 2; ++p) {
      const RotaryPart& r = a.part[p];
      const T* x = static_cast<const T*>(r.x) + token * r.x_token;
      T* out = static_cast<T*>(r.out) + token * r.out_token;
      for (int i = threadIdx.x; i < r.heads * a.pairs; i += kRotaryThreads) {
        const int h = i / a.pairs, k = i - h * a.pairs;
        const int first = kInterleaved ? 2 * k : k, second = kInterleaved ? 2 * k + 1 : k + a.pairs;
        const float u = rotary_in(x[h * r.x_head + first]), v = rotary_in(x[h * r.x_head + second]);
        const float2 cs = turn[k];
        out[h * r.out_head + first] = rotary_out<T>(u * cs.x - v * cs.y);
        out[h * r.out_head + second] = rotary_out<T>(u * cs.y + v * cs.x);
      }
      const int rest = r.copy ? a.dim - 2 * a.pairs : 0;
      for (int i = threadIdx.x; i < r.heads * rest; i += kRotaryThreads) {
        const int h = i / rest, d = 2 * a.pairs + i - h * rest;
        out[h * r.out_head + d] = x[h * r.x_head + d];
      }
    }
    __syncthreads();
  }
}

}  // namespace laya
