// Rotary positions: pairs of a head's values turned by position * f_k.
//
// Bound by the bytes of the heads, read once and written once.  A warp takes a token, or some of its heads where tokens are few.  Its
// lanes first load their places of the first heads; then they find the angles, each of other pairs (2^x and the product with the position in 64 bits, so
// that far positions keep their fraction of a turn, and sincospif), pass them on through shared memory, and go from head to head with the
// next ones' loads under way.  No table of angles is read, and no block waits for its warps.
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
  int positions_64, tokens, pairs;
  int places;         // of a head that are turned: vectors, or pairs of vectors
  int rest;           // vectors of a head that are copied
  int abreast;        // heads that a warp's lanes take side by side, one place each
  int shares;         // warps of a token, each with a part of the heads
  FastDiv by_places, by_rest, by_shares;
  float sine_sign, magnitude;
  // Turns per position of pair k: f = 2^(power + k step), by parts f (keep + (1 - keep) / factor) with keep = clamp(f above - below, 0, 1).
  double power, step, above, below, shrink;  // shrink: 1 / factor
  int by_parts;
};

template <typename T> __device__ __forceinline__ float rotary_in(T x) { return to_f32(x); }
template <> __device__ __forceinline__ float rotary_in<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T rotary_out(float x) { return from_f32<T>(x); }
template <> __device__ __forceinline__ float rotary_out<float>(float x) { return x; }

// V consecutive values, as one access where V > 1.
template <typename T, int V>
struct alignas(V == 1 ? sizeof(T) : 16) RotaryVector {
  T v[V];
};

// A place is, in the half layout, two vectors of V values half of the turned values apart; interleaved, one vector, or two values where V is 1.
//
// Heads of a lane at a time, with as many on the way, and blocks of an SM, as measured: vectors of the half layout one and five (16384 x 40 x 128
// bf16 70 us; two and four 84, four and two, without loads ahead, 121), interleaved 16-bit ones the same (78-80 us; two 88), of 32 bits two
// and four (9001 x 32 x 96 49 us; one 65), single values four and four (rows that are not whole vectors: 16384 x 40 x 128 bf16 125 us, 9001 x 32 x 96 of 32 bits 66).
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads, V > 1 && (!kInterleaved || sizeof(T) == 2) ? 5 : 4) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int P = kInterleaved && V > 1 ? V / 2 : V;  // pairs of a place
  constexpr bool kTwo = !kInterleaved || V == 1;        // two vectors
  constexpr int kHeads = V == 1 ? 4 : kTwo || sizeof(T) == 2 ? 1 : 2;
  using Vector = RotaryVector<T, V>;
  __shared__ float2 turn[kRotaryThreads / 32][kRotaryMostPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t work = blockIdx.x * (kRotaryThreads / 32) + warp;
  const int token = a.by_shares.div(work), share = work - token * a.shares;
  if (token >= a.tokens) return;
  pdl_wait();
  const int64_t position = a.positions_64 ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int*>(a.positions)[token];
  const T* x0 = static_cast<const T*>(a.part[0].x) + token * a.part[0].x_token;
  const T* x1 = static_cast<const T*>(a.part[1].x) + token * a.part[1].x_token;
  T* out0 = static_cast<T*>(a.part[0].out) + token * a.part[0].out_token;
  T* out1 = static_cast<T*>(a.part[1].out) + token * a.part[1].out_token;
  const int heads = a.part[0].heads + a.part[1].heads, step = a.abreast * a.shares;
  float2* mine = turn[warp];
  for (int place0 = 0; place0 < a.places; place0 += 32) {
    // Lanes past the last whole head, or the last place, have nothing to do.
    const int of = a.by_places.div(lane), place = a.places < 32 ? lane - of * a.places : place0 + lane;
    const int beside = a.places < 32 ? of : 0;
    const bool idle = beside >= a.abreast || place >= a.places;
    const int at0 = kTwo && kInterleaved ? 2 * place : place * V, at1 = kInterleaved ? at0 + 1 : a.pairs + at0;
    Vector now[kHeads][kTwo ? 2 : 1], next[kHeads][kTwo ? 2 : 1];
    auto load = [&](int h0, Vector (&v)[kHeads][kTwo ? 2 : 1]) {
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * step, g = h - a.part[0].heads;
        if (h < heads) {
          const T* x = g < 0 ? x0 + h * a.part[0].x_head : x1 + g * a.part[1].x_head;
          v[k][0] = *reinterpret_cast<const Vector*>(x + at0);
          if (kTwo) v[k][kTwo] = *reinterpret_cast<const Vector*>(x + at1);
        }
      }
    };
    int h0 = idle ? heads : share * a.abreast + beside;
    load(h0, now);
    if (place0 == 0) {
      for (int k = lane; k < a.pairs; k += 32) {
        double f = exp2(fma((double)k, a.step, a.power));
        if (a.by_parts) {
          const double keep = fmin(1.0, fmax(0.0, fma(f, a.above, -a.below)));
          f *= keep + (1.0 - keep) * a.shrink;
        }
        const double t = (double)position * f;
        // The angle within a turn, its sine and cosine in 32 bits (32-bit results 5.1e-8 off, 4.2e-8 with these in 64).
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        mine[k] = make_float2(c * a.magnitude, s * a.magnitude * a.sine_sign);
      }
      __syncwarp();
    }
    while (h0 < heads) {
      load(h0 + kHeads * step, next);
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * step, g = h - a.part[0].heads;
        if (h < heads) {
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const float2 cs = mine[place * P + p];
            T& u = kTwo ? now[k][0].v[p] : now[k][0].v[2 * p % V];
            T& v = kTwo ? now[k][kTwo].v[p] : now[k][0].v[(2 * p + 1) % V];
            const float fu = rotary_in(u), fv = rotary_in(v);
            u = rotary_out<T>(fu * cs.x - fv * cs.y);
            v = rotary_out<T>(fu * cs.y + fv * cs.x);
          }
          T* out = g < 0 ? out0 + h * a.part[0].out_head : out1 + g * a.part[1].out_head;
          *reinterpret_cast<Vector*>(out + at0) = now[k][0];
          if (kTwo) *reinterpret_cast<Vector*>(out + at1) = now[k][kTwo];
        }
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k)
#pragma unroll
        for (int i = 0; i < (kTwo ? 2 : 1); ++i) now[k][i] = next[k][i];
      h0 += kHeads * step;
    }
    __syncwarp();
  }
  if (a.rest)
    for (int q = 0; q < 2; ++q) {
      const RotaryPart& r = a.part[q];
      if (!r.copy) continue;
      const T* x = static_cast<const T*>(r.x) + token * r.x_token + 2 * a.pairs;
      T* out = static_cast<T*>(r.out) + token * r.out_token + 2 * a.pairs;
#pragma unroll 4
      for (int i = share * 32 + lane; i < r.heads * a.rest; i += 32 * a.shares) {
        const int h = a.by_rest.div(i), j = (i - h * a.rest) * V;
        *reinterpret_cast<Vector*>(out + h * r.out_head + j) = *reinterpret_cast<const Vector*>(x + h * r.x_head + j);
      }
    }
}

}  // namespace laya
