// Attention over packed sequences with caps, biases by distance and masks (see laya_op_attend in
// include/laya_b200.h for the definition).
#pragma once
#include <type_traits>

#include "common.cuh"

namespace laya {

constexpr int kAttendMostDim = 128;

struct AttendArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  const int *starts, *lengths, *k_starts, *k_lengths;
  int sequences, heads, kv_heads, group, dim;
  int q_tokens, k_tokens, max_queries;
  float scale, cap;
  int causal, left, right;
  const int *prefix, *documents, *k_documents;
  const float *slopes, *table;
  int reach;
  int* err;
};

struct AttendSequence {
  int q_start, queries, k_start, keys, prefix;
};

// The lengths of sequence b; none of it (and an error) where it does not lie in the tensors.
__device__ __forceinline__ AttendSequence attend_sequence(const AttendArgs& a, int b) {
  AttendSequence s{a.starts[b], a.lengths[b], a.k_starts[b], a.k_lengths[b], a.prefix ? a.prefix[b] : 0};
  const bool bad = s.q_start < 0 || s.queries < 0 || s.k_start < 0 || s.keys < 0 ||
                   (int64_t)s.q_start + s.queries > a.q_tokens || (int64_t)s.k_start + s.keys > a.k_tokens;
  if (bad) {
    if (a.err && threadIdx.x == 0) atomicCAS(a.err, 0, kErrBadIndex);
    s.queries = s.keys = 0;
  }
  s.queries = min(s.queries, a.max_queries);
  return s;
}

// One query of one head by one warp, in fp32 from global memory: a lane per key for the scores, a lane per value for the sum.
template <typename T>
__device__ void attend_row(const AttendArgs& a, const AttendSequence& s, int full_queries, int query, int head) {
  const int lane = threadIdx.x & 31;
  const int token = s.q_start + query, p = query + s.keys - full_queries;
  const T* q = static_cast<const T*>(a.q) + token * a.q_token + head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + s.k_start * a.k_token + head / a.group * a.k_head;
  const T* v = static_cast<const T*>(a.v) + s.k_start * a.v_token + head / a.group * a.v_head;
  const int doc = a.documents ? a.documents[token] : 0;
  float m = -INFINITY, l = 0.f, o[kAttendMostDim / 32] = {};
  for (int base = 0; base < s.keys; base += 32) {
    const int j = base + lane;
    bool see = j < s.keys;
    if (see && j >= s.prefix)
      see = (!a.causal || j <= p) && (a.left < 0 || j >= (int64_t)p - a.left) && (a.right < 0 || j <= (int64_t)p + a.right) &&
            (!a.documents || a.k_documents[s.k_start + j] == doc);
    if (!__any_sync(0xffffffffu, see)) continue;
    float x = -INFINITY;
    if (see) {
      float dot = 0.f;
      for (int d = 0; d < a.dim; ++d) dot = fmaf(to_f32(q[d]), to_f32(k[j * a.k_token + d]), dot);
      x = dot * a.scale;
      if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
      if (a.slopes) x -= a.slopes[head] * fabsf((float)(p - j));
      if (a.table) x += a.table[(int64_t)head * (2 * a.reach + 1) + min(max(j - p, -a.reach), a.reach) + a.reach];
    }
    float top = x;
    bool nan = x != x;
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    if (__any_sync(0xffffffffu, nan)) top = NAN;
    const float next = top != top || m != m ? NAN : fmaxf(m, top);
    if (next == -INFINITY) continue;
    const float alpha = m == -INFINITY ? 0.f : __expf(m - next);
    float e = see && x != -INFINITY ? expf(x - next) : 0.f;
    m = next;
    float sum = e;
#pragma unroll
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    l = l * alpha + sum;
#pragma unroll
    for (int i = 0; i < kAttendMostDim / 32; ++i) o[i] *= alpha;
    const uint32_t who = __ballot_sync(0xffffffffu, see && x != -INFINITY);
    for (uint32_t left = who; left; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const float w = __shfl_sync(0xffffffffu, e, src);
      const T* row = v + (base + src) * a.v_token;
#pragma unroll
      for (int i = 0; i < kAttendMostDim / 32; ++i)
        if (lane + 32 * i < a.dim) o[i] = fmaf(w, to_f32(row[lane + 32 * i]), o[i]);
    }
  }
  T* out = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kAttendMostDim / 32; ++i)
    if (lane + 32 * i < a.dim) out[lane + 32 * i] = from_f32<T>(o[i] * inv);
  if (a.lse && lane == 0) a.lse[(int64_t)token * a.heads + head] = m == -INFINITY ? -INFINITY : m + logf(l);
}

// A warp per query and head.
template <typename T>
__global__ void __launch_bounds__(128) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
  pdl_wait();
  const int b = blockIdx.z;
  const AttendSequence s = attend_sequence(a, b);
  const int query = blockIdx.x * 4 + threadIdx.x / 32;
  if (query < s.queries) attend_row<T>(a, s, a.lengths[b], query, blockIdx.y);
}

}  // namespace laya
