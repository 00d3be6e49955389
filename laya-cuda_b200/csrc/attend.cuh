// Attention over packed sequences with caps, biases by distance and masks (see laya_op_attend in
// include/laya_b200.h for the definition).
#pragma once
#include <limits.h>

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
  unsigned long long wait_ns;
  int pairs, splits;  // pairs of tiles for max_queries; CTAs (a cluster) that share a pair's keys
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

// ---------------------------------------------------------------------------------------------
// The kernel: a CTA takes two tiles of 128 rows, a row being one query of one head of a kv head's group, and walks the keys in
// blocks of 128.
//
// Warps 0-3 are the softmax of tile 0, warps 4-7 of tile 1 (a thread per row, warp w owning TMEM lanes 32 (w % 4) on), warp 8
// issues the tensor products, warp 9 finds the blocks that the masks leave and loads them.  TMEM: S of each tile (128 columns
// each; P, 16-bit, over its first 64), O of each.  The tensor core runs the products in issue order, so O_t += P_t V of a block
// and then S_t = Q_t K^T of the next are issued together as soon as P_t is there, and while tile 0's softmax works on its S
// the tensor core has tile 1's products to do.
// ---------------------------------------------------------------------------------------------
constexpr int kAtRows = 128;       // rows of a tile
constexpr int kAtKeys = 128;       // keys of a block
constexpr int kAtThreads = 320;
constexpr int kAtInfo = 4;         // blocks announced ahead
constexpr float kAtRescale = 8.f;  // O is rescaled when a row's maximum has grown by more than 2^8
enum AtClass : int { kAtEnd = -1, kAtSkip = 0, kAtMasked = 1, kAtFull = 2 };

template <int DP>
struct AttendCfg {
  static_assert(DP == 64 || DP == 128, "padded head size");
  static constexpr int kSlots = DP == 128 ? 4 : 8;       // K and V blocks in flight
  static constexpr int kTile = kAtKeys * DP * 2;         // a K or V block, and a tile of Q
  static constexpr int kHalf = kAtKeys * 128;            // [128 rows][64 values]
  static constexpr int kOffQ = 0, kOffRing = 2 * kTile;
  static constexpr int kOffDocs = kOffRing + kSlots * kTile;
  static constexpr int kOffBar = kOffDocs + kAtInfo * kAtKeys * 4;
  static constexpr int kBars = 2 + 2 * kSlots + 2 * kAtInfo + 2 + 2 + 2 + 1;
  static constexpr int kOffInfo = kOffBar + kBars * 8;
  static constexpr int kOffSums = kOffInfo + kAtInfo * 4 + 16;  // (maximum, sum) of each row, for a split
  static constexpr int kBytes = kOffSums + 2 * kAtRows * 8 + 1024;
  static_assert(kOffSums % 8 == 0, "alignment");
  static_assert(2 * kAtRows * DP * 4 <= kSlots * kTile, "a split's O fits the ring");
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// A [keys][64 values] tile with 128-byte swizzled rows as the operand whose rows are the values (N) and whose depth (K) is the keys: the next
// 8 keys are 1024 bytes on, the next 64 values a half on.
__device__ __forceinline__ uint64_t smem_desc_values(uint32_t saddr, int half) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(half >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

// The n lowest bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

struct AttendMaps {
  CUtensorMap q, k, v;
};

// What a row sees of the keys, besides the documents: [lo, hi] and all below prefix.
struct AttendSpan {
  int lo, hi;
};
__device__ __forceinline__ AttendSpan attend_span(const AttendArgs& a, int p, int keys) {
  AttendSpan s{0, keys - 1};
  if (a.left >= 0) s.lo = (int)min((int64_t)INT_MAX - 1, max((int64_t)0, (int64_t)p - a.left));
  if (a.causal) s.hi = min(s.hi, p);
  if (a.right >= 0) s.hi = (int)min((int64_t)s.hi, (int64_t)p + a.right);
  return s;
}

// T, the padded head size, and whether scores get a cap or a bias (kGeneral: natural units, any scale).
template <typename T, int DP, bool kGeneral>
__global__ void __launch_bounds__(kAtThreads, 1) attend_kernel(const __grid_constant__ AttendMaps maps, const __grid_constant__ AttendArgs a) {
  using Cfg = AttendCfg<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kLog2e = 1.4426950408889634f;
  // float16 numerators end at 2^-24: they are kept 2^7 larger, so that weights down to 2^-31 of the largest count.
  constexpr float kShift = kBf16 ? 0.f : 7.f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t *q_full = bar, *full = bar + 2, *empty = full + Cfg::kSlots, *info_full = empty + Cfg::kSlots, *info_empty = info_full + kAtInfo,
           *s_full = info_empty + kAtInfo, *p_full = s_full + 2, *o_full = p_full + 2, *drain = o_full + 2;
  volatile int* info = reinterpret_cast<volatile int*>(smem + Cfg::kOffInfo);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffInfo + kAtInfo * 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* docs = reinterpret_cast<int*>(smem + Cfg::kOffDocs);
  float2* sums = reinterpret_cast<float2*>(smem + Cfg::kOffSums);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned long long wait_ns = wait_limit(a.wait_ns);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) { mbar_init(q_full + t, 1); mbar_init(s_full + t, 1); mbar_init(p_full + t, 4); mbar_init(o_full + t, 1); }
    for (int i = 0; i < Cfg::kSlots; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
    for (int i = 0; i < kAtInfo; ++i) { mbar_init(info_full + i, 1); mbar_init(info_empty + i, 9); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  if (warp == 9 && lane == 0) { tma_prefetch_desc(&maps.q); tma_prefetch_desc(&maps.k); tma_prefetch_desc(&maps.v); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  // The work item: split x kv head x sequence x pair of tiles, the last queries first (they see the most keys under a causal mask).
  const int split = blockIdx.x % a.splits;
  uint32_t item = blockIdx.x / a.splits;
  const int kv = item % a.kv_heads;
  item /= a.kv_heads;
  const int b = item % a.sequences;
  const int pair = a.pairs - 1 - (int)(item / a.sequences);
  const AttendSequence s = attend_sequence(a, b);
  const int all_queries = s.queries ? a.lengths[b] : 0;
  const int offset = s.keys - all_queries;  // a query's position less its number
  const int per_tile = kAtRows / a.group, first = 2 * pair * per_tile;
  const int tokens[2] = {max(0, min(per_tile, s.queries - first)), max(0, min(per_tile, s.queries - first - per_tile))};
  const bool idle = tokens[0] == 0;  // of all CTAs of the cluster alike
  const int nk = (a.dim + 15) / 16;  // steps of 16 values
  const int halves = a.dim > 64 ? 2 : 1;

  if (!idle && warp == 9) {
    // ---- blocks and loads
    int doc_lo[2] = {INT_MAX, INT_MAX}, doc_hi[2] = {INT_MIN, INT_MIN};
    if (a.documents)
      for (int t = 0; t < 2; ++t) {
        for (int i = lane; i < tokens[t]; i += 32) {
          const int d = a.documents[s.q_start + first + t * per_tile + i];
          doc_lo[t] = min(doc_lo[t], d);
          doc_hi[t] = max(doc_hi[t], d);
        }
        doc_lo[t] = __reduce_min_sync(0xffffffffu, doc_lo[t]);
        doc_hi[t] = __reduce_max_sync(0xffffffffu, doc_hi[t]);
      }
    if (elect_one())
      for (int t = 0; t < 2; ++t)
        if (tokens[t]) {
          mbar_arrive_expect_tx(q_full + t, halves * 128 * a.group * per_tile);
          for (int h = 0; h < halves; ++h)
            tma_load_3d(smem + Cfg::kOffQ + t * Cfg::kTile + h * Cfg::kHalf, &maps.q, q_full + t, 64 * h, kv * a.group, s.q_start + first + t * per_tile);
        }
    __syncwarp();
    // Spans of the tiles' first and last queries: [lo0, hi1] is what some query sees, [lo1, hi0] what all do.
    AttendSpan outer[2], inner[2];
    int from = INT_MAX, to = -1;
    for (int t = 0; t < 2; ++t) {
      if (!tokens[t]) { outer[t] = inner[t] = {1, 0}; continue; }
      const int p0 = first + t * per_tile + offset;
      const AttendSpan x = attend_span(a, p0, s.keys), y = attend_span(a, p0 + tokens[t] - 1, s.keys);
      outer[t] = {x.lo, y.hi};
      inner[t] = {y.lo, x.hi};
      if (outer[t].lo <= outer[t].hi) { from = min(from, outer[t].lo); to = max(to, outer[t].hi); }
    }
    const int prefix = min(s.prefix, s.keys);
    if (prefix > 0) { from = 0; to = max(to, prefix - 1); }
    // This CTA's share of the blocks.
    int at = from <= to ? from / kAtKeys : 0, end = from <= to ? to / kAtKeys + 1 : 0;
    if (a.splits > 1) {
      const int share = (end - at + a.splits - 1) / a.splits;
      at += split * share;
      end = min(end, at + share);
    }
    int n = 0, issued = 0;
    bool ok = true;
    for (; at < end && ok; ++at) {
      const int kb = at * kAtKeys, last = min(kb + kAtKeys, s.keys) - 1;
      int d[4], lo = INT_MAX, hi = INT_MIN;
      if (a.documents) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = kb + lane + 32 * i;
          d[i] = j <= last ? a.k_documents[s.k_start + j] : 0;
          if (j <= last) { lo = min(lo, d[i]); hi = max(hi, d[i]); }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
      }
      int cls[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool in_prefix = kb < prefix, whole_prefix = kb + kAtKeys <= prefix;
        const bool meets = tokens[t] && kb <= outer[t].hi && last >= outer[t].lo && (!a.documents || (lo <= doc_hi[t] && hi >= doc_lo[t]));
        const bool whole = kb >= inner[t].lo && kb + kAtKeys - 1 <= inner[t].hi &&
                           (!a.documents || (lo == hi && doc_lo[t] == doc_hi[t] && lo == doc_lo[t]));
        cls[t] = !tokens[t] ? kAtSkip : whole_prefix || whole ? kAtFull : in_prefix || meets ? kAtMasked : kAtSkip;
      }
      if (cls[0] == kAtSkip && cls[1] == kAtSkip) continue;
      const int e = n % kAtInfo;
      ok = mbar_wait(info_empty + e, ((n / kAtInfo) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (a.documents)
#pragma unroll
        for (int i = 0; i < 4; ++i) docs[e * kAtKeys + lane + 32 * i] = d[i];
      if (lane == 0) info[e] = at << 4 | cls[1] << 2 | cls[0];
      __syncwarp();
      if (lane == 0) mbar_arrive(info_full + e);
#pragma unroll
      for (int kv_part = 0; kv_part < 2 && ok; ++kv_part) {
        const int load = 2 * n + kv_part, slot = load % Cfg::kSlots;
        ok = mbar_wait(empty + slot, ((load / Cfg::kSlots) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && elect_one()) {
          mbar_arrive_expect_tx(full + slot, halves * Cfg::kHalf);
          for (int h = 0; h < halves; ++h)
            tma_load_3d(smem + Cfg::kOffRing + slot * Cfg::kTile + h * Cfg::kHalf, kv_part ? &maps.v : &maps.k, full + slot, 64 * h, kv, s.k_start + kb);
        }
        __syncwarp();
        if (ok) ++issued;
      }
      if (ok) ++n;
    }
    if (ok) {
      const int e = n % kAtInfo;
      ok = mbar_wait(info_empty + e, ((n / kAtInfo) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (lane == 0 && ok) { info[e] = kAtEnd; mbar_arrive(info_full + e); }
    }
    __syncwarp();
    if (*abort_flag) {
      // Copies that nothing waits for any more land before the CTA ends.
      for (int t = 0; t < 2; ++t)
        if (tokens[t]) mbar_drain(q_full + t, 0);
      for (int load = max(0, issued - Cfg::kSlots); load < issued; ++load) mbar_drain(full + load % Cfg::kSlots, (load / Cfg::kSlots) & 1);
    }
  } else if (!idle && warp == 8) {
    // ---- tensor products
    constexpr uint32_t idesc_s = mma_idesc<kBf16>(kAtRows, kAtKeys);
    const uint32_t idesc_o = mma_idesc<kBf16>(kAtRows, 16) - (2u << 17) + ((uint32_t)(2 * nk) << 17) | 1u << 16;  // N = 16 nk; B by values
    const uint32_t q_addr = smem_u32(smem + Cfg::kOffQ), ring = smem_u32(smem + Cfg::kOffRing);
    bool ok = true, started[2] = {false, false};
    int p_phase[2] = {0, 0};
    auto wait = [&](uint64_t* which, int parity) {
      ok = ok && mbar_wait(which, parity, a.err, kErrAttnWait, abort_flag, wait_ns);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto read = [&](int n) {
      const int e = n % kAtInfo;
      wait(info_full + e, (n / kAtInfo) & 1);
      int x = kAtEnd;
      if (ok) x = info[e];
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(info_empty + e);
      return x;
    };
    auto scores = [&](int t, int n) {
      if (elect_one()) {
        const uint32_t k_addr = ring + (2 * n % Cfg::kSlots) * Cfg::kTile;
        for (int k = 0; k < nk; ++k) {
          const uint32_t o = (k >> 2) * Cfg::kHalf + (k & 3) * 32;
          tc_mma_f16(tmem + t * 128, smem_desc_sw128(q_addr + t * Cfg::kTile + o), smem_desc_sw128(k_addr + o), idesc_s, k > 0);
        }
        tc_commit(s_full + t);
      }
      __syncwarp();
    };
    int cur = read(0);
    if (cur != kAtEnd && ok) {
      for (int t = 0; t < 2; ++t)
        if (tokens[t]) wait(q_full + t, 0);
      wait(full, 0);
      tc_fence_after();
      if (ok)
        for (int t = 0; t < 2; ++t)
          if ((cur >> 2 * t) & 3) scores(t, 0);
      if (ok && elect_one()) tc_commit(empty);
      __syncwarp();
      for (int n = 0; ok; ++n) {
        const int next = read(n + 1);
        const int v_slot = (2 * n + 1) % Cfg::kSlots, k_next = (2 * n + 2) % Cfg::kSlots;
        bool v_here = false, k_here = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if ((cur >> 2 * t) & 3) {
            if (!v_here) {
              wait(full + v_slot, ((2 * n + 1) / Cfg::kSlots) & 1);
              v_here = true;
              // Rows past the last key may hold anything: a NaN there, times a weight of zero, would be a NaN.
              const int rows = s.keys - (cur >> 4) * kAtKeys;
              if (ok && rows < kAtKeys) {
                for (int h = 0; h < halves; ++h) {
                  uint4* tail = reinterpret_cast<uint4*>(smem + Cfg::kOffRing + v_slot * Cfg::kTile + h * Cfg::kHalf + rows * 128);
                  for (int i = lane; i < (kAtKeys - rows) * 8; i += 32) tail[i] = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            wait(p_full + t, p_phase[t]);
            p_phase[t] ^= 1;
            tc_fence_after();
            if (ok && elect_one()) {
              const uint32_t v_addr = ring + v_slot * Cfg::kTile;
#pragma unroll
              for (int k = 0; k < kAtKeys / 16; ++k)
                tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * k, smem_desc_values(v_addr + k * 2048, Cfg::kHalf), idesc_o,
                              started[t] || k > 0);
            }
            __syncwarp();
            started[t] = true;
          }
          if (ok && next != kAtEnd && ((next >> 2 * t) & 3)) {
            if (!k_here) { wait(full + k_next, ((2 * n + 2) / Cfg::kSlots) & 1); k_here = true; tc_fence_after(); }
            if (ok) scores(t, n + 1);
          }
        }
        if (ok && elect_one()) {
          tc_commit(empty + v_slot);
          if (next != kAtEnd) tc_commit(empty + k_next);
        }
        __syncwarp();
        if (next == kAtEnd) break;
        cur = next;
      }
    }
    if (elect_one()) {
      if (ok) { tc_commit(o_full); tc_commit(o_full + 1); }
      tc_commit(drain);
    }
    __syncwarp();
    mbar_drain(drain, 0);
  }

  // ---- softmax
  const int t = warp >> 2, row = (warp & 3) * 32 + lane;  // warps 0 .. 7
  const bool worker = !idle && warp < 8;
  const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t s_tmem = tmem + lane_addr + (t & 1) * 128, o_tmem = s_tmem + 256;
  const int tile_token = row / a.group, head = kv * a.group + row - tile_token * a.group;
  const int query = first + t * per_tile + tile_token;
  const bool live = worker && tile_token < tokens[t & 1] ;
  float m = -INFINITY, l = 0.f;  // the maximum that P is relative to (log2 units, natural ones with kGeneral), and the sum
  bool ok = true;
  if (worker) {
    const int p = query + offset;
    AttendSpan span = attend_span(a, p, s.keys);
    const int prefix = live ? min(s.prefix, s.keys) : 0;
    if (!live) span = {0, -1};
    const int doc = live && a.documents ? a.documents[s.q_start + query] : 0;
    const float scale_log2 = a.scale * kLog2e;
    const float slope = kGeneral && live && a.slopes ? a.slopes[head] : 0.f;
    const float* table = kGeneral && a.table ? a.table + (int64_t)(live ? head : 0) * (2 * a.reach + 1) + a.reach : nullptr;
    const float cap_in = kGeneral && a.cap > 0.f ? 2.f * kLog2e * a.scale / a.cap : 0.f;
    int s_phase = 0;
    for (int n = 0;; ++n) {
      const int e = n % kAtInfo;
      ok = mbar_wait(info_full + e, (n / kAtInfo) & 1, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      const int x = info[e];
      if (x == kAtEnd) break;
      const int cls = (x >> 2 * t) & 3, kb = (x >> 4) * kAtKeys;
      if (cls == kAtSkip) {
        __syncwarp();
        if (lane == 0) mbar_arrive(info_empty + e);
        continue;
      }
      ok = mbar_wait(s_full + t, s_phase, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      s_phase ^= 1;
      tc_fence_after();
      uint32_t sx[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32_async(s_tmem + 32 * c, sx[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_wait_ld(sx[c]);
      if (kGeneral) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (a.cap > 0.f) {
            // cap tanh(y) = cap - 2 cap / (exp(2 y) + 1): off by 2^-21 cap at most.
#pragma unroll
            for (int i = 0; i < 32; ++i)
              sx[c][i] = __float_as_uint(fmaf(-2.f * a.cap, rcp_approx(ex2_approx(__uint_as_float(sx[c][i]) * cap_in) + 1.f), a.cap));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) sx[c][i] = __float_as_uint(__uint_as_float(sx[c][i]) * a.scale);
          }
          const int d = kb + 32 * c - p;  // key less query
          if (a.slopes) {
            const float fd = (float)d;
#pragma unroll
            for (int i = 0; i < 32; ++i) sx[c][i] = __float_as_uint(fmaf(-slope, fabsf(fd + (float)i), __uint_as_float(sx[c][i])));
          }
          if (table) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              sx[c][i] = __float_as_uint(__uint_as_float(sx[c][i]) + __ldg(table + min(max(d + i, -a.reach), a.reach)));
          }
        }
      }
      if (cls == kAtMasked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int kc = kb + 32 * c;
          uint32_t bits = low_bits(span.hi + 1 - kc) & ~low_bits(span.lo - kc);
          if (a.documents) {
            uint32_t same = 0;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const int4 d = *reinterpret_cast<const int4*>(docs + e * kAtKeys + 32 * c + i);
              same |= (d.x == doc) << i | (d.y == doc) << (i + 1) | (d.z == doc) << (i + 2) | (d.w == doc) << (i + 3);
            }
            bits &= same;
          }
          bits |= low_bits(prefix - kc);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((bits >> i) & 1)) sx[c][i] = __float_as_uint(-INFINITY);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty + e);
      float mx[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mx[i] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 7] = max3(mx[(i >> 1) & 7], __uint_as_float(sx[c][i]), __uint_as_float(sx[c][i + 1]));
#pragma unroll
      for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) mx[i] = fmaxf(mx[i], mx[i + w]);
      const float top = kGeneral ? mx[0] : mx[0] * scale_log2;
      float alpha = 1.f;
      bool dirty = false;
      if (top > m + (kGeneral ? kAtRescale / kLog2e : kAtRescale)) {
        if (m != -INFINITY) { alpha = ex2_approx(kGeneral ? (m - top) * kLog2e : m - top); dirty = true; }
        m = top;
      }
      const float base = m == -INFINITY ? 0.f : m;
      float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 y = make_float2(__uint_as_float(sx[c][i]), __uint_as_float(sx[c][i + 1]));
          // Differences before the factor: scores of the type's lowest value stay equal to one another.
          if (kGeneral) y = fma2(sub2(y, make_float2(base, base)), make_float2(kLog2e, kLog2e), make_float2(kShift, kShift));
          else y = fma2(y, make_float2(scale_log2, scale_log2), make_float2(kShift - base, kShift - base));
          const float2 w = make_float2(ex2_approx(y.x), ex2_approx(y.y));
          sum[(i >> 1) & 3] = add2(sum[(i >> 1) & 3], w);
          pk[i >> 1] = pack2<T>(w.x, w.y);
        }
        tmem_st16(s_tmem + 16 * c, pk);
      }
      const float2 total = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
      l = l * alpha + (total.x + total.y);
      // O is settled: S of this block, which s_full announced, came after every product into O that was issued.
      if (__any_sync(0xffffffffu, dirty)) {
#pragma unroll 1
        for (int c = 0; c < (a.dim + 31) / 32; ++c) {
          uint32_t o[32];
          tmem_ld32_async(o_tmem + 32 * c, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(o_tmem + 32 * c, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + t);
    }
    ok = ok && mbar_wait(o_full + t, 0, a.err, kErrAttnWait, abort_flag, wait_ns);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
  }
  const int64_t token = s.q_start + query;
  if (a.splits == 1) {
    if (worker && ok) {
      // Rows without a visible key, and rows that no block was made for, hold nothing in O.
      const bool any = l > 0.f || l != l;
      const float inv = any ? 1.f / l : 0.f;
      bool fine = l - l == 0.f;
      T* out = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll 1
      for (int c = 0; c < a.dim; c += 32) {
        uint32_t o[32];
        tmem_ld32_async(o_tmem + c, o);
        tmem_wait_ld(o);
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = any ? __uint_as_float(o[i + 2 * k]) * inv : 0.f, y = any ? __uint_as_float(o[i + 2 * k + 1]) * inv : 0.f;
            if (c + i < a.dim) fine = fine && x - x == 0.f && y - y == 0.f;
            w[k] = pack2<T>(x, y);
          }
          if (live && c + i < a.dim) *reinterpret_cast<uint4*>(out + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      if (live && a.lse)
        a.lse[token * a.heads + head] = any ? (kGeneral ? m : m / kLog2e) + (log2f(l) - kShift) / kLog2e : -INFINITY;
      // A value that is not finite may come from a key that this row's mask hides (its weight of zero times that value): such rows
      // are computed once more, from the visible keys alone.
      for (uint32_t again = __ballot_sync(0xffffffffu, live && !fine); again; again &= again - 1) {
        const int src = __ffs(again) - 1;
        attend_row<T>(a, s, all_queries, __shfl_sync(0xffffffffu, query, src), __shfl_sync(0xffffffffu, head, src));
      }
    }
  } else {
    // Every CTA's rows into its own shared memory (all products are done, so the ring is free), then each warp of the cluster joins the
    // parts of its share of the rows.
    float* part = reinterpret_cast<float*>(smem + Cfg::kOffRing);
    if (worker) {
      const int slot = t * kAtRows + row;
      sums[slot] = make_float2(m, ok ? l : NAN);
#pragma unroll 1
      for (int c = 0; c < a.dim; c += 32) {
        uint32_t o[32];
        tmem_ld32_async(o_tmem + c, o);
        tmem_wait_ld(o);
        if (live)
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(part + slot * DP + (((c + i) / 4) ^ (row & 7)) * 4) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
    }
    tc_fence_before();
    cluster_sync();
    if (worker && !*abort_flag) {
      const uint32_t part_addr = smem_u32(part), sums_addr = smem_u32(sums);
      const int rows0 = tokens[0] * a.group, rows = rows0 + tokens[1] * a.group;
      for (int r = split * 8 + warp; r < rows; r += 8 * a.splits) {
        const int tile = r >= rows0, at = tile ? r - rows0 : r, slot = tile * kAtRows + at;
        float top = -INFINITY;
        for (int c = 0; c < a.splits; ++c) top = fmaxf(top, ld_cluster_v2(cluster_addr(sums_addr + slot * 8, c)).x);
        float sum = 0.f, o[DP / 32] = {};
        for (int c = 0; c < a.splits; ++c) {
          const float2 ml = ld_cluster_v2(cluster_addr(sums_addr + slot * 8, c));
          if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing: its O is not defined
          const float w = ex2_approx(kGeneral ? (ml.x - top) * kLog2e : ml.x - top);
          sum = fmaf(ml.y, w, sum);
#pragma unroll
          for (int i = 0; i < DP / 64; ++i) {
            const int d = 2 * lane + 64 * i;
            if (d < a.dim) {
              const float2 x = ld_cluster_v2(cluster_addr(part_addr + (slot * DP + ((d / 4) ^ (at & 7)) * 4 + d % 4) * 4, c));
              o[2 * i] = fmaf(x.x, w, o[2 * i]);
              o[2 * i + 1] = fmaf(x.y, w, o[2 * i + 1]);
            }
          }
        }
        const bool any = sum > 0.f || sum != sum;
        const float inv = any ? 1.f / sum : 0.f;
        bool fine = sum - sum == 0.f;
        const int tok = at / a.group, h = kv * a.group + at - tok * a.group, qi = first + tile * per_tile + tok;
        T* out = static_cast<T*>(a.out) + (int64_t)(s.q_start + qi) * a.out_token + h * a.out_head;
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) {
          const int d = 2 * lane + 64 * i;
          const float x = o[2 * i] * inv, y = o[2 * i + 1] * inv;
          fine = fine && x - x == 0.f && y - y == 0.f;
          if (d < a.dim) *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(x, y);
        }
        if (a.lse && lane == 0)
          a.lse[(int64_t)(s.q_start + qi) * a.heads + h] = any ? (kGeneral ? top : top / kLog2e) + (log2f(sum) - kShift) / kLog2e : -INFINITY;
        if (__any_sync(0xffffffffu, !fine)) attend_row<T>(a, s, all_queries, qi, h);
      }
    }
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

}  // namespace laya
