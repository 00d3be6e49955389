// Attention over packed sequences with caps, biases by distance and masks (see laya_op_attend in
// include/laya_b200.h for the definition).
#pragma once
#include <float.h>
#include <limits.h>

#include <type_traits>

#include "common.cuh"

namespace laya {

constexpr int kAttendMostDim = 128;
constexpr int kAtRows = 128;       // rows of a tile
constexpr int kAtKeys = 128;       // keys of a step

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
  int per_tile;       // queries of a tile, which holds all heads of a group for each
  int table_pad;      // values between the heads of a distance bias in shared memory
  int pairs_inside;   // a sequence's pairs one after the other, not all sequences' last ones first
  int longest_first;  // the sequences in the order of their keys' number (one pair; kAtMostOrdered of them at most)
  int pairs, splits;  // CTAs for max_queries of a kv head; CTAs (a cluster) that share a tile's keys
  FastDiv by_group, by_splits, by_kv, by_inner;  // by_inner: by pairs, or by sequences
};

struct AttendSequence {
  int q_start, queries, k_start, keys, prefix;
};

// The lengths of sequence b; none of it (and an error) where it does not lie in the tensors.  *all: its queries before the bound on them.
__device__ __forceinline__ AttendSequence attend_sequence(const AttendArgs& a, int b, int* all) {
  AttendSequence s{a.starts[b], a.lengths[b], a.k_starts[b], a.k_lengths[b], a.prefix ? a.prefix[b] : 0};
  const bool bad = s.q_start < 0 || s.queries < 0 || s.k_start < 0 || s.keys < 0 ||
                   (int64_t)s.q_start + s.queries > a.q_tokens || (int64_t)s.k_start + s.keys > a.k_tokens;
  if (bad) {
    if (a.err && threadIdx.x == 0) atomicCAS(a.err, 0, kErrBadIndex);
    s.queries = s.keys = 0;
  }
  *all = s.queries;
  s.queries = min(s.queries, a.max_queries);
  return s;
}

// The n lowest bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

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

// ---------------------------------------------------------------------------------------------
// Values that are not finite.
//
// A hidden key's score becomes -infinity whatever it was, but its weight of zero times an infinity or NaN of v would be a NaN.  So where a step holds hidden keys, two
// warps look its V over while the softmax is at work, put zeros in the place of what is not finite, and note the step.  What that took from rows that see such a key is put into their
// results at the end: attend_scan finds it, reading v of the noted steps once for all rows of a warp, attend_put writes it.  (Steps that all rows see are left as they are.)
// 4096 causal tokens, 4 heads of 128 over 2: 59 us; with a NaN in every key's v 88, with 100 NaN here and there 78 (50 ms when each row with a NaN was computed again by a warp).
// What it costs without any: windowed documents 160 -> 168 us, a packed batch 345 -> 356, ragged sequences up to 300 with heads of 64 69 -> 75 and with a window and a
// learned bias 312 -> 348; single tokens and long prompts nothing.
// ---------------------------------------------------------------------------------------------

// Pairs of 16-bit values.
template <typename T>
struct NotFinite {
  static constexpr uint32_t kTop = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;  // an infinity; NaN are above it
  static constexpr uint32_t kBits = kTop << 16 | kTop, kAdd = 0x80008000u - kBits;
  // Bits 15 and 31: which of the two are not finite (an addition to the exponent's bits carries there when all are set).
  static __device__ __forceinline__ uint32_t carries(uint32_t pair) { return (pair & kBits) + kAdd; }
  // sum + 0 pair: not finite any more once a value was not.
  static __device__ __forceinline__ uint32_t gather(uint32_t pair, uint32_t sum) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 r = __hfma2(reinterpret_cast<const __nv_bfloat162&>(pair), __nv_bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0)), reinterpret_cast<const __nv_bfloat162&>(sum));
      return reinterpret_cast<const uint32_t&>(r);
    } else {
      const __half2 r = __hfma2(reinterpret_cast<const __half2&>(pair), __half2(__ushort_as_half(0), __ushort_as_half(0)), reinterpret_cast<const __half2&>(sum));
      return reinterpret_cast<const uint32_t&>(r);
    }
  }
  static __device__ __forceinline__ uint32_t cleared(uint32_t pair) {
    const uint32_t c = carries(pair);
    return pair & ~((c >> 15 & 1) * 0xffffu | (c >> 31) * 0xffff0000u);
  }
};

// Channels that are NaN, infinity and -infinity for a key that a row sees: bit i of word c is channel 8 (i % 16) + c + 4 (i / 16).
struct AttendFound {
  uint32_t nan[4] = {}, up[4] = {}, down[4] = {};
  __device__ __forceinline__ bool any() const {
    uint32_t all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) all |= nan[c] | up[c] | down[c];
    return all != 0;
  }
};

// What the rows of a warp (a lane per row; those that ask) see that is not finite, among the keys 32 first .. 32 last + 31, every `stride`-th 32 of them.
template <typename T>
__device__ void attend_scan(const AttendArgs& a, AttendSequence s, int full_queries, int query, int kv, bool asks, int first, int last, int stride, AttendFound& found) {
  using F = NotFinite<T>;
  const int lane = threadIdx.x & 31;
  const AttendSpan span = attend_span(a, query + s.keys - full_queries, s.keys);
  const int below = max(0, min(s.prefix, s.keys)), doc = asks && a.documents ? a.documents[s.q_start + query] : 0;
  // Half a warp reads a key's channels.
  const int odd = lane >> 4, channel = 8 * (lane & 15);
  const T* v = static_cast<const T*>(a.v) + s.k_start * a.v_token + kv * a.v_head + channel;
  for (int block = first; block <= last; block += stride) {
    const int kc = 32 * block;
    uint32_t seen = low_bits(span.hi + 1 - kc) & ~low_bits(span.lo - kc);
    if (a.documents) {
      const int theirs = kc + lane < s.keys ? a.k_documents[s.k_start + kc + lane] : 0;
      uint32_t same = 0;
      for (int i = 0; i < 32; ++i) same |= (uint32_t)(__shfl_sync(0xffffffffu, theirs, i) == doc) << i;
      seen &= same;
    }
    seen = asks ? (seen | low_bits(below - kc)) & low_bits(s.keys - kc) : 0;
    const uint32_t some = __reduce_or_sync(0xffffffffu, seen);
    for (int i = 0; i < 32; i += 8) {
      if (!(some >> i & 0xff)) continue;
      uint4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = i + 2 * u + odd;
        w[u] = channel < a.dim && (some >> key & 1) ? *reinterpret_cast<const uint4*>(v + (kc + key) * a.v_token) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
        if (!__any_sync(0xffffffffu, ((F::carries(words[0]) | F::carries(words[1]) | F::carries(words[2]) | F::carries(words[3])) & 0x80008000u) != 0)) continue;
        const uint32_t sees = seen >> (i + 2 * u) & 3;  // the two keys, for this lane's row
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // Values c and c + 4 of the lanes' eight.
          const uint32_t x = words[c >> 1] >> 16 * (c & 1) & 0xffff, y = words[2 + (c >> 1)] >> 16 * (c & 1) & 0xffff;
          auto mark = [&](uint32_t& word, bool px, bool py) {
            const uint32_t bx = __ballot_sync(0xffffffffu, px), by = __ballot_sync(0xffffffffu, py);
            if (sees & 1) word |= (bx & 0xffff) | by << 16;
            if (sees & 2) word |= bx >> 16 | (by & 0xffff0000);
          };
          mark(found.nan[c], (x & 0x7fff) > F::kTop, (y & 0x7fff) > F::kTop);
          mark(found.up[c], x == F::kTop, y == F::kTop);
          mark(found.down[c], x == (F::kTop | 0x8000), y == (F::kTop | 0x8000));
        }
      }
    }
  }
}

// Puts what a row sees that is not finite into its result, by a warp: added to it, or, where all that it sees is known, in its place.
template <typename T>
__device__ void attend_put(const AttendArgs& a, int token, int head, const AttendFound& found, bool all) {
  const int lane = threadIdx.x & 31, bit = (lane >> 1) + 16 * (lane & 1);  // channels 4 lane .. 4 lane + 3
  if (4 * lane >= a.dim) return;
  T* out = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head + 4 * lane;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const bool up = found.up[c] >> bit & 1, down = found.down[c] >> bit & 1, nan = (found.nan[c] >> bit & 1) || (up && down);
    if (nan || up || down) out[c] = from_f32<T>((all ? 0.f : to_f32(out[c])) + (nan ? NAN : up ? INFINITY : -INFINITY));
  }
}

// ---------------------------------------------------------------------------------------------
// The kernel.  out = sum_j softmax(s)_j v_j in one pass over the keys: with m a running bound of a row's scores, the numerators P = exp(s - m) of a step
// and their sum l are relative to m; where a row's scores have grown by more than 2^8 beyond it, m follows and O and l are scaled by exp(m_old - m).
//
// A CTA takes tiles of 128 rows, a row being one query of one head of a kv head's group (so that the group reads its keys once), and walks the
// keys in steps of 128.  Warps 0-3 are the softmax of tile 0, warps 4-7 of tile 1 (a thread per row, warp w owning TMEM lanes 32 (w % 4) on); of the
// others one issues the tensor products, one finds the steps that the masks leave and loads them by TMA, and two look over V where a mask cuts a step.  TMEM: S of each tile (128 columns),
// O of each; P goes over S as 16-bit pairs.  The tensor core runs the products in issue order, so O += P V of a step and then S = Q K^T
// of the next are issued together as soon as P is there, and the other tile's softmax hides them.
//
// What bounds it: with prompts the softmax.  A step of a tile with heads of 128 is 2 x 128^3 multiply-adds, some 512 cycles of the tensor core, and 128 x 128
// exponentials, 1024 cycles of the special-function units that the two tiles share out: 16384 causal tokens, 16 heads of 128 over 4, bf16, inputs of unit variance, 980-1000 us
// (1.11 PFLOP/s of 1.66), not causal 8192 570 us (0.97); heads of 64, which have as many exponentials for half the products, 888 us (0.62); a cap doubles the work on the FMA
// pipe (1370 us); slopes cost 8%.  Single tokens: the caches' bytes, 5.8 TB/s (16 x 32768 keys, 8 kv heads of 128, 2.1 GB, 367 us); but one cache of 131072 keys is 64 CTAs' work,
// 168 us (3.2 TB/s), with 1 kv head 16 CTAs', 92 us.  A few queries over one cache: the chain of launch, first loads, products and the join (1 x 4000 keys 22 us, cold, 1 x 96 7 us).
// Documents are looked over ahead up to 256 steps of a CTA; past that each step costs a trip to memory (causal tokens in documents of 600, 8 heads of 128 over 2:
// 32768 215 us, 65536 1460).
//
// Tiles: with heads past 64 two to a CTA and one CTA per SM (one tile, two CTAs: 16384 causal 976 -> 999 us, with a cap 1441 -> 1482, 8192 tokens
// in documents 207 -> 229: K and V are loaded twice, into one buffer each).  Heads up to 64: one to a CTA and two CTAs per SM, whose starts and ends overlap
// (two tiles, before a sequence's tiles ran one after the other: 16384 causal 854 -> 915 us, 64 x 1024 444 -> 461, 1 x 1000 27 -> 32; with a distance bias 64 ragged sequences up to 1024 402 -> 369, but
// 64 x 250 74 -> 82 and 40 causal ones up to 500 63 -> 73).
//
// Where one tile holds all rows, both take them, and each every other step; the parts are joined at the end as those of a split
// are.  Where a quarter of a tile holds them (single tokens over a cache), each quarter has a copy of them and takes a quarter of
// a step's keys: a softmax thread then has 32 scores of a step to do and not 128.
// ---------------------------------------------------------------------------------------------
constexpr int kAtInfo = 4;         // steps announced ahead
constexpr float kAtRescale = 8.f;  // O is rescaled when a row's maximum has grown by more than 2^8
// kAtTail: all rows see all of its keys, which are fewer than a step's.
enum AtClass : int { kAtEnd = -1, kAtSkip = 0, kAtMasked = 1, kAtFull = 2, kAtTail = 3 };
// What is done to the scores: nothing, a cap, slopes (these in log2 units, a scale above zero), a distance bias in shared memory, or all else
// (these in natural units: log2e times the lowest number of a type would be -infinity; all else has a slower way only).
// Of a step as it is announced, with the classes of tile 0 and, two bits up, of tile 1: whether one is kAtMasked or kAtTail (the odd ones); whether one is kAtMasked.
__device__ __forceinline__ bool attend_cut(int x) { return (x & 5) != 0; }
__device__ __forceinline__ bool attend_hides(int x) { return (x & 3) == kAtMasked || (x >> 2 & 3) == kAtMasked; }
enum AtMode { kAtPlain, kAtCap, kAtSlopes, kAtTable, kAtGeneral };

constexpr int kAtMostSplits = 16;
constexpr int kAtMostOrdered = 128;  // sequences that are put in order
constexpr int kAtMostSummary = 256;  // steps whose documents are looked over ahead
constexpr int kAtMostTable = 4096;  // values of the distance bias that are kept in shared memory, clamped past the reach

// NT tiles per CTA, heads padded to DP values; kQuarters: all rows in a quarter of a tile.
template <int DP, int NT>
struct AttendCfg {
  static_assert((DP == 64 || DP == 128) && (NT == 1 || NT == 2), "padded head size, tiles");
  static constexpr int kSoftmax = 4 * NT;                // softmax warps
  static constexpr int kMmaWarp = kSoftmax, kLoadWarp = kSoftmax + 1, kCheckWarp = kSoftmax + 2, kThreads = 32 * (kSoftmax + 4), kCtas = NT == 1 ? 2 : 1;
  // Registers: what the launch gives all threads (128 with one tile, 168 with two), moved to the softmax, whose threads hold a step's 128 scores.
  // (224 and 56 with two tiles: a cap 3% faster, slopes and windows slower.)
  static constexpr int kSoftmaxRegs = NT == 1 ? 200 : 216, kOtherRegs = NT == 1 ? 56 : 72;
  static_assert(32 * (kSoftmax * kSoftmaxRegs + 4 * kOtherRegs) <= kThreads * (NT == 1 ? 128 : 168), "registers of the launch");
  static constexpr int kTmemO = 128 * NT, kTmemCols = NT == 1 ? 256 : 512;  // columns: O of tile 0, all
  static_assert(kTmemO + NT * DP <= kTmemCols, "tensor memory");
  static constexpr int kSlots = (DP == 128 ? 1 : 2) * NT;  // K tiles in flight, and V tiles
  static constexpr int kQTile = kAtRows * DP * 2, kQHalf = kAtRows * 128;  // halves: [rows][64 values]
  static constexpr int kTile = kAtKeys * DP * 2, kHalf = kAtKeys * 128;
  static constexpr int kOffQ = 0, kOffK = NT * kQTile, kOffV = kOffK + kSlots * kTile;
  static constexpr int kOffDocs = kOffV + kSlots * kTile;
  static constexpr int kOffBar = kOffDocs + kAtInfo * kAtKeys * 4;
  static constexpr int kBars = 2 + 4 * kSlots + 2 * kAtInfo + 10;
  static constexpr int kOffInfo = kOffBar + kBars * 8;
  static constexpr int kOffSums = kOffInfo + kAtInfo * 4 + 24;  // (maximum, sum) of each row, where results are joined
  static constexpr int kWeights = 2 * NT * kAtRows + 8 * kAtMostSplits;  // of the parts of the rows that a CTA joins
  static constexpr int kOffWeights = kOffSums + NT * kAtRows * 8;
  static constexpr int kOffTable = kOffWeights + kWeights * 4;
  static constexpr int kOffSummary = kOffTable + kAtMostTable * 4;
  static constexpr int kBytes = kOffSummary + kAtMostSummary * 8 + 1024;
  static_assert(kOffSums % 8 == 0, "alignment");
  static_assert(2 * kAtMostSplits <= 32, "a lane per part");
  static_assert(kAtMostOrdered < kWeights && kAtMostOrdered <= kThreads, "lengths in the place of the weights, a thread each");
  static_assert(NT * kAtRows * DP * 4 <= 2 * kSlots * kTile, "a part's O fits the K and V tiles");
  static_assert(kCtas * (kBytes + 1024) <= 228 * 1024, "shared memory");
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

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

struct AttendMaps {
  CUtensorMap q, k, v;
};

// out tanh(in s) for a raw product s, with out in some unit.
//   near  for |in s| <= 0.8 (less with large caps): s times a polynomial in s^2 by the Remez exchange algorithm, on the FMA pipe; off by 1.2e-7 of itself (a term
//         less made the logarithms of the sums ten times less exact than the exponentials do)
//   any   out - 2 out / (exp(2 in s) + 1) on the special-function unit; off by 2^-21 out
struct CapTerms {
  float in, out, c[6], most;  // most: the largest |s| for `near`
  // scale: in out, which has all its bits where `in` is below fp32's normal numbers.
  __device__ __forceinline__ CapTerms(float in_, float out_, float scale) : in(in_), out(out_) {
    constexpr float kC[6] = {0.99999994f, -0.333326757f, 0.13321048f, -0.0531143174f, 0.0190933011f, -0.00435529975f};
    float power = scale;
#pragma unroll
    for (int i = 0; i < 6; ++i) { c[i] = kC[i] * power; power *= in * in; }
    // Caps far above the scale (300 and more for 0.09) take the last factors below fp32's range: as far as the terms that are left reach.
    constexpr float kReach[6] = {5e-4f, 0.03f, 0.1f, 0.2f, 0.3f, 0.8f}, kLeast = 1e-36f;
    most = kReach[0];
#pragma unroll
    for (int i = 1; i < 6; ++i)
      if (fabsf(c[i]) > kLeast) most = kReach[i];
    most = fabsf(c[5]) < 1e30f ? most / fabsf(in) : -1.f;
  }
  __device__ __forceinline__ float2 slope(float2 s) const {  // out tanh(in s) / s
    const float2 z = mul2(s, s);
    float2 p = fma2(make_float2(c[5], c[5]), z, make_float2(c[4], c[4]));
#pragma unroll
    for (int i = 3; i >= 0; --i) p = fma2(p, z, make_float2(c[i], c[i]));
    return p;
  }
  __device__ __forceinline__ float any(float s) const {
    return fmaf(-2.f * out, rcp_approx(ex2_approx(s * (in * 2.8853900817779268f)) + 1.f), out);
  }
};

// T, the padded head size, and what is done to the scores.
template <typename T, int DP, int NT, int kMode, bool kQuarters>
__global__ void __launch_bounds__(AttendCfg<DP, NT>::kThreads, AttendCfg<DP, NT>::kCtas)
    attend_kernel(const __grid_constant__ AttendMaps maps, const __grid_constant__ AttendArgs a) {
  using Cfg = AttendCfg<DP, NT>;
  constexpr int kSlots = Cfg::kSlots;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value, kGeneral = kMode == kAtGeneral, kNatural = kMode >= kAtTable;
  constexpr float kUnit = kNatural ? 1.f : 1.4426950408889634f;  // of the scores: natural, or log2
  constexpr float kLog2e = 1.4426950408889634f;
  // float16 numerators end at 2^-24: they are kept 2^7 larger, so that weights down to 2^-31 of the largest count.
  constexpr float kShift = kBf16 ? 0.f : 7.f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t *q_full = bar, *k_full = bar + 2, *k_empty = k_full + kSlots, *v_full = k_empty + kSlots, *v_empty = v_full + kSlots,
           *info_full = v_empty + kSlots, *info_empty = info_full + kAtInfo, *s_full = info_empty + kAtInfo, *p_full = s_full + 2, *drain = p_full + 2, *table_full = drain + 2, *summary_full = table_full + 1, *v_ask = summary_full + 1, *v_clean = v_ask + 1;
  volatile int* info = reinterpret_cast<volatile int*>(smem + Cfg::kOffInfo);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::kOffInfo + kAtInfo * 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ask = reinterpret_cast<volatile int*>(tmem_slot + 4);  // a step whose V is to be looked over: its number among the CTA's, and of all (-1: no more)
  int* noted = reinterpret_cast<int*>(tmem_slot + 2);  // first and last step whose V held what is not finite
  int* docs = reinterpret_cast<int*>(smem + Cfg::kOffDocs);
  float2* sums = reinterpret_cast<float2*>(smem + Cfg::kOffSums);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned long long wait_ns = wait_limit(a.wait_ns);

  if (warp == 0) {
    for (int i = lane; i < Cfg::kBars; i += 32) {
      const uint64_t* of = bar + i;
      mbar_init(bar + i, of == v_clean ? 2 : of == v_ask ? 1 : of >= table_full ? Cfg::kSoftmax : of >= drain ? 3 : of >= p_full ? 4 : of >= info_empty && of < s_full ? Cfg::kSoftmax + 1 : 1);
    }
    if (lane == 0) {
      *abort_flag = 0;
      noted[0] = INT_MAX;
      noted[1] = -1;
    }
    fence_mbar_init();
  }
  if (warp == Cfg::kMmaWarp) { tmem_alloc(tmem_slot, Cfg::kTmemCols); tmem_relinquish(); }
  if (warp == Cfg::kLoadWarp && lane == 0) { tma_prefetch_desc(&maps.q); tma_prefetch_desc(&maps.k); tma_prefetch_desc(&maps.v); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  // The work item: split x kv head x sequence x group of tiles, the last queries first (they see the most keys under a causal mask); or with the
  // tiles inside the sequences.
  uint32_t item = a.by_splits.div(blockIdx.x);
  const int split = blockIdx.x - item * a.splits;
  const uint32_t of_kv = a.by_kv.div(item);
  const int kv = item - of_kv * a.kv_heads;
  const int outer_index = a.by_inner.div(of_kv), inner_index = of_kv - outer_index * (a.pairs_inside ? a.pairs : a.sequences);
  int b = a.pairs_inside ? outer_index : inner_index;
  if (kQuarters && a.longest_first) {
    // The sequence with b others before it.
    int *lengths = reinterpret_cast<int*>(smem + Cfg::kOffWeights), *found = lengths + kAtMostOrdered, me = threadIdx.x;
    if (me < a.sequences) lengths[me] = a.k_lengths[me];
    __syncthreads();
    if (me < a.sequences) {
      int before = 0;
#pragma unroll 8
      for (int i = 0; i < a.sequences; ++i) before += lengths[i] > lengths[me] || (lengths[i] == lengths[me] && i < me);
      if (before == b) *found = me;
    }
    __syncthreads();
    b = *found;
  }
  const int pair = a.pairs - 1 - (a.pairs_inside ? inner_index : outer_index);
  int all_queries;
  const AttendSequence s = attend_sequence(a, b, &all_queries);
  const int offset = s.keys - all_queries;  // a query's position less its number
  const int per_tile = a.per_tile, first = NT * pair * per_tile;
  const int tokens[2] = {max(0, min(per_tile, s.queries - first)), NT == 1 ? 0 : max(0, min(per_tile, s.queries - first - per_tile))};
  const bool idle = tokens[0] == 0, few = NT == 2 && tokens[1] == 0;  // of all CTAs of the cluster alike
  const int nk = (a.dim + 15) / 16;  // depth steps of 16 values
  const int halves = a.dim > 64 ? 2 : 1;

  // Spans of the tiles' first and last queries: [outer.lo, outer.hi] is what some query sees, [inner.lo, inner.hi] what all do.  The CTA
  // takes its share of the steps [at, end) from the first to the last key that some query sees.
  AttendSpan outer[2], inner[2];
  int from = INT_MAX, to = -1;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    outer[t] = inner[t] = {1, 0};
    if (!tokens[t]) continue;
    const int p0 = first + t * per_tile + offset;
    const AttendSpan x = attend_span(a, p0, s.keys), y = attend_span(a, p0 + tokens[t] - 1, s.keys);
    outer[t] = {x.lo, y.hi};
    inner[t] = {y.lo, x.hi};
    if (outer[t].lo <= outer[t].hi) { from = min(from, outer[t].lo); to = max(to, outer[t].hi); }
  }
  const int prefix = max(0, min(s.prefix, s.keys));
  if (prefix > 0) { from = 0; to = max(to, prefix - 1); }
  int at = from <= to ? from / kAtKeys : 0, end = from <= to ? to / kAtKeys + 1 : 0;
  if (a.splits > 1) {
    const int share = (end - at + a.splits - 1) / a.splits;
    at += split * share;
    end = min(end, at + share);
  }
  // Lowest and highest document of each of the CTA's steps, found by the softmax warps before there are scores: with documents most steps may
  // show nothing, and one at a time each takes a trip to memory.
  const bool summed = a.documents && end - at <= kAtMostSummary;
  int2* summary = reinterpret_cast<int2*>(smem + Cfg::kOffSummary);
  const bool dual = few && end - at > 1;            // both tiles take the rows of the first, each every other step
  const bool joined = !idle && (a.splits > 1 || dual || kQuarters);  // the rows' results are in parts
  float* part = reinterpret_cast<float*>(smem + Cfg::kOffK);  // unnormalised rows of O, once all products are done

  if (!idle && warp < Cfg::kSoftmax) {
    // ---- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kSoftmaxRegs));
    const int t = warp >> 2, quarter = warp & 3, tile = few ? 0 : t;
    const int row = quarter * 32 + lane, row_of_tile = kQuarters ? lane : row;
    constexpr int NC = kQuarters ? 1 : 4;     // chunks of 32 keys of a step that this thread takes,
    const int chunk0 = kQuarters ? quarter : 0;  // from this one on
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lane_addr + t * 128, o_tmem = tmem + lane_addr + Cfg::kTmemO + t * DP;
    const uint32_t p_tmem = s_tmem;
    const int tile_token = a.by_group.div(row_of_tile), head = kv * a.group + row_of_tile - tile_token * a.group;
    const int query = first + tile * per_tile + tile_token;
    const bool live = tile_token < tokens[tile];
    const bool warp_live = __any_sync(0xffffffffu, live);
    float m = -INFINITY, l = 0.f;  // the maximum that P is relative to (log2 units, natural ones with kNatural), and the sum
    const int p = query + offset;
    AttendSpan span = attend_span(a, p, s.keys);
    if (!live) span = {0, -1};
    const int below = live ? prefix : 0;
    const int doc = live && a.documents ? a.documents[s.q_start + query] : 0;
    // Finite factors stay finite in log2 units.
    auto in_units = [&](float x) { return fabsf(x) <= FLT_MAX ? fminf(fmaxf(x * kUnit, -FLT_MAX), FLT_MAX) : x; };
    const float scale = in_units(a.scale);
    const float slope = (kMode == kAtSlopes || kGeneral) && live && a.slopes ? in_units(a.slopes[head]) : 0.f;
    const bool tame = fabsf(slope) < 1e28f;  // its products with distances are finite
    const float* table = kGeneral && a.table ? a.table + (int64_t)(live ? head : 0) * (2 * a.reach + 1) + a.reach : nullptr;
    // The distance bias of the group's heads in shared memory, with the edges' values as far past the reach as a tile and a step make.
    const int wide = 2 * (a.reach + kAtKeys + kAtRows) + a.table_pad;
    constexpr bool table_here = kMode == kAtTable;
    const float* near = reinterpret_cast<const float*>(smem + Cfg::kOffTable) + (head - kv * a.group) * wide + a.reach + kAtKeys + kAtRows;
    if (table_here) {
      float* to = reinterpret_cast<float*>(smem + Cfg::kOffTable);
      for (int g = 0; g < a.group; ++g) {
        const float* of = a.table + (int64_t)(kv * a.group + g) * (2 * a.reach + 1) + a.reach;
#pragma unroll 4
        for (int i = threadIdx.x; i < wide; i += 32 * Cfg::kSoftmax)
          to[g * wide + i] = __ldg(of + min(max(i - (a.reach + kAtKeys + kAtRows), -a.reach), a.reach));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(table_full);
    }
    const bool capped = kMode == kAtCap || (kGeneral && a.cap > 0.f);
    // Caps near the ends of fp32's range stay finite: past 1e37 a cap's quotient is a step, and past 1e38 a cap is above all scores.
    const float most_cap = fminf(a.cap, 1e38f);
    const CapTerms cap(capped ? fminf(fmaxf(a.scale / most_cap, -1e37f), 1e37f) : 0.f, most_cap * kUnit, scale);
    if (summed) {
      for (int i0 = warp; i0 < end - at; i0 += 4 * Cfg::kSoftmax) {
        int d[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = i0 + u * Cfg::kSoftmax, j = (at + i) * kAtKeys + 32 * c + lane;
            // Past the last key the step's first document, which is in the step.
            if (i < end - at) d[u][c] = a.k_documents[s.k_start + (j < s.keys ? j : (at + i) * kAtKeys)];
          }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * Cfg::kSoftmax;
          if (i >= end - at) break;
          const int lo = __reduce_min_sync(0xffffffffu, min(min(d[u][0], d[u][1]), min(d[u][2], d[u][3])));
          const int hi = __reduce_max_sync(0xffffffffu, max(max(d[u][0], d[u][1]), max(d[u][2], d[u][3])));
          if (lane == 0) summary[i] = make_int2(lo, hi);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(summary_full);
    }
    bool ok = !table_here || mbar_wait(table_full, 0, a.err, kErrAttnWait, abort_flag, wait_ns);
    int count = 0;  // steps of this tile
    for (int n = 0;; ++n) {
      const int e = n % kAtInfo;
      ok = ok && mbar_wait(info_full + e, (n / kAtInfo) & 1, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      const int x = info[e];
      if (x == kAtEnd) break;
      const int cls = (x >> 2 * t) & 3, kb = (int)((uint32_t)x >> 8) * kAtKeys;
      if (cls == kAtSkip) {
        __syncwarp();
        if (lane == 0) mbar_arrive(info_empty + e);
        continue;
      }
      // `whole`: all rows of the warp see all of its keys; otherwise `bits` says for each chunk of 32 what this row sees.
      uint32_t bits[NC];
      bool whole = true;
      if (cls != kAtFull && warp_live) {
        const int mixed = x >> 4 & 15;  // chunks with keys of several documents
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int kc = kb + 32 * (chunk0 + c);
          bits[c] = low_bits(span.hi + 1 - kc) & ~low_bits(span.lo - kc);
          if (a.documents) {
            const int* dc = docs + e * kAtKeys + 32 * (chunk0 + c);
            uint32_t same = dc[0] == doc ? ~0u : 0u;
            if ((mixed >> (chunk0 + c)) & 1) {
              same = 0;
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const int4 d = *reinterpret_cast<const int4*>(dc + i);
                same |= (d.x == doc) << i | (d.y == doc) << (i + 1) | (d.z == doc) << (i + 2) | (d.w == doc) << (i + 3);
              }
            }
            bits[c] &= same;
          }
          bits[c] |= low_bits(below - kc);
          whole = whole && bits[c] == ~0u;
        }
        whole = __all_sync(0xffffffffu, whole || !live);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(info_empty + e);
      ok = mbar_wait(s_full + t, count & 1, a.err, kErrAttnWait, abort_flag, wait_ns);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      ++count;
      if (!warp_live) {
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + t);
        continue;
      }
      uint32_t sx[NC][32];
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_ld32_async(s_tmem + 32 * (chunk0 + c), sx[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_wait_ld(sx[c]);
      if (kQuarters) {
        // No P for the keys of the other quarters.
        uint32_t none[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) none[i] = 0u;
#pragma unroll
        for (int c = 1; c < 4; ++c) tmem_st16(p_tmem + 16 * ((chunk0 + c) & 3), none);
      }
      constexpr int kMine = 32 * NC;              // keys of this thread
      const int d = kb + 32 * chunk0 - p;  // the first less the query
      float sum = 0.f;
      // P from the exponents that f gives of the scores, to TMEM; the largest exponent.  P is rounded to the inputs' type, in which the tensor core takes it (bf16 results
      // are then off by 0.0020 of their size where the rounding of the results alone gives 0.0016, f16 ones by 0.00028 and 0.00021); their sum is not.  ex2.approx is
      // off by 2^-22.
      auto numerators = [&](auto f) {
        float2 part[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 v = f(make_float2(__uint_as_float(sx[c][i]), __uint_as_float(sx[c][i + 1])), 32 * c + i);
            mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], v.x, v.y);
            const float2 w = make_float2(ex2_approx(v.x), ex2_approx(v.y));
            part[(i >> 1) & 3] = add2(part[(i >> 1) & 3], w);
            pk[i >> 1] = pack2<T>(w.x, w.y);
          }
          tmem_st16(p_tmem + 16 * (chunk0 + c), pk);
        }
        const float2 both = add2(add2(part[0], part[1]), add2(part[2], part[3]));
        sum = both.x + both.y;
        return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      };
      // A step relative to the maximum of the steps before, from the products at once: the exponents' maximum, found beside them,
      // tells whether it will do (few steps raise it by more than kAtRescale).
      const float fd = (float)d;
      const float2 by = make_float2(scale, scale), unit = make_float2(kLog2e, kLog2e), shift = make_float2(kShift, kShift);
      // The distance bias of the first key, in the part of the table that is there: past the reach all values are the edge's.
      const float* bias = near + min(max(d, -(a.reach + kAtKeys + kAtRows)), a.reach + kAtRows);
      auto at_once = [&]() {
        const float base = m == -INFINITY ? 0.f : m;  // (rows of no query)
        const float2 less = make_float2(kShift - base, kShift - base), at_m = make_float2(base, base);
        float most = INFINITY;
        if (kMode == kAtPlain) {
          most = numerators([&](float2 y, int) { return fma2(y, by, less); });
        } else if (kMode == kAtCap) {
          float big = 0.f;
          most = numerators([&](float2 y, int) { big = max3(big, fabsf(y.x), fabsf(y.y)); return fma2(y, cap.slope(y), less); });
          if (!(big <= cap.most)) most = INFINITY;
        } else if (kMode == kAtSlopes) {
          // All keys on one side of the query.
          const bool left = d + kMine - 1 <= 0;
          if (__all_sync(0xffffffffu, tame && (left || d >= 0))) {
            const float g = left ? slope : -slope, at_d = fmaf(g, fd, kShift - base);
            const float2 from = make_float2(at_d, at_d), each = make_float2(g, g);
            most = numerators([&](float2 y, int i) { return fma2(y, by, fma2(each, make_float2((float)i, (float)(i + 1)), from)); });
          } else {
            most = numerators([&](float2 y, int i) {
              return fma2(y, by, fma2(make_float2(-slope, -slope), make_float2(fabsf(fd + (float)i), fabsf(fd + (float)(i + 1))), less));
            });
          }
        } else if (kMode == kAtTable) {
          most = numerators([&](float2 y, int i) { return fma2(sub2(fma2(y, by, make_float2(bias[i], bias[i + 1])), at_m), unit, shift); });
        }
        return __all_sync(0xffffffffu, most <= kShift + kAtRescale || !live);
      };
      bool done = false;
      // Masked steps and a row's first one take the other way: a second form of this one for masked steps made all 3% slower by its code's length, and
      // a first maximum from the raw products, so that first steps too come here, took longer than it saved (without it a learned bias 189 -> 180 us at 64 x 512, a
      // cap at 16384 causal, unit variance, 1436 -> 1389; plain ragged sequences of 64 306 -> 310).
      if (!kGeneral && whole && !__any_sync(0xffffffffu, m == -INFINITY && live)) done = at_once();
      if (!done) {
        if (!kGeneral) tmem_wait_st();  // before P is written again
        auto each = [&](auto f) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 y = f(make_float2(__uint_as_float(sx[c][i]), __uint_as_float(sx[c][i + 1])), 32 * c + i);
              sx[c][i] = __float_as_uint(y.x);
              sx[c][i + 1] = __float_as_uint(y.y);
            }
        };
        if (capped) {
          float big = 0.f;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2) big = max3(big, fabsf(__uint_as_float(sx[c][i])), fabsf(__uint_as_float(sx[c][i + 1])));
          if (__all_sync(0xffffffffu, big <= cap.most)) each([&](float2 y, int) { return mul2(y, cap.slope(y)); });
          else each([&](float2 y, int) {
            const float2 n = mul2(y, cap.slope(y));
            return make_float2(fabsf(y.x) <= cap.most ? n.x : cap.any(y.x), fabsf(y.y) <= cap.most ? n.y : cap.any(y.y));
          });
        }
        const float2 factor = capped ? make_float2(1.f, 1.f) : by;
        if ((kMode == kAtSlopes || kGeneral) && a.slopes) {
          each([&](float2 y, int i) { return fma2(y, factor, make_float2(-slope * fabsf(fd + (float)i), -slope * fabsf(fd + (float)(i + 1)))); });
        } else if (kMode == kAtTable) {
          each([&](float2 y, int i) { return fma2(y, factor, make_float2(bias[i], bias[i + 1])); });
        } else if (kGeneral && table) {
          each([&](float2 y, int i) {
            return fma2(y, factor, make_float2(__ldg(table + min(max(d + i, -a.reach), a.reach)), __ldg(table + min(max(d + i + 1, -a.reach), a.reach))));
          });
        } else if (kMode == kAtPlain || (kGeneral && !capped)) {
          each([&](float2 y, int) { return mul2(y, factor); });
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((bits[c] >> i) & 1)) sx[c][i] = __float_as_uint(-INFINITY);
        }
        float mx[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = -INFINITY;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 7] = max3(mx[(i >> 1) & 7], __uint_as_float(sx[c][i]), __uint_as_float(sx[c][i + 1]));
#pragma unroll
        for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
          for (int i = 0; i < w; ++i) mx[i] = fmaxf(mx[i], mx[i + w]);
        const float top = mx[0];
        float alpha = 1.f;
        bool dirty = false;
        if (top > m + (kNatural ? kAtRescale / kLog2e : kAtRescale)) {
          if (m != -INFINITY) { alpha = ex2_approx(kNatural ? (m - top) * kLog2e : m - top); dirty = true; }
          m = top;
        }
        l *= alpha;
        if (__any_sync(0xffffffffu, dirty)) {
          // O is settled: s_full followed the products before.
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
        const float base = m == -INFINITY ? 0.f : m;
        const float2 at_m = make_float2(base, base), less = make_float2(kShift - base, kShift - base);
        // Differences before the factor in natural units: scores of the type's lowest value stay equal to one another.
        numerators([&](float2 y, int) { return kNatural ? fma2(sub2(y, at_m), unit, shift) : add2(y, less); });
      }
      l += sum;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + t);
    }
    ok = ok && mbar_wait(drain + t, 0, a.err, kErrAttnWait, abort_flag, wait_ns);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (joined) {
      sums[t * kAtRows + row] = make_float2(m, ok ? l : NAN);
    } else if (ok && warp_live && !(few && t)) {
      // Rows without a visible key, and rows that no step was made for, hold nothing in O.
      const int64_t token = s.q_start + query;
      const bool any = l > 0.f || l != l;
      const float inv = any ? 1.f / l : 0.f;
      // Through the tile's Q in shared memory, which no product reads any more: 8 lanes then write 128 bytes of a row.
      uint8_t* stage = smem + Cfg::kOffQ + t * Cfg::kQTile;
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
            w[k] = pack2<T>(x, y);
          }
          const int at_c = c + i;  // 16 bytes: value at_c of the row
          *reinterpret_cast<uint4*>(stage + (at_c >> 6) * Cfg::kQHalf + row * 128 + (((at_c & 63) * 2) ^ ((row & 7) << 4))) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      for (int h = 0; h < halves; ++h) {
        const int at_c = 64 * h + (lane & 7) * 8;
#pragma unroll 4
        for (int i = 0; i < 32; i += 4) {
          const int r = (warp & 3) * 32 + i + (lane >> 3);
          const int tok = a.by_group.div(r), hd = kv * a.group + r - tok * a.group;
          if (tok < tokens[tile] && at_c < a.dim)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t)(s.q_start + first + tile * per_tile + tok) * a.out_token + hd * a.out_head + at_c) =
                *reinterpret_cast<const uint4*>(stage + h * Cfg::kQHalf + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        }
      }
      __syncwarp();
      if (live && a.lse)
        a.lse[token * a.heads + head] = any ? (kNatural ? m : m / kLog2e) + (log2f(l) - kShift) / kLog2e : -INFINITY;
      if (noted[1] >= 0) {
        AttendFound found;
        attend_scan<T>(a, s, all_queries, query, kv, live && l > 0.f, 4 * min(noted[0], noted[1]), min(4 * noted[1] + 3, (s.keys - 1) >> 5), 1, found);
        for (uint32_t rest = __ballot_sync(0xffffffffu, found.any()); rest; rest &= rest - 1) {
          const int src = __ffs(rest) - 1;
          AttendFound theirs;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            theirs.nan[c] = __shfl_sync(0xffffffffu, found.nan[c], src);
            theirs.up[c] = __shfl_sync(0xffffffffu, found.up[c], src);
            theirs.down[c] = __shfl_sync(0xffffffffu, found.down[c], src);
          }
          attend_put<T>(a, s.q_start + __shfl_sync(0xffffffffu, query, src), __shfl_sync(0xffffffffu, head, src), theirs, false);
        }
      }
    }
  } else if (!idle) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kOtherRegs));
    if (warp == Cfg::kLoadWarp) {
      // ---- steps and loads
      int doc_lo[2] = {INT_MAX, INT_MAX}, doc_hi[2] = {INT_MIN, INT_MIN};
      if (elect_one())
        for (int t = 0; t < NT; ++t)
          if (tokens[t]) {
            constexpr int kCopies = kQuarters ? 4 : 1;
            mbar_arrive_expect_tx(q_full + t, kCopies * halves * 128 * a.group * per_tile);
            for (int h = 0; h < halves; ++h)
              for (int c = 0; c < kCopies; ++c)
                tma_load_3d(smem + Cfg::kOffQ + t * Cfg::kQTile + h * Cfg::kQHalf + c * 32 * 128, &maps.q, q_full + t, 64 * h, kv * a.group,
                            s.q_start + first + t * per_tile);
          }
      __syncwarp();
      if (a.documents)
        for (int t = 0; t < NT; ++t) {
          for (int i = lane; i < tokens[t]; i += 32) {
            const int d = a.documents[s.q_start + first + t * per_tile + i];
            doc_lo[t] = min(doc_lo[t], d);
            doc_hi[t] = max(doc_hi[t], d);
          }
          doc_lo[t] = __reduce_min_sync(0xffffffffu, doc_lo[t]);
          doc_hi[t] = __reduce_max_sync(0xffffffffu, doc_hi[t]);
        }
      int n = 0, k_issued = 0, v_issued = 0;
      bool ok = !summed || mbar_wait(summary_full, 0, a.err, kErrAttnWait, abort_flag, wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      auto load = [&](const CUtensorMap* map, uint64_t* full, uint64_t* empty, int off, int kb, int& issued) {
        const int slot = n % kSlots;
        ok = ok && mbar_wait(empty + slot, ((n / kSlots) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        if (elect_one()) {
          mbar_arrive_expect_tx(full + slot, halves * Cfg::kHalf);
          for (int h = 0; h < halves; ++h) tma_load_3d(smem + off + slot * Cfg::kTile + h * Cfg::kHalf, map, full + slot, 64 * h, kv, s.k_start + kb);
        }
        __syncwarp();
        ++issued;
      };
      // What a step with documents lo .. hi is to each tile: kAtClass of tile 0, and of tile 1 two bits up.
      auto classify = [&](int step, int lo, int hi) {
        const int kb = step * kAtKeys, last = min(kb + kAtKeys, s.keys) - 1;
        int both = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const bool one = !a.documents || (lo == hi && doc_lo[t] == doc_hi[t] && lo == doc_lo[t]);
          const bool to_last = last < prefix || (kb >= inner[t].lo && last <= inner[t].hi && one);
          const bool meets = kb < prefix || (kb <= outer[t].hi && last >= outer[t].lo && (!a.documents || (lo <= doc_hi[t] && hi >= doc_lo[t])));
          both |= (!tokens[t] ? kAtSkip : to_last ? (last == kb + kAtKeys - 1 ? kAtFull : kAtTail) : meets ? kAtMasked : kAtSkip) << 2 * t;
        }
        return both;
      };
      // With slopes the nearest keys first, whose scores the later ones then seldom exceed.
      auto step_of = [&](int i) { return a.slopes ? at + end - 1 - i : i; };
      // 32 steps at a time, each by a lane, then those that show something.  (Documents that are not known yet: all may be.)
      uint32_t shown = 0;
      int lane_lo = 0, lane_hi = 0, lane_class = 0;
      for (int i = at; i < end && ok; ++i) {
        const int in_group = (i - at) & 31;
        if (in_group == 0) {
          lane_lo = INT_MIN;
          lane_hi = INT_MAX;
          lane_class = 0;
          if (i + lane < end) {
            const int mine = step_of(i + lane);
            if (summed) { lane_lo = summary[mine - at].x; lane_hi = summary[mine - at].y; }
            lane_class = classify(mine, lane_lo, lane_hi);
          }
          shown = __ballot_sync(0xffffffffu, lane_class != 0);
        }
        const uint32_t left = shown >> in_group;
        if (!left) { i += 31 - in_group; continue; }  // on to the next 32
        const int next = __ffs(left) - 1 + in_group;
        i += next - in_group;
        const int step = step_of(i);
        int both = __shfl_sync(0xffffffffu, lane_class, next), lo = __shfl_sync(0xffffffffu, lane_lo, next), hi = __shfl_sync(0xffffffffu, lane_hi, next);
        const int kb = step * kAtKeys, last = min(kb + kAtKeys, s.keys) - 1;
        int d[4] = {lo, lo, lo, lo}, mixed = 0;
        if (a.documents && lo != hi) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int j = kb + lane + 32 * c;
            d[c] = a.k_documents[s.k_start + (j <= last ? j : kb)];
          }
          if (!summed) {
            lo = __reduce_min_sync(0xffffffffu, min(min(d[0], d[1]), min(d[2], d[3])));
            hi = __reduce_max_sync(0xffffffffu, max(max(d[0], d[1]), max(d[2], d[3])));
            if (kb >= prefix && (lo > doc_hi[0] || hi < doc_lo[0]) && (NT == 1 || lo > doc_hi[1] || hi < doc_lo[1])) continue;  // (most steps of many documents)
            both = classify(step, lo, hi);
            if (!both) continue;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (!__all_sync(0xffffffffu, d[c] == __shfl_sync(0xffffffffu, d[c], 0))) mixed |= 1 << c;
        }
        int cls[2] = {both & 3, both >> 2};
        if (dual && (n & 1)) { cls[1] = cls[0]; cls[0] = kAtSkip; }
        const int e = n % kAtInfo;
        ok = mbar_wait(info_empty + e, ((n / kAtInfo) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (a.documents) {
#pragma unroll
          for (int i = 0; i < 4; ++i) docs[e * kAtKeys + lane + 32 * i] = d[i];
        }
        if (lane == 0) info[e] = (int)((uint32_t)step << 8 | mixed << 4 | cls[1] << 2 | cls[0]);
        __syncwarp();
        if (lane == 0) mbar_arrive(info_full + e);
        load(&maps.k, k_full, k_empty, Cfg::kOffK, kb, k_issued);
        load(&maps.v, v_full, v_empty, Cfg::kOffV, kb, v_issued);
        ++n;
      }
      if (ok) {
        const int e = n % kAtInfo;
        ok = mbar_wait(info_empty + e, ((n / kAtInfo) & 1) ^ 1, a.err, kErrAttnWait, abort_flag, wait_ns);
        if (lane == 0 && ok) { info[e] = kAtEnd; mbar_arrive(info_full + e); }
      }
      __syncwarp();
      // Every copy has landed before this warp ends, and the CTA with it: all have been used by then, unless a role gave up, be it after this point.
      for (int t = 0; t < NT; ++t)
        if (tokens[t]) mbar_drain(q_full + t, 0);
      for (int i = max(0, k_issued - kSlots); i < k_issued; ++i) mbar_drain(k_full + i % kSlots, (i / kSlots) & 1);
      for (int i = max(0, v_issued - kSlots); i < v_issued; ++i) mbar_drain(v_full + i % kSlots, (i / kSlots) & 1);
    } else if (warp == Cfg::kMmaWarp) {
      // ---- tensor products, by one thread
      if (elect_one()) {
        constexpr uint32_t idesc_s = mma_idesc<kBf16>(kAtRows, kAtKeys);
        const uint32_t idesc_o = mma_idesc<kBf16>(kAtRows, 0) | (uint32_t)(2 * nk) << 17 | 1u << 16;  // N = 16 nk; B by values
        const uint32_t q_addr = smem_u32(smem + Cfg::kOffQ), k_addr = smem_u32(smem + Cfg::kOffK), v_addr = smem_u32(smem + Cfg::kOffV);
        bool ok = true;
        int used[2] = {0, 0};  // products P V of each tile
        int checked = 0;       // steps whose V was looked over
        auto wait = [&](uint64_t* which, int parity) { ok = ok && mbar_wait(which, parity, a.err, kErrAttnWait, abort_flag, wait_ns); };
        auto read = [&](int n) {
          const int e = n % kAtInfo;
          wait(info_full + e, (n / kAtInfo) & 1);
          int x = kAtEnd;
          if (ok) {
            x = info[e];
            mbar_arrive(info_empty + e);
          }
          return x;
        };
        auto takes = [](int x, int t) { return x != kAtEnd && ((x >> 2 * t) & 3); };
        // S of step n for tile t, over the P whose product has been issued.
        auto scores = [&](int n, int t) {
          if (!ok) return;
          tc_fence_after();
          const uint32_t qt = q_addr + (dual ? 0 : t * Cfg::kQTile), kt = k_addr + n % kSlots * Cfg::kTile;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)  // (not to nk: rolled, the issue of a product took 80 cycles, more than the product)
            if (k < nk)
              tc_mma_f16(tmem + t * 128, smem_desc_sw128(qt + (k >> 2) * Cfg::kQHalf + (k & 3) * 32),
                         smem_desc_sw128(kt + (k >> 2) * Cfg::kHalf + (k & 3) * 32), idesc_s, k > 0);
          tc_commit(s_full + t);
        };
        auto values = [&](int n, int t) {
          wait(p_full + t, used[t] & 1);
          if (!ok) return;
          tc_fence_after();
          const uint32_t pt = tmem + t * 128;
#pragma unroll
          for (int k = 0; k < kAtKeys / 16; ++k)
            tc_mma_f16_ts(tmem + Cfg::kTmemO + t * DP, pt + 8 * k, smem_desc_values(v_addr + n % kSlots * Cfg::kTile + k * 2048, Cfg::kHalf), idesc_o,
                          used[t] > 0 || k > 0);
          ++used[t];
        };
        int cur = read(0);
        // Also where no step follows: the softmax warps, which wait for `drain` alone, then write their rows over Q.
        for (int t = 0; t < NT; ++t)
          if (tokens[t]) wait(q_full + t, 0);
        if (cur != kAtEnd) {
          wait(k_full, 0);
          for (int t = 0; t < NT; ++t)
            if (takes(cur, t)) scores(0, t);
          if (ok) tc_commit(k_empty);
        }
        for (int n = 0; ok && cur != kAtEnd; ++n) {
          wait(v_full + n % kSlots, (n / kSlots) & 1);  // (V of a step is loaded before K of the next)
          const bool asked = ok && attend_cut(cur);
          if (asked) {
            ask[0] = 2 * n + attend_hides(cur);
            ask[1] = (int)((uint32_t)cur >> 8);
            mbar_arrive(v_ask);
          }
          const int next = read(n + 1), k_next = (n + 1) % kSlots;
          if (next != kAtEnd) wait(k_full + k_next, ((n + 1) / kSlots) & 1);
          // A tile that has no part in this step need not wait for it.
          for (int t = 0; t < NT; ++t)
            if (!takes(cur, t) && takes(next, t)) scores(n + 1, t);
          if (asked) wait(v_clean, checked++ & 1);
          for (int t = 0; t < NT; ++t)
            if (takes(cur, t)) {
              values(n, t);
              if (takes(next, t)) scores(n + 1, t);
            }
          if (ok) {
            tc_commit(v_empty + n % kSlots);
            if (next != kAtEnd) tc_commit(k_empty + k_next);
          }
          cur = next;
        }
        ask[1] = -1;
        mbar_arrive(v_ask);
        for (int t = 0; t < NT; ++t) tc_commit(drain + t);
        for (int t = 0; t < NT; ++t) mbar_drain(drain + t, 0);
      }
      __syncwarp();
    } else {
      // ---- V of steps with hidden keys: no value that is not finite, and zeros past the last key, whose rows may hold anything.  A warp takes half of the keys.
      using F = NotFinite<T>;
      for (int checked = 0;; ++checked) {
        // (Between two of them all steps that the CTA has may lie.)
        const bool ok = mbar_wait(v_ask, checked & 1, a.err, kErrAttnWait, abort_flag, wait_ns * (unsigned long long)(max(0, end - at) + 2));
        if (!__all_sync(0xffffffffu, ok)) break;
        const int n = ask[0] >> 1, step = ask[1], slot = n % kSlots, rows = s.keys - step * kAtKeys;
        if (step < 0 || !__all_sync(0xffffffffu, mbar_wait(v_full + slot, (n / kSlots) & 1, a.err, kErrAttnWait, abort_flag, wait_ns))) break;
        uint8_t* tile = smem + Cfg::kOffV + slot * Cfg::kTile;
        for (int h = 0; rows < kAtKeys && h < halves; ++h)
          for (int i = rows * 8 + threadIdx.x - 32 * Cfg::kCheckWarp; i < kAtKeys * 8; i += 64) reinterpret_cast<uint4*>(tile + h * Cfg::kHalf)[i] = make_uint4(0, 0, 0, 0);
        bool found = false;
        if (ask[0] & 1) {
          const int key0 = (warp - Cfg::kCheckWarp) * 64;  // 4 keys at a time
          uint32_t sum[4] = {};
          for (int h = 0; h < halves; ++h) {
            const uint4* v = reinterpret_cast<const uint4*>(tile + h * Cfg::kHalf + key0 * 128) + lane;
#pragma unroll 4  // (8 are no faster)
            for (int i = 0; i < 16; ++i) {
              const uint4 w = key0 + 4 * i + (lane >> 3) < rows ? v[32 * i] : make_uint4(0, 0, 0, 0);
              sum[0] = F::gather(w.x, sum[0]);
              sum[1] = F::gather(w.y, sum[1]);
              sum[2] = F::gather(w.z, sum[2]);
              sum[3] = F::gather(w.w, sum[3]);
            }
          }
          found = ((F::carries(sum[0]) | F::carries(sum[1]) | F::carries(sum[2]) | F::carries(sum[3])) & 0x80008000u) != 0;
          if (found)
            for (int h = 0; h < halves; ++h) {
              uint4* v = reinterpret_cast<uint4*>(tile + h * Cfg::kHalf + key0 * 128) + lane;
#pragma unroll 1
              for (int i = 0; i < 16; ++i)
                if (key0 + 4 * i + (lane >> 3) < rows) {
                  const uint4 w = v[32 * i];
                  v[32 * i] = make_uint4(F::cleared(w.x), F::cleared(w.y), F::cleared(w.z), F::cleared(w.w));
                }
            }
        }
        if (found) {
          atomicMin(noted, step);
          atomicMax(noted + 1, step);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
      __syncwarp();
      if (lane == 0)
        for (int t = 0; t < NT; ++t) mbar_arrive(drain + t);
    }
  }
  if (joined) {
    // Every part of the rows into its CTA's shared memory: all products are done, so the tiles of K and V are free.
    __syncthreads();
    tc_fence_after();
    if (warp < Cfg::kSoftmax) {
      const int t = warp >> 2, row = (warp & 3) * 32 + lane, slot = t * kAtRows + row;
      const bool live = (int)a.by_group.div(kQuarters ? lane : row) < tokens[few ? 0 : t];
      if (__any_sync(0xffffffffu, live)) {
#pragma unroll 1
        for (int c = 0; c < a.dim; c += 32) {
          uint32_t o[32];
          tmem_ld32_async(tmem + ((uint32_t)((warp & 3) * 32) << 16) + Cfg::kTmemO + t * DP + c, o);
          tmem_wait_ld(o);
          if (live)
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(part + slot * DP + (((c + i) / 4) ^ (row & 7)) * 4) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    }
    tc_fence_before();
    if (a.splits > 1) cluster_sync();
    else __syncthreads();
    // Each CTA joins its share of the rows: their parts' weights, then the rows.  `sound` has a word for each row, whether its sum is finite and above zero.
    const int rows0 = tokens[0] * a.group, rows = rows0 + tokens[1] * a.group, parts = (kQuarters ? 8 : few ? 2 : 1) * a.splits;
    const int share = (rows + a.splits - 1) / a.splits, row0 = split * share, mine = max(0, min(share, rows - row0));
    float* weights = reinterpret_cast<float*>(smem + Cfg::kOffWeights);  // [parts][share]
    volatile int* sound = docs;
    static_assert(kAtInfo * kAtKeys >= 2 * kAtRows, "a word per row");
    const uint32_t part_addr = smem_u32(part), sums_addr = smem_u32(sums);
    auto slot_of = [&](int r, int c) { return kQuarters ? (c & 7) * 32 + r : few ? (c & 1) * kAtRows + r : r >= rows0 ? kAtRows + r - rows0 : r; };
    auto rank_of = [&](int c) { return kQuarters ? c >> 3 : few ? c >> 1 : c; };
    auto place = [&](int r, int* query, int* head) {
      const int at_row = r >= rows0 ? r - rows0 : r, tok = a.by_group.div(at_row);
      *query = first + (r >= rows0 ? per_tile : 0) + tok;
      *head = kv * a.group + at_row - tok * a.group;
    };
    if (!*abort_flag)
      for (int i = warp; i < mine; i += Cfg::kThreads / 32) {
        // A lane per part, several where there are more than 32.
        constexpr int kEach = kQuarters ? 8 * kAtMostSplits / 32 : 1;
        const int r = row0 + i;
        float2 ml[kEach];
        float top = -INFINITY, sum = 0.f, w[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          ml[k] = make_float2(-INFINITY, 0.f);
          if (lane + 32 * k < parts) ml[k] = ld_cluster_v2(cluster_addr(sums_addr + slot_of(r, lane + 32 * k) * 8, rank_of(lane + 32 * k)));
          top = fmaxf(top, ml[k].x);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          // A part that saw nothing has no weight (-1 here), and its O holds anything.  A weight of 0 counts: its part may hold a NaN.
          w[k] = ml[k].x == -INFINITY && ml[k].y == 0.f ? -1.f : ex2_approx(kNatural ? (ml[k].x - top) * kLog2e : ml[k].x - top);
          sum = fmaf(ml[k].y, w[k], sum);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const bool any = sum > 0.f || sum != sum;
        const float inv = any ? 1.f / sum : 0.f;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
          if (lane + 32 * k < parts) weights[(lane + 32 * k) * share + i] = w[k] < 0.f ? -1.f : w[k] * inv;
        if (lane == 0) {
          sound[i] = sum > 0.f && sum - sum == 0.f;
          if (a.lse) {
            int qi, h;
            place(r, &qi, &h);
            a.lse[(int64_t)(s.q_start + qi) * a.heads + h] = any ? (kNatural ? top : top / kLog2e) + (log2f(sum) - kShift) / kLog2e : -INFINITY;
          }
        }
      }
    __syncthreads();
    // The steps that the CTAs of the cluster have noted.
    auto noted_by = [&](int rank) { return ld_cluster_v2(cluster_addr(smem_u32(noted), rank)); };
    bool odd = a.splits == 1 ? noted[1] >= 0 : threadIdx.x < a.splits && __float_as_int(noted_by(threadIdx.x).y) >= 0;
    if (!*abort_flag)
      for (int i = threadIdx.x; i < mine * (DP / 4); i += Cfg::kThreads) {
        const int at_row = i / (DP / 4), dv = i % (DP / 4), r = row0 + at_row;
        if (4 * dv >= a.dim) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int c = 0; c < parts; ++c) {
          const float w = weights[c * share + at_row];
          const int slot = slot_of(r, c);
          const float4 x = ld_cluster_v4(cluster_addr(part_addr + (slot * DP + (dv ^ (slot & 7)) * 4) * 4, rank_of(c)));
          if (!(w < 0.f)) { o.x = fmaf(x.x, w, o.x); o.y = fmaf(x.y, w, o.y); o.z = fmaf(x.z, w, o.z); o.w = fmaf(x.w, w, o.w); }
        }
        // Each quarter's copy of a row has weights of zero for the other quarters' keys, whose infinities make NaN.
        if (kQuarters && (o.x != o.x || o.y != o.y || o.z != o.z || o.w != o.w) && sound[at_row]) odd = true;
        int qi, h;
        place(r, &qi, &h);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.q_start + qi) * a.out_token + h * a.out_head + 4 * dv) =
            make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
      }
    if (__syncthreads_or(odd)) {
      // All warps read v for 32 rows at a time, and put together what they find in the weights' place.
      constexpr int kWarps = Cfg::kThreads / 32, kWords = 12;
      uint32_t* marks = reinterpret_cast<uint32_t*>(weights);
      static_assert(32 * kWords <= Cfg::kWeights, "three masks of 128 channels for each of 32 rows");
      int lo = 0, hi = (s.keys - 1) >> 5;
      if (!kQuarters) {
        int first_noted = INT_MAX, last_noted = -1;
        for (int c = 0; c < a.splits; ++c) {
          const float2 of = noted_by(c);
          first_noted = min(first_noted, __float_as_int(of.x));
          last_noted = max(last_noted, __float_as_int(of.y));
        }
        lo = 4 * max(0, min(first_noted, last_noted));
        hi = min(hi, 4 * last_noted + 3);
      }
      for (int g = 0; g < mine; g += 32) {
        int qi, h;
        place(row0 + min(g + lane, mine - 1), &qi, &h);
        __syncthreads();  // (the marks of the 32 rows before have been read)
        for (int i = threadIdx.x; i < 32 * kWords; i += Cfg::kThreads) marks[i] = 0;
        __syncthreads();
        AttendFound found;
        attend_scan<T>(a, s, all_queries, qi, kv, g + lane < mine && sound[min(g + lane, mine - 1)], lo + warp, hi, kWarps, found);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (found.nan[c]) atomicOr(marks + kWords * lane + c, found.nan[c]);
          if (found.up[c]) atomicOr(marks + kWords * lane + 4 + c, found.up[c]);
          if (found.down[c]) atomicOr(marks + kWords * lane + 8 + c, found.down[c]);
        }
        __syncthreads();
        for (int i = warp; i < min(32, mine - g); i += kWarps) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            found.nan[c] = marks[kWords * i + c];
            found.up[c] = marks[kWords * i + 4 + c];
            found.down[c] = marks[kWords * i + 8 + c];
          }
          place(row0 + g + i, &qi, &h);
          attend_put<T>(a, s.q_start + qi, h, found, kQuarters);
        }
      }
    }
  }
  if (a.splits > 1) {
    if (idle) cluster_sync();
    cluster_sync();  // no CTA ends while another reads its parts
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == Cfg::kMmaWarp) tmem_dealloc(tmem, Cfg::kTmemCols);
}

}  // namespace laya
