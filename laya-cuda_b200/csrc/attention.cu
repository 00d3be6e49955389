// Entry points of the rotary positions and of attention over packed sequences (see include/laya_b200.h): checks of
// arguments and launches.
#include <algorithm>
#include <cmath>

#include "attend.cuh"
#include "host.cuh"
#include "rotary.cuh"

using namespace laya;

namespace {

// A tensor [tokens][heads][dim], strides in elements.
void check_heads(const char* what, const void* p, int64_t token, int64_t head, int dtype) {
  if (!p) fail(LAYA_ERR_INVALID, "%s is null", what);
  if (token < 0 || head < 0) fail(LAYA_ERR_INVALID, "%s: a stride is negative; it must be at least 0", what);
  if (reinterpret_cast<uintptr_t>(p) % dtype_size(dtype)) fail(LAYA_ERR_INVALID, "%s is not aligned to its elements", what);
}

void check_strides(const char* what, int tokens, int heads, int dim, int64_t token, int64_t head) {
  if ((tokens > 1 && token < dim) || (heads > 1 && head < dim))
    fail(LAYA_ERR_INVALID, "%s: strides %lld and %lld must be at least a head's %d values", what, (long long)token, (long long)head, dim);
}

// Tokens and heads apart from one another, as what is written must be.
void check_apart(const char* what, int tokens, int heads, int dim, int64_t token, int64_t head) {
  check_strides(what, tokens, heads, dim, token, head);
  if (tokens <= 1 || heads <= 1) return;
  using Wide = __int128;
  if (token >= (Wide)(heads - 1) * head + dim || head >= (Wide)(tokens - 1) * token + dim) return;
  // Neither lies within a step of the other: j steps of one meet i of the other where they are less than a head apart.
  const int few = std::min(tokens, heads), many = std::max(tokens, heads);
  const int64_t by = tokens < heads ? token : head, of = tokens < heads ? head : token;
  for (int j = 1; j < few; ++j) {
    const Wide at = (Wide)j * by;
    for (Wide i = std::max<Wide>(1, at / of); i <= at / of + 1 && i < many; ++i)
      if (at - i * of < dim && i * of - at < dim)
        fail(LAYA_ERR_INVALID, "%s: with strides %lld and %lld heads of %d values overlap", what, (long long)token, (long long)head, dim);
  }
}

// 16-byte vectors, which the tensor maps and the stores of attention take.  The stride of a dimension of one says nothing and is
// made one that they take.
void check_vectors(const char* what, const void* p, int tokens, int heads, int dim, int64_t* token, int64_t* head, int dtype, bool written) {
  if (heads == 1) *head = dim;
  if (tokens == 1) *token = heads * *head;
  check_heads(what, p, *token, *head, dtype);
  if (written) check_apart(what, tokens, heads, dim, *token, *head);
  else check_strides(what, tokens, heads, dim, *token, *head);
  if (reinterpret_cast<uintptr_t>(p) & 15) fail(LAYA_ERR_INVALID, "%s must be 16-byte aligned", what);
  if (*token % 8 || *head % 8) fail(LAYA_ERR_INVALID, "%s: strides %lld and %lld must each be a multiple of 8", what, (long long)*token, (long long)*head);
  if (*token >= (1ll << 38) || *head >= (1ll << 38)) fail(LAYA_ERR_INVALID, "%s: a stride is too large", what);
}

template <typename F>
void with_half(int dtype, F f) {
  if (dtype == LAYA_DTYPE_F16) f((__half*)nullptr);
  else f((__nv_bfloat16*)nullptr);
}

// A tensor [tokens][heads][dim] of 16-bit values in boxes of 64 values x box_heads x box_tokens, 128-byte swizzle.  Values past
// dim and rows past the last read as zeros.
CUtensorMap heads_map(bool bf16, const void* p, int dim, int heads, int tokens, int64_t head, int64_t token, int box_heads, int box_tokens) {
  CUtensorMap map;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)token * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode_fn()(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims, strides,
                           box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(LAYA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return map;
}

// Clusters of more than 8 CTAs, once per device.
template <typename K>
void allow_wide_clusters(K kern, int dev, std::atomic<uint64_t>& done) {
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  CK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename T, int DP, int NT, int kMode, bool kQuarters>
void launch_attend_kernel(const AttendArgs& a, const AttendMaps& maps, int64_t ctas, int dev, cudaStream_t st) {
  static std::atomic<uint64_t> done{0}, wide{0};
  using Cfg = AttendCfg<DP, NT>;
  auto kern = attend_kernel<T, DP, NT, kMode, kQuarters>;
  allow_smem(kern, Cfg::kBytes, dev, done);
  if (a.splits > 8) allow_wide_clusters(kern, dev, wide);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (a.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  CK(cudaLaunchKernelEx(&cfg, kern, maps, a));
}

template <typename T, int DP, int NT, bool kQuarters>
void launch_attend(AttendArgs a, int max_keys, int dev, cudaStream_t st) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  a.per_tile = (kQuarters ? kAtRows / 4 : kAtRows) / a.group;
  a.pairs = (a.max_queries + NT * a.per_tile - 1) / (NT * a.per_tile);
  const int64_t items = (int64_t)a.pairs * a.sequences * a.kv_heads;
  // Keys are split over the CTAs of a cluster while that finds idle SMs and leaves each four steps.  Clusters of 16 only for a few kv heads: four of them
  // fit the GPU at once (1 x 131072 keys with 1 kv head 94 us, 177 with 8 CTAs; with 8 kv heads 208 us, 175 with 8).
  const int blocks = (max_keys + kAtKeys - 1) / kAtKeys, sms = sm_count(dev);
  a.splits = 1;
  while (a.splits < kAtMostSplits && items * a.splits * 2 <= sms && a.splits * 4 <= blocks && (a.splits < 8 || items <= 4)) a.splits *= 2;
  // Single tokens over long caches, whose lengths differ: also past one CTA per SM, while parts keep 16 steps, so that the longest cache is not what all
  // wait for (8 kv heads; 16 caches, one of 32768 keys and the others 4096 on: 330 -> 260 us, all of 32768 356 -> 373; 6 up to 16384 92 -> 63, all 100 -> 113;
  // 24 up to 16384 186 -> 168, all 350 -> 295).  Clusters of 8 for few more than the SMs: 3 up to 65536 167 -> 111, all 177 -> 194; 4 of 32768 110 -> 165.
  if (kQuarters)
    while (a.splits < 8 && 3 * items * a.splits * 2 <= (a.splits < 4 ? 9 : 4) * sms && a.splits * 32 <= blocks) a.splits *= 2;
  const int64_t ctas = items * a.splits;
  // The longest caches first where not all CTAs run at once: 64 caches up to 16384 442 -> 365 us, 32 283 -> 195; short ones lose more by it than they
  // gain (64 up to 1000 61 -> 64).
  a.longest_first = kQuarters && ctas > sms && a.sequences <= kAtMostOrdered && blocks >= 32;
  if (ctas > INT32_MAX) fail(LAYA_ERR_INVALID, "%d queries of %d sequences and %d heads are too many for one call", a.max_queries, a.sequences, a.heads);
  // The heads of a group on different banks for the rows of a warp.
  a.table_pad = a.group > 1 ? (32 - 2 * a.reach % 32 + 32 / std::min(a.group, 32)) % 32 : 0;
  const bool table_fits = a.table && (int64_t)a.group * (2ll * (a.reach + kAtKeys + kAtRows) + a.table_pad) <= kAtMostTable;
  a.by_group = FastDiv(a.group);
  a.by_splits = FastDiv(a.splits);
  a.by_kv = FastDiv(a.kv_heads);
  // Where all of a sequence's tiles see the same keys, they run one after the other and find them in the L2 cache: 64 ragged sequences up to 1024 (12 heads of
  // 64) 315 -> 280 us, with a learned bias 394 -> 345, 24 up to 4096 (8 kv heads of 128) 3179 -> 2680 when it was taken.  A causal mask wants the longest tiles of all
  // sequences first (64 x 512 128 us, 150 otherwise), a window gains nothing (314, 321).
  a.pairs_inside = !a.causal && a.left < 0 && a.right < 0 && (int64_t)a.sequences * a.kv_heads >= sms;
  a.by_inner = FastDiv(a.pairs_inside ? a.pairs : a.sequences);
  AttendMaps maps;
  maps.q = heads_map(kBf16, a.q, a.dim, a.heads, a.q_tokens, a.q_head, a.q_token, a.group, a.per_tile);
  // Without a key there is nothing to load: any map will do.
  maps.k = a.k_tokens ? heads_map(kBf16, a.k, a.dim, a.kv_heads, a.k_tokens, a.k_head, a.k_token, 1, kAtKeys) : maps.q;
  maps.v = a.k_tokens ? heads_map(kBf16, a.v, a.dim, a.kv_heads, a.k_tokens, a.v_head, a.v_token, 1, kAtKeys) : maps.q;
  const bool positive = a.scale > 0.f, capped = a.cap > 0.f;
  if (table_fits && !capped) launch_attend_kernel<T, DP, NT, kAtTable, kQuarters>(a, maps, ctas, dev, st);
  else if (a.table || !positive || (a.slopes && capped)) launch_attend_kernel<T, DP, NT, kAtGeneral, kQuarters>(a, maps, ctas, dev, st);
  else if (a.slopes) launch_attend_kernel<T, DP, NT, kAtSlopes, kQuarters>(a, maps, ctas, dev, st);
  else if (capped) launch_attend_kernel<T, DP, NT, kAtCap, kQuarters>(a, maps, ctas, dev, st);
  else launch_attend_kernel<T, DP, NT, kAtPlain, kQuarters>(a, maps, ctas, dev, st);
}

}  // namespace

extern "C" {

int laya_op_rotary(const laya_rotary* p, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  if (p->tokens < 0 || p->head_dim < 1) fail(LAYA_ERR_INVALID, "bad shape: %d tokens, heads of %d", p->tokens, p->head_dim);
  if (p->dims < 2 || p->dims % 2 || p->dims > std::min(p->head_dim, LAYA_ROTARY_MOST_DIMS))
    fail(LAYA_ERR_INVALID, "dims %d is not even and between 2 and %d", p->dims, std::min(p->head_dim, LAYA_ROTARY_MOST_DIMS));
  dtype_size(p->dtype);
  if (p->scaling < LAYA_ROTARY_NONE || p->scaling > LAYA_ROTARY_PARTS) fail(LAYA_ERR_INVALID, "unknown scaling %d", p->scaling);
  if (!(p->theta > 0) || !std::isfinite(p->theta)) fail(LAYA_ERR_INVALID, "theta must be positive");
  if (p->scaling != LAYA_ROTARY_NONE && (!(p->factor > 0) || !std::isfinite(p->factor))) fail(LAYA_ERR_INVALID, "factor must be positive");
  if (p->scaling == LAYA_ROTARY_NTK && p->dims <= 2) fail(LAYA_ERR_INVALID, "ntk scaling needs dims above 2");
  if (p->scaling == LAYA_ROTARY_PARTS && (!(p->length > 0) || !(p->low < p->high)))
    fail(LAYA_ERR_INVALID, "scaling by parts needs a length and low < high");
  RotaryArgs a = {};
  const int size = (int)dtype_size(p->dtype), wide = 16 / size;
  bool vectors = true, any = false;
  for (int i = 0; i < 2; ++i) {
    const laya_heads& h = p->part[i];
    if (h.heads < 0) fail(LAYA_ERR_INVALID, "bad shape: %d heads", h.heads);
    if (!h.heads || !p->tokens) continue;
    check_heads("x", h.x, h.x_token, h.x_head, p->dtype);
    check_heads("out", h.out, h.out_token, h.out_head, p->dtype);
    check_apart("out", p->tokens, h.heads, p->head_dim, h.out_token, h.out_head);
    const bool in_place = h.x == h.out;
    if (in_place && ((p->tokens > 1 && h.x_token != h.out_token) || (h.heads > 1 && h.x_head != h.out_head)))
      fail(LAYA_ERR_INVALID, "out is x, but with other strides");
    a.part[i] = {h.x, h.out, h.x_token, h.x_head, h.out_token, h.out_head, h.heads, !in_place};
    vectors = vectors && ((reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.out)) & 15) == 0 &&
              (h.x_token | h.x_head | h.out_token | h.out_head) % wide == 0;
    any = true;
  }
  if (!any) return LAYA_OK;
  if (!p->positions) fail(LAYA_ERR_INVALID, "positions is null");
  if (reinterpret_cast<uintptr_t>(p->positions) % (p->positions_64 ? 8 : 4)) fail(LAYA_ERR_INVALID, "positions is not aligned to its elements");
  a.positions = p->positions;
  a.positions_64 = p->positions_64;
  a.tokens = p->tokens;
  a.pairs = p->dims / 2;
  // Vectors of 16 bytes where all of a head's parts are whole ones.
  vectors = vectors && (p->interleaved ? p->dims : a.pairs) % wide == 0 && (p->head_dim - p->dims) % wide == 0;
  const int v = vectors ? wide : 1;
  a.places = p->interleaved && vectors ? p->dims / v : a.pairs / v;
  a.rest = (p->head_dim - p->dims) / v;
  if (((int64_t)a.part[0].heads + a.part[1].heads) * std::max(1, a.rest) > INT32_MAX / 2)
    fail(LAYA_ERR_INVALID, "%d and %d heads of %d are too many for one call", a.part[0].heads, a.part[1].heads, p->head_dim);
  a.abreast = std::max(1, 32 / a.places);
  a.by_places = FastDiv(a.places);
  a.by_rest = FastDiv(std::max(1, a.rest));
  a.sine_sign = p->backward ? -1.f : 1.f;
  a.magnitude = p->magnitude;
  constexpr double kTurn = 6.283185307179586;
  const double theta = p->theta * (p->scaling == LAYA_ROTARY_NTK ? std::pow(p->factor, p->dims / (p->dims - 2.0)) : 1.0);
  if (!(theta > 0) || !std::isfinite(theta)) fail(LAYA_ERR_INVALID, "factor %g takes theta %g out of range", p->factor, p->theta);
  a.step = -2.0 / p->dims * std::log2(theta);
  a.power = -std::log2(p->scaling == LAYA_ROTARY_LINEAR ? kTurn * p->factor : kTurn);
  a.by_parts = p->scaling == LAYA_ROTARY_PARTS;
  if (a.by_parts) {
    a.above = p->length / (p->high - p->low);
    a.below = p->low / (p->high - p->low);
    a.shrink = 1.0 / p->factor;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(current_device(st));
  // A warp per token, more while the warps do not fill the SMs and a token has heads for them.
  const int rounds = (int)(((int64_t)a.part[0].heads + a.part[1].heads + a.abreast - 1) / a.abreast);
  a.shares = 1;
  while (a.shares < rounds && (int64_t)a.tokens * a.shares * 2 <= 16ll * sms) a.shares *= 2;
  a.by_shares = FastDiv(a.shares);
  const int64_t warps = (int64_t)a.tokens * a.shares;  // at most 2^31 - 1: several to a token only where tokens are few
  const dim3 grid((unsigned)((warps + kRotaryThreads / 32 - 1) / (kRotaryThreads / 32)));
  with_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int V = 16 / sizeof(T);
    auto kern = vectors ? (p->interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>)
                        : (p->interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
    launch_k(kern, grid, dim3(kRotaryThreads), 0, st, a);
  });
  OP_API_END
}

int laya_op_attend(const laya_attend* p, int* err, void* stream) {
  OP_API_BEGIN
  if (!p) fail(LAYA_ERR_INVALID, "null argument");
  if (p->sequences < 0 || p->sequences > 65535 || p->q_tokens < 0 || p->k_tokens < 0 || p->max_queries < 0 || p->max_keys < 0)
    fail(LAYA_ERR_INVALID, "bad shape: %d sequences (65535 at most), %d and %d tokens, at most %d and %d of a sequence", p->sequences,
         p->q_tokens, p->k_tokens, p->max_queries, p->max_keys);
  // Positions and steps of keys past the last one are counted in 32 bits.
  constexpr int kMost = INT32_MAX - 255;
  if (p->q_tokens > kMost || p->k_tokens > kMost) fail(LAYA_ERR_INVALID, "%d and %d tokens: at most %d", p->q_tokens, p->k_tokens, kMost);
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads / p->kv_heads > 128 || p->heads > 65535)
    fail(LAYA_ERR_INVALID, "%d heads over %d kv heads: a multiple of at most 128 times", p->heads, p->kv_heads);
  if (p->head_dim < 8 || p->head_dim > kAttendMostDim || p->head_dim % 8)
    fail(LAYA_ERR_INVALID, "heads of %d values: a multiple of 8 up to %d", p->head_dim, kAttendMostDim);
  if (p->dtype != LAYA_DTYPE_F16 && p->dtype != LAYA_DTYPE_BF16) fail(LAYA_ERR_INVALID, "dtype %d is not F16 or BF16", p->dtype);
  if (!std::isfinite(p->scale)) fail(LAYA_ERR_INVALID, "scale must be finite");
  if (!(p->cap >= 0.f) || !std::isfinite(p->cap)) fail(LAYA_ERR_INVALID, "cap must be at least 0");
  if (p->window_left < -1 || p->window_right < -1) fail(LAYA_ERR_INVALID, "window bounds must be at least 0, or -1 for none");
  if (p->slopes && p->distance_bias) fail(LAYA_ERR_INVALID, "slopes and distance_bias cannot both be given");
  // (Twice the reach and a step to either side of it are counted in 32 bits.)
  constexpr int kMostReach = (1 << 30) - 1024;
  if (p->distance_bias && (p->reach < 0 || p->reach > kMostReach)) fail(LAYA_ERR_INVALID, "reach %d must be at least 0 and at most %d", p->reach, kMostReach);
  if (!p->documents != !p->k_documents) fail(LAYA_ERR_INVALID, "documents and k_documents go together");
  if (!p->k_starts != !p->k_lengths) fail(LAYA_ERR_INVALID, "k_starts and k_lengths go together");
  if (!p->sequences || !p->q_tokens || !p->max_queries) return LAYA_OK;
  if (!p->starts || !p->lengths) fail(LAYA_ERR_INVALID, "starts or lengths is null");
  const struct { const char* name; const void* p; } vectors[] = {
      {"starts", p->starts}, {"lengths", p->lengths}, {"k_starts", p->k_starts}, {"k_lengths", p->k_lengths}, {"prefix", p->prefix}, {"documents", p->documents},
      {"k_documents", p->k_documents}, {"slopes", p->slopes}, {"distance_bias", p->distance_bias}, {"lse", p->lse}, {"err", err}};
  for (const auto& v : vectors)
    if (reinterpret_cast<uintptr_t>(v.p) % 4) fail(LAYA_ERR_INVALID, "%s is not aligned to its elements", v.name);
  AttendArgs a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.lse = p->lse;
  a.q_token = p->q_token; a.q_head = p->q_head; a.k_token = p->k_token; a.k_head = p->k_head;
  a.v_token = p->v_token; a.v_head = p->v_head; a.out_token = p->out_token; a.out_head = p->out_head;
  check_vectors("q", p->q, p->q_tokens, p->heads, p->head_dim, &a.q_token, &a.q_head, p->dtype, false);
  check_vectors("out", p->out, p->q_tokens, p->heads, p->head_dim, &a.out_token, &a.out_head, p->dtype, true);
  if (p->k_tokens) {
    check_vectors("k", p->k, p->k_tokens, p->kv_heads, p->head_dim, &a.k_token, &a.k_head, p->dtype, false);
    check_vectors("v", p->v, p->k_tokens, p->kv_heads, p->head_dim, &a.v_token, &a.v_head, p->dtype, false);
  }
  a.starts = p->starts; a.lengths = p->lengths;
  a.k_starts = p->k_starts ? p->k_starts : p->starts;
  a.k_lengths = p->k_lengths ? p->k_lengths : p->lengths;
  a.sequences = p->sequences; a.heads = p->heads; a.kv_heads = p->kv_heads; a.group = p->heads / p->kv_heads; a.dim = p->head_dim;
  a.q_tokens = p->q_tokens; a.k_tokens = p->k_tokens; a.max_queries = std::min(p->max_queries, p->q_tokens);
  a.scale = p->scale; a.cap = p->cap; a.causal = p->causal; a.left = p->window_left; a.right = p->window_right;
  a.prefix = p->prefix; a.documents = p->documents; a.k_documents = p->k_documents;
  a.slopes = p->slopes; a.table = p->distance_bias; a.reach = p->reach;
  a.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  current_device(st);
  a.wait_ns = wait_ns();
  with_half(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int dev = current_device(st), max_keys = std::min(p->max_keys, p->k_tokens);
    // All rows of a sequence's kv head in a quarter of a tile: single tokens, and a few where the group is small.
    const bool quarters = (int64_t)a.max_queries * a.group <= kAtRows / 4;
    if (a.dim > 64 && quarters) launch_attend<T, 128, 2, true>(a, max_keys, dev, st);
    else if (a.dim > 64) launch_attend<T, 128, 2, false>(a, max_keys, dev, st);
    else if (quarters) launch_attend<T, 64, 2, true>(a, max_keys, dev, st);
    else launch_attend<T, 64, 1, false>(a, max_keys, dev, st);
  });
  OP_API_END
}

}  // extern "C"
