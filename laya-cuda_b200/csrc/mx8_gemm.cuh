// tcgen05 products of MX8 matrices (tcgen05.mma kind::mxf8f6f4 with block scales in tensor memory)
// with the layer's epilogue (mx8_linear.cuh).
//
// Operands are K-major E4M3 tiles of 128 columns (128-byte swizzle, four MMAs of K = 32 each), read by
// TMA; the scale tiles of mx8.cuh travel beside them (512 bytes per 128 rows) and are copied into
// tensor memory by tcgen05.cp (32 lanes x 16 bytes, repeated for the four lane quarters), where an
// MMA takes byte k of each 32-bit column for its k-th block of 32.  No copy is multicast.
#pragma once
#include "mx8_linear.cuh"

namespace laya {

constexpr int kMxBK = 128;                 // columns of K per stage, one scale tile
constexpr int kMxOperandBytes = 128 * kMxBK;

// mbar_wait for a converged warp, with the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code, volatile int* abort,
                                          unsigned long long limit_ns) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const unsigned long long start = global_ns();
  for (;;) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool given_up = *abort != 0, late = global_ns() - start > limit_ns;
    if (__any_sync(0xffffffffu, given_up || late)) {
      if (late && !given_up) {
        *abort = 1;
        if (err) atomicCAS(err, 0, code);
      }
      __syncwarp();
      return false;
    }
  }
}

// The two halves of cluster_sync: arrive (releasing what this thread wrote), and wait for all to have.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// tc_commit_pair onto the barrier at the same offset in both CTAs of the pair.
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

struct MxMaps {
  CUtensorMap x, xs, w, ws, g, gs;  // values {128 columns, rows}, scales {512 bytes, 1, tiles}; g, gs: gated only
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y,
                                                 int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Instruction descriptor of kind::mxf8f6f4: E4M3 operands, both K-major, E8M0 scales; `k` selects
// the byte of the scale columns.
__host__ __device__ constexpr uint32_t mx_idesc(int M, int N, int k) {
  return ((uint32_t)k << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) | ((uint32_t)k << 29);
}

// Shared-memory descriptor of a scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <bool kPair>
__device__ __forceinline__ void mx_copy_scales(uint32_t taddr, uint64_t d) {
  if (kPair) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

template <bool kPair>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                       uint32_t b_scales, uint32_t accumulate) {
  if (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scales), "r"(b_scales)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scales), "r"(b_scales)
        : "memory");
}

// ---------------------------------------------------------------------------------------------
// Many rows: CTA pairs (cta_group::2), 256 x BN output tiles, persistent.  Each CTA holds its
// 128 rows of X, half of the tile's rows of W (gated: rank 0 the rows of G and rank 1 those of W, the
// tile's output being 256 x BN / 2), its X scales and all of the tile's weight scales.
//
// Warps: 0 TMA producer, 1 tensor-memory allocator and (in the leader) MMA issuer, 2..9 epilogue (two
// per lane quarter, each with half of the columns).  Tensor memory: two accumulators, so that the
// epilogue of a tile overlaps the next tile's MMAs, and scale columns.  With BN = 256
// the accumulators take 2 x 256 of the 512 columns and would leave none for the scales, so they
// share 32 columns, [224, 256): the epilogue reads those first and the next tile's MMAs wait for
// that (barrier `shared`) instead of for half of the tile's columns.
//
// A k-tile's MMAs take 512 cycles with BN = 256 (the tensor core's rate for 8-bit operands) and its stage's
// copies arrive in less, so the MMAs run back to back but for some 900 cycles from one tile to the next.
// 16384 x 4096 x 4096 with a bf16 residual: 192-213 us (2.6-2.9 PFLOP/s), 244 us when it runs for seconds (the card then draws its
// 990 W and the clock falls to 1.15 GHz); 8192 x 2048 x 2 x 5632 gated into MX8: 128-135 us, 155 for seconds.
// Sixteen epilogue warps instead of eight: slower (96 registers each; 46 us for 34 with K = 64).
//
// Barriers as in gemm_pair_kernel: full[s] in the leader (both CTAs' copies), empty[s] and
// tfull[a] in both (committed by the leader), tempty[a] and shared in the leader.
// ---------------------------------------------------------------------------------------------
constexpr int kMxThreadsPair = 320;
constexpr int kMxEpiWarps = 8;
constexpr int kMxEpiBytes = kMxEpiWarps * 4096;

template <int BN>
struct MxPairCfg {
  static constexpr int kStageB = BN / 2 * kMxBK;
  static constexpr int kWeightTiles = (BN + 127) / 128;  // scale tiles of the weight rows
  static constexpr int kStageScales = (1 + kWeightTiles) * kMxTileBytes;
  static constexpr int kStageBytes = kMxOperandBytes + kStageB + kStageScales;
  static constexpr int kStages = (196 * 1024 - 1024) / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + kMxEpiBytes + 1024 /*align*/ + 512 /*barriers*/;
  static constexpr uint32_t kAcc1 = BN == 256 ? 224 : BN;  // column of the second accumulator
  static constexpr bool kShared = kAcc1 < BN;
  // Scale columns: a set per stage where there is room, so that a stage's are free when it is filled
  // again; else two, and a set is waited for.
  static constexpr int kSetCols = 4 + 4 * kWeightTiles;
  static constexpr bool kSetPerStage = kAcc1 + BN + kStages * kSetCols <= 512;
  static constexpr int kSets = kSetPerStage ? kStages : 2;
  static constexpr uint32_t kScales = 512 - kSets * ((kSetCols + 7) & ~7);
  static constexpr int kSetStride = (kSetCols + 7) & ~7;
  static_assert(kAcc1 + BN <= kScales, "accumulators and scale columns overlap");
};

template <int BN, bool kGated, int kRes>
__global__ void __launch_bounds__(kMxThreadsPair, 1)
    mx8_linear_pair_kernel(const __grid_constant__ MxMaps maps, const __grid_constant__ MxLinearArgs args) {
  using Cfg = MxPairCfg<BN>;
  static_assert(!kGated || BN == 256, "gated tiles pair 128 rows of G with 128 of W");
  constexpr int S = Cfg::kStages;
  constexpr int kOutCols = kGated ? BN / 2 : BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * kMxOperandBytes;
  uint8_t* epi = sB + S * Cfg::kStageB;
  uint8_t* sS = epi + kMxEpiBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sS + S * Cfg::kStageScales);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* tfull = bars + 2 * S;
  uint64_t* tempty = bars + 2 * S + 2;
  uint64_t* shared = bars + 2 * S + 4;
  uint64_t* drain = bars + 2 * S + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* issued_blocks = abort_flag + 1;  // [2]: k-blocks whose copies each CTA of the pair issued
  const unsigned long long wait_ns = wait_limit(args.wait_ns);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  const int m_blocks = (args.M + 255) / 256;
  const int n_blocks = (args.N + kOutCols - 1) / kOutCols;
  const int k_blocks = mx_col_tiles(args.K);
  const int tiles = m_blocks * n_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 2 * kMxEpiWarps); }
    mbar_init(shared, kMxEpiWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    issued_blocks[0] = issued_blocks[1] = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.x); tma_prefetch_desc(&maps.xs);
    tma_prefetch_desc(&maps.w); tma_prefetch_desc(&maps.ws);
    if (kGated) { tma_prefetch_desc(&maps.g); tma_prefetch_desc(&maps.gs); }
  }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised before any cross-CTA arrival
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    int stage = 0; uint32_t phase = 0;
    uint32_t issued = 0, last_par = 0;
    int count = 0;
    bool ok = true;
    const CUtensorMap* wmap = kGated && leader ? &maps.g : &maps.w;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int mb = t / n_blocks, nb = t - mb * n_blocks;
      const int arow = mb * 256 + (int)rank * 128;
      const int brow = kGated ? nb * 128 : nb * BN + (int)rank * (BN / 2);
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!warp_wait(&empty[stage], phase ^ 1, args.err, kErrGemmProducerWait, abort_flag, wait_ns)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t bar = cluster_addr(smem_u32(&full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::kStageBytes);
          uint8_t* sc = sS + stage * Cfg::kStageScales;
          tma_load_2d_pair(sA + stage * kMxOperandBytes, &maps.x, bar, kb * kMxBK, arow);
          tma_load_2d_pair(sB + stage * Cfg::kStageB, wmap, bar, kb * kMxBK, brow);
          tma_load_3d_pair(sc, &maps.xs, bar, 0, kb, arow / 128);
          if (kGated) {
            tma_load_3d_pair(sc + kMxTileBytes, &maps.gs, bar, 0, kb, nb);
            tma_load_3d_pair(sc + 2 * kMxTileBytes, &maps.ws, bar, 0, kb, nb);
          } else {
            tma_load_3d_pair(sc + kMxTileBytes, &maps.ws, bar, 0, kb, nb * Cfg::kWeightTiles);
          }
        }
        ++count;
        issued |= 1u << stage;
        last_par = (last_par & ~(1u << stage)) | (phase << stage);
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
    }
    if (lane == 0) {
      if (leader) {
        // Both CTAs' copies complete on the leader's full barriers: wait for them by time only, on
        // every path, so that nothing is still landing when the pair exits.
        for (int s = 0; s < S; ++s)
          if (issued & (1u << s)) mbar_drain(&full[s], (last_par >> s) & 1);
      }
      issued_blocks[rank] = count;
      const uint32_t there = cluster_addr(smem_u32(const_cast<int*>(issued_blocks + rank)), rank ^ 1);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(count) : "memory");
    }
  } else if (warp == 1) {
    if (leader) {
      const uint64_t adesc = smem_desc_sw128(smem_u32(sA)), bdesc = smem_desc_sw128(smem_u32(sB));
      const uint64_t sdesc = mx_scale_desc(smem_u32(sS));
      int stage = 0; uint32_t phase = 0;
      int set = 0;
      bool ok = true;
      int i = 0;  // this pair's tile
      int done_stage = 0; uint32_t done_phase = 0;  // the k-block two before the current one
      int blocks = 0;
      for (int t = pair; t < tiles && ok; t += pairs, ++i) {
        const int acc = i & 1;
        const uint32_t d = tmem + (acc ? Cfg::kAcc1 : 0);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!warp_wait(&full[stage], phase, args.err, kErrGemmMmaWait, abort_flag, wait_ns)) { ok = false; break; }
          // The scale columns of this set were last read by the MMAs two k-blocks ago.
          if (!Cfg::kSetPerStage && blocks >= 2) {
            if (!warp_wait(&empty[done_stage], done_phase, args.err, kErrGemmMmaWait, abort_flag, wait_ns)) { ok = false; break; }
            if (++done_stage == S) { done_stage = 0; done_phase ^= 1; }
          }
          ++blocks;
          tc_fence_after();
          const uint32_t ts = tmem + Cfg::kScales + (Cfg::kSetPerStage ? stage : set) * Cfg::kSetStride;
          auto copy_scales = [&] {
            const uint64_t sc = sdesc + (uint64_t)(stage * (Cfg::kStageScales >> 4));
            mx_copy_scales<true>(ts, sc);
#pragma unroll
            for (int j = 0; j < Cfg::kWeightTiles; ++j) mx_copy_scales<true>(ts + 4 + 4 * j, sc + (1 + j) * (kMxTileBytes >> 4));
          };
          if (kb == 0) {
            // The accumulator is waited for last: its columns are free about 500 cycles after the previous tile's
            // MMAs (commit, epilogue's first read, arrival), and all else is ready then.
            if (elect_one()) copy_scales();
            __syncwarp();
            if (!warp_wait(&tempty[acc], ((i >> 1) & 1) ^ 1, args.err, kErrGemmMmaWait, abort_flag, wait_ns)) { ok = false; break; }
            if (Cfg::kShared && i > 0 && !warp_wait(shared, (i - 1) & 1, args.err, kErrGemmMmaWait, abort_flag, wait_ns)) { ok = false; break; }
            tc_fence_after();
          }
          if (elect_one()) {
            if (kb > 0) copy_scales();
            const uint64_t a = adesc + (uint64_t)(stage * (kMxOperandBytes >> 4));
            const uint64_t b = bdesc + (uint64_t)(stage * (Cfg::kStageB >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx_mma<true>(d, a + 2 * k, b + 2 * k, mx_idesc(256, BN, k), ts, ts + 4, (kb > 0 || k > 0) ? 1u : 0u);
            tc_commit_both(&empty[stage]);
            if (kb == k_blocks - 1) tc_commit_both(&tfull[acc]);
          }
          __syncwarp();
          set ^= 1;
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (elect_one()) {
        tc_commit_pair(cluster_addr(smem_u32(drain), 0));
        mbar_drain(drain, 0);
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = epi + (warp - 2) * 4096;
    const uint32_t bar_shared = cluster_addr(smem_u32(shared), 0);
    constexpr int kChunks = kOutCols / 64;  // 32-column chunks of this warp
    // The shared columns are the second half's last of accumulator 0 and the first half's first of
    // accumulator 1: outwards in, so that they are read first.
    auto chunk = [&](int j) { return half ? 2 * kChunks - 1 - j : j; };
    struct Tile {
      int row, col;  // this lane's row, the tile's first column
    };
    auto tile_at = [&](int t) {
      const int mb = t / n_blocks, nb = t - mb * n_blocks;
      return Tile{mb * 256 + (int)rank * 128 + quarter * 32 + lane, nb * kOutCols};
    };
    // The residual is loaded kDepth chunks ahead of its use, over tiles' ends too, and brought into L2 a tile
    // ahead.  (One chunk ahead, a chunk waits 1,000 to 1,700 cycles for it.)
    constexpr int kDepth =
        kRes == MX_RES_HALF || (!kGated && (kRes == MX_RES_FULL || kRes == MX_RES_ANY_HALF)) ? 2 : 1;
    MxResidualRow<kRes> in[kDepth];
    auto prefetch = [&](const Tile& t) {
      if constexpr (kRes != MX_RES_NONE) {
        constexpr int kSize = mx_res_size(kRes);
        const int c0 = t.col + half * kChunks * 32;
        const char* p = static_cast<const char*>(args.residual) + ((size_t)t.row * args.ldr + c0) * kSize;
        if (t.row < args.M) {
#pragma unroll
          for (int j = 0; j < kChunks * kSize / 2; ++j)  // 64 bytes each
            if (c0 + j * (64 / kSize) < args.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + 64 * j));
        }
      }
    };
    int i = 0;
    Tile now = tile_at(pair);
    if (pair < tiles) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) mx_fetch_row<kRes>(args, now.row, now.col + chunk(d) * 32, in[d]);
      prefetch(now);
    }
    for (int t = pair; t < tiles; t += pairs, ++i) {
      const int acc = i & 1;
      const bool more = t + pairs < tiles;
      const Tile next = more ? tile_at(t + pairs) : now;
      if (more) prefetch(next);
      if (!warp_wait(&tfull[acc], (i >> 1) & 1, args.err, kErrGemmEpilogueWait, abort_flag, wait_ns)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + (acc ? Cfg::kAcc1 : 0);
      uint32_t scales = 0;  // MX8: this row's scale bytes of the warp's chunks
#pragma unroll 1
      for (int j0 = 0; j0 < kChunks; j0 += kDepth) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
          const int j = j0 + d, c = chunk(j);
          uint32_t r[32], u[kGated ? 32 : 1];
          tmem_ld32_async(tbase + c * 32, r);
          if constexpr (kGated) {
            tmem_ld32_async(tbase + 128 + c * 32, u);
            tmem_wait_ld(u);
          }
          tmem_wait_ld(r);
          if (j == 0 && Cfg::kShared && half != acc) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(bar_shared);
          }
          if (j == kChunks - 1) {
            // The accumulator has been read; the stores that follow need no ordering with the next MMAs.
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(cluster_addr(smem_u32(&tempty[acc]), 0));
          }
          float v[32], g[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            v[k] = __uint_as_float(kGated ? u[kGated ? k : 0] : r[k]);
            if (kGated) g[k] = __uint_as_float(r[k]);
          }
          const uint32_t byte = mx_finish_row<kGated, kRes>(args, now.row, now.col + c * 32, v, g, in[d], buf);
          scales |= byte << (8 * (c & 3));
          const bool here = j + kDepth < kChunks;
          if (kRes != MX_RES_NONE && (here || more)) {
            const Tile& at = here ? now : next;
            mx_fetch_row<kRes>(args, at.row, at.col + chunk(here ? j + kDepth : j + kDepth - kChunks) * 32, in[d]);
          }
        }
      }
      if (args.out_type == MX_MX8 && now.row < args.M) {
        // Four chunks are a scale tile's four blocks, two its first or last two.
        const int col = now.col + half * kChunks * 32, col_tiles = mx_col_tiles(args.N), tile = col / kMxTileCols;
        uint8_t* p = args.out_scales + mx_scale_tile(now.row, tile, col_tiles) + mx_scale_row(now.row);
        if (tile < col_tiles) {
          if (kChunks == 4) *reinterpret_cast<uint32_t*>(p) = scales;
          else reinterpret_cast<uint16_t*>(p)[(col / 64) & 1] = (uint16_t)(scales >> (col & 64 ? 16 : 0));
        }
      }
      now = next;
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();  // both CTAs done with tensor memory and with the peer's barriers
  tc_fence_after();
  if (issued_blocks[0] != issued_blocks[1]) {
    // One CTA gave up on a wait before the other.  Copies that the peer issued for stages the
    // leader never armed still land on the leader's barriers: arm those and wait (by time only).
    if (leader && threadIdx.x == 0)
      for (int b = issued_blocks[0]; b < issued_blocks[1]; ++b) {
        mbar_arrive_expect_tx(&full[b % S], Cfg::kStageBytes);
        mbar_drain(&full[b % S], (b / S) & 1);
      }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------------------------------------
// Few rows: the weights are the 128-row operand and the tokens the BN-column one, so a tile is 128
// features x BN rows of X and reads each weight byte once.  The K tiles are split over the CTAs of a
// cluster (as many as keep the SMs busy); each CTA leaves its partial sums in shared memory, and
// every CTA adds and finishes its share of the rows from all of them in rank order, so the result
// does not depend on timing.  What bounds it is the chain of latencies from the launch to the last
// store: one row, 4096 x 4096, takes 5.4 us, of which its 17 MB would be 2.6 from HBM.
//
// One thread issues a k-block (wait, 2 scale copies, 4 MMAs, commit) in about 320 cycles whatever BN is, longer
// than its MMAs take, so two warps issue, each into an accumulator of its own: not gated, k-blocks in
// turn (the accumulators are added when they are read); gated, one the products with W and one
// those with G.  Likewise two warps load: k-blocks in turn, or W and its scales / G and X.
//
// Warps: 0..3 read tensor memory, 4 and 7 TMA producers, 5 and 6 MMA issuers (5 allocates tensor
// memory); all eight finish rows.
// ---------------------------------------------------------------------------------------------
constexpr int kMxThreadsFew = 256;
constexpr int kMxMaxSplit = 4;

template <int BN, bool kGated>
struct MxFewCfg {
  static constexpr int kWeights = kGated ? 2 : 1;
  static constexpr int kStageB = BN * kMxBK;
  static constexpr int kStageScales = (kWeights + 1) * kMxTileBytes;
  static constexpr int kStageBytes = kWeights * kMxOperandBytes + kStageB + kStageScales;
  // Not gated: as many stages as leave room for two CTAs per SM (64 x 4096 x 4096: 6.8 us, with twice the
  // stages and one CTA 8.2), an even number of them, so that a stage always belongs to the same producer and
  // issuer.  Gated stages are larger, and two of them too few (64 x 4096 x 2 x 4096: 12.9 us, with four 11.4).
  static constexpr int kStages = kGated ? 200 * 1024 / kStageBytes : 111 * 1024 / kStageBytes & ~1;
  static constexpr int kPartialBytes = kWeights * BN * 128 * 4;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 /*align*/ + 256 /*barriers*/;
  // Tensor memory: two accumulators, then each stage's scale columns (weights' 4 and X's 4, for each issuer of the stage).
  static constexpr int kScales = 2 * BN;
  static constexpr int kScaleCols = 8 * kWeights;
  static constexpr int kUsedCols = kScales + kStages * kScaleCols;
  static constexpr int kTmemCols = kUsedCols <= 64 ? 64 : kUsedCols <= 128 ? 128 : 256;
  static_assert(kUsedCols <= 256, "two CTAs share an SM's tensor memory");
  static_assert(kPartialBytes <= kStages * kStageBytes, "partial sums reuse the stages");
};

template <int BN, bool kGated>
__global__ void __launch_bounds__(kMxThreadsFew, kGated ? 1 : 2)
    mx8_linear_few_kernel(const __grid_constant__ MxMaps maps, const __grid_constant__ MxLinearArgs args) {
  using Cfg = MxFewCfg<BN, kGated>;
  constexpr int S = Cfg::kStages;
  constexpr int W = Cfg::kWeights;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S * W * kMxOperandBytes;
  uint8_t* sS = sB + S * Cfg::kStageB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sS + S * Cfg::kStageScales);
  uint64_t* full = bars;
  uint64_t* empty = bars + S;
  uint64_t* tfull = bars + 2 * S;
  uint64_t* drain = bars + 2 * S + 1;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* partial = reinterpret_cast<float*>(smem);  // [W][BN][128], over the stages once they are consumed
  const unsigned long long wait_ns = wait_limit(args.wait_ns);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int split = (int)gridDim.z, rank = (int)cluster_rank();
  const int f0 = blockIdx.x * 128, t0 = blockIdx.y * BN;
  const int k_tiles = mx_col_tiles(args.K);
  const int kb0 = (int)((int64_t)k_tiles * rank / split), kb1 = (int)((int64_t)k_tiles * (rank + 1) / split);
  const int k_blocks = kb1 - kb0;  // at least 1: split <= k_tiles
  const int issuers = kGated || k_blocks > 1 ? 2 : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) { mbar_init(&full[s], W); mbar_init(&empty[s], W); }
    mbar_init(tfull, issuers);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 4 && lane == 0) { tma_prefetch_desc(&maps.w); tma_prefetch_desc(&maps.ws); }
  if (warp == 7 && lane == 0) {
    tma_prefetch_desc(&maps.x); tma_prefetch_desc(&maps.xs);
    if (kGated) { tma_prefetch_desc(&maps.g); tma_prefetch_desc(&maps.gs); }
  }
  if (warp == 5) { tmem_alloc(tmem_slot, Cfg::kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 4 || warp == 7) {
    const int who = warp == 4 ? 0 : 1;
    uint32_t issued = 0, last_par = 0;
    for (int b = kGated ? 0 : who; b < k_blocks; b += kGated ? 1 : 2) {
      const int stage = b % S; const uint32_t phase = (b / S) & 1;
      if (!warp_wait(&empty[stage], phase ^ 1, args.err, kErrGemmProducerWait, abort_flag, wait_ns)) break;
      if (elect_one()) {
        const int kb = kb0 + b;
        uint8_t* a = sA + stage * W * kMxOperandBytes;
        uint8_t* sc = sS + stage * Cfg::kStageScales;
        if (!kGated || who == 0) {
          mbar_arrive_expect_tx(&full[stage], kGated ? kMxOperandBytes + 2 * kMxTileBytes : Cfg::kStageBytes);
          tma_load_2d(a, &maps.w, &full[stage], kb * kMxBK, f0);
          tma_load_3d(sc, &maps.ws, &full[stage], 0, kb, f0 / 128);
          tma_load_3d(sc + W * kMxTileBytes, &maps.xs, &full[stage], 0, kb, t0 / 128);
        }
        if (kGated && who == 1) {
          mbar_arrive_expect_tx(&full[stage], kMxOperandBytes + kMxTileBytes + Cfg::kStageB);
          tma_load_2d(a + kMxOperandBytes, &maps.g, &full[stage], kb * kMxBK, f0);
          tma_load_3d(sc + kMxTileBytes, &maps.gs, &full[stage], 0, kb, f0 / 128);
        }
        if (!kGated || who == 1) tma_load_2d(sB + stage * Cfg::kStageB, &maps.x, &full[stage], kb * kMxBK, t0);
      }
      issued |= 1u << stage;
      last_par = (last_par & ~(1u << stage)) | (phase << stage);
    }
    if (lane == 0)
      for (int s = 0; s < S; ++s)
        if (issued & (1u << s)) mbar_drain(&full[s], (last_par >> s) & 1);
  } else if (warp == 5 || warp == 6) {
    const int who = warp - 5;
    const uint64_t adesc = smem_desc_sw128(smem_u32(sA) + (kGated ? who * kMxOperandBytes : 0));
    const uint64_t bdesc = smem_desc_sw128(smem_u32(sB));
    const uint64_t sdesc = mx_scale_desc(smem_u32(sS));
    const uint32_t d = tmem + who * BN;
    const int first = kGated ? 0 : who, step = kGated ? 1 : 2;
    for (int b = first; b < k_blocks; b += step) {
      const int stage = b % S;
      if (!warp_wait(&full[stage], (b / S) & 1, args.err, kErrGemmMmaWait, abort_flag, wait_ns)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = adesc + (uint64_t)(stage * W * (kMxOperandBytes >> 4));
        const uint64_t x = bdesc + (uint64_t)(stage * (Cfg::kStageB >> 4));
        const uint64_t sc = sdesc + (uint64_t)(stage * (Cfg::kStageScales >> 4));
        // The stage's own scale columns: its last MMAs were done before it was filled again.
        const uint32_t ts = tmem + Cfg::kScales + stage * Cfg::kScaleCols + (kGated ? 8 * who : 0);
        mx_copy_scales<false>(ts, sc + (kGated ? who * (kMxTileBytes >> 4) : 0));
        mx_copy_scales<false>(ts + 4, sc + W * (kMxTileBytes >> 4));
        // Tokens t0 .. t0 + BN - 1 are the lanes from column (t0 % 128) / 32 of their scale tile on.
        const uint32_t xs = ts + 4 + (t0 % 128) / 32;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mx_mma<false>(d, a + 2 * k, x + 2 * k, mx_idesc(128, BN, k), ts, xs, (b > first || k > 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
        if (b + step >= k_blocks) tc_commit(tfull);
      }
      __syncwarp();
    }
    if (elect_one()) {
      tc_commit(&drain[who]);
      mbar_drain(&drain[who], 0);
    }
  } else {
    // This CTA's sums: lane = feature, columns = rows of X.
    if (warp_wait(tfull, 0, args.err, kErrGemmEpilogueWait, abort_flag, wait_ns)) {
      tc_fence_after();
      const uint32_t tbase = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll
      for (int c = 0; c < BN / 16; ++c) {
        float v[16], u[16];
        tmem_ld16x2(tbase + c * 16, tbase + (issuers > 1 ? BN : 0) + c * 16, v, u);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float* p = partial + (c * 16 + i) * 128 + warp * 32 + lane;
          if (kGated) {
            p[0] = v[i];
            p[BN * 128] = u[i];
          } else {
            p[0] = issuers > 1 ? v[i] + u[i] : v[i];
          }
        }
      }
      tc_fence_before();
    }
  }
  // Rows of X are dealt to the cluster's warps, which finish R at a time.  The loads of a turn are in flight
  // together, and the first turn's inputs are loaded between the arrival at the barrier that follows the
  // sums and the wait for it.
  const int rows = min(BN, args.M - t0), step = 8 * split, col = f0 + 4 * lane;
  int t = rank * 8 + warp;
  auto whole = [&](int r) { return f0 + 128 <= args.N && t + (r - 1) * step < rows; };
  cluster_arrive();  // this CTA's sums are in its shared memory
  if (split == 1) {
    constexpr int R = kGated ? 4 : 8;
    MxInputs<R> in;
    mx_fetch<kGated, R>(args, t0 + t, step, t0 + rows, col, whole(R), in);
    cluster_wait();
    for (; t < rows; t += R * step) {
      float v[R][4], g[R][4];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float* p = partial + min(t + k * step, BN - 1) * 128 + 4 * lane;
        const float4 s = *reinterpret_cast<const float4*>(p);
        v[k][0] = s.x; v[k][1] = s.y; v[k][2] = s.z; v[k][3] = s.w;
        if constexpr (kGated) {
          const float4 u = *reinterpret_cast<const float4*>(p + BN * 128);
          g[k][0] = u.x; g[k][1] = u.y; g[k][2] = u.z; g[k][3] = u.w;
        }
      }
      mx_finish<kGated, R>(args, t0 + t, step, t0 + rows, col, v, g, in);
      if (t + R * step < rows) {
        t += R * step;
        mx_fetch<kGated, R>(args, t0 + t, step, t0 + rows, col, whole(R), in);
        t -= R * step;
      }
    }
  } else {
    constexpr int R = kGated ? 1 : 2;
    MxInputs<R> in;
    mx_fetch<kGated, R>(args, t0 + t, step, t0 + rows, col, whole(R), in);
    cluster_wait();
    const uint32_t mine = smem_u32(partial) + lane * 16;
    bool read = t >= rows;
    if (read) cluster_arrive();
    for (; t < rows; t += R * step) {
      float4 s[R][kMxMaxSplit], u[kGated ? R : 1][kMxMaxSplit];
#pragma unroll
      for (int r = 0; r < kMxMaxSplit; ++r) {
        if (r >= split) break;
        const uint32_t there = cluster_addr(mine, r);
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const uint32_t at = there + min(t + k * step, BN - 1) * 512;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(s[k][r].x), "=f"(s[k][r].y), "=f"(s[k][r].z), "=f"(s[k][r].w) : "r"(at));
          if constexpr (kGated)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(u[k][r].x), "=f"(u[k][r].y), "=f"(u[k][r].z), "=f"(u[k][r].w) : "r"(at + BN * 512));
        }
      }
      float v[R][4] = {}, g[R][4] = {};
#pragma unroll
      for (int r = 0; r < kMxMaxSplit; ++r) {
        if (r >= split) break;
#pragma unroll
        for (int k = 0; k < R; ++k) {
          v[k][0] += s[k][r].x; v[k][1] += s[k][r].y; v[k][2] += s[k][r].z; v[k][3] += s[k][r].w;
          if constexpr (kGated) {
            g[k][0] += u[k][r].x; g[k][1] += u[k][r].y; g[k][2] += u[k][r].z; g[k][3] += u[k][r].w;
          }
        }
      }
      const bool last = t + R * step >= rows;
      if (last) cluster_arrive();  // this warp has read the other CTAs' sums
      mx_finish<kGated, R>(args, t0 + t, step, t0 + rows, col, v, g, in);
      if (!last) {
        t += R * step;
        mx_fetch<kGated, R>(args, t0 + t, step, t0 + rows, col, whole(R), in);
        t -= R * step;
      }
    }
    cluster_wait();  // no CTA leaves while its sums are read
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, Cfg::kTmemCols);
}

}  // namespace laya
