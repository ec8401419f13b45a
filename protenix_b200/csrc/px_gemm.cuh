// A persistent product D(m, n) = sum_k A(m, k) B(n, k) of 16-bit operands on the tensor cores, whose epilogue is a parameter: the
// passes of the cross entropy (cross_entropy.cu).
//
// Operands lie along k ([m][k], K-major) or across it ([k][m], MN-major); TMA fills tiles of 128 m (n) by 64 k in 128-byte
// swizzle either way, and zeroes what lies outside, so no size needs to be a multiple of anything but the row strides (16 bytes).
// One CTA works on 128 x kN, or a pair of them (cta_group::2) on 256 x kN, each with its own 128 rows of A and half of B: the pair asks L2 for
// 64 bytes a cycle where a CTA alone with kN = 256 asks for 96.
//
// Roles: warp 0 copies, warp 1 issues products, kSets sets of kSetWarps (4 or 8) are the epilogue: a warp has a quarter of the lanes and all or half of
// the columns; two sets take the tiles in turn, each with an accumulator of its own.
// Accumulators are double-buffered.
//
// 8192 rows, 2048 channels, 65536 classes, bf16, pairs: the sums of the forward pass at 1600 to 1650 TFLOP/s (a library product 1655), 1024 channels 1580, 512 1380 (tensor
// pipe 78 % busy), 256 770: below some 700 channels the exponentials' threads take longer than the products (a tile of 256 x 256 costs them some 4 us).  One
// set of eight epilogue warps 824, 580 and 504 us for 1024, 512 and 256 channels, one of sixteen 774, 575 and 452, two of eight 758, 475 and 357.
#pragma once
#include "px_pair.cuh"
#include "px_rowpipe.cuh"

namespace px {

constexpr int kGemmM = 128, kGemmK = 64;          // rows of a CTA's tile, k of a stage

template <int kCtas_, int kN_, bool kAMn_, bool kBMn_, int kStages_, int kSets_ = 1, int kSetWarps_ = 8, int kStgBytes_ = 4096, bool kEpiMemory = false>
struct GemmShape {
  static constexpr int kCtas = kCtas_, kN = kN_, kStages = kStages_, kSets = kSets_, kSetWarps = kSetWarps_, kEpiWarps = kSets * kSetWarps, kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kParts = kSetWarps / 4, kPartCols = kN / kParts, kStgBytes = kStgBytes_;      // columns of an epilogue warp
  static constexpr bool kAMn = kAMn_, kBMn = kBMn_;
  static constexpr int kBRows = kN / kCtas;       // rows of B that a CTA loads
  static constexpr int kABytes = kGemmM * kGemmK * 2, kBBytes = kBRows * kGemmK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kCols = 2 * kN;
  static constexpr int kStg = kStages * kStageBytes, kExtra = kStg + kEpiWarps * kStgBytes, kExtraBytes = kEpiMemory ? 1536 * (kParts - 1) * kSets + 4 * kEpiWarps * kPartCols : 0;
  static constexpr int kBars = kExtra + kExtraBytes;
  static constexpr size_t kSmem = kBars + 256 + 1024;
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(kBRows % 64 == 0 && kN <= 256 && kPartCols >= 64, "tile");
  static constexpr uint32_t idesc(bool f16) { return umma_idesc_16(kGemmM * kCtas, kN, f16, f16, kAMn, kBMn); }
};

// The tiles of a product: `batch` products of tiles_m x tiles_n tiles, each over `nk` steps of 64 k in `splits` parts.  symmetric: only
// tiles (i, j) with i <= j (square ones).  Tiles run through `group` rows of tiles column by column, so that what is worked on at once reads few operands.
struct GemmTiles {
  int tiles_m, tiles_n, batch, splits, nk, nk_split, group, symmetric, total;
};
struct GemmTile {
  int z, split, mt, nt, k0, nk;
};
__device__ __forceinline__ GemmTile gemm_tile(const GemmTiles& t, int tile) {
  GemmTile a;
  const int per = t.symmetric ? t.tiles_m * (t.tiles_m + 1) / 2 : t.tiles_m * t.tiles_n;
  const int zs = tile / per, r = tile - zs * per;
  a.z = zs / t.splits;
  a.split = zs - a.z * t.splits;
  if (t.symmetric) {
    // column nt holds nt + 1 tiles
    int nt = (int)((sqrtf(8.f * (float)r + 1.f) - 1.f) * 0.5f);
    while (nt * (nt + 1) / 2 > r) --nt;
    while ((nt + 1) * (nt + 2) / 2 <= r) ++nt;
    a.nt = nt;
    a.mt = r - nt * (nt + 1) / 2;
  } else {
    const int whole = t.group * t.tiles_n, g = r / whole, first = g * t.group, rows = min(t.group, t.tiles_m - first), in = r - g * whole;
    a.nt = in / rows;
    a.mt = first + in - a.nt * rows;
  }
  a.k0 = a.split * t.nk_split;
  a.nk = min(t.nk_split, t.nk - a.k0);
  return a;
}

struct GemmOperands {
  CUtensorMap a, b, b_other;         // b_other: taken in place of b where *other is not zero
  const uint32_t* other;             // or NULL
  uint32_t idesc;
};

struct GemmBarriers {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem_base, peer_stop;
};

static_assert(sizeof(GemmBarriers) <= 256, "barriers");

// What an epilogue gets for a tile: its place, the accumulator's address with this warp's lanes in it, and what it may use in shared memory.
struct GemmEpiTile {
  GemmTile at;
  int m0, n0;                        // first of this warp's 32 rows, first of its columns
  uint32_t acc;                      // tensor memory, lanes and first column of this warp
  int quarter, part, lane, set;
  unsigned char* stg;                // kStgBytes of this warp's own, for blocks of 32 rows that leave by TMA
  float* own;                        // kEpiMemory: a number for each column of this warp, its own
  float* shared;                     // 384 numbers for each part but the first, shared by the warps of a set
};
template <class S>
__device__ __forceinline__ void gemm_epi_sync(int set) { asm volatile("bar.sync %0, %1;\n" ::"r"(1 + set), "n"(32 * S::kSetWarps) : "memory"); }

template <class S, class Epi>
__global__ void __launch_bounds__(S::kThreads, 1)
gemm_kernel(const __grid_constant__ GemmOperands ops, const __grid_constant__ Epi epi, const GemmTiles tiles) {
  constexpr bool kPair = S::kCtas == 2;
  constexpr int kStages = S::kStages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = smem_aligned(smem_raw);
  GemmBarriers& bars = *reinterpret_cast<GemmBarriers*>(ring + S::kBars);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_rank() : 0;
  const int first_tile = blockIdx.x / S::kCtas, tile_step = gridDim.x / S::kCtas;

  const bool skip = cta_begin();
  if (threadIdx.x == 32) prefetch_maps(ops.a, ops.b);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars.acc_full[b], 1);
      mbar_init(&bars.acc_empty[b], S::kSetWarps * S::kCtas);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(S::kCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(S::kCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  }
  bool stop;
  tc_fence_before();
  if constexpr (kPair) {
    // both CTAs work or neither does
    stop = __syncthreads_or(skip) != 0;
    if (threadIdx.x == 0)
      asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(map_to_rank(smem_u32(&bars.peer_stop), rank ^ 1)), "r"((uint32_t)stop) : "memory");
    tc_cluster_sync();
    stop = stop || *reinterpret_cast<volatile uint32_t*>(&bars.peer_stop) != 0;
  } else {
    stop = __syncthreads_or(skip) != 0;
  }
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = bars.tmem_base;
  if (blockIdx.x == 0 && threadIdx.x == 64) epi.begin();

  if (stop) {
    // nothing
  } else if (warp == 0) {
    uint32_t it = 0;
    bool ok = true;
    const bool other = ops.other && *ops.other != 0;
    const CUtensorMap* const map_b = other ? &ops.b_other : &ops.b;
    for (int tile = first_tile; tile < tiles.total && ok; tile += tile_step) {
      const GemmTile t = gemm_tile(tiles, tile);
      const int m0 = (t.mt * S::kCtas + (int)rank) * kGemmM, n0 = t.nt * S::kN + (int)rank * S::kBRows;
      for (int kt = 0; kt < t.nk && ok; ++kt, ++it) {
        const int s = it % kStages;
        const uint32_t ph = (it / kStages) & 1;
        ok = mbar_wait_warp(&bars.empty[s], ph ^ 1, 1u);
        if (!ok) break;
        if (elect_lane()) {
          const uint32_t sa = smem_u32(ring + s * S::kStageBytes), sb = sa + S::kABytes;
          const int k = (t.k0 + kt) * kGemmK;
          if (rank == 0) mbar_expect_tx(&bars.full[s], S::kCtas * S::kStageBytes);
          const uint32_t bar = kPair ? map_to_rank(smem_u32(&bars.full[s]), 0) : 0;
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (kPair)
              tma_load_3d_pair(dst, map, bar, x, y, z);
            else
              tma_load_3d(dst, map, &bars.full[s], x, y, z);
          };
          if constexpr (S::kAMn) {
#pragma unroll
            for (int j = 0; j < kGemmM / 64; ++j) load(sa + j * 8192, &ops.a, m0 + 64 * j, k, t.z);
          } else {
            load(sa, &ops.a, k, m0, t.z);
          }
          if constexpr (S::kBMn) {
#pragma unroll
            for (int j = 0; j < S::kBRows / 64; ++j) load(sb + j * 8192, map_b, n0 + 64 * j, k, t.z);
          } else {
            load(sb, map_b, k, n0, t.z);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t it = 0, count = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles.total && ok; tile += tile_step, ++count) {
        const GemmTile t = gemm_tile(tiles, tile);
        const uint32_t ab = count & 1, aph = (count >> 1) & 1;
        ok = mbar_wait_warp(&bars.acc_empty[ab], aph ^ 1, 2u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + ab * S::kN;
        for (int kt = 0; kt < t.nk; ++kt, ++it) {
          const int s = it % kStages;
          const uint32_t ph = (it / kStages) & 1;
          ok = mbar_wait_warp(&bars.full[s], ph, 4u);
          if (!ok) break;
          tc_fence_after();
          if (elect_lane()) {
            const uint32_t sa = smem_u32(ring + s * S::kStageBytes), sb = sa + S::kABytes;
            const uint64_t da = S::kAMn ? umma_desc_mn_sw128(sa, 8192, 1024) : umma_desc_sw128(sa);
            const uint64_t db = S::kBMn ? umma_desc_mn_sw128(sb, 8192, 1024) : umma_desc_sw128(sb);
#pragma unroll
            for (int ks = 0; ks < kGemmK / 16; ++ks) {     // 16 k: two 16-byte pieces of a row, or sixteen rows of 128 bytes
              const uint64_t a = da + (S::kAMn ? 128 : 2) * ks, b = db + (S::kBMn ? 128 : 2) * ks;
              const uint32_t more = (kt | ks) ? 1u : 0u;
              if constexpr (kPair)
                umma_pair(d, a, b, ops.idesc, more);
              else
                umma_bf16(d, a, b, ops.idesc, more);
            }
            if constexpr (kPair)
              umma_commit_pair(&bars.empty[s]);
            else
              umma_commit(&bars.empty[s]);
            if (kt == t.nk - 1) {
              if constexpr (kPair)
                umma_commit_pair(&bars.acc_full[ab]);
              else
                umma_commit(&bars.acc_full[ab]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
  } else {
    const int q = warp & 3;                                // the quarter of the lanes that this warp may access goes by its index
    bool ok = true;
    GemmEpiTile e;
    e.quarter = q, e.set = (warp - 2) / S::kSetWarps, e.part = (warp - 2) % S::kSetWarps >> 2, e.lane = lane;
    uint32_t count = e.set;
    e.stg = ring + S::kStg + (warp - 2) * S::kStgBytes;
    e.own = reinterpret_cast<float*>(ring + S::kExtra) + (warp - 2) * S::kPartCols;
    e.shared = reinterpret_cast<float*>(ring + S::kExtra) + S::kEpiWarps * S::kPartCols + 384 * (S::kParts - 1) * e.set;
    for (int tile = first_tile + e.set * tile_step; tile < tiles.total; tile += S::kSets * tile_step, count += S::kSets) {
      e.at = gemm_tile(tiles, tile);
      const uint32_t ab = count & 1, aph = (count >> 1) & 1;
      e.m0 = (e.at.mt * S::kCtas + (int)rank) * kGemmM + 32 * q;
      e.n0 = e.at.nt * S::kN + e.part * S::kPartCols;
      e.acc = tmem_base + ((uint32_t)(32 * q) << 16) + ab * S::kN + e.part * S::kPartCols;
      const typename Epi::Row row = epi.template before<S>(e);      // what it fetches is on its way while the product is
      ok = ok && mbar_wait_warp(&bars.acc_full[ab], aph, 8u);
      if (!Epi::kMeets && !ok) break;                      // an epilogue whose warps meet goes through all tiles
      tc_fence_after();
      // called once by a whole warp, when it has read the last of the accumulator
      epi.template tile<S>(e, row, [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair)
            mbar_arrive_cluster(map_to_rank(smem_u32(&bars.acc_empty[ab]), 0));
          else
            mbar_arrive(&bars.acc_empty[ab]);
        }
      });
    }
    if (lane == 0) tma_store_wait_read<0>();
  }

  // teardown: everybody meets, then the allocating warp frees the tensor memory
  __syncwarp();
  tc_fence_before();
  cta_teardown_sync();
  if constexpr (kPair) tc_cluster_sync();          // nobody leaves while its pair may still signal or read it
  if (warp == 0) {
    tc_fence_after();
    if constexpr (kPair)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(S::kCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(S::kCols) : "memory");
  }
  if constexpr (kPair) tc_cluster_sync();
}

// The map of an operand: `rows` rows of `inner` elements, `stride` elements apart, `batch` of them `plane` elements apart.  K-major operands
// come in boxes of box_rows rows (their tile), MN-major ones in boxes of 64 k.
static inline bool gemm_map(CUtensorMap* map, bool f16, const void* base, int64_t inner, int64_t rows, int64_t batch, int64_t stride, int64_t plane, int box_rows) {
  return make_map_3d(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, (uint64_t)inner, (uint64_t)rows, (uint64_t)batch,
                     (uint64_t)stride * 2, (uint64_t)plane * 2, 64, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <class S, class Epi>
static int32_t gemm_launch(const GemmOperands& ops, const Epi& epi, GemmTiles t, cudaStream_t st) {
  const int64_t per = t.symmetric ? (int64_t)t.tiles_m * (t.tiles_m + 1) / 2 : (int64_t)t.tiles_m * t.tiles_n;
  const int64_t total = per * t.batch * t.splits;
  if (total > 0x7fffffff) return PX_ERR_UNSUPPORTED;
  t.total = (int)total;
  static SmemLimit limit;
  if (!limit.set(gemm_kernel<S, Epi>, S::kSmem)) return PX_ERR_LAUNCH;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = S::kCtas, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(even_grid(total, sm_count() / S::kCtas) * S::kCtas));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = S::kCtas > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, gemm_kernel<S, Epi>, ops, epi, t) == cudaSuccess) return PX_OK;
  cudaGetLastError();
  return PX_ERR_LAUNCH;
}

}  // namespace px
