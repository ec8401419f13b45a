// Newton-Schulz orthogonalisation of matrices: X = G / (|G| + eps), |.| the root of the sum of squares, then for each step
//   A = X X^T,   X <- (a I + b A + c A^2) X
// (for tall matrices from the other side: A = X^T X, X <- X (a I + b A + c A^2), the same result without a transposition).  An odd polynomial of the
// singular values: the steps drive them towards one and leave the singular vectors.
//
// Three products a step on the tensor cores (px_gemm.cuh).  Iterates of 16 bits are not enough: the polynomial multiplies small singular values by up
// to 3.4 a step, and the rounding noise of an iterate with them.  For 384 x 1536 in a simulation the result is off by 1.2e-2 (noise), 0.11 (falling
// spectrum) and 0.34 (rank 8) with bf16 iterates, 1.5e-3 to 4e-2 with fp16 ones, 7e-6 to 6e-5 with fp32 throughout.  So every
// operand is two fp16 planes, v = hi + 2^-11 lo (22 bits), and three of the four products are formed: 3e-7 to 8e-6.
// Values are stored times 2^10 (planes keep their bits down to 2^-34 of an element; iterates and polynomials may grow to 60).
//
// A and the polynomial are symmetric: only tiles on and above the diagonal are formed, the epilogue stores each a second time transposed, which
// saves half of two of the three products.
//
// 4096 x 4096, bf16: 160 + 170 + 290 us a step (X X^T, polynomial, P X), the last at 1430 TFLOP/s of plane products; 24 x 384 x 1536: 23 + 14 + 46.  What bounds them: the power
// limit for the former; for short sums shared memory (a stage of 256 columns reads and takes in 208 KB in the 1536 cycles of its products, the planes of a tile
// are 256 KB more) and some 6 us that a launch takes to begin and end.
#include <algorithm>

#include "px_gemm.cuh"

namespace px {

constexpr float kPlaneScale = 1024.f;
constexpr int kOrthoEpiWarps = 8, kOrthoThreads = 64 + 32 * kOrthoEpiWarps;
constexpr int kOrthoStgBytes = 4096;      // staged block of a warp

// An accumulator is cut after each 16 k, which takes half a step off a sum of positive terms on average, 5.8e-8 of it (2.3e-7 measured for a sum of squares of 128
// and the product behind it), and the polynomial multiplies a common factor by up to 30 where singular values lie close together: what the
// cuts of a growing sum over k, in accumulators of `chunk` times 64, take off on average is put back.  64 x 700 in fp32 is off by 4.5e-6 without, plain fp32 products give 1.8e-6.
__host__ __device__ constexpr float uncut(int64_t k, int chunk) { return 1.f + 2.9e-8f * (float)(((k + 15) / 16 < 4 * chunk ? (k + 15) / 16 : 4 * chunk) + 1); }

// ---- norm and first iterate ------------------------------------------------------------------------------------------
constexpr int kNormBlocks = 1024;      // of a matrix, at most
// Blocks of a matrix, each of which leaves a sum.
static int norm_parts(int64_t batch, int64_t elements) {
  return (int)std::min<int64_t>(std::min<int64_t>(kNormBlocks, std::max<int64_t>(8, 8 * sm_count() / batch)), (elements + 2047) / 2048);
}
// kVec elements at a time: 16 bytes where matrices begin at a multiple of that (24 x 384 x 1536, bf16: by elements 14 us).
template <typename T, int kVec>
__global__ void __launch_bounds__(256) ortho_norm_kernel(const T* __restrict__ g, double* __restrict__ sums, int64_t elements) {
  __shared__ double part[8];
  struct alignas(sizeof(T) * kVec) Vec {
    T v[kVec];
  };
  pdl_wait();
  const Vec* p = reinterpret_cast<const Vec*>(g + blockIdx.y * elements);
  double s0 = 0.0, s1 = 0.0;
  const int64_t step = (int64_t)gridDim.x * 256, all = elements / kVec;
  constexpr int kAtOnce = kVec == 1 ? 8 : 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += kAtOnce * step) {
    Vec v[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i + j * step < all) v[j] = p[i + j * step];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i + j * step >= all) break;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const double x = (double)(float)v[j].v[k];
        double& s = ((j * kVec + k) & 1) ? s1 : s0;
        s = fma(x, x, s);
      }
    }
  }
  s0 += s1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s0;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s0 += part[w];
    sums[blockIdx.y * gridDim.x + blockIdx.x] = s0;
  }
}
// v = hi + 2^-11 lo, two values at a time
__device__ __forceinline__ void split_planes2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16x2_inf(x, y);
  const float2 h = unpack_f16x2(hi);
  // 2048 v - 2048 hi, both exact
  const float2 r = apart2(fma2(pair2(h.x, h.y), pair2(-2048.f, -2048.f), mul2(pair2(x, y), pair2(2048.f, 2048.f))));
  lo = pack_f16x2_inf(r.x, r.y);
}
// The planes of G 2^10 / (|G| + eps), eight columns a thread; columns behind n are zero.
template <typename T>
__global__ void __launch_bounds__(256) ortho_split_kernel(const T* __restrict__ g, const double* __restrict__ sums, uint4* __restrict__ planes, int64_t m, int64_t n,
                                                          int64_t ld, int parts, double eps) {
  __shared__ double by;
  pdl_wait();
  const int64_t z = blockIdx.y;
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 32) s += sums[z * parts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) by = (double)kPlaneScale / (sqrt(s) + eps);
  }
  __syncthreads();
  const double scale = by;
  const bool plain = scale > 1e-30 && scale < 1e30;        // fp32 holds the factor, and a value times it
  const float scale32 = (float)scale;
  const int64_t per = ld / 8, all = m * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per, col = (i - row * per) * 8;
    const T* p = g + (z * m + row) * n + col;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < n ? (plain ? (float)p[j] * scale32 : (float)((double)(float)p[j] * scale)) : 0.f;
    uint4 hi, lo;
    split_planes2(v[0], v[1], hi.x, lo.x), split_planes2(v[2], v[3], hi.y, lo.y);
    split_planes2(v[4], v[5], hi.z, lo.z), split_planes2(v[6], v[7], hi.w, lo.w);
    planes[2 * z * all + i] = hi;
    planes[(2 * z + 1) * all + i] = lo;
  }
}
// The planes of A from the sums over parts of the long side, fp32 [matrix][part][s][ld]; eight columns a thread.
__global__ void __launch_bounds__(256) ortho_gram_kernel(const float* __restrict__ parts, uint4* __restrict__ planes, int s, int ld, int splits) {
  pdl_wait();
  const int64_t z = blockIdx.y, all = (int64_t)s * ld / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const float* const p = parts + z * splits * s * ld + 8 * i;
    float v[8] = {};
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 a = *reinterpret_cast<const float4*>(p + (int64_t)k * s * ld), b = *reinterpret_cast<const float4*>(p + (int64_t)k * s * ld + 4);
      v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    }
    const int col = (int)(8 * i % ld);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j >= s) v[j] = 0.f;                        // nothing was stored there
    uint4 hi, lo;
    split_planes2(v[0], v[1], hi.x, lo.x), split_planes2(v[2], v[3], hi.y, lo.y);
    split_planes2(v[4], v[5], hi.z, lo.z), split_planes2(v[6], v[7], hi.w, lo.w);
    planes[2 * z * all + i] = hi;
    planes[(2 * z + 1) * all + i] = lo;
  }
}
// The other way, for results whose rows TMA cannot store.
template <typename T>
__global__ void __launch_bounds__(256) ortho_join_kernel(const __half* __restrict__ planes, T* __restrict__ out, int64_t m, int64_t n, int64_t ld) {
  pdl_wait();
  const int64_t z = blockIdx.y, all = m * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / n, at = (2 * z * m + row) * ld + (i - row * n);
    out[z * all + i] = (T)((__half2float(planes[at]) + __half2float(planes[at + m * ld]) * (1.f / 2048.f)) * (1.f / kPlaneScale));
  }
}

// ---- the product -----------------------------------------------------------------------------------------------------
// D = A B^T of operands in two planes: D1 = hi hi, D2 = hi lo + lo hi, D = D1 + 2^-11 D2.  The tensor core truncates where it adds, which shortens a sum
// of positive terms by some 5e-8 a step of 16 k (384 x 1536 in fp32: 1.6e-5 off with one accumulator for all of K, plain fp32 products 3e-6 to 7e-6).  So D1
// gets a fresh accumulator for each `chunk` stages of 64 k, which the epilogue's warps add to their registers, rounding to nearest, while the stage's products
// with a low plane run; D2, 2^-11 as large, is added up in tensor memory.  Of chunk = 1, 2, 4, 8 the results of eight 1024 x 1024 matrices are off by 0.9, 1.4, 2.5,
// 4.7e-6 (plain fp32 products 3.1e-6) and take 708, 634, 582, 552 us: 1 where the result is fp32, 2 for fp16 and 8 for bf16, whose own rounding is 2e-4 and 1.7e-3.
//
// Tiles of 128 x 128, or 256 x 256 for a pair of CTAs.  What bounds them is shared memory: a product of 128 x 128 x 16 reads 8 KB in 64 cycles, as much as there is,
// and 64 KB a stage come in besides (0.71 us a stage, 768 cycles of it products); those of 256 columns, which only a pair has, read 12 KB in 128.
template <int kCtas_, bool kAMn_, bool kBMn_>
struct PlaneShape {
  static constexpr int kCtas = kCtas_, kSide = 128 * kCtas, kStages = 3, kCols = 64 * kCtas;      // kCols: of an epilogue warp
  static constexpr bool kAMn = kAMn_, kBMn = kBMn_;
  static constexpr int kPlaneBytes = kGemmM * kGemmK * 2, kStageBytes = 4 * kPlaneBytes;      // A hi, A lo, B hi, B lo: 128 rows each
  static constexpr int kStg = kStages * kStageBytes, kBars = kStg + kOrthoEpiWarps * kOrthoStgBytes;
  static constexpr size_t kSmem = kBars + 256 + 1024;
  static constexpr uint32_t kIdesc = umma_idesc_f16(kSide, kSide, kAMn, kBMn);
  static_assert(kSmem <= 232448, "shared memory budget");
};
struct PlaneBarriers {
  uint64_t full[3], empty[3], part_full, part_empty, rest_full, rest_empty;
  uint32_t tmem_base, peer_stop;
};

static_assert(sizeof(PlaneBarriers) <= 256, "barriers");

// What becomes of the product: planes of a factor times it (and the polynomial's other terms), symmetric ones stored twice; or the result.
struct OrthoEnd {
  CUtensorMap out;              // planes: boxes of 32 x 32 (z = 2 matrix + plane); result: of 32 rows of 32 columns
  const __half* gram;           // planes of A, for the polynomial; or NULL
  float factor, a, b;           // v = factor D + b A + a I
  int rows, cols, ld;           // ld: of gram
  int type, symmetric, result;  // type: of the result, whichever product this is

  // A plane of a block, which has a buffer of 2 KB; the one before may still be on its way out of the other.
  __device__ __forceinline__ void store(unsigned char* stg, int lane, int x, int y, int z) const {
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(&out, smem_u32(stg), x, y, z);
      tma_store_commit();
    }
  }
  __device__ __forceinline__ void room(int lane) const {
    if (lane == 0) tma_store_wait_read<1>();
    __syncwarp();
  }
  // The planes of A at 32 columns from col on of a row.
  __device__ __forceinline__ void fetch(uint4 (&h)[4], uint4 (&l)[4], int row, int col, int z) const {
    const __half* p = gram + ((int64_t)2 * z * rows + row) * ld + col;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = l[k] = make_uint4(0, 0, 0, 0);
      if (row < rows && col + 8 * k < ld) h[k] = *reinterpret_cast<const uint4*>(p + 8 * k), l[k] = *reinterpret_cast<const uint4*>(p + (int64_t)rows * ld + 8 * k);
    }
  }
  // v: 32 columns from col on of row m0 + lane
  __device__ __forceinline__ void block(float* v, int m0, int col, int z, bool twice, unsigned char* stg, int lane) const {
    const int row = m0 + lane;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= factor;
    if (gram) {
      uint4 h[4], l[4];
      fetch(h, l, row, col, z);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t hs[4] = {h[k].x, h[k].y, h[k].z, h[k].w}, ls[4] = {l[k].x, l[k].y, l[k].z, l[k].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 x = unpack_f16x2(hs[w]), y = unpack_f16x2(ls[w]);
          v[8 * k + 2 * w] = fmaf(b, fmaf(y.x, 1.f / 2048.f, x.x), v[8 * k + 2 * w]);
          v[8 * k + 2 * w + 1] = fmaf(b, fmaf(y.y, 1.f / 2048.f, x.y), v[8 * k + 2 * w + 1]);
        }
      }
      if (m0 == col) {                       // blocks of 32 x 32: the diagonal is that of the block, or not in it
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += lane == j ? a * kPlaneScale : 0.f;
      }
    }
    if (result) {
      if (lane == 0) tma_store_wait_read<0>();
      __syncwarp();
      if (type == PX_F32) {
#pragma unroll
        for (int p = 0; p < 8; ++p)
          *reinterpret_cast<float4*>(stg + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t o[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) o[w] = type == PX_F16 ? pack_f16x2_inf(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]) : pack_bf16x2(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]);
          *reinterpret_cast<uint4*>(stg + lane * 64 + ((p ^ (lane >> 1 & 3)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(&out, smem_u32(stg), col, m0, z);
        tma_store_commit();
      }
      return;
    }
    uint32_t w[2][16];
#pragma unroll
    for (int j = 0; j < 16; ++j) split_planes2(v[2 * j], v[2 * j + 1], w[0][j], w[1][j]);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      room(lane);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4*>(stg + 2048 * p + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[p][4 * k], w[p][4 * k + 1], w[p][4 * k + 2], w[p][4 * k + 3]);
      store(stg + 2048 * p, lane, col, m0, 2 * z + p);
    }
    if (twice) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        room(lane);
        // lane = column of the transposed block
#pragma unroll
        for (int j = 0; j < 32; ++j)
          *reinterpret_cast<uint16_t*>(stg + 2048 * p + j * 64 + (((lane >> 3) ^ (j >> 1 & 3)) << 4) + 2 * (lane & 7)) = (uint16_t)(w[p][j / 2] >> (16 * (j & 1)));
        store(stg + 2048 * p, lane, m0, col, 2 * z + p);
      }
    }
  }
};

template <class S>
__global__ void __launch_bounds__(kOrthoThreads, 1)
plane_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ OrthoEnd end, const GemmTiles tiles, int chunk) {
  constexpr bool kPair = S::kCtas == 2;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kTmem = 2 * S::kSide;      // D1, D2
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = smem_aligned(smem_raw);
  PlaneBarriers& bars = *reinterpret_cast<PlaneBarriers*>(ring + S::kBars);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_rank() : 0;
  const int first_tile = blockIdx.x / S::kCtas, tile_step = gridDim.x / S::kCtas;

  const bool skip = cta_begin();
  if (threadIdx.x == 32) prefetch_maps(map_a, map_b, end.out);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.part_full, 1);
    mbar_init(&bars.part_empty, kOrthoEpiWarps * S::kCtas);
    mbar_init(&bars.rest_full, 1);
    mbar_init(&bars.rest_empty, kOrthoEpiWarps * S::kCtas);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(kTmem) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(kTmem) : "memory");
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

  if (stop) {
    // nothing
  } else if (warp == 0) {
    uint32_t it = 0;
    bool ok = true;
    for (int tile = first_tile; tile < tiles.total && ok; tile += tile_step) {
      const GemmTile t = gemm_tile(tiles, tile);
      const int m0 = t.mt * S::kSide + (int)rank * 128, n0 = t.nt * S::kSide + (int)rank * 128;
      const bool same = end.symmetric && t.mt == t.nt;      // rows against themselves: one operand is fetched
      for (int kt = 0; kt < t.nk && ok; ++kt, ++it) {
        const int s = it % kStages;
        ok = mbar_wait_warp(&bars.empty[s], ((it / kStages) & 1) ^ 1, 1u);
        if (!ok) break;
        if (elect_lane()) {
          const uint32_t sa = smem_u32(ring + s * S::kStageBytes);
          if (rank == 0) mbar_expect_tx(&bars.full[s], S::kCtas * (same ? S::kStageBytes / 2 : S::kStageBytes));
          const uint32_t bar = kPair ? map_to_rank(smem_u32(&bars.full[s]), 0) : 0;
          auto load = [&](uint32_t dst, const CUtensorMap* map, bool across, int from, int z) {
            for (int j = 0; j < (across ? 2 : 1); ++j) {
              const int x = across ? from + 64 * j : (t.k0 + kt) * kGemmK, y = across ? (t.k0 + kt) * kGemmK : from;
              if constexpr (kPair)
                tma_load_3d_pair(dst + 8192 * j, map, bar, x, y, z);
              else
                tma_load_3d(dst + 8192 * j, map, &bars.full[s], x, y, z);
            }
          };
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            load(sa + p * S::kPlaneBytes, &map_a, S::kAMn, m0, 2 * t.z + p);
            if (!same) load(sa + (2 + p) * S::kPlaneBytes, &map_b, S::kBMn, n0, 2 * t.z + p);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t it = 0, part = 0, count = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles.total && ok; tile += tile_step, ++count) {
        const GemmTile t = gemm_tile(tiles, tile);
        ok = mbar_wait_warp(&bars.rest_empty, (count & 1) ^ 1, 2u);
        for (int kt = 0; kt < t.nk && ok; ++kt, ++it) {
          const int s = it % kStages;
          const bool begins = (kt & (chunk - 1)) == 0, ends = ((kt + 1) & (chunk - 1)) == 0 || kt == t.nk - 1;
          ok = mbar_wait_warp(&bars.full[s], (it / kStages) & 1, 4u) && (!begins || mbar_wait_warp(&bars.part_empty, (part & 1) ^ 1, 8u));
          if (!ok) break;
          tc_fence_after();
          if (elect_lane()) {
            const uint32_t sa = smem_u32(ring + s * S::kStageBytes), sb = sa + (end.symmetric && t.mt == t.nt ? 0 : 2 * S::kPlaneBytes);
            const uint64_t da = S::kAMn ? umma_desc_mn_sw128(sa, 8192, 1024) : umma_desc_sw128(sa);
            const uint64_t db = S::kBMn ? umma_desc_mn_sw128(sb, 8192, 1024) : umma_desc_sw128(sb);
            constexpr uint64_t kLo = S::kPlaneBytes >> 4;
            auto mma = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t more) {
              if constexpr (kPair)
                umma_pair(d, a, b, S::kIdesc, more);
              else
                umma_bf16(d, a, b, S::kIdesc, more);
            };
            auto commit = [&](uint64_t* bar) {
              if constexpr (kPair)
                umma_commit_pair(bar);
              else
                umma_commit(bar);
            };
#pragma unroll
            for (int ks = 0; ks < kGemmK / 16; ++ks) mma(tmem_base, da + (S::kAMn ? 128 : 2) * ks, db + (S::kBMn ? 128 : 2) * ks, !begins || ks > 0);
            if (ends) commit(&bars.part_full);
#pragma unroll
            for (int ks = 0; ks < kGemmK / 16; ++ks) {
              const uint64_t a = da + (S::kAMn ? 128 : 2) * ks, b = db + (S::kBMn ? 128 : 2) * ks;
              mma(tmem_base + S::kSide, a, b + kLo, (kt | ks) ? 1u : 0u);
              mma(tmem_base + S::kSide, a + kLo, b, 1u);
            }
            commit(&bars.empty[s]);
            if (kt == t.nk - 1) commit(&bars.rest_full);
          }
          __syncwarp();
          if (ends) ++part;
        }
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    unsigned char* const stg = ring + S::kStg + (warp - 2) * kOrthoStgBytes;
    const uint32_t lanes = tmem_base + ((uint32_t)(32 * q) << 16) + S::kCols * half;
    auto arrive = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair)
          mbar_arrive_cluster(map_to_rank(smem_u32(bar), 0));
        else
          mbar_arrive(bar);
      }
    };
    uint32_t part = 0, count = 0;
    bool ok = true;
    for (int tile = first_tile; tile < tiles.total && ok; tile += tile_step, ++count) {
      const GemmTile t = gemm_tile(tiles, tile);
      float sum[S::kCols];
#pragma unroll
      for (int j = 0; j < S::kCols; ++j) sum[j] = 0.f;
      for (int kt = 0; kt < t.nk && ok; kt += chunk, ++part) {
        ok = mbar_wait_warp(&bars.part_full, part & 1, 16u);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < S::kCols; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 2) add2(sum[c + j], sum[c + j + 1], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        }
        arrive(&bars.part_empty);
      }
      ok = ok && mbar_wait_warp(&bars.rest_full, count & 1, 32u);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < S::kCols; c += 32) {
        uint32_t r[32];
        tmem_ld32(lanes + S::kSide + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[c + j] = fmaf(__uint_as_float(r[j]), 1.f / 2048.f, sum[c + j]);
      }
      arrive(&bars.rest_empty);
      const int m0 = t.mt * S::kSide + (int)rank * 128 + 32 * q, n0 = t.nt * S::kSide + S::kCols * half;
      if (m0 < end.rows) {
#pragma unroll
        for (int c = 0; c < S::kCols; c += 32)
          if (n0 + c < end.cols) end.block(&sum[c], m0, n0 + c, t.z * tiles.splits + t.split, end.symmetric && t.mt != t.nt, stg, lane);
      }
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
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kTmem) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kTmem) : "memory");
  }
  if constexpr (kPair) tc_cluster_sync();
}

}  // namespace px

#include "px_ortho_small.cuh"

namespace px {

PX_DEFINE_FAMILY_HOOKS(update)

// ---- host ------------------------------------------------------------------------------------------------------------
static int64_t ortho_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// planes [batch][2][rows][ld], of which `inner` columns count, with the maps of their copies: as an operand along k or across it, and on their way out
struct Planes {
  __half* at;
  CUtensorMap along, across, out;
  bool set(__half* to, int64_t rows, int64_t inner, int64_t ld, int64_t batch) {
    at = to;
    return gemm_map(&along, true, at, inner, rows, 2 * batch, ld, rows * ld, kGemmM) && gemm_map(&across, true, at, inner, rows, 2 * batch, ld, rows * ld, kGemmK) &&
           make_map_3d(&out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, at, (uint64_t)inner, (uint64_t)rows, (uint64_t)(2 * batch), (uint64_t)ld * 2, (uint64_t)rows * ld * 2, 32, 32,
                       CU_TENSOR_MAP_SWIZZLE_64B);
  }
};
template <class S>
static int32_t launch_planes(const CUtensorMap& ma, const CUtensorMap& mb, OrthoEnd end, GemmTiles t, int64_t m, int64_t n, int64_t k, int dtype, cudaStream_t st) {
  const int chunk = dtype == PX_F32 ? 1 : dtype == PX_F16 ? 2 : 8;
  end.factor *= uncut(k, chunk);
  t.tiles_m = (int)(ortho_up(m, S::kSide) / S::kSide), t.tiles_n = (int)(ortho_up(n, S::kSide) / S::kSide);
  const int64_t total = (int64_t)t.batch * t.splits * (t.symmetric ? (int64_t)t.tiles_m * (t.tiles_m + 1) / 2 : (int64_t)t.tiles_m * t.tiles_n);
  if (total > 0x7fffffff) return PX_ERR_UNSUPPORTED;
  t.total = (int)total;
  static SmemLimit limit;
  if (!limit.set(plane_product_kernel<S>, S::kSmem)) return PX_ERR_LAUNCH;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = S::kCtas, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(even_grid(total, sm_count() / S::kCtas) * S::kCtas));
  cfg.blockDim = dim3(kOrthoThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = S::kCtas > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, plane_product_kernel<S>, ma, mb, end, t, chunk) == cudaSuccess) return PX_OK;
  cudaGetLastError();
  return PX_ERR_LAUNCH;
}
template <bool kAMn, bool kBMn>
static int32_t ortho_product(const Planes& a, const Planes& b, int64_t batch, int64_t m, int64_t n, int64_t k, const OrthoEnd& end, int dtype, cudaStream_t st) {
  const CUtensorMap &ma = kAMn ? a.across : a.along, &mb = kBMn ? b.across : b.along;
  GemmTiles t = {};
  t.batch = (int)batch, t.splits = 1, t.group = 8, t.symmetric = end.symmetric;
  t.nk = t.nk_split = (int)(ortho_up(k, kGemmK) / kGemmK);
  // Cycles of both forms: a stage of 64 k takes some 1500 of either, more of a pair whose accumulator is read after each (fp32 results); a tile's epilogue 6000
  // and 9000.
  const auto cycles = [&](int64_t side, int64_t room, int64_t stage, int64_t epilogue) {
    const int64_t tm = ortho_up(m, side) / side, tn = ortho_up(n, side) / side, tiles = batch * (end.symmetric ? tm * (tm + 1) / 2 : tm * tn);
    return (tiles + room - 1) / room * (t.nk * stage + epilogue);
  };
  if (cycles(256, sm_count() / 2, dtype == PX_F32 ? 2200 : 1500, 9000) < cycles(128, sm_count(), 1500, 6000)) return launch_planes<PlaneShape<2, kAMn, kBMn>>(ma, mb, end, t, m, n, k, dtype, st);
  return launch_planes<PlaneShape<1, kAMn, kBMn>>(ma, mb, end, t, m, n, k, dtype, st);
}

// Parts that the long side is cut into where A has few tiles: as many as the SMs take at once, of two stages at least, if they and the kernel that adds them up
// (some 10000 cycles) are the faster: 256 x 16384 816 -> 214 us, 256 x 4096 287 -> 156, 1024 x 4096 420 -> 354.  Parts of all of A: one half stored two ways would
// have to be read across.
static int gram_splits(int64_t batch, int64_t s, int64_t length) {
  const int64_t side = (s + 127) / 128, tiles = batch * side * side, nk = (length + kGemmK - 1) / kGemmK, most = std::min<int64_t>(sm_count() / tiles, nk / 2);
  if (most < 2) return 1;
  const int64_t part = (nk + most - 1) / most, splits = (nk + part - 1) / part;
  return part * 1500 + 10000 + splits * batch * s * s / 400 < nk * 1500 ? (int)splits : 1;
}

struct OrthoPlan {
  int64_t ld, s, lds, sums, x[2], gram, poly, parts, bytes;
  int splits;
};
static OrthoPlan ortho_plan(int64_t batch, int64_t m, int64_t n) {
  OrthoPlan p;
  p.s = std::min(m, n);
  p.ld = ortho_up(n, 8), p.lds = ortho_up(p.s, 8);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += ortho_up(bytes, 1024);
    return here;
  };
  p.sums = take(batch * norm_parts(batch, m * n) * 8);
  for (int64_t& x : p.x) x = take(batch * 2 * m * p.ld * 2);
  p.gram = take(batch * 2 * p.s * p.lds * 2);
  p.poly = take(batch * 2 * p.s * p.lds * 2);
  p.splits = gram_splits(batch, p.s, std::max(m, n));
  p.parts = take(p.splits > 1 ? p.splits * batch * p.s * p.lds * 4 : 0);
  p.bytes = at;
  return p;
}
template <typename T>
static bool ortho_first(const void* g, double* sums, uint4* planes, int64_t batch, int64_t m, int64_t n, int64_t ld, double eps, cudaStream_t st) {
  const int parts = norm_parts(batch, m * n);
  constexpr int kVec = 16 / sizeof(T);
  const bool wide = m * n % kVec == 0 && ((uintptr_t)g & 15) == 0;
  if (!launch_pdl(wide ? ortho_norm_kernel<T, kVec> : ortho_norm_kernel<T, 1>, dim3(parts, (unsigned)batch), 256, 0, st, (const T*)g, sums, m * n)) return false;
  const int64_t blocks = std::min<int64_t>((m * ld / 8 + 255) / 256, std::max<int64_t>(1, 8 * sm_count() / batch));
  return launch_pdl(ortho_split_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), 256, 0, st, (const T*)g, (const double*)sums, planes, m, n, ld, parts, eps);
}
template <typename T>
static bool ortho_last(const __half* planes, void* out, int64_t batch, int64_t m, int64_t n, int64_t ld, cudaStream_t st) {
  const int64_t blocks = std::min<int64_t>((m * n + 255) / 256, std::max<int64_t>(1, 8 * sm_count() / batch));
  return launch_pdl(ortho_join_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), 256, 0, st, planes, (T*)out, m, n, ld);
}

}  // namespace px

using namespace px;

extern "C" int64_t px_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n) {
  return batch <= 0 || m <= 0 || n <= 0 ? 0 : ortho_plan(batch, m, n).bytes;
}

// All steps in one launch take none; 1024 bytes, so that a call has a workspace whatever its form.
extern "C" int64_t px_orthogonalize_steps_workspace_bytes(int64_t batch, int64_t m, int64_t n, int32_t steps) {
  if (batch <= 0 || m <= 0 || n <= 0) return 0;
  int slices;
  return small_ortho_ctas(batch, std::min(m, n), std::max(m, n), steps, &slices) ? 1024 : ortho_plan(batch, m, n).bytes;
}

extern "C" int32_t px_orthogonalize(const void* g, void* out, int64_t batch, int64_t m, int64_t n, const float* coefficients, int32_t steps, double eps, int32_t dtype,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (batch < 0 || m < 0 || n < 0 || steps < 1 || !coefficients || !(eps >= 0.0)) return PX_ERR_BAD_ARG;
  if (dtype != PX_F32 && dtype != PX_BF16 && dtype != PX_F16) return PX_ERR_UNSUPPORTED;
  if (batch > 65535 || m > (1 << 20) || n > (1 << 20) || steps > 1000) return PX_ERR_UNSUPPORTED;
  if (batch == 0 || m == 0 || n == 0) return PX_OK;
  if (!g || !out || !workspace || ((uintptr_t)workspace & 255) || (((uintptr_t)g | (uintptr_t)out) & (dtype == PX_F32 ? 3 : 1))) return PX_ERR_BAD_ARG;
  if (workspace_bytes < px_orthogonalize_steps_workspace_bytes(batch, m, n, steps)) return PX_ERR_WORKSPACE;
  const OrthoPlan p = ortho_plan(batch, m, n);
  if (!have_context()) return PX_ERR_LAUNCH;
  const cudaStream_t st = (cudaStream_t)stream;
  int slices = 1;
  if (const int ctas = small_ortho_ctas(batch, p.s, std::max(m, n), steps, &slices)) {
    SmallOrtho a = {};
    a.g = g, a.out = out, a.stride = m * n, a.ld = (int)n, a.side = (int)p.s, a.length = (int)std::max(m, n);
    a.steps = steps, a.ctas = ctas, a.eps = eps;
    std::copy(coefficients, coefficients + 3 * steps, a.abc);
    const int size = dtype == PX_F32 ? 4 : 2;
    a.type = dtype, a.wide_access = n * size % 16 == 0 && (((uintptr_t)g | (uintptr_t)out) & 15) == 0;
    const bool ok = launch_small_ortho(a, batch, slices, m > n, st);
    return ok ? PX_OK : PX_ERR_LAUNCH;
  }
  char* const ws = (char*)workspace;
  const bool wide = m <= n;
  double* sums = (double*)(ws + p.sums);
  Planes planes[2], gram, poly;
  if (!planes[0].set((__half*)(ws + p.x[0]), m, n, p.ld, batch) || !planes[1].set((__half*)(ws + p.x[1]), m, n, p.ld, batch) ||
      !gram.set((__half*)(ws + p.gram), p.s, p.s, p.lds, batch) || !poly.set((__half*)(ws + p.poly), p.s, p.s, p.lds, batch))
    return PX_ERR_LAUNCH;
  const bool ok = dtype == PX_F32    ? ortho_first<float>(g, sums, (uint4*)planes[0].at, batch, m, n, p.ld, eps, st)
                  : dtype == PX_BF16 ? ortho_first<bf16>(g, sums, (uint4*)planes[0].at, batch, m, n, p.ld, eps, st)
                                     : ortho_first<__half>(g, sums, (uint4*)planes[0].at, batch, m, n, p.ld, eps, st);
  if (!ok) return PX_ERR_LAUNCH;
  const int size = dtype == PX_F32 ? 4 : 2;
  const bool direct = n * size % 16 == 0 && ((uintptr_t)out & 15) == 0;      // what TMA can store
  for (int i = 0; i < steps; ++i) {
    const Planes &x = planes[i & 1], &next = planes[1 - (i & 1)];
    OrthoEnd e = {};
    e.out = gram.out, e.factor = 1.f / kPlaneScale, e.rows = e.cols = (int)p.s, e.ld = (int)p.lds, e.symmetric = 1, e.type = dtype;
    int32_t status;
    if (p.splits > 1) {
      OrthoEnd part = e;
      part.symmetric = 0, part.result = 1, part.type = PX_F32;
      if (!make_map_3d(&part.out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, ws + p.parts, (uint64_t)p.s, (uint64_t)p.s, (uint64_t)(batch * p.splits), (uint64_t)p.lds * 4,
                       (uint64_t)p.s * p.lds * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B))
        return PX_ERR_LAUNCH;
      GemmTiles t = {};
      t.batch = (int)batch, t.splits = p.splits, t.group = 8, t.nk = (int)(ortho_up(std::max(m, n), kGemmK) / kGemmK);
      t.nk_split = (t.nk + p.splits - 1) / p.splits;
      status = wide ? launch_planes<PlaneShape<1, false, false>>(x.along, x.along, part, t, p.s, p.s, (int64_t)t.nk_split * kGemmK, dtype, st)
                    : launch_planes<PlaneShape<1, true, true>>(x.across, x.across, part, t, p.s, p.s, (int64_t)t.nk_split * kGemmK, dtype, st);
      const int64_t blocks = std::min<int64_t>((p.s * p.lds / 8 + 255) / 256, std::max<int64_t>(1, 8 * sm_count() / batch));
      if (!status && !launch_pdl(ortho_gram_kernel, dim3((unsigned)blocks, (unsigned)batch), 256, 0, st, (const float*)(ws + p.parts), (uint4*)gram.at, (int)p.s, (int)p.lds, p.splits))
        status = PX_ERR_LAUNCH;
    } else {
      status = wide ? ortho_product<false, false>(x, x, batch, p.s, p.s, n, e, dtype, st) : ortho_product<true, true>(x, x, batch, p.s, p.s, m, e, dtype, st);
    }
    if (status) return status;
    e.out = poly.out, e.gram = gram.at, e.a = coefficients[3 * i], e.b = coefficients[3 * i + 1], e.factor = coefficients[3 * i + 2] / kPlaneScale;
    status = ortho_product<false, false>(gram, gram, batch, p.s, p.s, p.s, e, dtype, st);
    if (status) return status;
    e = {};
    e.out = next.out, e.factor = 1.f / kPlaneScale, e.rows = (int)m, e.cols = (int)n, e.type = dtype;
    if (i == steps - 1 && direct) {
      e.result = 1, e.factor = 1.f / (kPlaneScale * kPlaneScale);
      const CUtensorMapDataType type = dtype == PX_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == PX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
      if (!make_map_3d(&e.out, type, out, (uint64_t)n, (uint64_t)m, (uint64_t)batch, (uint64_t)n * size, (uint64_t)m * n * size, 32, 32,
                       dtype == PX_F32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
        return PX_ERR_LAUNCH;
    }
    status = wide ? ortho_product<false, true>(poly, x, batch, m, n, m, e, dtype, st) : ortho_product<false, false>(x, poly, batch, m, n, n, e, dtype, st);
    if (status) return status;
  }
  if (direct) return PX_OK;
  const bool done = dtype == PX_F32    ? ortho_last<float>(planes[steps & 1].at, out, batch, m, n, p.ld, st)
                    : dtype == PX_BF16 ? ortho_last<bf16>(planes[steps & 1].at, out, batch, m, n, p.ld, st)
                                       : ortho_last<__half>(planes[steps & 1].at, out, batch, m, n, p.ld, st);
  return done ? PX_OK : PX_ERR_LAUNCH;
}
