// Newton-Schulz orthogonalisation of matrices whose short side is at most 128: all steps in one launch, a CTA (or a cluster of up to eight) a matrix.
//
// The iterate stays in shared memory: a CTA has one or two slices of 128 along the long side, X_s [128][128] in two fp16 planes, rows along the short
// side (tall matrices are turned on the way in and out).  A step is A = sum over slices and CTAs of X_s X_s^T, P = a I + b A + c A^2 (every CTA forms it,
// in the place of A), X_s <- P X_s.  Three products of 128 x 128 x 128 a slice or less, each waiting for the one before: what bounds it is that chain, some
// 2 us a product with its epilogue, instead of a launch of 7 us each.
//
// A's parts of the CTAs are exchanged through distributed shared memory: each CTA adds up 128 / k rows from all k parts, in the order of their ranks, and
// writes the planes of the sum to all of them.  Accumulators are as in plane_product_kernel: a fresh one for each 64 k (two slices: the last of four goes on
// with the second), joined in registers, and one for the products with a low plane.
#pragma once
#include "px_pair.cuh"
#include "px_rowpipe.cuh"

namespace px {

constexpr int kSmallSteps = 32, kSmallOrthoThreads = 256;
constexpr int kSmallPlane = 2 * 128 * 128;                 // [128][128] fp16, two panels of 64 columns

struct SmallOrtho {
  const void* g;
  void* out;
  int64_t stride;               // of a matrix
  int ld;                       // its columns
  int side, length;             // short and long side
  int steps, ctas;
  double eps;
  float abc[3 * kSmallSteps];
};

template <int kSlices>
struct SmallOrthoShape {
  static constexpr int kX = 0, kA = kSlices * 2 * kSmallPlane, kBars = kA + 2 * kSmallPlane;
  static constexpr size_t kSmem = kBars + 512 + 1024;
  static_assert(kSmem <= 232448, "shared memory budget");
};
struct SmallOrthoBarriers {
  uint64_t done;
  uint32_t tmem_base, stop[8];
  double part[8], sums[8];      // of this CTA's warps; of the cluster's CTAs
};

__device__ __forceinline__ int plane_offset(int row, int piece) {      // of the 16 bytes with columns 8 piece ..
  return (piece >> 3) * (kSmallPlane / 2) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}
template <typename T>
__device__ __forceinline__ float small_value(const void* g, int64_t at) { return (float)((const T*)g)[at]; }

template <typename T, int kSlices, bool kTall>
__global__ void __launch_bounds__(kSmallOrthoThreads, 1) small_ortho_kernel(const __grid_constant__ SmallOrtho p) {
  typedef SmallOrthoShape<kSlices> S;
  constexpr float kScale = kPlaneScale;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  SmallOrthoBarriers& bars = *reinterpret_cast<SmallOrthoBarriers*>(sm + S::kBars);
  const int warp = warp_index(), lane = threadIdx.x & 31, q = warp & 3, half = warp >> 2;
  const int rank = p.ctas > 1 ? (int)cluster_rank() : 0;
  const int64_t matrix = blockIdx.x / p.ctas;

  bool skip = cta_begin();
  if (threadIdx.x == 0) {
    mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  skip = __syncthreads_or(skip) != 0;
  if (p.ctas > 1) {
    // all CTAs of a cluster work or none does
    tc_cluster_sync();
    if (threadIdx.x < p.ctas)
      asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(map_to_rank(smem_u32(&bars.stop[rank]), threadIdx.x)), "r"((uint32_t)skip) : "memory");
    tc_cluster_sync();
    for (int r = 0; r < p.ctas; ++r) skip = skip || *reinterpret_cast<volatile uint32_t*>(&bars.stop[r]) != 0;
  }
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = bars.tmem_base;

  if (!skip) {
    // ---- the first iterate -------------------------------------------------------------------------------------------
    const void* const g = (const T*)p.g + matrix * p.stride;
    const int first = rank * kSlices * 128;                // of this CTA's columns along the long side
    // eight values along the long side: row r of the slices, columns c0 ..
    auto read = [&](int i, float (&v)[8]) {
      const int r = kTall ? i & 127 : i / (16 * kSlices), c0 = first + 8 * (kTall ? i >> 7 : i % (16 * kSlices));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = c0 + j;
        v[j] = r < p.side && c < p.length ? small_value<T>(g, kTall ? (int64_t)c * p.ld + r : (int64_t)r * p.ld + c) : 0.f;
      }
    };
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < 2048 * kSlices; i += kSmallOrthoThreads) {
      float v[8];
      read(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fma((double)v[j], (double)v[j], s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) bars.part[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = 0.0;
      for (int w = 0; w < 8; ++w) s += bars.part[w];
      if (p.ctas == 1) bars.sums[0] = s;
      else
        for (int r = 0; r < p.ctas; ++r) asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(map_to_rank(smem_u32(&bars.sums[rank]), r)), "d"(s) : "memory");
    }
    if (p.ctas > 1) tc_cluster_sync();
    else __syncthreads();
    s = 0.0;
    for (int r = 0; r < p.ctas; ++r) s += bars.sums[r];
    const double by = (double)kScale / (sqrt(s) + p.eps);
#pragma unroll 2
    for (int i = threadIdx.x; i < 2048 * kSlices; i += kSmallOrthoThreads) {
      float v[8];
      read(i, v);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_planes2((float)((double)v[2 * j] * by), (float)((double)v[2 * j + 1] * by), hi[j], lo[j]);
      const int r = kTall ? i & 127 : i / (16 * kSlices), piece = kTall ? i >> 7 : i % (16 * kSlices);
      unsigned char* const x = sm + S::kX + (piece >> 4) * 2 * kSmallPlane + plane_offset(r, piece & 15);
      *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(x + kSmallPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }

    // ---- the steps ---------------------------------------------------------------------------------------------------
    constexpr uint32_t idesc_kk = umma_idesc_f16(128, 128), idesc_kn = umma_idesc_f16(128, 128, false, true);
    constexpr uint64_t kLo = kSmallPlane >> 4, kPanel = kSmallPlane >> 5;
    uint32_t parity = 0;
    // Accumulators: leading ones at columns 0, 128 and 384, the rest at 256.
    auto product = [&](auto issue) {
      tc_fence_before();
      asm volatile("fence.proxy.async;\n" ::: "memory");
      __syncthreads();
      if (warp == 0) {
        tc_fence_after();
        asm volatile("fence.proxy.async;\n" ::: "memory");
        if (elect_lane()) {
          issue();
          umma_commit(&bars.done);
        }
        __syncwarp();
      }
      // where the wait gives up the work goes on, on values that the flag has declared void: the barriers of the cluster want everybody
      mbar_wait(&bars.done, parity, 1u);
      __syncwarp();
      parity ^= 1;
      tc_fence_after();
    };
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16) + 64 * half;
    const int row = 32 * q + lane;
    // 32 columns of the sums of all accumulators, from column 64 half + c on
    auto sums = [&](int c, bool third, float (&v)[32]) {
      uint32_t a[32];
      tmem_ld32(lanes + 256 + c, a);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(a[j]) * (1.f / 2048.f);
      for (int k = 0; k < (third ? 3 : 2); ++k) {
        tmem_ld32(lanes + (k == 2 ? 384 : 128 * k) + c, a);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(a[j]);
      }
    };
    // planes of 32 values of this thread's row, from column 64 half + c on
    auto put = [&](unsigned char* to, int c, const float (&v)[32]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_planes2(v[8 * k + 2 * j], v[8 * k + 2 * j + 1], hi[j], lo[j]);
        unsigned char* const x = to + plane_offset(row, 8 * half + c / 8 + k);
        *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(x + kSmallPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    };
    unsigned char* const gram = sm + S::kA;
    for (int step = 0; step < p.steps; ++step) {
      // A
      product([&] {
#pragma unroll
        for (int n = 0; n < 2 * kSlices; ++n) {            // panels of 64 k
          const uint64_t x = umma_desc_sw128(smem_u32(sm + S::kX + (n >> 1) * 2 * kSmallPlane)) + (n & 1) * kPanel;
          const uint32_t lead = tmem + (n == 2 ? 384 : 128 * (n & 1));
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            umma_bf16(lead, x + 2 * ks, x + 2 * ks, idesc_kk, (ks > 0 || n == 3) ? 1u : 0u);
            umma_bf16(tmem + 256, x + 2 * ks, x + kLo + 2 * ks, idesc_kk, (n | ks) ? 1u : 0u);
            umma_bf16(tmem + 256, x + kLo + 2 * ks, x + 2 * ks, idesc_kk, 1u);
          }
        }
      });
      if (p.ctas == 1) {
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          sums(c, kSlices == 2, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= 1.f / kScale;
          put(gram, c, v);
        }
      } else {
        // this CTA's part in fp32, where A will be: 16-byte pieces exchanged by row
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          sums(c, kSlices == 2, v);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *reinterpret_cast<float4*>(gram + row * 512 + (((16 * half + c / 4 + k) ^ (row & 31)) << 4)) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
        tc_cluster_sync();
        const int share = 128 / p.ctas, groups = share * 16 / kSmallOrthoThreads;      // 4, 2 or 1 of eight columns a thread
        uint4 hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i < groups) {
            const int at = threadIdx.x + kSmallOrthoThreads * i, r = rank * share + (at >> 4), piece = at & 15;
            float v[8] = {};
            for (int k = 0; k < p.ctas; ++k) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float4 x;
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                             : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                             : "r"(map_to_rank(smem_u32(gram + r * 512 + (((2 * piece + j) ^ (r & 31)) << 4)), k))
                             : "memory");
                v[4 * j] += x.x, v[4 * j + 1] += x.y, v[4 * j + 2] += x.z, v[4 * j + 3] += x.w;
              }
            }
            constexpr float f = 1.f / kScale;
            split_planes2(f * v[0], f * v[1], hi[i].x, lo[i].x), split_planes2(f * v[2], f * v[3], hi[i].y, lo[i].y);
            split_planes2(f * v[4], f * v[5], hi[i].z, lo[i].z), split_planes2(f * v[6], f * v[7], hi[i].w, lo[i].w);
          }
        }
        tc_cluster_sync();                                 // all parts are read
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i < groups) {
            const int at = threadIdx.x + kSmallOrthoThreads * i, r = rank * share + (at >> 4), piece = at & 15;
            const uint32_t to = smem_u32(gram + plane_offset(r, piece));
            for (int k = 0; k < p.ctas; ++k) {
              const uint32_t there = map_to_rank(to, k);
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(there), "r"(hi[i].x), "r"(hi[i].y), "r"(hi[i].z), "r"(hi[i].w) : "memory");
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(there + kSmallPlane), "r"(lo[i].x), "r"(lo[i].y), "r"(lo[i].z), "r"(lo[i].w) : "memory");
            }
          }
        }
        asm volatile("fence.proxy.async;\n" ::: "memory");
        tc_cluster_sync();
      }

      // the polynomial, in the place of A
      const float a = p.abc[3 * step], b = p.abc[3 * step + 1], c2 = p.abc[3 * step + 2] / kScale;
      product([&] {
        const uint64_t x = umma_desc_sw128(smem_u32(gram));
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint64_t y = x + (ks >> 2) * kPanel + 2 * (ks & 3);
          umma_bf16(tmem + 128 * (ks >> 2), y, y, idesc_kk, (ks & 3) ? 1u : 0u);
          umma_bf16(tmem + 256, y, y + kLo, idesc_kk, ks ? 1u : 0u);
          umma_bf16(tmem + 256, y + kLo, y, idesc_kk, 1u);
        }
      });
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        float v[32];
        sums(c, false, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned char* const x = gram + plane_offset(row, 8 * half + c / 8 + k);
          const uint4 h = *reinterpret_cast<const uint4*>(x), l = *reinterpret_cast<const uint4*>(x + kSmallPlane);
          const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 xh = unpack_f16x2(hs[w]), xl = unpack_f16x2(ls[w]);
            const int j = 8 * k + 2 * w, col = 64 * half + c + j;
            v[j] = fmaf(c2, v[j], b * fmaf(xl.x, 1.f / 2048.f, xh.x)) + (row == col ? a * kScale : 0.f);
            v[j + 1] = fmaf(c2, v[j + 1], b * fmaf(xl.y, 1.f / 2048.f, xh.y)) + (row == col + 1 ? a * kScale : 0.f);
          }
        }
        put(gram, c, v);
      }

      // X, a slice at a time
      const bool last = step == p.steps - 1;
#pragma unroll 1
      for (int n = 0; n < kSlices; ++n) {
        unsigned char* const slice = sm + S::kX + n * 2 * kSmallPlane;
        product([&] {
          const uint64_t y = umma_desc_sw128(smem_u32(gram)), x = umma_desc_mn_sw128(smem_u32(slice), kSmallPlane / 2, 1024);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint64_t u = y + (ks >> 2) * kPanel + 2 * (ks & 3), w = x + 128 * ks;
            umma_bf16(tmem + 128 * (ks >> 2), u, w, idesc_kn, (ks & 3) ? 1u : 0u);
            umma_bf16(tmem + 256, u, w + kLo, idesc_kn, ks ? 1u : 0u);
            umma_bf16(tmem + 256, u + kLo, w, idesc_kn, 1u);
          }
        });
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          sums(c, false, v);
          if (!last) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= 1.f / kScale;
            put(slice, c, v);
          } else if (row < p.side) {
            T* const out = (T*)p.out + matrix * p.stride;
            const int col0 = first + 128 * n + 64 * half + c;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col0 + j < p.length) out[kTall ? (int64_t)(col0 + j) * p.ld + row : (int64_t)row * p.ld + col0 + j] = (T)(v[j] * (1.f / (kScale * kScale)));
          }
        }
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  cta_teardown_sync();
  if (p.ctas > 1) tc_cluster_sync();                       // nobody leaves while its cluster may still read or write here
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <typename T, int kSlices, bool kTall>
static bool launch_small_ortho(const SmallOrtho& p, int64_t batch, cudaStream_t st) {
  typedef SmallOrthoShape<kSlices> S;
  static SmemLimit limit;
  if (!limit.set(small_ortho_kernel<T, kSlices, kTall>, S::kSmem)) return false;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.ctas, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * p.ctas));
  cfg.blockDim = dim3(kSmallOrthoThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = p.ctas > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, small_ortho_kernel<T, kSlices, kTall>, p) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}
// CTAs of a matrix: one slice each where the matrices then have room at once, otherwise two; 0: not this kernel.
static inline int small_ortho_ctas(int64_t batch, int64_t side, int64_t length, int steps, int* slices) {
  if (side > 128 || steps > kSmallSteps) return 0;
  const auto fit = [](int64_t n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 0; };
  const int one = fit((length + 127) / 128), two = fit((length + 255) / 256);
  if (!two) return 0;
  *slices = one && (one == two || batch * one <= sm_count()) ? 1 : 2;
  return *slices == 1 ? one : two;
}
template <typename T>
static bool launch_small_ortho(const SmallOrtho& p, int64_t batch, int slices, bool tall, cudaStream_t st) {
  if (slices == 1) return tall ? launch_small_ortho<T, 1, true>(p, batch, st) : launch_small_ortho<T, 1, false>(p, batch, st);
  return tall ? launch_small_ortho<T, 2, true>(p, batch, st) : launch_small_ortho<T, 2, false>(p, batch, st);
}

}  // namespace px
