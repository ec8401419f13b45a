// Newton-Schulz orthogonalisation of matrices whose short side is at most 128: all steps in one launch, a CTA (or a cluster of up to eight) a matrix.
//
// The iterate stays in shared memory: a CTA has one or two slices of 128 along the long side, X_s [128][128] in two fp16 planes, rows along the short
// side (tall matrices are turned on the way in and out).  A step is A = sum over slices and CTAs of X_s X_s^T, P = a I + b A + c A^2 (every CTA forms it,
// in the place of A), X_s <- P X_s.  Three products of 128 x 128 x 128 a slice or less, each waiting for the one before: what bounds it is that chain, some
// 2.5 us a product with its epilogue, instead of a launch of 7 us each.  Nine warps share the registers of four partitions: 168 a thread, and every form keeps some 200
// to 240 bytes of a thread in local memory.
//
// A's parts of the CTAs are exchanged through distributed shared memory: each CTA adds up 128 / k rows from all k parts, in the order of their ranks, and
// writes the planes of the sum to all of them.  Accumulators are as in plane_product_kernel: a fresh one for each 64 k, joined in
// registers (two slices: the second's take the place of the first's, which the other warps read while the low planes are multiplied), and one for the products
// with a low plane.
#pragma once
#include "px_pair.cuh"
#include "px_rowpipe.cuh"

namespace px {

constexpr int kSmallSteps = 32, kSmallOrthoThreads = 256;      // and a warp that issues the products
constexpr int kSmallPlane = 2 * 128 * 128;                 // [128][128] fp16, two panels of 64 columns

struct SmallOrtho {
  const void* g;
  void* out;
  int64_t stride;               // of a matrix
  int ld;                       // its columns
  int side, length;             // short and long side
  int steps, ctas, type;
  int wide_access;              // rows of the matrix are aligned to 16 bytes
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
  uint64_t lead, done;          // the leading products (of the first slice); all of them
  uint64_t drained;             // the first have been read
  uint32_t tmem_base, stop[8];
  double part[8], sums[8];      // of this CTA's warps; of the cluster's CTAs
};
static_assert(sizeof(SmallOrthoBarriers) <= 512, "barriers");

__device__ __forceinline__ int plane_offset(int row, int piece) {      // of the 16 bytes with columns 8 piece ..
  return (piece >> 3) * (kSmallPlane / 2) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}
// A slice as 128 rows of 128 floats, the way in and out, and A's parts.  Pieces of 16 bytes are exchanged by row, so that neither eight rows of a piece nor
// a piece of every eighth row meet in a bank.
__device__ __forceinline__ int float_offset(int row, int col) { return row * 512 + (((col >> 2) ^ ((row ^ (row >> 3)) & 31)) << 4) + 4 * (col & 3); }
__device__ __forceinline__ float small_value(const void* g, int64_t at, int type) {
  return type == PX_F32 ? ((const float*)g)[at] : type == PX_F16 ? __half2float(((const __half*)g)[at]) : __bfloat162float(((const bf16*)g)[at]);
}
// 16 bytes of a matrix as 4 or 8 values
__device__ __forceinline__ int small_values(const uint4& u, int type, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (type == PX_F32) {
      v[j] = __uint_as_float(w[j]);
    } else {
      const float2 x = type == PX_F16 ? unpack_f16x2(w[j]) : unpack_bf16x2(w[j]);
      v[2 * j] = x.x, v[2 * j + 1] = x.y;
    }
  }
  return type == PX_F32 ? 4 : 8;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory"); }

// A from its parts in the kCtas CTAs of a cluster: every row goes to the CTA that adds it up (row / kShare), which writes the planes of the sum to all of
// them.  `sum`: this thread's row, columns 64 half ..; f: what A is multiplied by; the parts lie where A will be, part k from row k kShare on.
// Rows and columns from `side` on (kAll: there are none) are left as they are: no sum takes them in, and no result that counts comes of them.
template <int kCtas, bool kAll>
__device__ __forceinline__ void exchange_gram(unsigned char* gram, int rank, int row, int half, const float (&sum)[64], float f, int side) {
  constexpr int kShare = 128 / kCtas, kGroups = 8 / kCtas;      // rows of a CTA; eight columns each of a thread
  cluster_wait();                                               // nobody multiplies by what lies there any more
  if (kAll || row < side) {
    const int to = row / kShare, r = rank * kShare + row % kShare;
    const uint32_t there = map_to_rank(smem_u32(gram), to);
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (kAll || 64 * half + 4 * k < side) asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(there + float_offset(r, 64 * half + 4 * k)), "f"(sum[4 * k]), "f"(sum[4 * k + 1]),
                   "f"(sum[4 * k + 2]), "f"(sum[4 * k + 3])
                   : "memory");
  }
  __syncwarp();
  tc_cluster_sync();
  uint4 hi[kGroups], lo[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = threadIdx.x + kSmallOrthoThreads * i, r = at >> 4, piece = at & 15;
    if (!kAll && (rank * kShare + r >= side || 8 * piece >= side)) continue;
    float v[8] = {};
#pragma unroll
    for (int k = 0; k < kCtas; ++k) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(gram + float_offset(k * kShare + r, 8 * piece + 4 * j));
        v[4 * j] += x.x, v[4 * j + 1] += x.y, v[4 * j + 2] += x.z, v[4 * j + 3] += x.w;
      }
    }
    split_planes2(f * v[0], f * v[1], hi[i].x, lo[i].x), split_planes2(f * v[2], f * v[3], hi[i].y, lo[i].y);
    split_planes2(f * v[4], f * v[5], hi[i].z, lo[i].z), split_planes2(f * v[6], f * v[7], hi[i].w, lo[i].w);
  }
  __syncwarp();
  tc_cluster_sync();                                            // all parts are read
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = threadIdx.x + kSmallOrthoThreads * i, r = rank * kShare + (at >> 4), piece = at & 15;
    if (!kAll && (r >= side || 8 * piece >= side)) continue;
    const uint32_t to = smem_u32(gram + plane_offset(r, piece));
#pragma unroll
    for (int k = 0; k < kCtas; ++k) {
      const uint32_t there = map_to_rank(to, k);
      asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(there), "r"(hi[i].x), "r"(hi[i].y), "r"(hi[i].z), "r"(hi[i].w) : "memory");
      asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(there + kSmallPlane), "r"(lo[i].x), "r"(lo[i].y), "r"(lo[i].z), "r"(lo[i].w) : "memory");
    }
  }
  asm volatile("fence.proxy.async;\n" ::: "memory");
  __syncwarp();
  tc_cluster_sync();
}

template <int kSlices, bool kTall, bool kShort>
__global__ void __launch_bounds__(kSmallOrthoThreads + 32, 1) small_ortho_kernel(const __grid_constant__ SmallOrtho p) {
  typedef SmallOrthoShape<kSlices> S;
  constexpr float kScale = kPlaneScale;
  const float uncut_gram = uncut(p.length, 1), uncut_side = uncut(p.side, 1);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  SmallOrthoBarriers& bars = *reinterpret_cast<SmallOrthoBarriers*>(sm + S::kBars);
  const int warp = warp_index(), lane = threadIdx.x & 31, q = warp & 3, half = warp >> 2;
  const int rank = p.ctas > 1 ? (int)cluster_rank() : 0;
  const int64_t matrix = blockIdx.x / p.ctas;

  bool skip = cta_begin();
  if (threadIdx.x == 0) {
    mbar_init(&bars.lead, 1);
    mbar_init(&bars.done, 1);
    mbar_init(&bars.drained, 8);
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

  constexpr uint32_t idesc_kk = umma_idesc_f16(128, 128), idesc_kn = umma_idesc_f16(128, 128, false, true);
  // Steps of 16 k that hold anything, of sums over the short side and of A's (kShort: the side is 112 or less): 48 x 16 x 16 take 29 us with them alone, 35 with
  // all, 4 x 20 x 500 52 and 73.  Counts that the compiler does not know cost 128 x 128 2 of 37 us.
  const int side_steps = kShort ? (p.side + 15) / 16 : 8, gram_steps = kShort && kSlices == 1 && p.ctas == 1 ? (p.length + 15) / 16 : 8 * kSlices;
  constexpr uint64_t kLo = kSmallPlane >> 4, kPanel = kSmallPlane >> 5;
  unsigned char* const gram = sm + S::kA;
  // Before a product all threads meet: its operands are in shared memory, and the accumulators have been read.
  auto meet = [&] {
    tc_fence_before();
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncthreads();
  };

  if (skip) {
    // nothing
  } else if (warp == 8) {
    // ---- products: accumulators of the leading ones at columns 0 and 128, of the rest at 256 ------------------------
    const uint64_t gram_at = umma_desc_sw128(smem_u32(gram));
    auto issue = [&](auto leading, auto rest) {
      meet();
      tc_fence_after();
      if (elect_lane()) {
        leading();
        umma_commit(&bars.lead);
        rest();
        umma_commit(&bars.done);
      }
      __syncwarp();
    };
    // operand u along k, w along k (K-major) or across it
    auto one = [&](uint64_t u, uint64_t w, bool across, uint32_t idesc) {
      issue(
          [&] {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (ks < side_steps) umma_bf16(tmem + 128 * (ks >> 2), u + (ks >> 2) * kPanel + 2 * (ks & 3), w + (across ? 128 * ks : (ks >> 2) * kPanel + 2 * (ks & 3)), idesc, (ks & 3) ? 1u : 0u);
          },
          [&] {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              if (ks >= side_steps) break;
              const uint64_t x = u + (ks >> 2) * kPanel + 2 * (ks & 3), y = w + (across ? 128 * ks : (ks >> 2) * kPanel + 2 * (ks & 3));
              umma_bf16(tmem + 256, x, y + kLo, idesc, ks ? 1u : 0u);
              umma_bf16(tmem + 256, x + kLo, y, idesc, 1u);
            }
          });
    };
    auto slice_at = [&](int n) { return umma_desc_sw128(smem_u32(sm + S::kX + (n >> 1) * 2 * kSmallPlane)) + (n & 1) * kPanel; };      // panels of 64 k
    // the barriers of the other warps' way in
    __syncthreads();
    if (p.ctas > 1) tc_cluster_sync();
    else __syncthreads();
    for (int n = 0; n < kSlices; ++n) __syncthreads();
    if (p.ctas > 1) cluster_arrive();
    for (int step = 0; step < p.steps; ++step) {
      auto lead = [&](int slice) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint64_t x = slice_at(2 * slice + n);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (8 * slice + 4 * n + ks < gram_steps) umma_bf16(tmem + 128 * n, x + 2 * ks, x + 2 * ks, idesc_kk, ks ? 1u : 0u);
        }
      };
      meet();
      tc_fence_after();
      if (elect_lane()) {
        lead(0);
        umma_commit(&bars.lead);
#pragma unroll
        for (int n = 0; n < 2 * kSlices; ++n) {
          const uint64_t x = slice_at(n);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            if (4 * n + ks >= gram_steps) break;
            umma_bf16(tmem + 256, x + 2 * ks, x + kLo + 2 * ks, idesc_kk, (n | ks) ? 1u : 0u);
            umma_bf16(tmem + 256, x + kLo + 2 * ks, x + 2 * ks, idesc_kk, 1u);
          }
        }
        if (kSlices == 1) umma_commit(&bars.done);
      }
      __syncwarp();
      if (kSlices == 2) {
        mbar_wait_warp(&bars.drained, step & 1, 4u);
        tc_fence_after();
        if (elect_lane()) {
          lead(1);
          umma_commit(&bars.done);
        }
        __syncwarp();
      }
      if (p.ctas > 1) {
        cluster_wait();
        for (int k = 0; k < (p.ctas == 2 ? 1 : 3); ++k) tc_cluster_sync();
      }
      one(gram_at, gram_at, false, idesc_kk);
      for (int n = 0; n < kSlices; ++n) one(gram_at, umma_desc_mn_sw128(smem_u32(sm + S::kX + n * 2 * kSmallPlane), kSmallPlane / 2, 1024), true, idesc_kn);
      if (p.ctas > 1 && step < p.steps - 1) cluster_arrive();
    }
    __syncthreads();
  } else {
    // ---- the first iterate -------------------------------------------------------------------------------------------
    const int size = p.type == PX_F32 ? 4 : 2;
    const char* const g = (const char*)p.g + matrix * p.stride * size;
    const int first = rank * kSlices * 128;                // of this CTA's columns along the long side
    // lines along the rows of the matrix, `unit` elements at a time: a line is a row of the slices, or (tall) a column of them
    const int unit = p.wide_access ? 16 / size : 1, across = (kTall ? 128 : 128 * kSlices) / unit, lines = kTall ? 128 * kSlices : 128;
    const int end = kTall ? p.side : min(p.length - first, 128 * kSlices), last_line = kTall ? min(p.length - first, lines) : p.side;
    const int64_t from = kTall ? (int64_t)first * p.ld : first;
    double s4[4] = {};
    for (int i0 = threadIdx.x; i0 < across * lines; i0 += 8 * kSmallOrthoThreads) {
      uint4 u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kSmallOrthoThreads, line = i / across, at = (i - line * across) * unit;
        u[k] = make_uint4(0, 0, 0, 0);
        if (line < last_line && at < end) {
          const int64_t e = from + (int64_t)line * p.ld + at;
          if (unit > 1) u[k] = __ldg(reinterpret_cast<const uint4*>(g + e * size));      // rows are whole pieces of 16 bytes
          else u[k].x = __float_as_uint(small_value(g, e, p.type));
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kSmallOrthoThreads, line = i / across, at = (i - line * across) * unit;
        float v[8];
        if (unit > 1) small_values(u[k], p.type, v);
        else v[0] = __uint_as_float(u[k].x);
        auto place = [&](int j) {
          const int r = kTall ? at + j : line, c = kTall ? line : at + j;
          return sm + S::kX + (c >> 7) * 2 * kSmallPlane + float_offset(r, c & 127);
        };
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          if (j >= unit) break;
          if (unit == 1) {
            s4[0] = fma((double)v[0], (double)v[0], s4[0]);
            *reinterpret_cast<float*>(place(0)) = v[0];
            break;
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) s4[w] = fma((double)v[j + w], (double)v[j + w], s4[w]);
          if (kTall) {
#pragma unroll
            for (int w = 0; w < 4; ++w) *reinterpret_cast<float*>(place(j + w)) = v[j + w];
          } else {
            *reinterpret_cast<float4*>(place(j)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
      }
    }
    double s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
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
    const bool plain = by > 1e-30 && by < 1e30;            // fp32 holds the factor, and a value times it
    const float by32 = (float)by;
    auto times = [&](float v) { return plain ? v * by32 : (float)((double)v * by); };
    // the planes take the place of the floats: a slice's are all read before the first is written
#pragma unroll 1
    for (int n = 0; n < kSlices; ++n) {
      unsigned char* const slice = sm + S::kX + n * 2 * kSmallPlane;
      uint4 hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = threadIdx.x + kSmallOrthoThreads * i, r = at >> 4, c = 8 * (at & 15);
        const float4 u = *reinterpret_cast<const float4*>(slice + float_offset(r, c)), v = *reinterpret_cast<const float4*>(slice + float_offset(r, c + 4));
        split_planes2(times(u.x), times(u.y), hi[i].x, lo[i].x), split_planes2(times(u.z), times(u.w), hi[i].y, lo[i].y);
        split_planes2(times(v.x), times(v.y), hi[i].z, lo[i].z), split_planes2(times(v.z), times(v.w), hi[i].w, lo[i].w);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = threadIdx.x + kSmallOrthoThreads * i, x = plane_offset(at >> 4, at & 15);
        *reinterpret_cast<uint4*>(slice + x) = hi[i];
        *reinterpret_cast<uint4*>(slice + kSmallPlane + x) = lo[i];
      }
    }

    // ---- the steps ---------------------------------------------------------------------------------------------------
    uint32_t parity = 0;
    float sum[64];                // of this thread's row, columns 64 half ..
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16) + 64 * half;
    const int row = 32 * q + lane;
    // Where a wait gives up the work goes on, on values that the flag has declared void: the barriers of the cluster want everybody.
    auto leading = [&](bool first, bool both) {
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t a[32], b[32];
        tmem_ld32(lanes + c, a);
        tmem_ld32(lanes + 128 + c, b);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float s = both ? __uint_as_float(a[j]) + __uint_as_float(b[j]) : __uint_as_float(a[j]);      // or nothing was added up there
          sum[c + j] = first ? s : sum[c + j] + s;
        }
      }
    };
    auto product = [&](bool two, int steps) {
      meet();
      // the leading accumulators are added up while the other products run
      mbar_wait(&bars.lead, parity, 1u);
      __syncwarp();
      tc_fence_after();
      leading(true, steps > 4);
      if (two) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.drained);
      }
      mbar_wait(&bars.done, parity, 2u);
      __syncwarp();
      parity ^= 1;
      tc_fence_after();
      if (two) leading(false, true);
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t a[32];
        tmem_ld32(lanes + 256 + c, a);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[c + j] = fmaf(__uint_as_float(a[j]), 1.f / 2048.f, sum[c + j]);
      }
    };
    // planes of `by` times the sums
    auto put = [&](unsigned char* to, float by) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_planes2(by * sum[8 * k + 2 * j], by * sum[8 * k + 2 * j + 1], hi[j], lo[j]);
        unsigned char* const x = to + plane_offset(row, 8 * half + k);
        *reinterpret_cast<uint4*>(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(x + kSmallPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    };
    auto put_floats = [&](unsigned char* to, float by) {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        *reinterpret_cast<float4*>(to + float_offset(row, 64 * half + 4 * k)) = make_float4(by * sum[4 * k], by * sum[4 * k + 1], by * sum[4 * k + 2], by * sum[4 * k + 3]);
    };
    if (p.ctas > 1) cluster_arrive();
    for (int step = 0; step < p.steps; ++step) {
      // A
      product(kSlices == 2, gram_steps);
      if (p.ctas == 1) {
        put(gram, uncut_gram / kScale);
      } else {
        const int live = 16 * side_steps;
        if (p.ctas == 2) {
          // each sends its whole part to the other, and both add up
          cluster_wait();                                // the other does not multiply by what lies there any more
          const uint32_t there = map_to_rank(smem_u32(gram), rank ^ 1);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (!kShort || (row < live && 64 * half + 4 * k < live))
              asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(there + float_offset(row, 64 * half + 4 * k)), "f"(sum[4 * k]), "f"(sum[4 * k + 1]),
                           "f"(sum[4 * k + 2]), "f"(sum[4 * k + 3])
                           : "memory");
          __syncwarp();
          tc_cluster_sync();
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (kShort && (row >= live || 64 * half + 4 * k >= live)) break;
            const float4 x = *reinterpret_cast<const float4*>(gram + float_offset(row, 64 * half + 4 * k));
            sum[4 * k] += x.x, sum[4 * k + 1] += x.y, sum[4 * k + 2] += x.z, sum[4 * k + 3] += x.w;
          }
          __syncwarp();
          asm volatile("bar.sync 1, %0;\n" ::"n"(kSmallOrthoThreads) : "memory");
          put(gram, uncut_gram / kScale);
        } else if (p.ctas == 4) {
          exchange_gram<4, !kShort>(gram, rank, row, half, sum, uncut_gram / kScale, live);
        } else {
          exchange_gram<8, !kShort>(gram, rank, row, half, sum, uncut_gram / kScale, live);
        }
      }

      // the polynomial, in the place of A
      const float a = p.abc[3 * step], b = p.abc[3 * step + 1], c2 = p.abc[3 * step + 2] * (uncut_side / kScale);
      product(false, side_steps);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned char* const x = gram + plane_offset(row, 8 * half + k);
        const uint4 h = *reinterpret_cast<const uint4*>(x), l = *reinterpret_cast<const uint4*>(x + kSmallPlane);
        const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 xh = unpack_f16x2(hs[w]), xl = unpack_f16x2(ls[w]);
          const int j = 8 * k + 2 * w;
          sum[j] = fmaf(c2, sum[j], b * fmaf(xl.x, 1.f / 2048.f, xh.x));
          sum[j + 1] = fmaf(c2, sum[j + 1], b * fmaf(xl.y, 1.f / 2048.f, xh.y));
        }
      }
      // the diagonal crosses half of the warps, in 32 of their columns
      if (q == 2 * half) {
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] += lane == j ? a * kScale : 0.f;
      } else if (q == 2 * half + 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[32 + j] += lane == j ? a * kScale : 0.f;
      }
      put(gram, 1.f);

      // X, a slice at a time
      const bool last = step == p.steps - 1;
#pragma unroll 1
      for (int n = 0; n < kSlices; ++n) {
        unsigned char* const slice = sm + S::kX + n * 2 * kSmallPlane;
        product(false, side_steps);
        if (last) put_floats(slice, uncut_side / (kScale * kScale));
        else put(slice, uncut_side / kScale);
      }
      if (p.ctas > 1 && !last) cluster_arrive();           // this CTA has multiplied by the polynomial; waited for before its place is written
    }

    // ---- the result, along the rows of the matrix ----------------------------------------------------------------------
    __syncthreads();
    char* const out = (char*)p.out + matrix * p.stride * size;
#pragma unroll 4
    for (int i = threadIdx.x; i < across * lines; i += kSmallOrthoThreads) {
      const int line = i / across, at = (i - line * across) * unit;
      if (line >= last_line || at >= end) continue;
      float v[8];
      auto place = [&](int j) {
        const int r = kTall ? at + j : line, c = kTall ? line : at + j;
        return sm + S::kX + (c >> 7) * 2 * kSmallPlane + float_offset(r, c & 127);
      };
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        if (j >= unit) break;
        if (unit == 1) {
          v[0] = *reinterpret_cast<const float*>(place(0));
        } else if (kTall) {
#pragma unroll
          for (int w = 0; w < 4; ++w) v[j + w] = *reinterpret_cast<const float*>(place(j + w));
        } else {
          const float4 x = *reinterpret_cast<const float4*>(place(j));
          v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
        }
      }
      char* const to = out + (from + (int64_t)line * p.ld + at) * size;
      if (unit == 1) {
        if (p.type == PX_F32) *(float*)to = v[0];
        else if (p.type == PX_F16) *(__half*)to = __float2half_rn(v[0]);
        else *(bf16*)to = __float2bfloat16_rn(v[0]);
      } else if (p.type == PX_F32) {
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      } else if (p.type == PX_F16) {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack_f16x2_inf(v[0], v[1]), pack_f16x2_inf(v[2], v[3]), pack_f16x2_inf(v[4], v[5]), pack_f16x2_inf(v[6], v[7]));
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
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

template <int kSlices, bool kTall, bool kShort>
static bool launch_small_ortho(const SmallOrtho& p, int64_t batch, cudaStream_t st) {
  typedef SmallOrthoShape<kSlices> S;
  static SmemLimit limit;
  if (!limit.set(small_ortho_kernel<kSlices, kTall, kShort>, S::kSmem)) return false;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.ctas, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * p.ctas));
  cfg.blockDim = dim3(kSmallOrthoThreads + 32);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = p.ctas > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, small_ortho_kernel<kSlices, kTall, kShort>, p) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}
// CTAs of a matrix, 0: not this kernel.  us of five steps, bf16, with one slice a CTA | two: one CTA 37 to 42 | 59 to 61, two 60 to 64 | 83 to 86, four 67 to 74 | 94,
// eight 72 to 79 | 92 to 100, as often as the clusters take turns (148, 74, 32 or 14 fit); by products of their own launches, 33 to 40 matrices of 128 x 512 (four CTAs
// in two turns: 134) 131 to 140, 16 of 128 x 1024 (eight in two turns: 144) 149, 37 (four with two slices, in two turns: 176) 167.
static inline int small_ortho_ctas(int64_t batch, int64_t side, int64_t length, int steps, int* slices) {
  if (side > 128 || steps > kSmallSteps) return 0;
  static constexpr int kFit[4] = {148, 74, 32, 14}, kUs[4][2] = {{40, 60}, {62, 84}, {72, 95}, {78, 98}};
  const int64_t sms = sm_count();
  // launches of 6 us, and 0.7 us for each 64 k of the rounds of tiles
  const auto rounds = [&](int64_t tiles) { return (batch * tiles + sms - 1) / sms; };
  const int64_t along = (length + 127) / 128, sk = (side + 63) / 64;
  double best = 90.0 + 3.5 * (double)(rounds(1) * ((length + 63) / 64 + sk) + rounds(along) * sk);
  int ctas = 0;
  for (int i = 0; i < 4; ++i) {
    for (int n = 1; n <= 2; ++n) {
      if (along > (n << i) || (i && along <= (n << (i - 1)))) continue;      // too few, or more than are needed
      const int64_t fit = std::max<int64_t>(1, kFit[i] * sms / 148);
      const double us = (double)((batch + fit - 1) / fit * kUs[i][n - 1]);
      if (us < best) best = us, ctas = 1 << i, *slices = n;
    }
  }
  return ctas;
}
template <bool kShort>
static bool launch_small_ortho(const SmallOrtho& p, int64_t batch, int slices, bool tall, cudaStream_t st) {
  if (slices == 1) return tall ? launch_small_ortho<1, true, kShort>(p, batch, st) : launch_small_ortho<1, false, kShort>(p, batch, st);
  return tall ? launch_small_ortho<2, true, kShort>(p, batch, st) : launch_small_ortho<2, false, kShort>(p, batch, st);
}
static bool launch_small_ortho(const SmallOrtho& p, int64_t batch, int slices, bool tall, cudaStream_t st) {
  return p.side <= 112 ? launch_small_ortho<true>(p, batch, slices, tall, st) : launch_small_ortho<false>(p, batch, slices, tall, st);
}

}  // namespace px
