// The cross entropy of a head with up to 128 channels and 128 classes (bins over pairs of tokens): one pass over x forward, one backward.
//
// The weight stays in shared memory and the rows go through once.  Forward, a tile of 128 rows: logits = x W^T into tensor memory, a thread a row
// forms the loss.  Backward: logits again, a thread a row writes dl in 16 bits to shared memory, and both gradients are products with that same
// tile, dx = dl W (dl along the classes, W across) and dW^T += x^T dl (both across), dW^T staying in tensor memory until the CTA's last tile.  The
// sums of the CTAs are joined in their order (backward, rows beyond what a CTA's dW^T may add up go through another launch).  Bytes: x once forward; x and dx once backward.  (Through the general path dl would be written and read
// twice, 16 bits a class: 768^2 rows, 128 channels, 64 classes 664 us in all.)
//
// Rows that are ignored: dl zero by selection, and their x is zeroed in shared memory before the product for dW reads it.
//
// Roles: warp 0 copies rows in, warp 1 issues products, sets of four warps are the rows of the softmax and take the tiles in turn (four sets
// forward, two backward); backward four more warps round dx and store it.  The logits of tile i + 1 are issued before the gradients of tile i.
//
// 768^2 rows, 128 channels, 64 classes, bf16, a bias, a fifth of the rows ignored: 34 us forward (4.6 TB/s of a copy's 6.5), 72 backward (4.3), 125 a training pass.  What
// bounds both is the chain of a tile in its rows' threads (copy, product, tensor memory, exponentials, 47 % of the issue slots); backward with one set of
// softmax warps, which fetched targets and references when it came to them, 120.
#pragma once
#include "px_head.cuh"

namespace px {

constexpr int kSmallC = 128, kSmallV = 128;
constexpr int kSmallPanel = 128 * 128;                    // [128 rows][64 channels or classes] in 16 bits

struct SmallArgs {
  CUtensorMap x, w, dx;
  const int64_t* target;
  HeadBias bias;
  float2* norm;
  float* losses;                                          // forward: of the rows, or NULL
  double2* sums;                                          // forward: [CTAs] sum and number of the losses
  LossOut out;                                            // backward
  float* part_w;                                          // backward: [CTAs][128][kVp], or NULL
  float* part_b;                                          // backward: [8 CTAs][kVp], or NULL
  int64_t ignore;
  int rows, classes, panels, tiles, f16, want_dx;
  float smooth, uncut;
  uint32_t idesc_logits, idesc_dx, idesc_dw;
};

template <bool kBackward, int kVp>
struct SmallShape {
  static constexpr int kStages = kBackward ? 3 : 5, kSets = kBackward ? 2 : 4;
  static constexpr int kThreads = 64 + 128 * kSets + (kBackward ? 128 : 0);
  static constexpr int kXBytes = 2 * kSmallPanel, kWBytes = 2 * kVp * 128, kDlBytes = kVp / 64 * kSmallPanel;
  static constexpr int kW = kStages * kXBytes, kDl = kW + kWBytes, kStg = kDl + (kBackward ? 2 * kDlBytes : 0);
  static constexpr int kBias = kStg + (kBackward ? 4 * 2 * 4096 : 0), kBars = kBias + kVp * 4;
  static constexpr size_t kSmem = kBars + 256 + 1024;
  static_assert(kSmem <= 232448, "shared memory budget");
  // tensor memory: logits (one for each set, which then sees every phase of its barrier), dx (twice, where there is room), dW^T
  static constexpr int kDxs = kVp == 128 ? 1 : 2;
  static constexpr uint32_t kDx = kSets * kVp, kDw = kDx + 128 * kDxs, kCols = kBackward ? 512 : kSets * kVp;
  static_assert(!kBackward || kDw + kVp <= 512, "tensor memory");
};
struct SmallBarriers {
  uint64_t w_full, x_full[5], x_empty[5], logit_full[4], logit_empty[4], dl_full[2], dl_empty[2], dx_full[2], dx_empty[2], done;
  uint32_t tmem_base;
};
static_assert(sizeof(SmallBarriers) <= 256, "barriers");

template <bool kBackward, int kVp>
__global__ void __launch_bounds__(SmallShape<kBackward, kVp>::kThreads, 1) small_head_kernel(const __grid_constant__ SmallArgs a) {
  typedef SmallShape<kBackward, kVp> S;
  constexpr int kLogits = S::kSets, kDxs = S::kDxs;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  SmallBarriers& bars = *reinterpret_cast<SmallBarriers*>(sm + S::kBars);
  float* bias = reinterpret_cast<float*>(sm + S::kBias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool skip = cta_begin();
  if (threadIdx.x == 32) prefetch_maps(a.x, a.w, a.dx);
  if (threadIdx.x == 0) {
    mbar_init(&bars.w_full, 1);
    mbar_init(&bars.done, 1);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&bars.x_full[s], 1);
      mbar_init(&bars.x_empty[s], 1);
    }
    for (int b = 0; b < kLogits; ++b) {
      mbar_init(&bars.logit_full[b], 1);
      mbar_init(&bars.logit_empty[b], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars.dl_full[b], 4);
      mbar_init(&bars.dl_empty[b], 1);
      mbar_init(&bars.dx_full[b], 1);
      mbar_init(&bars.dx_empty[b], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(S::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  const bool work = cta_ready(skip, warp == 0, bars.tmem_base, S::kCols);
  if (!work) return;
  const uint32_t tmem = bars.tmem_base;
  if (threadIdx.x < kVp) {
    const float b = a.bias.at && (int)threadIdx.x < a.classes ? bias_value(a.bias, threadIdx.x) : 0.f;
    bias[threadIdx.x] = (int)threadIdx.x < a.classes ? b : -CUDART_INF_F;      // classes that are not there: no exponential
  }
  __syncthreads();

  if (warp == 0) {
    if (elect_lane()) {
      mbar_expect_tx(&bars.w_full, a.panels * kVp * 128);
      for (int p = 0; p < a.panels; ++p) tma_load_3d(smem_u32(sm + S::kW + p * kVp * 128), &a.w, &bars.w_full, 64 * p, 0, 0);
    }
    __syncwarp();
    int i = 0;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++i) {
      const int s = i % S::kStages;
      if (!mbar_wait_warp(&bars.x_empty[s], ((i / S::kStages) & 1) ^ 1, 1u)) break;
      if (elect_lane()) {
        mbar_expect_tx(&bars.x_full[s], a.panels * kSmallPanel);
        for (int p = 0; p < a.panels; ++p) tma_load_3d(smem_u32(sm + s * S::kXBytes + p * kSmallPanel), &a.x, &bars.x_full[s], 64 * p, 128 * tile, 0);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const int mine = a.tiles > (int)blockIdx.x ? (a.tiles - (int)blockIdx.x - 1) / (int)gridDim.x + 1 : 0;
    bool ok = mbar_wait_warp(&bars.w_full, 0, 2u);
    auto logits = [&](int i) {
      const int s = i % S::kStages, b = i % kLogits;
      ok = ok && mbar_wait_warp(&bars.x_full[s], (i / S::kStages) & 1, 4u) && mbar_wait_warp(&bars.logit_empty[b], ((i / kLogits) & 1) ^ 1, 8u);
      if (!ok) return;
      tc_fence_after();
      if (elect_lane()) {
        for (int p = 0; p < a.panels; ++p) {
          const uint64_t da = umma_desc_sw128(smem_u32(sm + s * S::kXBytes + p * kSmallPanel)), db = umma_desc_sw128(smem_u32(sm + S::kW + p * kVp * 128));
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma_bf16(tmem + b * kVp, da + 2 * ks, db + 2 * ks, a.idesc_logits, (p | ks) ? 1u : 0u);
        }
        if (!kBackward) umma_commit(&bars.x_empty[s]);
        umma_commit(&bars.logit_full[b]);              // last: what is waited for
      }
      __syncwarp();
    };
    if (mine > 0) logits(0);
    for (int i = 0; i < mine && ok; ++i) {
      if (i + 1 < mine) logits(i + 1);
      if constexpr (kBackward) {
        const int s = i % S::kStages, b = i & 1, d = i % kDxs;
        ok = ok && mbar_wait_warp(&bars.dl_full[b], (i >> 1) & 1, 16u) && mbar_wait_warp(&bars.dx_empty[d], ((i / kDxs) & 1) ^ 1, 32u);
        if (!ok) break;
        tc_fence_after();
        if (elect_lane()) {
          const uint32_t dl = smem_u32(sm + S::kDl + b * S::kDlBytes);
          const uint64_t al = umma_desc_sw128(dl), wl = umma_desc_mn_sw128(smem_u32(sm + S::kW), kVp * 128, 1024);
#pragma unroll
          for (int ks = 0; ks < kVp / 16; ++ks)
            umma_bf16(tmem + S::kDx + 128 * d, al + (ks >> 2) * (kSmallPanel >> 4) + 2 * (ks & 3), wl + 128 * ks, a.idesc_dx, ks > 0);
          umma_commit(&bars.dx_full[d]);
          const uint64_t xt = umma_desc_mn_sw128(smem_u32(sm + s * S::kXBytes), kSmallPanel, 1024), bl = umma_desc_mn_sw128(dl, kSmallPanel, 1024);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) umma_bf16(tmem + S::kDw, xt + 128 * ks, bl + 128 * ks, a.idesc_dw, (i | ks) ? 1u : 0u);
          umma_commit(&bars.x_empty[s]);
          umma_commit(&bars.dl_empty[b]);
          if (i == mine - 1) umma_commit(&bars.done);
        }
        __syncwarp();
      }
    }
    // Nothing else waits for the last products of a backward pass that wants no dW: they write tensor memory and arrive on barriers, so this warp stays until
    // they are through.
    if (kBackward && ok && mine > 0) mbar_wait_warp(&bars.done, 0, 1024u);
  } else if (warp < 2 + 4 * S::kSets) {
    // rows of the softmax
    const int q = warp & 3, set = (warp - 2) >> 2;
    constexpr int sets = S::kSets;
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
    double total = 0.0;
    int counted = 0;
    float db[kVp / 32] = {};
    float out = 0.f, each = 1.f;
    if constexpr (kBackward) {
      out = a.out();
      each = a.out.scale ? a.out.scale->each : 1.f;
    }
    int i = set;
    bool ok = true;
    int64_t next_t = a.ignore;
    float2 next_n = {};
    auto fetch = [&](int tile) {                            // a tile ahead
      const int row = 128 * tile + 32 * q + lane;
      if (tile < a.tiles && row < a.rows) {
        next_t = a.target[row];
        if (kBackward) next_n = a.norm[row];
      }
    };
    fetch(blockIdx.x + set * gridDim.x);
    for (int tile = blockIdx.x + set * gridDim.x; tile < a.tiles && ok; tile += sets * gridDim.x, i += sets) {
      const int b = i % kLogits, s = i % S::kStages, row = 128 * tile + 32 * q + lane;
      const int64_t t = next_t;
      const float2 n = next_n;
      fetch(tile + sets * gridDim.x);
      const bool counts = row < a.rows && row_counts(t, a.ignore), valid = t >= 0 && t < a.classes;
      const int mine = counts && valid ? (int)t : -1;
      ok = mbar_wait_warp(&bars.logit_full[b], (i / kLogits) & 1, 64u);
      if (!ok) break;
      tc_fence_after();
      if constexpr (!kBackward) {
        float m = -CUDART_INF_F, sum = 0.f, all = 0.f, hit = 0.f;
#pragma unroll
        for (int c = 0; c < kVp; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + b * kVp + c, r);
          tmem_wait_ld();
          if (c + 32 == kVp) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.logit_empty[b]);
          }
          float v[32];
          logits_of(r, a.uncut, v);
          add_bias(v, bias + c);
          if (a.smooth > 0.f) {
#pragma unroll
            for (int j = 0; j < 32; ++j) all += c + j < a.classes ? v[j] : 0.f;
          }
          if (mine >= c && mine < c + 32) hit = pick(v, mine - c);
          float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int j = 4; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], v[j]);
          const float next = fmaxf(m, kLog2e * fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), ref = reference(next);
          float e[4] = {sum * fast_exp2(m - ref), 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 32; ++j) e[j & 3] += fast_exp2(fmaf(v[j], kLog2e, -ref));
          sum = (e[0] + e[1]) + (e[2] + e[3]);
          m = next;
        }
        const float ref = reference(m);
        float loss = 0.f;
        if (counts) {
          loss = row_loss(sum, ref, hit, valid, a.smooth, all, a.classes);
          total += loss;
          ++counted;
        }
        if (row < a.rows) {
          a.norm[row] = make_float2(ref, sum);
          if (a.losses) a.losses[row] = loss;
        }
      } else {
        const int bl = i & 1;
        float factor = 0.f, ref = 0.f, over = 0.f;
        if (counts) {
          factor = a.out.scale ? a.out.grad[row] * each : 1.f;
          if (!valid) factor = CUDART_NAN_F;
          if (a.f16) factor *= kDlScaleF16;
          ref = -n.x, over = factor / n.y;
        }
        const float less = factor * a.smooth / (float)a.classes, less_hit = -less - factor * (1.f - a.smooth);
        ok = mbar_wait_warp(&bars.dl_empty[bl], ((i >> 1) & 1) ^ 1, 128u);
        if (!ok) break;
        unsigned char* const dl = sm + S::kDl + bl * S::kDlBytes;
        const int r128 = 32 * q + lane;
#pragma unroll
        for (int c = 0; c < kVp; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + b * kVp + c, r);
          tmem_wait_ld();
          if (c + 32 == kVp) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.logit_empty[b]);
          }
          float v[32];
          logits_of(r, a.uncut, v);
          add_bias(v, bias + c);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = fmaf(over, fast_exp2(fmaf(v[j], kLog2e, ref)), mine == c + j ? less_hit : -less);
          if (c + 32 > a.classes) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j >= a.classes) v[j] = 0.f;
          }
          if (!counts) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            uint32_t o[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) o[w] = a.f16 ? pack_f16x2_inf(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]) : pack_bf16x2(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]);
            *reinterpret_cast<uint4*>(dl + (c >> 6) * kSmallPanel + r128 * 128 + (((((c & 63) >> 3) + p) ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (a.part_b) {
            column_sums(v, lane);
            db[c / 32] += v[0];
          }
        }
        if (!counts) {
          for (int p = 0; p < 8 * a.panels; ++p)
            *reinterpret_cast<uint4*>(sm + s * S::kXBytes + (p >> 3) * kSmallPanel + r128 * 128 + ((p & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.dl_full[bl]);
      }
    }
    if constexpr (!kBackward) {
      if (a.sums) {
        // the CTA's sum in the order of its warps
        double2* const x = reinterpret_cast<double2*>(sm + S::kW);      // the weight is not read any more once all warps are here
        double n = counted;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o), n += __shfl_xor_sync(0xffffffffu, n, o);
        asm volatile("bar.sync 1, 512;\n" ::: "memory");
        if (lane == 0) x[warp - 2] = make_double2(total, n);
        asm volatile("bar.sync 1, 512;\n" ::: "memory");
        if (warp == 2 && lane == 0) {
          for (int w = 1; w < 16; ++w) total += x[w].x, n += x[w].y;
          a.sums[blockIdx.x] = make_double2(total, n);
        }
      }
    } else {
      if (a.part_b) {
#pragma unroll
        for (int c = 0; c < kVp / 32; ++c) a.part_b[((int64_t)blockIdx.x * 8 + (warp - 2)) * kVp + 32 * c + lane] = db[c] * out;
      }
      if (a.part_w && set == 0) {
        const bool any = (int)blockIdx.x < a.tiles;
        if (any) ok = ok && mbar_wait_warp(&bars.done, 0, 256u);
        tc_fence_after();
        float* const to = a.part_w + ((int64_t)blockIdx.x * 128 + 32 * q + lane) * kVp;
#pragma unroll
        for (int c = 0; c < kVp; c += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + S::kDw + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(to + c + j) =
                make_float4(out * __uint_as_float(r[j]), out * __uint_as_float(r[j + 1]), out * __uint_as_float(r[j + 2]), out * __uint_as_float(r[j + 3]));
        }
      }
    }
  } else {
    // dx
    const int q = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16) + S::kDx;
    const float out = a.out();
    int i = 0;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++i) {
      const int d = i % kDxs, row = 128 * tile + 32 * q + lane;
      const bool zero = row < a.rows && !row_counts(a.target[row], a.ignore);
      if (!mbar_wait_warp(&bars.dx_full[d], (i / kDxs) & 1, 512u)) break;
      tc_fence_after();
      for (int p = 0; p < a.panels; ++p) {
        unsigned char* const stg = sm + S::kStg + (2 * q + p) * 4096;
        if (p == 0) {
          if (lane == 0) tma_store_wait_read<0>();      // both panels of the tile before
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          uint32_t r[32];
          tmem_ld32(lanes + 128 * d + 64 * p + h, r);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t o[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float u = zero ? 0.f : out * __uint_as_float(r[8 * k + 2 * w]), v = zero ? 0.f : out * __uint_as_float(r[8 * k + 2 * w + 1]);
              o[w] = a.f16 ? pack_f16x2_inf(u, v) : pack_bf16x2(u, v);
            }
            *reinterpret_cast<uint4*>(stg + lane * 128 + (((h / 8 + k) ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        if (p == a.panels - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.dx_empty[d]);
        }
        if (a.want_dx) {
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (lane == 0 && 128 * tile + 32 * q < a.rows) {
            tma_store_3d(&a.dx, smem_u32(stg), 64 * p, 128 * tile + 32 * q, 0);
            tma_store_commit();
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_read<0>();
  }

  __syncwarp();
  tc_fence_before();
  cta_teardown_sync();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kCols) : "memory");
  }
}

// The total of what the CTAs of a forward pass have left, in their order.
__global__ void __launch_bounds__(32) small_total_kernel(const double2* __restrict__ sums, int ctas, float* __restrict__ total, float* __restrict__ inverse, int mean) {
  pdl_wait();
  double l = 0.0, c = 0.0;
  for (int i = threadIdx.x; i < ctas; i += 32) l += sums[i].x, c += sums[i].y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o), c += __shfl_xor_sync(0xffffffffu, c, o);
  if (threadIdx.x == 0) {
    *total = (float)(mean ? l / c : l);                   // the mean of nothing is NaN
    *inverse = mean ? (float)(1.0 / fmax(c, 1.0)) : 1.f;
  }
}
// dW and db from what the CTAs of a backward pass have left: a block for 32 classes of a channel (or, the last ones, of the bias), its warps along the
// CTAs, in a fixed order.
__global__ void __launch_bounds__(256) small_join_kernel(const float* __restrict__ part_w, const float* __restrict__ part_b, uint16_t* __restrict__ dw, void* __restrict__ db,
                                                         int ctas, int vp, int c, int classes, int f16, int db_type) {
  __shared__ float x[8][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, groups = vp / 32, v = (blockIdx.x % groups) * 32 + lane, ch = blockIdx.x / groups;
  const float* const p = ch < c ? part_w + (int64_t)ch * vp + v : part_b + v;
  const int64_t step = ch < c ? 128 * vp : vp;
  const int n = ch < c ? ctas : 8 * ctas;
  if (!(ch < c ? part_w : part_b)) return;
  float s[4] = {};
  for (int k = w; k < n; k += 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + 8 * j < n) s[j] += p[(k + 8 * j) * step];
  }
  x[w][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (w == 0 && v < classes) {
    float all = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) all += x[k][lane];
    if (ch == c)
      bias_store(db, db_type, v, all);
    else
      dw[(int64_t)v * c + ch] = f16 ? __half_as_ushort(__float2half_rn(all)) : __bfloat16_as_ushort(__float2bfloat16_rn(all));
  }
}

}  // namespace px
