// Gradients of windowed attention (part of window_attention.cu).  With P recomputed from the forward pass's lse:
//   dV = P^T dO;  dP = dO V^T;  delta_i = dO_i . O_i;  dS = P (dP - delta);  dQ = scale dS K;  dK = scale dS^T Q;
//   dbias[head][b] = sum of dS over the pairs of bucket b.
// Two kernels of one form, each with its own rows in shared memory and a loop over streamed tiles of 64, so that every sum has one owner and a
// fixed order (no atomics): window_dq_kernel owns 128 queries and streams keys; it also sums delta (and leaves it for the other) and the bias's
// gradient.  window_dkv_kernel owns 128 keys and streams the queries that see them, those of all heads of the group one after the other.
// The price is S and dP twice: seven products a tile pair in place of five.
//
// Eight compute warps, a thread = one row x 32 of the 64 columns (no reduction along a row is needed here), one warp for copies and
// products.  dS and P are rounded to the operands' type for the products they enter and stay fp32 in the bias's gradient.
//
// Keys that are sinks are seen by all later queries.  Their CTA takes the queries of the window, like any other; the
// queries beyond are cut into chunks of about as many tiles, a CTA each, and window_sink_kernel adds the chunks up in their order.
#pragma once
#include "px_window.cuh"

namespace px {

constexpr int kWBwdThreads = 288;

struct WindowBwdArgs {
  const float* lse;              // [batch * heads][npad], base 2; +inf for rows that see nothing and beyond the last
  float* delta;                  // the same shape
  float* dbias;                  // partial sums [batch * heads * tiles][2 r + 1] or NULL
  float* sinks;                  // partial sums [batch * kv_heads][sink_tiles][1 + chunks][2][128][dn] (dK, dV)
  float scale;
  int sink_tiles, chunks, chunk; // chunk: streamed tiles of one
};

struct WindowBwdBars {
  uint64_t own_full, first_full[2], second_full[2], ready, given, done;      // streamed operands; S and dP; P and dS; the products with them
  uint32_t tmem_base;
};

// ---- dQ, delta, dbias ------------------------------------------------------------------------------------------------
// TMEM: S (64) | dP (64) | dQ (64 or 128); dS in the place of S.
template <int kPanels>
struct WindowDqLayout {
  static constexpr int stages = kPanels == 1 ? 2 : 1, tile = kPanels * kWCols * 128;
  static constexpr int q = 0, dout = kPanels * kWRows * 128, k = 2 * dout, v = k + stages * tile, bars = v + stages * tile;
  static constexpr int part = bars + 128, bias = part + 2 * kWRows * 4;
  static constexpr int bytes(int r, bool grad) { return bias + bias_floats(r) * 4 * (grad ? 9 : 1) + (grad ? 8 * 32 * 4 : 0); }
};
static_assert(sizeof(WindowBwdBars) <= 128, "room for the barriers");

template <bool kF16, int kPanels, bool kBiasGrad>
__global__ void __launch_bounds__(kWBwdThreads, 2)
window_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const WindowArgs a, const WindowBwdArgs g, const RowsOut dout, const RowsOut o,
                 const RowsOut dq) {
  typedef WindowDqLayout<kPanels> L;
  constexpr uint32_t kCols = 256;
  constexpr int kStages = L::stages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowBwdBars& bars = *reinterpret_cast<WindowBwdBars*>(sm + L::bars);
  float* const part = reinterpret_cast<float*>(sm + L::part);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int q0 = (int)(blockIdx.x % a.tiles) * kWRows, bh = blockIdx.x / a.tiles, head = bh % a.heads, batch = bh / a.heads;
  const KeyTiles tiles(a, q0);

  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    prefetch_maps(map_q, map_do, map_k, map_v);
    mbar_init(&bars.own_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.first_full[s], 1);
      mbar_init(&bars.second_full[s], 1);
    }
    mbar_init(&bars.ready, 1);
    mbar_init(&bars.given, 8);
    mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) tmem_alloc(&bars.tmem_base, kCols);
  if (!cta_ready(skip, warp == 8, bars.tmem_base, kCols)) return;
  const uint32_t tmem = bars.tmem_base;
  const int ext = bias_floats(a.r);
  if (a.r >= 0) {
    bias_fill(a, head, bias);
    if (kBiasGrad)
      for (int k = threadIdx.x; k < 8 * ext; k += kWBwdThreads) bias[ext + k] = 0.f;
  }
  __syncthreads();

  float low = 0.f, high = 0.f;                     // sums of dS over offsets that are clipped
  if (warp == 8) {
    // ------------------------------------------------------------------ copies and products
    const int kv = head / a.group;
    const uint32_t q_at = smem_u32(sm), do_at = smem_u32(sm + L::dout), k_at = smem_u32(sm + L::k), v_at = smem_u32(sm + L::v);
    const uint32_t idesc_s = umma_idesc_16(128, kWCols, kF16, kF16), idesc_q = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const int steps = (a.d + 15) / 16;
    const auto load = [&](int t, uint64_t* full, const CUtensorMap* map, uint32_t at) {      // one lane
      const int s = t % kStages;
      mbar_expect_tx(&full[s], L::tile);
      load_rows<kPanels>(at + s * L::tile, map, &full[s], kWCols, tiles.key(t), kv, batch);
    };
    const auto issue = [&](int t) {
      const int s = t % kStages, parity = (t / kStages) & 1;
      if (!mbar_wait_warp(&bars.first_full[s], parity, 2u) || !mbar_wait_warp(&bars.second_full[s], parity, 4u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows(tmem, q_at, k_at + s * L::tile, kWCols, steps, idesc_s);
        mma_rows(tmem + kWCols, do_at, v_at + s * L::tile, kWCols, steps, idesc_s);
        umma_commit(&bars.ready);
      }
      __syncwarp();
      return true;
    };
    if (elect_lane()) {
      mbar_expect_tx(&bars.own_full, 2 * kPanels * kWRows * 128);
      load_rows<kPanels>(q_at, &map_q, &bars.own_full, kWRows, q0, head, batch);
      load_rows<kPanels>(do_at, &map_do, &bars.own_full, kWRows, q0, head, batch);
      for (int t = 0; t < kStages && t < tiles.count; ++t) {
        load(t, bars.first_full, &map_k, k_at);
        load(t, bars.second_full, &map_v, v_at);
      }
    }
    __syncwarp();
    bool ok = mbar_wait_warp(&bars.own_full, 0, 1u) && issue(0);
    for (int t = 0; t < tiles.count && ok; ++t) {
      ok = mbar_wait_warp(&bars.given, t & 1, 8u);            // dS(t) is there; S(t) and dP(t) are complete: V's tile is free
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        mma_streamed(tmem + 2 * kWCols, tmem, k_at + (t % kStages) * L::tile, idesc_q, t == 0);
        umma_commit(&bars.done);
        if (t + kStages < tiles.count) load(t + kStages, bars.second_full, &map_v, v_at);
      }
      __syncwarp();
      ok = mbar_wait_warp(&bars.done, t & 1, 16u);            // K's tile and the place of S are free
      if (!ok) break;
      if (t + kStages < tiles.count && elect_lane()) load(t + kStages, bars.first_full, &map_k, k_at);
      __syncwarp();
      if (t + 1 < tiles.count) ok = issue(t + 1);
    }
  } else {
    // ------------------------------------------------------------------ one query row x 32 keys a thread
    const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane, i = q0 + row;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    // delta = dO . O, each thread over its half of the 16-byte pieces of the row
    float sum = 0.f;
    if (i < a.n) {
      const uint16_t *x = dout.at(batch, head, i), *y = o.at(batch, head, i);
      for (int c = 8 * half; c < a.d; c += 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + c)), v = __ldg(reinterpret_cast<const uint4*>(y + c));
        const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 p = unpack16x2<kF16>(us[e]), q = unpack16x2<kF16>(vs[e]);
          sum = fmaf(p.x, q.x, fmaf(p.y, q.y, sum));
        }
      }
    }
    part[half * kWRows + row] = sum;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    const float delta = part[row] + part[kWRows + row];
    if (half == 0) g.delta[(size_t)bh * a.npad + i] = delta;      // 0 beyond the last row
    const float lse = g.lse[(size_t)bh * a.npad + i];
    float* const sums = bias + ext * (1 + warp);                   // by offset, as the bias lies
    float* const stage = bias + ext * 9 + 32 * warp;
    bool ok = true;
    for (int t = 0; t < tiles.count; ++t) {
      const int k0 = tiles.key(t), kh = k0 + 32 * half;
      const uint64_t keys = key_bits(a, batch, k0, lane);
      const bool whole = keys == ~0ull && window_covers(a, q0, k0);
      ok = mbar_wait(&bars.ready, t & 1, 32u);
      __syncwarp();
      tc_fence_after();
      float s[32], d[32];
      tmem_ld32(t_lane + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
      tmem_ld32(t_lane + kWCols + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
      tmem_wait_ld();
      // all of S has to be read before any of dS goes where it lies
      tc_fence_before();
      ok = barrier_all(2 + quarter, 64, ok);
      if (!ok) break;
      tc_fence_after();
      const int lowest = kh - (q0 + 32 * quarter + 31), highest = kh + 31 - (q0 + 32 * quarter);      // offsets of this warp's block
      const bool flat_low = a.r >= 0 && clipped_low(a, highest), flat_high = a.r >= 0 && clipped_high(a, lowest);
      const bool near = a.r >= 0 && !flat_low && !flat_high;
      const float shift = (flat_low ? bias[0] : flat_high ? bias[ext - 1] : 0.f) - lse;
      if (near) {
        const float* b = bias + (kh - i + a.r + kWBiasBeyond);
#pragma unroll
        for (int c = 0; c < 32; ++c) s[c] = fast_exp2(fmaf(s[c], a.c, shift + b[c]));
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) s[c] = fast_exp2(fmaf(s[c], a.c, shift));
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) d[c] = s[c] * (d[c] - delta);
      if (!whole) {
        const uint32_t seen = (uint32_t)(visible_bits(a, i, k0, keys) >> (32 * half));
#pragma unroll
        for (int c = 0; c < 32; ++c) d[c] = (seen >> c & 1u) ? d[c] : 0.f;
      }
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) w[e] = pack16x2<kF16>(d[2 * e], d[2 * e + 1]);
      tmem_st16(t_lane + 16 * half, w);
      if (keys != bits_between(0, a.n - 1 - k0)) {  // masked keys: their rows of K
        mbar_wait(&bars.first_full[t % kStages], (t / kStages) & 1, 128u);      // complete: S(t) is; orders these writes behind the copy's
        const int r64 = threadIdx.x & 63;
        if (!(keys >> r64 & 1)) clear_row<kPanels>(sm + L::k + (t % kStages) * L::tile, r64, threadIdx.x >> 6, 4);
        fence_async_shared();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.given);
      if (kBiasGrad) {
        if (near) {
          // Sums along the diagonals of a 32 x 32 block: the running sum moves one lane on with each column, and leaves by the last lane.
          float run = 0.f;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            run = __shfl_up_sync(0xffffffffu, run, 1);
            run = (lane == 0 ? 0.f : run) + d[c];
            if (lane == 31) stage[c] = run;         // offset c - 31 of the block is complete
          }
          __syncwarp();
          float* const at = sums + (kh - (q0 + 32 * quarter) + a.r + kWBiasBeyond);
          at[lane - 31] += stage[lane];
          __syncwarp();
          if (lane < 31) at[31 - lane] += run;
          __syncwarp();
        } else {
          float v = 0.f;
#pragma unroll
          for (int c = 0; c < 32; ++c) v += d[c];
          if (flat_low) low += v;
          else high += v;
        }
      }
    }
    ok = ok && mbar_wait(&bars.done, (tiles.count - 1) & 1, 64u);
    ok = __all_sync(0xffffffffu, ok);
    if (ok && dq.data) {
      tc_fence_after();
      uint16_t* const out = dq.at(batch, head, i);
      for (int c = 16 * half; c < a.d; c += 32) {
        uint32_t x[16];
        tmem_ld16(t_lane + 2 * kWCols + c, x);
        tmem_wait_ld();
        if (i < a.n) {
          store8<kF16>(out + c, x, g.scale);
          if (c + 8 < a.d) store8<kF16>(out + c + 8, x + 8, g.scale);
        }
      }
    }
    if (kBiasGrad) {
      low = warp_sum(low);
      high = warp_sum(high);
      if (lane == 0) part[warp] = low, part[8 + warp] = high;
    }
  }
  tc_fence_before();
  cta_teardown_sync();
  if (warp == 8) {
    tc_fence_after();
    tmem_free(tmem, kCols);
  }
  if (kBiasGrad) {
    float* const out = g.dbias + (size_t)blockIdx.x * (2 * a.r + 1);
    for (int b = threadIdx.x; b < 2 * a.r + 1; b += kWBwdThreads) {
      float v = 0.f;
      for (int k = 0; k < 8; ++k) {
        const float* const s = bias + ext * (1 + k);
        v += s[b + kWBiasBeyond];
        if (b == 0) {
          for (int e = 0; e < kWBiasBeyond; ++e) v += s[e];
          v += part[k];
        }
        if (b == 2 * a.r) {
          for (int e = b + kWBiasBeyond + 1; e < ext; ++e) v += s[e];
          v += part[8 + k];
        }
      }
      out[b] = v;
    }
  }
}

// dbias[head][b] of the CTAs' sums, in their order: 32 buckets a block, 32 slices of the CTAs of a head.
__global__ void __launch_bounds__(1024) window_dbias_kernel(const float* __restrict__ partial, void* __restrict__ dbias, int type, int batches, int heads,
                                                            int tiles, int buckets) {
  __shared__ float slice[32][33];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, b = blockIdx.x * 32 + lane, head = blockIdx.y;
  float v = 0.f;
  if (b < buckets)
    for (int k = s; k < batches * tiles; k += 32)
      v += partial[((size_t)((k / tiles) * heads + head) * tiles + k % tiles) * buckets + b];
  slice[s][lane] = v;
  __syncthreads();
  if (s == 0 && b < buckets) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) sum += slice[e][lane];
    const size_t at = (size_t)head * buckets + b;
    if (type == PX_F32) ((float*)dbias)[at] = sum;
    else if (type == PX_BF16) ((bf16*)dbias)[at] = __float2bfloat16_rn(sum);
    else ((__half*)dbias)[at] = __float2half_rn(sum);
  }
}

// ---- dK, dV ----------------------------------------------------------------------------------------------------------
// TMEM: S^T (64) | dP^T (64) | dV | dK (64 or 128 each); P^T and dS^T in the places of S^T and dP^T.
template <int kPanels>
struct WindowDkvLayout {
  static constexpr int tile = kPanels * kWCols * 128, stat = 2 * kWCols * 4;
  static constexpr int k = 0, v = kPanels * kWRows * 128, q = 2 * v, dout = q + 2 * tile, stats = dout + 2 * tile, bars = stats + 2 * stat;
  static constexpr int bias = bars + 128;
  static constexpr int bytes(int r) { return bias + bias_floats(r) * 4; }
};

// The queries of one CTA: streamed tiles first .. first + count - 1 of `per` a head, over the heads of the group.
struct QueryTiles {
  int first, per, begin, count;      // begin: the first of the items head-of-group * per + tile
  __device__ __forceinline__ int query(int it) const { return (first + (begin + it) % per) * kWCols; }
  __device__ __forceinline__ int member(int it) const { return (begin + it) / per; }
};
__host__ __device__ __forceinline__ int last_of_window(int n, int left, int k0) {      // last streamed tile of the window of 128 keys
  return (k0 + kWRows - 1 + left < n - 1 ? k0 + kWRows - 1 + left : n - 1) / kWCols;
}

template <bool kF16, int kPanels>
__global__ void __launch_bounds__(kWBwdThreads, kPanels == 1 ? 2 : 1)
window_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const WindowArgs a, const WindowBwdArgs g, const RowsOut dk, const RowsOut dv) {
  typedef WindowDkvLayout<kPanels> L;
  constexpr uint32_t kCols = kPanels == 1 ? 256 : 512;
  constexpr int kAcc = 64 * kPanels;             // columns of an accumulator
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowBwdBars& bars = *reinterpret_cast<WindowBwdBars*>(sm + L::bars);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  // the chunks of the sinks first: they are the longest
  const int extra = g.sink_tiles * g.chunks, blocks = a.tiles + extra, bkv = blockIdx.x / blocks, at = blockIdx.x % blocks;
  const int kv = bkv % a.kv_heads, batch = bkv / a.kv_heads;
  const int own = at < extra ? at / g.chunks : at - extra, k0 = own * kWRows;
  const int last = last_of_window(a.n, a.left, k0);
  QueryTiles tiles;
  if (at < extra) {
    tiles.first = last + 1;
    tiles.per = max((a.n - 1) / kWCols - last, 1);
    tiles.begin = at % g.chunks * g.chunk;
    tiles.count = min(g.chunk, ((a.n - 1) / kWCols - last) * a.group - tiles.begin);       // none where the chunks of an earlier tile are more
  } else {
    tiles.first = max(0, k0 - a.right) / kWCols;
    tiles.per = last - tiles.first + 1;
    tiles.begin = 0;
    tiles.count = tiles.per * a.group;
  }

  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    prefetch_maps(map_q, map_do, map_k, map_v);
    mbar_init(&bars.own_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.first_full[s], 1);
      mbar_init(&bars.second_full[s], 1);
    }
    mbar_init(&bars.ready, 1);
    mbar_init(&bars.given, 8);
    mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) tmem_alloc(&bars.tmem_base, kCols);
  if (!cta_ready(skip, warp == 8, bars.tmem_base, kCols)) return;
  const uint32_t tmem = bars.tmem_base;
  const int own_key = min(k0 + (int)(threadIdx.x & 127), a.n - 1);
  const bool masked = a.mask && __ldg(a.mask + (size_t)batch * a.n + own_key) == 0;
  const bool any_masked = __syncthreads_or(masked) != 0;

  if (warp == 8) {
    // ------------------------------------------------------------------ copies and products
    const uint32_t k_at = smem_u32(sm), v_at = smem_u32(sm + L::v), q_at = smem_u32(sm + L::q), do_at = smem_u32(sm + L::dout);
    const uint32_t idesc_s = umma_idesc_16(128, kWCols, kF16, kF16), idesc_d = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const int steps = (a.d + 15) / 16;
    const auto load = [&](int t) {      // one lane: Q, dO and the rows' statistics
      const int s = t & 1, head = kv * a.group + tiles.member(t), q0 = tiles.query(t);
      mbar_expect_tx(&bars.first_full[s], 2 * L::tile + L::stat);
      load_rows<kPanels>(q_at + s * L::tile, &map_q, &bars.first_full[s], kWCols, q0, head, batch);
      load_rows<kPanels>(do_at + s * L::tile, &map_do, &bars.first_full[s], kWCols, q0, head, batch);
      const size_t row = (size_t)(batch * a.heads + head) * a.npad + q0;
      bulk_load(sm + L::stats + s * L::stat, g.lse + row, kWCols * 4, &bars.first_full[s]);
      bulk_load(sm + L::stats + s * L::stat + kWCols * 4, g.delta + row, kWCols * 4, &bars.first_full[s]);
    };
    const auto issue = [&](int t) {
      const int s = t & 1;
      if (!mbar_wait_warp(&bars.first_full[s], (t >> 1) & 1, 2u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows(tmem, k_at, q_at + s * L::tile, kWCols, steps, idesc_s);
        mma_rows(tmem + kWCols, v_at, do_at + s * L::tile, kWCols, steps, idesc_s);
        umma_commit(&bars.ready);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    if (tiles.count > 0) {
      if (elect_lane()) {
        mbar_expect_tx(&bars.own_full, 2 * kPanels * kWRows * 128);
        load_rows<kPanels>(k_at, &map_k, &bars.own_full, kWRows, k0, kv, batch);
        load_rows<kPanels>(v_at, &map_v, &bars.own_full, kWRows, k0, kv, batch);
        for (int t = 0; t < 2 && t < tiles.count; ++t) load(t);
      }
      __syncwarp();
      ok = mbar_wait_warp(&bars.own_full, 0, 1u) && issue(0);
    }
    for (int t = 0; t < tiles.count && ok; ++t) {
      ok = mbar_wait_warp(&bars.given, t & 1, 8u);
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        const int s = t & 1;
        mma_streamed(tmem + 2 * kWCols, tmem, do_at + s * L::tile, idesc_d, t == 0);
        mma_streamed(tmem + 2 * kWCols + kAcc, tmem + kWCols, q_at + s * L::tile, idesc_d, t == 0);
        umma_commit(&bars.done);
      }
      __syncwarp();
      ok = mbar_wait_warp(&bars.done, t & 1, 16u);            // the streamed tile and the places of S^T and dP^T are free
      if (!ok) break;
      if (t + 2 < tiles.count && elect_lane()) load(t + 2);
      __syncwarp();
      if (t + 1 < tiles.count) ok = issue(t + 1);
    }
  } else {
    // ------------------------------------------------------------------ one key row x 32 queries a thread
    const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane, j = k0 + row;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    bool ok = true;
    int filled = -1;                               // the group's head whose bias is in shared memory
    const int wide = a.r >= 0 && a.group > 1;      // the bias changes on the way: all eight warps keep together
    for (int t = 0; t < tiles.count; ++t) {
      const int q0 = tiles.query(t), qh = q0 + 32 * half, s = t & 1, member = tiles.member(t);
      if (a.r >= 0 && member != filled) {
        // all are past the tile before (barrier below), but not all are through with it
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        for (int k = threadIdx.x; k < bias_floats(a.r); k += 256)
          bias[k] = bias_value(a, kv * a.group + member, min(max(k - kWBiasBeyond, 0), 2 * a.r));
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        filled = member;
      }
      ok = mbar_wait(&bars.ready, t & 1, 32u);
      // the statistics came with the operands; this wait only makes the copy's writes visible here
      ok = mbar_wait(&bars.first_full[s], (t >> 1) & 1, 64u) && ok;
      __syncwarp();
      tc_fence_after();
      float p[32], d[32];
      tmem_ld32(t_lane + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&p[0]));
      tmem_ld32(t_lane + kWCols + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
      tmem_wait_ld();
      tc_fence_before();
      ok = barrier_all(wide ? 1 : 2 + quarter, wide ? 256 : 64, ok);      // both halves have read what is overwritten below
      if (!ok) break;
      tc_fence_after();
      const float4* const lse4 = reinterpret_cast<const float4*>(sm + L::stats + s * L::stat) + 8 * half;
      const float4* const delta4 = lse4 + kWCols / 4;
      const int lowest = k0 + 32 * quarter - (qh + 31), highest = k0 + 32 * quarter + 31 - qh;
      const bool flat_low = a.r >= 0 && clipped_low(a, highest), flat_high = a.r >= 0 && clipped_high(a, lowest);
      const float flat = flat_low ? bias[0] : flat_high ? bias[bias_floats(a.r) - 1] : 0.f;
      const bool near = a.r >= 0 && !flat_low && !flat_high;
      const float* const b = bias + (near ? j - qh + a.r + kWBiasBeyond : 0);
      const bool whole = !any_masked && k0 + kWRows - 1 <= q0 + a.right && q0 + kWCols - 1 <= k0 + a.left && q0 + kWCols <= a.n;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 l4 = lse4[c], e4 = delta4[c];
        const float l[4] = {l4.x, l4.y, l4.z, l4.w}, e[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float add = (near ? b[-(4 * c + x)] : flat) - l[x];
          p[4 * c + x] = fast_exp2(fmaf(p[4 * c + x], a.c, add));
          d[4 * c + x] = p[4 * c + x] * (d[4 * c + x] - e[x]);
        }
      }
      bool nothing = false;                        // a query of this tile that sees nothing: its rows of Q and dO may hold anything
      if (!whole) {
        // queries j - right .. j + left, all from j - right on for a sink, none for a masked key
        const int from = j - a.right - qh, to = masked ? -1 : j < a.sinks ? 31 : min(31, j + a.left - qh);
        const uint32_t seen = (uint32_t)bits_between(from, to);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const bool see = seen >> c & 1u;
          p[c] = see ? p[c] : 0.f;
          d[c] = see ? d[c] : 0.f;
        }
      }
      {
        const float* const all = reinterpret_cast<const float*>(sm + L::stats + s * L::stat);
        nothing = __any_sync(0xffffffffu, all[lane] == CUDART_INF_F || all[32 + lane] == CUDART_INF_F);
        if (nothing) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 l4 = lse4[c];
            const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (l[x] == CUDART_INF_F) p[4 * c + x] = d[4 * c + x] = 0.f;
          }
          const int r64 = threadIdx.x & 63;
          if (all[r64] == CUDART_INF_F) {
            clear_row<kPanels>(sm + L::q + s * L::tile, r64, threadIdx.x >> 6, 4);
            clear_row<kPanels>(sm + L::dout + s * L::tile, r64, threadIdx.x >> 6, 4);
          }
          fence_async_shared();
        }
      }
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) w[e] = pack16x2<kF16>(p[2 * e], p[2 * e + 1]);
      tmem_st16(t_lane + 16 * half, w);
#pragma unroll
      for (int e = 0; e < 16; ++e) w[e] = pack16x2<kF16>(d[2 * e], d[2 * e + 1]);
      tmem_st16(t_lane + kWCols + 16 * half, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.given);
    }
    if (tiles.count > 0) {
      ok = ok && mbar_wait(&bars.done, (tiles.count - 1) & 1, 128u);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
      const int dn = (a.d + 15) & ~15;
      // where the key is a sink with chunks, this is one of the sums that window_sink_kernel adds up: its own first, then the chunks
      const bool summed = g.chunks > 0 && own < g.sink_tiles;
      float* const to = g.sinks + (((size_t)bkv * g.sink_tiles + own) * (1 + g.chunks) + (at < extra ? 1 + at % g.chunks : 0)) * 2 * kWRows * dn +
                        (size_t)row * dn;
      for (int which = 0; which < 2; ++which) {      // dK, dV
        const RowsOut& out = which ? dv : dk;
        const float scale = which ? 1.f : g.scale;
        if (!out.data) continue;
        for (int c = 16 * half; c < a.d; c += 32) {
          uint32_t x[16];
          if (tiles.count > 0) {
            tmem_ld16(t_lane + 2 * kWCols + (which ? 0 : kAcc) + c, x);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 0u;
          }
          if (summed) {
            float* const f = to + which * kWRows * dn + c;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(f + e) = make_float4(__uint_as_float(x[e]) * scale, __uint_as_float(x[e + 1]) * scale,
                                                              __uint_as_float(x[e + 2]) * scale, __uint_as_float(x[e + 3]) * scale);
          } else if (j < a.n) {
            uint16_t* const p = out.at(batch, kv, j) + c;
            store8<kF16>(p, x, scale);
            if (c + 8 < a.d) store8<kF16>(p + 8, x + 8, scale);
          }
        }
      }
    }
  }
  tc_fence_before();
  cta_teardown_sync();
  if (warp == 8) {
    tc_fence_after();
    tmem_free(tmem, kCols);
  }
}

// Rows of dK and dV that the chunks of the sinks have parts of: thread = 8 values.
template <bool kF16>
__global__ void __launch_bounds__(256) window_sink_kernel(const WindowArgs a, const WindowBwdArgs g, const RowsOut dk, const RowsOut dv) {
  const int dn = (a.d + 15) & ~15, pieces = a.d / 8, rows = min(a.n, g.sink_tiles * kWRows), per = (2 * rows * pieces + 255) / 256;
  const int bkv = blockIdx.x / per, u = blockIdx.x % per * 256 + threadIdx.x;
  if (u >= 2 * rows * pieces) return;
  const int c = u % pieces * 8, j = u / pieces % rows, which = u / pieces / rows;
  const RowsOut& out = which ? dv : dk;
  if (!out.data) return;
  const float* from = g.sinks + ((size_t)bkv * g.sink_tiles + j / kWRows) * (1 + g.chunks) * 2 * kWRows * dn + (size_t)which * kWRows * dn +
                      (size_t)(j % kWRows) * dn + c;
  float v[8] = {};
  for (int k = 0; k <= g.chunks; ++k, from += 2 * kWRows * dn) {
    const float4 x = *reinterpret_cast<const float4*>(from), y = *reinterpret_cast<const float4*>(from + 4);
    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
  }
  store8<kF16>(out.at(bkv / a.kv_heads, bkv % a.kv_heads, j) + c, reinterpret_cast<const uint32_t*>(v), 1.f);
}

}  // namespace px
