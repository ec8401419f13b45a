// Gradients of windowed attention (part of window_attention.cu).  With P recomputed from the forward pass's lse:
//   dV = P^T dO;  dP = dO V^T;  delta_i = dO_i . O_i;  dS = P (dP - delta);  dQ = scale dS K;  dK = scale dS^T Q;
//   dbias[head][b] = sum of dS over the pairs of bucket b.
// A small kernel for delta, then two of one form, each with its own rows in shared memory and a loop over streamed tiles of 64, so that every sum has one
// owner and a fixed order (no atomics): window_dq_kernel owns 128 queries and streams keys; it also sums the bias's gradient. window_dkv_kernel owns 128 keys
// and streams the queries that see them, those of all heads of the group one after the other.  The price is S and dP twice: seven products a tile
// pair in place of five.
//
// The two are independent but for the sums of the bias, so the second lets its blocks in as soon as the last of the first's has begun: window_dq_kernel
// signals its dependents once its wait for window_delta_kernel is over, and a block of window_dkv_kernel waits for that grid only at its end (or, where it adds
// the bias's sums up, before it begins).  Neither fills a whole number of rounds over the SMs, and now they share the rest.
//
// Compute warps: a thread = one row x 32 of the 64 columns (no reduction along a row is needed here), x 16 where the block is alone on its SM.  Copies and
// products have one warp in the first kernel and two in the second, whose four products a step take an issuing warp some 1000 cycles beside busy ones
// (177 -> 168 us for a causal window of 1024 over 8192 tokens; in the first kernel two warps were slower, 142 us against 114).  dS and P are rounded to the
// operands' type for the products they enter and stay fp32 in the bias's gradient.  A dS or a gradient that fp16 cannot hold becomes infinite and what it enters
// infinite or NaN: clipped it would pass for a number, and a loss scaler would not learn that its scale is too large.
//
// What bounds them is, as forward, what the warps issue for a tile (exponentials, products, rounding, the bias's sums), and the latency of each
// warp's chain: issue slots 32 to 54 %, tensor pipe 26 to 48 %, with 16 row warps an SM, whose S, dP, P, dS and sums fill tensor memory.  At 8192 tokens, 16 heads of 64 over 4 of keys, causal window of 1024, from the first kernel's beginning to the last one's end: 252 us
// (280 one behind the other) for seven products of 16 GFLOP; 8 heads of 128 over 2: 207 us.  2 x 1237 tokens, 16 heads of 24, window 200 + 200: 60 (80).
// Atoms, five samples of 3987 with 4 heads of 32, windows of 128, a bias by offset: 55 (64).
//
// Keys that are sinks are seen by all later queries.  Their CTA takes the queries of the window, like any other; the
// queries beyond are cut into chunks of about as many tiles, a CTA each, and the last of these CTAs adds the chunks up in their order.
#pragma once
#include <type_traits>

#include "px_window.cuh"

namespace px {

constexpr int kWDqThreads = 288;      // eight warps of rows, one for copies and products

struct WindowBwdArgs {
  const float* nlse;             // [batch * heads][npad], base 2, negative; -inf for rows that see nothing and beyond the last
  float* ndelta;                 // -delta, the same shape
  float* dbias;                  // partial sums [batch * heads * tiles][2 r + 1] or NULL
  float* sinks;                  // partial sums [batch * kv_heads][sink_tiles][1 + chunks][2][128][dn] (dK, dV)
  unsigned int* arrived;         // [batch * kv_heads][sink_tiles]: how many of the sums are there
  void* dbias_out;               // [heads][2 r + 1], the type of the bias, or NULL
  float scale;
  int sink_tiles, chunks, chunk; // chunk: streamed tiles of one
  int bias_blocks, batches;      // blocks of 32 buckets a head
  bool own, early;               // dK or dV is wanted; window_dkv_kernel begins beside window_dq_kernel
};

// -delta = -dO . O, O with what its rounding has taken off: a group of lanes a row, a lane = 16 bytes; zeros beyond the last row.  Memory-bound.
__host__ __device__ constexpr int delta_rows(int lanes) { return lanes == 4 ? 2 : 4; }                      // of a group
__host__ __device__ constexpr int delta_block(int lanes) { return 256 / lanes * delta_rows(lanes); }     // of a block: 128 or 64, which divide npad
template <bool kF16, int kLanes>
__global__ void __launch_bounds__(256) window_delta_kernel(const WindowArgs a, const WindowBwdArgs g, const RowsOut dout, const RowsOut o, const RowsOut rest) {
  pdl_wait();
  if (blockIdx.x == 0)      // for window_dkv_kernel
    for (int k = threadIdx.x; k < g.batches * a.kv_heads * g.sink_tiles; k += 256) g.arrived[k] = 0u;
  constexpr int kRows = delta_rows(kLanes);
  const int lane = threadIdx.x % kLanes, c = 8 * lane, blocks = a.npad / delta_block(kLanes), bh = blockIdx.x / blocks, head = bh % a.heads, batch = bh / a.heads;
  const int first = (int)(blockIdx.x % blocks) * delta_block(kLanes) + threadIdx.x / kLanes;
  uint4 u[kRows], v[kRows], z[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int i = first + r * (256 / kLanes);
    const bool there = i < a.n && c < a.d;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    u[r] = there ? __ldg(reinterpret_cast<const uint4*>(dout.at(batch, head, i) + c)) : none;
    v[r] = there ? __ldg(reinterpret_cast<const uint4*>(o.at(batch, head, i) + c)) : none;
    z[r] = there && rest.data ? __ldg(reinterpret_cast<const uint4*>(rest.at(batch, head, i) + c)) : none;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const uint32_t us[4] = {u[r].x, u[r].y, u[r].z, u[r].w}, vs[4] = {v[r].x, v[r].y, v[r].z, v[r].w}, zs[4] = {z[r].x, z[r].y, z[r].z, z[r].w};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = unpack16x2<kF16>(us[k]), q = unpack16x2<kF16>(vs[k]), x = unpack16x2<kF16>(zs[k]);
      sum = fmaf(p.x, q.x + x.x, fmaf(p.y, q.y + x.y, sum));
    }
#pragma unroll
    for (int w = kLanes / 2; w > 0; w /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    if (lane == 0) g.ndelta[(size_t)bh * a.npad + first + r * (256 / kLanes)] = -sum;
  }
}

struct WindowBwdBars {
  // streamed operands; S and dP, complete and in registers; P and dS; the products with them
  uint64_t own_full, first_full[4], second_full[2], ready, taken, given, done;
  uint32_t tmem_base;
};

// ---- dQ, delta, dbias ------------------------------------------------------------------------------------------------
// TMEM: S (64) | dP (64) | dS (32) | dQ (64): the next S and dP are made while this dS is.  Heads beyond 64: S | dP | dQ (128), dS in the place of S.
// kD: the head size that there is room for, 64 or 128.
template <int kD>
struct WindowDqLayout {
  // K's tiles serve two products: three of them, or the next S would wait for one that was asked for only when the dS before was through
  static constexpr int panels = kD / 64, k_stages = kD == 64 ? 3 : 1, v_stages = kD == 64 ? 2 : 1, tile = panels * kWCols * 128;
  static constexpr bool ahead = kD == 64;
  static constexpr int cols = 256, col_ds = ahead ? 2 * kWCols : 0, col_q = ahead ? 2 * kWCols + kWCols / 2 : 2 * kWCols;
  static_assert(col_q + kD <= cols, "tensor memory of a CTA");
  static constexpr int q = 0, dout = panels * kWRows * 128, k = 2 * dout, v = k + k_stages * tile, bars = v + v_stages * tile;
  static constexpr int part = bars + 128, bias = part + 2 * kWRows * 4;
  static constexpr int bytes(int r, bool grad) { return bias + bias_floats(r) * 4 * (grad ? 9 : 1) + (grad ? 8 * 32 * 4 : 0); }
};
static_assert(sizeof(WindowBwdBars) <= 128, "room for the barriers");

template <bool kF16, int kD, bool kBiasGrad>
__global__ void __launch_bounds__(kWDqThreads, 2)
window_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const WindowArgs a, const WindowBwdArgs g, const RowsOut dq) {
  typedef WindowDqLayout<kD> L;
  constexpr uint32_t kCols = L::cols;
  constexpr int kK = L::k_stages, kV = L::v_stages, kPanels = L::panels;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowBwdBars& bars = *reinterpret_cast<WindowBwdBars*>(sm + L::bars);
  float* const part = reinterpret_cast<float*>(sm + L::part);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int q0 = (int)(blockIdx.x % a.tiles) * kWRows, bh = blockIdx.x / a.tiles, head = bh % a.heads, batch = bh / a.heads;
  const KeyTiles<kWCols> tiles(a, q0);

  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    prefetch_maps(map_q, map_do, map_k, map_v);
    mbar_init(&bars.own_full, 1);
    for (int s = 0; s < 4; ++s) mbar_init(&bars.first_full[s], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&bars.second_full[s], 1);
    mbar_init(&bars.ready, 1);
    mbar_init(&bars.taken, 8);
    mbar_init(&bars.given, 8);
    mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) tmem_alloc(&bars.tmem_base, kCols);
  if (!cta_ready(skip, warp == 8, bars.tmem_base, kCols)) return;
  // window_delta_kernel is complete: when all blocks have come this far, those of window_dkv_kernel may begin
  if (g.early) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const uint32_t tmem = bars.tmem_base;
  const int ext = bias_floats(a.r);

  // Sums of this thread's dS over offsets that are clipped and over the others, and of its P over the clipped ones.
  float low = 0.f, high = 0.f, inner = 0.f, p_low = 0.f, p_high = 0.f;
  if (warp == 8) {
    // ------------------------------------------------------------------ copies and products
    const int kv = head / a.group;
    const uint32_t q_at = smem_u32(sm), do_at = smem_u32(sm + L::dout), k_at = smem_u32(sm + L::k), v_at = smem_u32(sm + L::v);
    const uint32_t idesc_s = umma_idesc_16(128, kWCols, kF16, kF16), idesc_q = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const int steps = (a.d + 15) / 16;
    const auto load_k = [&](int t) {      // one lane
      mbar_expect_tx(&bars.first_full[t % kK], L::tile);
      load_rows<kPanels>(k_at + t % kK * L::tile, &map_k, &bars.first_full[t % kK], kWCols, tiles.key(t), kv, batch);
    };
    const auto load_v = [&](int t) {
      mbar_expect_tx(&bars.second_full[t % kV], L::tile);
      load_rows<kPanels>(v_at + t % kV * L::tile, &map_v, &bars.second_full[t % kV], kWCols, tiles.key(t), kv, batch);
    };
    const auto issue = [&](int t) {
      if (!mbar_wait_warp(&bars.first_full[t % kK], (t / kK) & 1, 2u) || !mbar_wait_warp(&bars.second_full[t % kV], (t / kV) & 1, 4u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows<kPanels, kWCols>(tmem, q_at, k_at + t % kK * L::tile, steps, idesc_s);
        mma_rows<kPanels, kWCols>(tmem + kWCols, do_at, v_at + t % kV * L::tile, steps, idesc_s);
        umma_commit(&bars.ready);
      }
      __syncwarp();
      return true;
    };
    if (elect_lane()) {
      mbar_expect_tx(&bars.own_full, 2 * kPanels * kWRows * 128);
      load_rows<kPanels>(q_at, &map_q, &bars.own_full, kWRows, q0, head, batch);
      load_k(0);
      load_rows<kPanels>(do_at, &map_do, &bars.own_full, kWRows, q0, head, batch);
      load_v(0);
      for (int t = 1; t < kK && t < tiles.count; ++t) {
        load_k(t);
        if (t < kV) load_v(t);
      }
    }
    __syncwarp();
    bool ok = mbar_wait_warp(&bars.own_full, 0, 1u) && issue(0);
    for (int t = 0; t < tiles.count && ok; ++t) {
      ok = mbar_wait_warp(&bars.taken, t & 1, 8u);            // S(t) and dP(t) are complete and in registers: V's tile is free
      if (!ok) break;
      if (t + kV < tiles.count && elect_lane()) load_v(t + kV);
      __syncwarp();
      if (L::ahead) {
        if (t + 1 < tiles.count && !(ok = issue(t + 1))) break;
        if (t > 0 && t - 1 + kK < tiles.count) {              // K's tile of the step before is free
          ok = mbar_wait_warp(&bars.done, (t - 1) & 1, 16u);
          if (!ok) break;
          if (elect_lane()) load_k(t - 1 + kK);
          __syncwarp();
        }
      }
      ok = mbar_wait_warp(&bars.given, t & 1, 8u);
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        mma_streamed(tmem + L::col_q, tmem + L::col_ds, k_at + t % kK * L::tile, idesc_q, t == 0);
        umma_commit(&bars.done);
      }
      __syncwarp();
      if (!L::ahead) {
        ok = mbar_wait_warp(&bars.done, t & 1, 16u);          // K's tile and the place of S are free
        if (!ok) break;
        if (t + 1 < tiles.count && elect_lane()) load_k(t + 1);
        __syncwarp();
        if (t + 1 < tiles.count) ok = issue(t + 1);
      }
    }
  } else {
    // ------------------------------------------------------------------ one query row x 32 keys a thread
    const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane, i = q0 + row, qw = q0 + 32 * quarter;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    const float nlse = g.nlse[(size_t)bh * a.npad + i], ndelta = g.ndelta[(size_t)bh * a.npad + i];
    if (a.r >= 0) {
      bias_fill(a, head, bias, 256);
      if (kBiasGrad)
        for (int k = threadIdx.x; k < 8 * ext; k += 256) bias[ext + k] = 0.f;
    }
    if (a.r >= 0) barrier_of(1, 256);
    float* const sums = bias + ext * (1 + warp);                   // by offset, as the bias lies
    float* const stage = bias + ext * 9 + 32 * warp;
    const f32x2 scale = both2(a.c), ndelta2 = both2(ndelta);
    const float flat_low = a.r < 0 ? 0.f : bias[0], flat_high = a.r < 0 ? 0.f : bias[ext - 1];
    bool ok = true;
    for (int t = 0; t < tiles.count; ++t) {
      const int k0 = tiles.key(t), kh = k0 + 32 * half;
      const uint32_t keys = a.mask || kh + 32 > a.n ? key_bits(a, batch, kh, lane) : 0xffffffffu;
      const bool dead = keys == 0 || block_dead(a, qw, kh);
      ok = mbar_wait(&bars.ready, t & 1, 32u);
      __syncwarp();
      tc_fence_after();
      float s[32], d[32];
      uint32_t w[16];
      if (!dead) {
        tmem_ld32(t_lane + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld32(t_lane + kWCols + 32 * half, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
        tmem_wait_ld();
      }
      tc_fence_before();
      // where dS goes to the place of S, all of S has to be read before
      ok = L::ahead ? __all_sync(0xffffffffu, ok) != 0 : barrier_all(2 + quarter, 64, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive(&bars.taken);
      const bool is_low = kh + 31 - qw <= -a.r, near = a.r >= 0 && !is_low && kh - qw - 31 < a.r;
      if (!dead) {
        if (near) {
          const float* const y = bias_row(a, bias, i, kh);
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = fmaf(s[c], a.c, y[c] + nlse);
        } else {
          const float shift = nlse + (is_low ? flat_low : flat_high);
          const f32x2 shift2 = pair2(shift, shift);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 x = apart2(fma2(pair2(s[c], s[c + 1]), scale, shift2));
            s[c] = x.x, s[c + 1] = x.y;
          }
        }
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          s[c] = fast_exp2(s[c]), s[c + 1] = fast_exp2(s[c + 1]);
          const float2 x = apart2(mul2(add2(pair2(d[c], d[c + 1]), ndelta2), pair2(s[c], s[c + 1])));
          d[c] = x.x, d[c + 1] = x.y;
        }
        if (keys != 0xffffffffu || !block_whole(a, qw, kh)) {
          const uint32_t seen = visible_bits(a, i, kh, keys);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            d[c] = (seen >> c & 1u) ? d[c] : 0.f;
            if (kBiasGrad) s[c] = (seen >> c & 1u) ? s[c] : 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack16x2_inf<kF16>(d[2 * e], d[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = 0u;
      }
      if (L::ahead && t > 0) {                      // the product before has read its dS
        ok = mbar_wait(&bars.done, (t - 1) & 1, 64u);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      tc_fence_after();
      tmem_st16(t_lane + L::col_ds + 16 * half, w);
      // masked keys of the tile: their rows of K become zeros, those of this half by its four warps
      if (keys != 0xffffffffu && keys != bits_between(0, a.n - 1 - kh)) {
        mbar_wait(&bars.first_full[t % kK], (t / kK) & 1, 128u);      // complete: S(t) is; orders these writes behind the copy's
        if (!(keys >> lane & 1)) clear_row<kPanels, kWCols>(sm + L::k + t % kK * L::tile, 32 * half + lane, quarter, 4);
        fence_async_shared();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.given);
      if (kBiasGrad && !dead) {
        f32x2 v = pair2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 32; c += 2) v = add2(v, pair2(d[c], d[c + 1]));
        const float2 x = apart2(v);
        if (near) {
          inner += x.x + x.y;
          // Sums along the diagonals of a 32 x 32 block, 8 columns at a time (four chains beside one another: a single one waits for its shuffles):
          // the running sum moves one lane on with each column, and leaves by the last lane.
          float run[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float up = __shfl_up_sync(0xffffffffu, run[e], 1);
              run[e] = (lane == 0 ? 0.f : up) + d[8 * e + c];
              if (lane == 31) stage[8 * e + c] = run[e];      // offset 8 e + c - 31 of the block, as far as these columns go
            }
          __syncwarp();
          float* const at = sums + (kh - qw + a.r + kWBiasBeyond);
          at[lane - 31] += stage[lane];
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (lane < 31) at[8 * e + 7 - lane] += run[e];
            __syncwarp();
          }
        } else {
          f32x2 p = pair2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 32; c += 2) p = add2(p, pair2(s[c], s[c + 1]));
          const float2 y = apart2(p);
          if (is_low) low += x.x + x.y, p_low += y.x + y.y;
          else high += x.x + x.y, p_high += y.x + y.y;
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
        tmem_ld16(t_lane + L::col_q + c, x);
        tmem_wait_ld();
        if (i < a.n) {
          store8<kF16>(out + c, x, g.scale);
          if (c + 8 < a.d) store8<kF16>(out + c + 8, x + 8, g.scale);
        }
      }
    }
    if (kBiasGrad) {
      // dS adds up to zero along a row; what is left is the error of delta, which lies in every dS of the row as P times it.  In the sums over the clipped
      // offsets, where many keys of a row come together, it is taken out (37 sinks, two other keys: dbias off by 4.2e-3 in bf16 without,
      // 2.9e-3 with it; 2 to 6 % of the kernel).
      part[half * kWRows + row] = low + high + inner;
      ok = barrier_all(2 + quarter, 64, ok);
      const float left_over = part[row] + part[kWRows + row];
      low = fmaf(-left_over, p_low, low), high = fmaf(-left_over, p_high, high);
      barrier_of(1, 256);                          // `part` has been read
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
    // the two ends first, with what lies beyond them, a warp each
    if (warp < 2) {
      const float* const s = bias + ext + (warp == 0 ? 0 : 2 * a.r + 1 + kWBiasBeyond);
      float v = lane < 8 ? part[8 * warp + lane] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += s[ext * k + lane] + s[ext * k + 32 + lane];
      v = warp_sum(v);
      if (lane == 0) part[32 + warp] = v;
    }
    __syncthreads();
    float* const out = g.dbias + (size_t)blockIdx.x * (2 * a.r + 1);
    for (int b = threadIdx.x; b < 2 * a.r + 1; b += kWDqThreads) {
      float v = (b == 0 ? part[32] : 0.f) + (b == 2 * a.r ? part[33] : 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) v += bias[ext * (1 + k) + b + kWBiasBeyond];
      out[b] = v;
    }
  }
}

// dbias[head][b] of the CTAs' sums, in their order: 32 buckets (block `of` of a head's), a slice of the CTAs of the head for each warp.
template <int kThreads>
__device__ __forceinline__ void sum_dbias(const WindowArgs& a, const WindowBwdArgs& g, int head, int of, float* slice) {
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, buckets = 2 * a.r + 1, b = of * 32 + lane;
  constexpr int kSlices = kThreads / 32;
  float v = 0.f;
  if (b < buckets)
#pragma unroll 4
    for (int k = s; k < g.batches * a.tiles; k += kSlices)
      v += g.dbias[((size_t)((k / a.tiles) * a.heads + head) * a.tiles + k % a.tiles) * buckets + b];
  slice[s * 32 + lane] = v;
  __syncthreads();
  if (s == 0 && b < buckets) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < kSlices; ++e) sum += slice[e * 32 + lane];
    const size_t at = (size_t)head * buckets + b;
    if (a.bias_type == PX_F32) ((float*)g.dbias_out)[at] = sum;
    else if (a.bias_type == PX_BF16) ((bf16*)g.dbias_out)[at] = __float2bfloat16_rn(sum);
    else ((__half*)g.dbias_out)[at] = __float2half_rn(sum);
  }
}

// ---- dK, dV ----------------------------------------------------------------------------------------------------------
// TMEM, heads up to 32: S^T (64) | dP^T (64) | P^T (32) | dS^T (32) | dV (32) | dK (32), two CTAs an SM; beyond 64 the same with dV and dK of 128 and one CTA.
// Heads of 33 to 64: S^T | dP^T | dV (64) | dK (64), P^T and dS^T in shared memory.  The next S^T and dP^T are made while these P^T and dS^T are.
template <int kD>
struct WindowDkvLayout {
  // Streamed tiles: three or more, or the next S^T waits for one that was asked for only when the dS^T before was through (heads of 128: two 167 us, four 148);
  // heads of 33 to 64 have room for two.
  static constexpr int panels = kD > 64 ? 2 : 1, stages = kD == 64 ? 2 : kD == 32 ? 3 : 4, tile = panels * kWCols * 128, stat = 2 * kWCols * 4;
  static constexpr bool p_shared = kD == 64;
  static constexpr int cols = kD == 128 ? 512 : 256, ctas = kD == 128 ? 1 : 2;
  // Warps of rows: 16 an SM whatever the head size, a thread = 32 of the 64 columns or, where the CTA is alone, 16.  Then one warp for S^T and dP^T, one for
  // the products with P^T and dS^T.
  static constexpr int warps = 16 / ctas, groups = warps / 4, rows = 32 * warps, threads = rows + 64;
  static constexpr int col_p = 2 * kWCols, col_ds = col_p + kWCols / 2;
  static constexpr int col_v = p_shared ? 2 * kWCols : 3 * kWCols, col_k = col_v + kD;
  static_assert(col_k + kD <= cols, "tensor memory of a CTA");
  static constexpr int k = 0, v = panels * kWRows * 128, q = 2 * v, dout = q + stages * tile, p = dout + stages * tile;
  static constexpr int ds = p + (p_shared ? kWRows * 128 : 0), stats = ds + (p_shared ? kWRows * 128 : 0), bars = stats + stages * stat;
  static constexpr int bias = bars + 128;
  static constexpr int bytes(int r) { return bias + bias_floats(r) * 4; }
};

// P in fp16 is rounded times this (P is 1 at most, 2^15 fits) and dV divided by it: weights are normal numbers down to 2^-29, where 2^-14 would be the last and all weights of a
// wide window could be off alike (10.5 steps of 2^-24: 5 %; a loss scale does not reach P).
constexpr float kWPUp = 32768.f;

// The rows of dK and dV of one key tile, from the parts that its CTAs have left: a thread = 8 values.
template <bool kF16, int kThreads>
__device__ __forceinline__ void sum_sinks(const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dk, const RowsOut& dv, int bkv, int own) {
  const int dn = (a.d + 15) & ~15, pieces = a.d / 8, rows = min(a.n - own * kWRows, kWRows);
  for (int u = threadIdx.x; u < 2 * rows * pieces; u += kThreads) {
    const int c = u % pieces * 8, row = u / pieces % rows, which = u / pieces / rows;
    const RowsOut& out = which ? dv : dk;
    if (!out.data) continue;
    const float* from = g.sinks + ((size_t)bkv * g.sink_tiles + own) * (1 + g.chunks) * 2 * kWRows * dn + (size_t)which * kWRows * dn + (size_t)row * dn + c;
    float v[8] = {};
#pragma unroll 4
    for (int k = 0; k <= g.chunks; ++k, from += 2 * kWRows * dn) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(from)), y = __ldcg(reinterpret_cast<const float4*>(from + 4));
      v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    store8<kF16>(out.at(bkv / a.kv_heads, bkv % a.kv_heads, own * kWRows + row) + c, reinterpret_cast<const uint32_t*>(v), 1.f);
  }
}

// The queries of one CTA: streamed tiles first .. first + count - 1 of `per` a head, over the heads of the group.
struct QueryTiles {
  int first, per, begin, count;      // begin: the first of the items head-of-group * per + tile
};
struct QueryItem {                   // one of them, stepped along
  int tile, member;
  __device__ __forceinline__ explicit QueryItem(const QueryTiles& t) : tile(t.begin % t.per), member(t.begin / t.per) {}
  __device__ __forceinline__ void next(const QueryTiles& t) {
    if (++tile == t.per) tile = 0, ++member;
  }
};
__host__ __device__ __forceinline__ int last_of_window(int n, int left, int k0) {      // last streamed tile of the window of 128 keys
  return (k0 + kWRows - 1 + left < n - 1 ? k0 + kWRows - 1 + left : n - 1) / kWCols;
}

template <bool kF16, int kD>
__global__ void __launch_bounds__(WindowDkvLayout<kD>::threads, WindowDkvLayout<kD>::ctas)
window_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const WindowArgs a, const WindowBwdArgs g, const RowsOut dk, const RowsOut dv) {
  typedef WindowDkvLayout<kD> L;
  constexpr uint32_t kCols = L::cols;
  constexpr int kPanels = L::panels, kStages = L::stages, kFirst = L::warps;      // kFirst: the first control warp
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowBwdBars& bars = *reinterpret_cast<WindowBwdBars*>(sm + L::bars);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  // the chunks of the sinks, which may be the longest, then the key tiles, then the sums of the bias, which need all of window_dq_kernel
  const int extra = g.sink_tiles * g.chunks, kv_all = a.kv_heads * g.batches;
  int block = blockIdx.x - (g.own ? (a.tiles + extra) * kv_all : 0);
  if (block >= 0) {
    pdl_wait();
    sum_dbias<L::threads>(a, g, block / g.bias_blocks, block % g.bias_blocks, reinterpret_cast<float*>(sm));
    return;
  }
  block = blockIdx.x;
  const bool chunk = block < extra * kv_all;
  if (!chunk) block -= extra * kv_all;
  const int each = chunk ? extra : a.tiles, bkv = block / each, at = block % each;      // at: of the chunks, or the key tile
  const int kv = bkv % a.kv_heads, batch = bkv / a.kv_heads;
  const int own = chunk ? at / g.chunks : at, k0 = own * kWRows;
  const int last = last_of_window(a.n, a.left, k0);
  QueryTiles tiles;
  if (chunk) {
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
    for (int s = 0; s < 4; ++s) mbar_init(&bars.first_full[s], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&bars.second_full[s], 1);
    mbar_init(&bars.ready, 1);
    mbar_init(&bars.taken, L::warps);
    mbar_init(&bars.given, L::warps);
    mbar_init(&bars.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == kFirst) tmem_alloc(&bars.tmem_base, kCols);
  // as cta_ready, but beside window_dq_kernel: what this kernel reads was complete before that one's blocks signalled
  tc_fence_before();
  const bool stop = __syncthreads_or(skip) != 0;
  tc_fence_after();
  if (!g.early || stop) pdl_wait();
  if (stop) {
    if (warp == kFirst) tmem_free(bars.tmem_base, kCols);
    return;
  }
  const uint32_t tmem = bars.tmem_base;

  if (warp >= kFirst) {
    // ------------------------------------------------------------------ copies and products
    const uint32_t k_at = smem_u32(sm), v_at = smem_u32(sm + L::v), q_at = smem_u32(sm + L::q), do_at = smem_u32(sm + L::dout);
    const uint32_t idesc_s = umma_idesc_16(128, kWCols, kF16, kF16), idesc_d = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const int steps = (a.d + 15) / 16;
    QueryItem coming(tiles);
    const auto load = [&](int s) {      // one lane: Q, dO and the rows' statistics of the item that comes next
      const int head = kv * a.group + coming.member, q0 = (tiles.first + coming.tile) * kWCols;
      mbar_expect_tx(&bars.first_full[s], 2 * L::tile + L::stat);
      load_rows<kPanels>(q_at + s * L::tile, &map_q, &bars.first_full[s], kWCols, q0, head, batch);
      load_rows<kPanels>(do_at + s * L::tile, &map_do, &bars.first_full[s], kWCols, q0, head, batch);
      const size_t row = (size_t)(batch * a.heads + head) * a.npad + q0;
      bulk_load(sm + L::stats + s * L::stat, g.nlse + row, kWCols * 4, &bars.first_full[s]);
      bulk_load(sm + L::stats + s * L::stat + kWCols * 4, g.ndelta + row, kWCols * 4, &bars.first_full[s]);
    };
    const auto issue = [&](int t) {
      const int s = t % kStages;
      if (!mbar_wait_warp(&bars.first_full[s], (t / kStages) & 1, 2u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows<kPanels, kWCols>(tmem, k_at, q_at + s * L::tile, steps, idesc_s);
        mma_rows<kPanels, kWCols>(tmem + kWCols, v_at, do_at + s * L::tile, steps, idesc_s);
        umma_commit(&bars.ready);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    if (warp == kFirst) {
      if (tiles.count > 0) {
        if (elect_lane()) {
          mbar_expect_tx(&bars.own_full, 2 * kPanels * kWRows * 128);
          load_rows<kPanels>(k_at, &map_k, &bars.own_full, kWRows, k0, kv, batch);
          load_rows<kPanels>(v_at, &map_v, &bars.own_full, kWRows, k0, kv, batch);
        }
        __syncwarp();
        for (int t = 0; t < kStages && t < tiles.count; ++t) {
          if (elect_lane()) load(t);
          __syncwarp();
          coming.next(tiles);
        }
        ok = mbar_wait_warp(&bars.own_full, 0, 1u) && issue(0);
      }
      for (int t = 0; t + 1 < tiles.count && ok; ++t) ok = mbar_wait_warp(&bars.taken, t & 1, 8u) && issue(t + 1);
    } else {
      for (int t = 0; t < kStages; ++t) coming.next(tiles);
      for (int t = 0; t < tiles.count && ok; ++t) {
        ok = mbar_wait_warp(&bars.given, t & 1, 8u);
        if (!ok) break;
        tc_fence_after();
        const int s = t % kStages;
        if (elect_lane()) {
          if (L::p_shared) {
            mma_streamed_ss(tmem + L::col_v, smem_u32(sm + L::p), do_at + s * L::tile, idesc_d, t == 0);
            mma_streamed_ss(tmem + L::col_k, smem_u32(sm + L::ds), q_at + s * L::tile, idesc_d, t == 0);
          } else {
            mma_streamed(tmem + L::col_v, tmem + L::col_p, do_at + s * L::tile, idesc_d, t == 0);
            mma_streamed(tmem + L::col_k, tmem + L::col_ds, q_at + s * L::tile, idesc_d, t == 0);
          }
          umma_commit(&bars.done);
        }
        __syncwarp();
        if (t + kStages < tiles.count) {                      // the streamed tile is free then
          ok = mbar_wait_warp(&bars.done, t & 1, 16u);
          if (ok && elect_lane()) load(s);
          __syncwarp();
          coming.next(tiles);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ one key row x 32 queries a thread, or 16 of the 32
    constexpr int kHalves = L::groups == 2 ? 2 : 1;
    const int quarter = warp & 3, group = warp >> 2, half = group / (L::groups / 2), row = 32 * quarter + lane, j = k0 + row, kw = k0 + 32 * quarter;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    const bool masked = a.mask && __ldg(a.mask + (size_t)batch * a.n + min(j, a.n - 1)) == 0;
    const bool any_masked = a.mask && barrier_any(1, L::rows, masked);
    const f32x2 scale = both2(a.c);
    constexpr float up = kF16 ? kWPUp : 1.f;
    // blocks of queries from qh on that see all of this warp's keys, and those whose bias is the first or the last entry for all
    const int whole_from = any_masked ? 0x3fffffff : kw + 31 - a.right, whole_to = min(kw + 32 <= a.sinks ? a.n : kw - 31 + a.left, a.n - 32);
    const int low_from = kw + 31 + a.r, high_to = kw - 31 - a.r;
    bool ok = true;                                // of the warp: one whose wait ran out goes on to the barriers alone
    int filled = -1;                               // the group's head whose bias is in shared memory
    QueryItem now(tiles);
    for (int t = 0; t < tiles.count; ++t, now.next(tiles)) {
      const int qh = (tiles.first + now.tile) * kWCols + 32 * half, s = t % kStages;
      if (a.r >= 0 && now.member != filled) {
        barrier_of(1, L::rows);                        // all are through with the tile before
        bias_fill(a, kv * a.group + now.member, bias, L::rows);
        barrier_of(1, L::rows);
        filled = now.member;
      }
      if (!ok) continue;
      const bool dead = qh >= a.n || block_dead(a, qh, kw);
      ok = mbar_wait(&bars.ready, t & 1, 32u);
      // the statistics came with the operands; this wait only makes the copy's writes visible here
      ok = mbar_wait(&bars.first_full[s], (t / kStages) & 1, 64u) && ok;
      __syncwarp();
      tc_fence_after();
      uint32_t wp[8 * kHalves], wd[8 * kHalves], nothing = 0, seen = 0xffffffffu;
      bool near = false;
      float flat = 0.f;
      const float* y = bias;
      if (a.r >= 0) {
        const bool high = qh <= high_to;
        near = !high && qh < low_from;
        flat = near ? 0.f : bias[high ? bias_floats(a.r) - 1 : 0];
        if (near) y = bias_row(a, bias, qh, j);                 // of query qh + c: y[-c]
      }
      if (qh < whole_from || qh > whole_to)
        // queries j - right .. j + left, all from j - right on for a sink, none for a masked key
        seen = bits_between(j - a.right - qh, masked ? -1 : j < a.sinks ? 31 : j + a.left - qh);
      if (a.mask) {
        const float* const mine = reinterpret_cast<const float*>(sm + L::stats + s * L::stat) + 32 * half;
        nothing = __ballot_sync(0xffffffffu, mine[lane] == -CUDART_INF_F);      // queries that see nothing
        seen &= ~nothing;
      }
      const bool seen_all = __all_sync(0xffffffffu, seen == 0xffffffffu);
#pragma unroll
      for (int k = 0; k < kHalves; ++k) {                       // 16 columns at a time, for the registers' sake
        const int h = kHalves == 2 ? k : group & 1;
        float p[16], d[16];
        if (!dead) {
          tmem_ld16(t_lane + 32 * half + 16 * h, *reinterpret_cast<uint32_t(*)[16]>(&p[0]));
          tmem_ld16(t_lane + kWCols + 32 * half + 16 * h, *reinterpret_cast<uint32_t(*)[16]>(&d[0]));
          tmem_wait_ld();
        }
        if (k == kHalves - 1) {
          tc_fence_before();
          ok = __all_sync(0xffffffffu, ok) != 0;
          if (!ok) break;
          if (lane == 0) mbar_arrive(&bars.taken);
        }
        if (dead) {
#pragma unroll
          for (int e = 0; e < 8; ++e) wp[8 * k + e] = wd[8 * k + e] = 0u;
          continue;
        }
        const ulonglong2* const nlse4 = reinterpret_cast<const ulonglong2*>(sm + L::stats + s * L::stat) + 8 * half + 4 * h;
        const ulonglong2* const ndelta4 = nlse4 + kWCols / 4;
        if (near) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const ulonglong2 l4 = nlse4[c];
            const int b = 16 * h + 4 * c;
            const float2 u = apart2(fma2(pair2(p[4 * c], p[4 * c + 1]), scale, add2(l4.x, pair2(y[-b], y[-b - 1]))));
            const float2 v = apart2(fma2(pair2(p[4 * c + 2], p[4 * c + 3]), scale, add2(l4.y, pair2(y[-b - 2], y[-b - 3]))));
            p[4 * c] = u.x, p[4 * c + 1] = u.y, p[4 * c + 2] = v.x, p[4 * c + 3] = v.y;
          }
        } else {
          const f32x2 flat2 = pair2(flat, flat);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const ulonglong2 l4 = nlse4[c];
            const float2 u = apart2(fma2(pair2(p[4 * c], p[4 * c + 1]), scale, add2(l4.x, flat2)));
            const float2 v = apart2(fma2(pair2(p[4 * c + 2], p[4 * c + 3]), scale, add2(l4.y, flat2)));
            p[4 * c] = u.x, p[4 * c + 1] = u.y, p[4 * c + 2] = v.x, p[4 * c + 3] = v.y;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const ulonglong2 e4 = ndelta4[c];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[4 * c + x] = fast_exp2(p[4 * c + x]);
          const float2 u = apart2(mul2(add2(pair2(d[4 * c], d[4 * c + 1]), e4.x), pair2(p[4 * c], p[4 * c + 1])));
          const float2 v = apart2(mul2(add2(pair2(d[4 * c + 2], d[4 * c + 3]), e4.y), pair2(p[4 * c + 2], p[4 * c + 3])));
          d[4 * c] = u.x, d[4 * c + 1] = u.y, d[4 * c + 2] = v.x, d[4 * c + 3] = v.y;
        }
        if (seen_all) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            wp[8 * k + e] = pack16x2<kF16>(up * p[2 * e], up * p[2 * e + 1]);
            wd[8 * k + e] = pack16x2_inf<kF16>(d[2 * e], d[2 * e + 1]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool a0 = seen >> (16 * h + 2 * e) & 1u, a1 = seen >> (16 * h + 2 * e + 1) & 1u;
            wp[8 * k + e] = pack16x2<kF16>(a0 ? up * p[2 * e] : 0.f, a1 ? up * p[2 * e + 1] : 0.f);
            wd[8 * k + e] = pack16x2_inf<kF16>(a0 ? d[2 * e] : 0.f, a1 ? d[2 * e + 1] : 0.f);
          }
        }
      }
      if (!ok) continue;
      if (nothing) {                                // whatever their rows of Q and dO hold becomes zeros; those of this half by four of its warps
        if ((nothing >> lane & 1u) && (kHalves == 2 || (group & 1) == 0)) {
          clear_row<kPanels, kWCols>(sm + L::q + s * L::tile, 32 * half + lane, quarter, 4);
          clear_row<kPanels, kWCols>(sm + L::dout + s * L::tile, 32 * half + lane, quarter, 4);
        }
      }
      if (t > 0) {                                  // the products before have read their P^T and dS^T
        ok = mbar_wait(&bars.done, (t - 1) & 1, 64u);
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) continue;
      }
      tc_fence_after();
      if constexpr (L::p_shared) {
        panel_store(sm + L::p, row, half, wp);
        panel_store(sm + L::ds, row, half, wd);
      } else {
        if constexpr (kHalves == 2) {
          tmem_st16(t_lane + L::col_p + 16 * half, wp);
          tmem_st16(t_lane + L::col_ds + 16 * half, wd);
        } else {
          tmem_st8(t_lane + L::col_p + 8 * group, wp);
          tmem_st8(t_lane + L::col_ds + 8 * group, wd);
        }
        tmem_wait_st();
      }
      if (L::p_shared || nothing) fence_async_shared();
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
      // where the key is a sink with chunks, this is one of the sums that the last of its CTAs adds up: its own first, then the chunks
      const bool summed = g.chunks > 0 && own < g.sink_tiles;
      float* const to = g.sinks + (((size_t)bkv * g.sink_tiles + own) * (1 + g.chunks) + (chunk ? 1 + at % g.chunks : 0)) * 2 * kWRows * dn +
                        (size_t)row * dn;
      for (int which = 0; which < 2; ++which) {      // dK, dV
        const RowsOut& out = which ? dv : dk;
        const float scale = which ? (kF16 ? 1.f / kWPUp : 1.f) : g.scale;
        if (!out.data) continue;
        for (int c = 16 * group; c < a.d; c += 16 * L::groups) {
          uint32_t x[16];
          if (tiles.count > 0) {
            tmem_ld16(t_lane + (which ? L::col_v : L::col_k) + c, x);
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
  const bool summed = g.chunks > 0 && own < g.sink_tiles;
  if (summed) __threadfence();      // this CTA's sums are seen before its arrival is
  tc_fence_before();
  cta_teardown_sync();
  if (warp == kFirst) {
    tc_fence_after();
    tmem_free(tmem, kCols);
  }
  if (summed) {
    // whoever arrives last adds the sums up, in their order
    uint32_t& count = bars.tmem_base;      // no longer needed
    if (threadIdx.x == 0) count = atomicAdd(g.arrived + (size_t)bkv * g.sink_tiles + own, 1u);
    __syncthreads();
    if (count == (uint32_t)g.chunks) {
      __threadfence();
      sum_sinks<kF16, L::threads>(a, g, dk, dv, bkv, own);
    }
  }
  if (g.early) pdl_wait();      // the grid ends behind window_dq_kernel's, as whatever comes next expects
}

}  // namespace px
