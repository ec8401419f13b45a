// Attention with a sliding window, first tokens that stay visible and a learned bias by offset, on the 5th-generation tensor cores.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax over visible j of  scale q_i . k_j + bias[head][clip(j - i, -r, r) + r]
//   j is visible to i when mask[j] and j <= i + right and (j >= i - left or j < sinks);  a row that sees nothing gives 0.
//
// q, k, v: [batch][head][n][d], any strides along batch, head and row, bf16 or fp16, d a multiple of 8 up to 128; heads of k and v may serve a
// group of q's heads each.
//
// One CTA = 128 queries of a head, streamed over the 64-key tiles that they see.  Warps 0..3: one thread a query row.  Warp 4
// loads Q once and K, V tiles by TMA (panels of 64 elements, 128-byte swizzle, a ring of two each) and issues S = Q K^T and, once the rows have left P
// (16 bits), O += P V with V read as it lies, along its rows.  The next S is made while this one, by then in registers, becomes P.
// Softmax is online in base 2 with a reference maximum that moves (and O with it) only when a tile exceeds it by more than 8: P is 2^8 at most (2^15 in fp16, see kWUpF16).
// Logits, statistics and O are fp32; P is rounded to the type of V, which the product needs (relative error of half a step, 2^-8 or 2^-11 at most,
// with either sign); the denominators sum the fp32 values.
//
// Blocks of 32 queries x 32 keys out of sight cost nothing but zeros.  Tiles that a warp's rows see whole and with one bias for all, the larger part of a
// wide window, take a loop of their own without tests; elsewhere a row's visible keys are a word of 32 bits, and where the offsets are not all clipped
// alike the bias is read from shared memory, where the head's row lies continued beyond its ends, so that a thread's values lie side by side.
//
// What bounds it: the chain of a tile in a row's thread (maximum, exponentials, rounding: some 330 instructions where nothing is tested, 2000 cycles beside
// the other warps), not a unit: at 8192 tokens, 16 heads of 64, causal window of 1024, 88 us (370 TFLOP/s), the special-function unit is
// busy for two fifths of the time and the tensor pipe for a fifth; at 16384 tokens, 8 heads of 128, window of 2048, both for half: 141 us in a loop over the same
// inputs (920 TFLOP/s), 165 to 170 where the inputs change from pass to pass (770 TFLOP/s).
// So as many CTAs an SM as tensor memory, shared memory and registers allow: four (heads up to 32), three, two, with four row warps each.  Short windows (atoms: four tiles a CTA) pay as much for a CTA's beginning and
// end.  Built, measured and not kept: 128 keys a tile for heads of 64 (2 % slower), eight warps of rows with 32 keys each (10 to 40 %), copies issued by the row
// warps (7 %), window and bias in one table with -inf (1 to 8 %), the maximum looked for only where a tile's sum is large (heads of 128 1.5 % faster, of 64 4 % slower).
// A second allocation of tensor memory for P (heads of 64) would be asked for while holding the first, which could wait for good beside other kernels.
#include <type_traits>

#include "px_window.cuh"

namespace px {

constexpr float kWRescaleGap = 8.0f;
// P in fp16 is 2^7 times as large as against the reference maximum, 2^15 at most: weights are normal numbers down to 2^-21 of the row's largest at least, where 2^-14
// would be the last and those of many keys could be off alike (10.5 steps of 2^-24: 5 %).  The denominator has the same factor.
constexpr float kWUpF16 = 7.0f;
constexpr int kWFwdThreads = 160;

struct WindowFwdBars {
  uint64_t q_full, k_full[2], v_full[2], s_full, s_free, p_ready, pv_done;
  uint32_t tmem_base;
};
static_assert(sizeof(WindowFwdBars) <= 128, "room for the barriers");

// kD: the head size that the accumulator has room for, 32, 64 or 128.
template <int kD>
struct WindowFwdLayout {
  static constexpr int panels = kD > 64 ? 2 : 1, keys = 64, ctas = kD == 32 ? 4 : kD == 64 ? 3 : 2;
  // TMEM: S | P | O.  Heads of 33 to 64: S | O, and P in shared memory, so that 128 columns are enough.
  static constexpr bool p_shared = kD == 64;
  static constexpr int cols = kD == 128 ? 256 : 128, col_p = keys, col_o = p_shared ? keys : keys + keys / 2;
  static_assert(col_o + kD <= cols, "tensor memory of a CTA");
  static constexpr int q = 0, tile = panels * keys * 128;
  static constexpr int k = panels * kWRows * 128, v = k + 2 * tile, p = v + 2 * tile, bars = p + (p_shared ? kWRows * 128 : 0);
  static constexpr int bias = bars + 128;
  static constexpr int bytes(int r) { return bias + bias_floats(r) * 4; }
};

template <bool kF16, int kD>
__global__ void __launch_bounds__(kWFwdThreads, WindowFwdLayout<kD>::ctas)
window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const WindowArgs a, const RowsOut o, const RowsOut rest, float* __restrict__ nlse) {
  typedef WindowFwdLayout<kD> L;
  constexpr uint32_t kCols = L::cols;
  constexpr int kPanels = L::panels, kKT = L::keys, kBlocks = kKT / 32;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowFwdBars& bars = *reinterpret_cast<WindowFwdBars*>(sm + L::bars);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int q0 = (int)(blockIdx.x % a.tiles) * kWRows, bh = blockIdx.x / a.tiles, head = bh % a.heads, batch = bh / a.heads;
  const KeyTiles<kKT> tiles(a, q0);

  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    prefetch_maps(map_q, map_k, map_v);
    mbar_init(&bars.q_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.v_full[s], 1);
    }
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.s_free, 4);
    mbar_init(&bars.p_ready, 4);
    mbar_init(&bars.pv_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 4) tmem_alloc(&bars.tmem_base, kCols);
  if (!cta_ready(skip, warp == 4, bars.tmem_base, kCols)) return;
  const uint32_t tmem = bars.tmem_base;
  if (warp == 4) {
    // ------------------------------------------------------------------ copies and products
    const int kv = head / a.group;
    const uint32_t q_at = smem_u32(sm), k_at = smem_u32(sm + L::k), v_at = smem_u32(sm + L::v);
    const uint32_t idesc_s = umma_idesc_16(128, kKT, kF16, kF16), idesc_o = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const auto load_k = [&](int t) {      // one lane
      mbar_expect_tx(&bars.k_full[t & 1], L::tile);
      load_rows<kPanels>(k_at + (t & 1) * L::tile, &map_k, &bars.k_full[t & 1], kKT, tiles.key(t), kv, batch);
    };
    const auto load_v = [&](int t) {
      mbar_expect_tx(&bars.v_full[t & 1], L::tile);
      load_rows<kPanels>(v_at + (t & 1) * L::tile, &map_v, &bars.v_full[t & 1], kKT, tiles.key(t), kv, batch);
    };
    const auto issue_s = [&](int t) {
      if (!mbar_wait_warp(&bars.k_full[t & 1], (t >> 1) & 1, 2u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows<kPanels, kKT>(tmem, q_at, k_at + (t & 1) * L::tile, (a.d + 15) / 16, idesc_s);
        umma_commit(&bars.s_full);
      }
      __syncwarp();
      return true;
    };
    if (elect_lane()) {
      mbar_expect_tx(&bars.q_full, kPanels * kWRows * 128);
      load_rows<kPanels>(q_at, &map_q, &bars.q_full, kWRows, q0, head, batch);
      for (int t = 0; t < 2 && t < tiles.count; ++t) {
        load_k(t);
        load_v(t);
      }
    }
    __syncwarp();
    bool ok = mbar_wait_warp(&bars.q_full, 0, 1u) && issue_s(0);
    for (int t = 0; t < tiles.count && ok; ++t) {
      ok = mbar_wait_warp(&bars.s_free, t & 1, 4u);           // S(t) is complete and in registers: its K tile and its place are free
      if (!ok) break;
      if (t + 2 < tiles.count && elect_lane()) load_k(t + 2);
      __syncwarp();
      if (t + 1 < tiles.count && !(ok = issue_s(t + 1))) break;
      if (t > 0 && t + 1 < tiles.count) {                     // the V tile of the step before is free
        ok = mbar_wait_warp(&bars.pv_done, (t - 1) & 1, 16u);
        if (!ok) break;
        if (elect_lane()) load_v(t + 1);
        __syncwarp();
      }
      ok = mbar_wait_warp(&bars.p_ready, t & 1, 8u) && mbar_wait_warp(&bars.v_full[t & 1], (t >> 1) & 1, 8u);
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        if (L::p_shared) mma_streamed_ss(tmem + L::col_o, smem_u32(sm + L::p), v_at + (t & 1) * L::tile, idesc_o, t == 0);
        else mma_streamed(tmem + L::col_o, tmem + L::col_p, v_at + (t & 1) * L::tile, idesc_o, t == 0);
        umma_commit(&bars.pv_done);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ one query row a thread
    const int row = threadIdx.x, i = q0 + row, qw = q0 + 32 * warp;
    const uint32_t t_s = tmem + ((uint32_t)(32 * warp) << 16), t_p = t_s + L::col_p, t_o = t_s + L::col_o;
    if (a.r >= 0) {
      bias_fill(a, head, bias, 128);
      barrier_of(1, 128);
    }
    constexpr float kUp = kF16 ? kWUpF16 : 0.f;      // in base 2
    float m = -CUDART_INF_F;
    f32x2 l = pair2(0.f, 0.f);
    const f32x2 scale = both2(a.c);
    const PlainKeys runs(a, qw, bias, bias_floats(a.r));
    // One tile: S into registers, P out of them.  kPlain: all of it is seen, with one bias.
    const auto work = [&](int t, int k0, auto plain) {
      constexpr bool kPlain = decltype(plain)::value;
      uint32_t keys[kBlocks];
      bool dead[kBlocks], hidden = false;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        dead[b] = false;
        if (kPlain) continue;
        keys[b] = key_bits(a, batch, k0 + 32 * b, lane);
        dead[b] = keys[b] == 0 || block_dead(a, qw, k0 + 32 * b);
        hidden = hidden || keys[b] != bits_between(0, a.n - 1 - (k0 + 32 * b));
      }
      bool ok = mbar_wait(&bars.s_full, t & 1, 32u);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return false;
      tc_fence_after();
      float s[kKT];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) tmem_ld32(t_s + 32 * b, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * b]));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.s_free);
      // logits = s * mul + add, in base 2
      float mt = -CUDART_INF_F, add[kBlocks];
      f32x2 mul[kBlocks];
      if (kPlain) {
        mt = max32(s);
#pragma unroll
        for (int b = 1; b < kBlocks; ++b) mt = fmaxf(mt, max32(s + 32 * b));
        add[0] = runs.flat(k0 + kKT - 1);
        mt = fmaf(mt, a.c, add[0]);
      } else {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          if (dead[b]) continue;
          const int kb = k0 + 32 * b;
          float* const x = s + 32 * b;
          const BlockBias bb(a, bias, qw, kb);
          mul[b] = scale, add[b] = bb.flat;
          if (bb.near) {
            const float* const y = bias_row(a, bias, i, kb);
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = fmaf(x[c], a.c, y[c]);
            mul[b] = pair2(1.f, 1.f), add[b] = 0.f;
          }
          if (keys[b] != 0xffffffffu || !block_whole(a, qw, kb)) {
            const uint32_t seen = visible_bits(a, i, kb, keys[b]);
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = (seen >> c & 1u) ? x[c] : -CUDART_INF_F;
          }
          mt = fmaxf(mt, fmaf(max32(x), bb.near ? 1.f : a.c, add[b]));
        }
      }
      const bool up = mt > m + kWRescaleGap;
      const bool move = __any_sync(0xffffffffu, up) && t > 0;      // the first product overwrites O
      const float m_old = m;
      m = up ? mt : m;
      const float shift = (m == -CUDART_INF_F ? 0.f : -m) + kUp;
      f32x2 sum = pair2(0.f, 0.f);
      uint32_t w[kKT / 2];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        if (dead[b]) {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[16 * b + e] = 0u;
          continue;
        }
        const float sh = add[kPlain ? 0 : b] + shift;
        const f32x2 sh2 = pair2(sh, sh), by2 = kPlain ? scale : mul[b];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x = apart2(fma2(pair2(s[32 * b + 2 * e], s[32 * b + 2 * e + 1]), by2, sh2));
          const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
          sum = add2(sum, pair2(p0, p1));
          w[16 * b + e] = pack16x2<kF16>(p0, p1);
        }
      }
      if (t > 0) {                                                  // P and O are at rest
        ok = mbar_wait(&bars.pv_done, (t - 1) & 1, 128u);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return false;
        tc_fence_after();
      }
      if (move) {
        const float alpha = up ? fast_exp2(m_old - m) : 1.f;
        l = mul2(l, pair2(alpha, alpha));
        for (int c = 0; c < a.d; c += 16) {
          uint32_t x[16];
          tmem_ld16(t_o + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
          tmem_st16(t_o + c, x);
        }
      }
      l = add2(l, sum);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        if (L::p_shared) panel_store(sm + L::p, row, b, *reinterpret_cast<const uint32_t(*)[16]>(&w[16 * b]));
        else tmem_st16(t_p + 16 * b, *reinterpret_cast<const uint32_t(*)[16]>(&w[16 * b]));
      }
      if (hidden) {                                                 // masked keys: their rows of V
        if (!mbar_wait_warp(&bars.v_full[t & 1], (t >> 1) & 1, 64u)) return false;
        constexpr int kParts = 128 / kKT;
        const int r = row % kKT;
        uint32_t word = keys[0];
#pragma unroll
        for (int b = 1; b < kBlocks; ++b) word = r >> 5 == b ? keys[b] : word;
        if (!(word >> (r & 31) & 1)) clear_row<kPanels, kKT>(sm + L::v + (t & 1) * L::tile, r, row / kKT, kParts);
      }
      if (L::p_shared || hidden) fence_async_shared();
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_ready);
      return true;
    };
    bool ok = true;
    for (int t = 0; t < tiles.count && ok; ++t) {
      const int k0 = tiles.key(t);
      ok = runs.plain(k0, k0 + kKT - 1) ? work(t, k0, std::true_type()) : work(t, k0, std::false_type());
    }
    ok = ok && mbar_wait(&bars.pv_done, (tiles.count - 1) & 1, 128u);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      const float2 both = apart2(l);
      const float denominator = both.x + both.y;
      const bool empty = denominator == 0.f;      // not by m, which a row of NaN leaves at -inf, too
      const float inv = empty ? 0.f : 1.f / denominator;
      uint16_t *const out = o.at(batch, head, i), *const more = rest.data ? rest.at(batch, head, i) : nullptr;
      for (int c = 0; c < a.d; c += 16) {
        uint32_t x[16];
        tmem_ld16(t_o + c, x);
        tmem_wait_ld();
        if (i < a.n) {
          store8<kF16>(out + c, more ? more + c : nullptr, x, inv);
          if (c + 8 < a.d) store8<kF16>(out + c + 8, more ? more + c + 8 : nullptr, x + 8, inv);
        }
      }
      // Rows that see nothing, and those beyond the last, have weights of zero in the backward pass.
      if (nlse) nlse[(size_t)bh * a.npad + i] = i < a.n && !empty ? kUp - m - log2f(denominator) : -CUDART_INF_F;
    }
  }
  tc_fence_before();
  cta_teardown_sync();
  if (warp == 4) {
    tc_fence_after();
    tmem_free(tmem, kCols);
  }
}

}  // namespace px

#include "px_window_bwd.cuh"

namespace px {

PX_DEFINE_FAMILY_HOOKS(window)

// [batch][head][n][d] 16-bit values: boxes of 64 elements x 64 rows.
static bool rows_map(CUtensorMap* map, const px_rows& t, const px_window& w, int64_t heads) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  // the stride of an axis of length one is not used, but checked
  const auto stride = [&](int64_t s, int64_t len) { return (cuuint64_t)(len > 1 ? s * 2 : (w.d * 2 + 15) / 16 * 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)w.d, (cuuint64_t)w.n, (cuuint64_t)heads, (cuuint64_t)w.batch};
  const cuuint64_t strides[3] = {stride(t.row, w.n), stride(t.head, heads), stride(t.batch, w.batch)};
  const cuuint32_t box[4] = {64, 64, 1, 1}, one[4] = {1, 1, 1, 1};
  return enc(map, w.dtype == PX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.data), dims,
             strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr float kWMaxScale = 2.35e38f;      // the kernels multiply by scale * log2(e), which has to be finite
static int32_t window_check(const px_window* w) {
  if (!w || w->batch < 0 || w->n < 0 || w->heads <= 0 || w->kv_heads <= 0 || w->d <= 0 || w->left < 0 || w->right < 0 || w->sinks < 0 ||
      w->heads % w->kv_heads != 0 || !(w->scale > 0.f) || !(w->scale <= kWMaxScale))
    return PX_ERR_BAD_ARG;
  if ((w->dtype != PX_BF16 && w->dtype != PX_F16) || w->d % 8 != 0 || w->d > 128 || w->n > (1 << 24) || w->r_max > kWMaxR) return PX_ERR_UNSUPPORTED;
  if (w->heads / w->kv_heads * (w->n / kWCols + 1) > 0x3fffffffll) return PX_ERR_UNSUPPORTED;
  if (w->batch * w->heads * ((w->n + kWRows - 1) / kWRows) > 0x3fffffffll || w->batch > 65535 || w->heads > 65535) return PX_ERR_UNSUPPORTED;
  if (w->r_max >= 0 && (!w->bias || (w->bias_dtype != PX_F32 && w->bias_dtype != PX_BF16 && w->bias_dtype != PX_F16))) return PX_ERR_BAD_ARG;
  return PX_OK;
}
// Rows that the kernels can address: 16-byte aligned, strides of the axes longer than one multiples of 8 elements, a row at least (a tensor map
// asks for it) and below 2^40 bytes.
static bool rows_fit(const px_rows* t, const px_window& w, int64_t heads) {
  const auto fits = [&](int64_t s, int64_t len) { return len <= 1 || (s >= w.d && s % 8 == 0 && s < (1ll << 38)); };
  return t && t->data && ((uintptr_t)t->data & 15) == 0 && fits(t->row, w.n) && fits(t->head, heads) && fits(t->batch, w.batch);
}
static RowsOut rows_out(const px_rows* t) {
  return t ? RowsOut{(uint16_t*)t->data, t->batch, t->head, t->row} : RowsOut{nullptr, 0, 0, 0};
}
static WindowArgs window_args(const px_window& w) {
  WindowArgs a = {};
  const auto cut = [&](int64_t v) { return (int)(v < w.n ? v : w.n); };
  a.n = (int)w.n, a.d = (int)w.d, a.heads = (int)w.heads, a.kv_heads = (int)w.kv_heads, a.group = (int)(w.heads / w.kv_heads);
  a.tiles = (int)((w.n + kWRows - 1) / kWRows), a.npad = a.tiles * kWRows;
  a.left = cut(w.left), a.right = cut(w.right), a.sinks = cut(w.sinks), a.r = w.r_max < 0 ? -1 : (int)w.r_max;
  a.c = w.scale * kLog2e, a.mask = w.mask, a.bias = w.bias, a.bias_type = w.bias_dtype;
  return a;
}

template <bool kF16, int kD>
static bool launch_window_fwd(const px_window& w, const px_rows& q, const px_rows& k, const px_rows& v, const WindowArgs& a, const RowsOut& o,
                              const RowsOut& rest, float* lse, cudaStream_t st) {
  typedef WindowFwdLayout<kD> L;
  CUtensorMap mq, mk, mv;
  if (!rows_map(&mq, q, w, w.heads) || !rows_map(&mk, k, w, w.kv_heads) || !rows_map(&mv, v, w, w.kv_heads)) return false;
  static SmemLimit limit;
  if (!limit.set(window_fwd_kernel<kF16, kD>, L::bytes(kWMaxR) + 1024)) return false;
  return launch_pdl(window_fwd_kernel<kF16, kD>, dim3((unsigned)((int64_t)a.tiles * w.heads * w.batch)), kWFwdThreads, (size_t)L::bytes(a.r) + 1024,
                    st, mq, mk, mv, a, o, rest, lse);
}

}  // namespace px

using namespace px;

extern "C" int64_t px_window_lse_floats(int64_t batch, int64_t heads, int64_t n) { return batch * heads * ((n + kWRows - 1) / kWRows * kWRows); }

extern "C" int32_t px_window_fwd(const px_window* w, const px_rows* q, const px_rows* k, const px_rows* v, const px_rows* o, const px_rows* o_rest,
                                 float* lse, void* stream) {
  const int32_t status = window_check(w);
  if (status != PX_OK) return status;
  if (w->batch == 0 || w->n == 0) return PX_OK;
  if (!rows_fit(q, *w, w->heads) || !rows_fit(k, *w, w->kv_heads) || !rows_fit(v, *w, w->kv_heads) || !rows_fit(o, *w, w->heads) ||
      (o_rest && !rows_fit(o_rest, *w, w->heads)))
    return PX_ERR_BAD_ARG;
  if (!have_context()) return PX_ERR_LAUNCH;
  const auto go = w->dtype == PX_F16 ? (w->d <= 32 ? launch_window_fwd<true, 32> : w->d <= 64 ? launch_window_fwd<true, 64> : launch_window_fwd<true, 128>)
                                     : (w->d <= 32   ? launch_window_fwd<false, 32>
                                        : w->d <= 64 ? launch_window_fwd<false, 64>
                                                     : launch_window_fwd<false, 128>);
  return go(*w, *q, *k, *v, window_args(*w), rows_out(o), rows_out(o_rest), lse, (cudaStream_t)stream) ? PX_OK : PX_ERR_LAUNCH;
}

namespace px {

// How the queries beyond the window that see sinks are cut: key tiles that hold sinks, chunks each, streamed tiles a chunk.
static void sink_chunks(const WindowArgs& a, int* tiles, int* chunks, int* chunk) {
  *tiles = (a.sinks + kWRows - 1) / kWRows;
  int most = 0;
  if (*tiles > 0) most = ((a.n - 1) / kWCols - last_of_window(a.n, a.left, 0)) * a.group;      // the first tile has the most
  const int window = ((kWRows + a.left + a.right) / kWCols + 2) * a.group;      // about what the other CTAs have
  *chunk = std::max(window, std::max(16, (most + 15) / 16));
  if (*tiles > 16 && *chunk < (most + 1) / 2) *chunk = (most + 1) / 2;      // CTAs enough, and each chunk takes memory for its sums
  *chunks = most > 0 ? (most + *chunk - 1) / *chunk : 0;
  if (*chunks > 0) *chunk = (most + *chunks - 1) / *chunks;      // alike
  if (*chunks == 0) *tiles = 0;
}
static int64_t al256(int64_t n) { return (n + 255) / 256 * 256; }
struct WindowSpace {
  int64_t delta, dbias, sinks, arrived, total;      // where they begin; bytes
};
static WindowSpace window_space(const px_window& w, const WindowArgs& a, bool bias_grad) {
  int tiles, chunks, chunk;
  sink_chunks(a, &tiles, &chunks, &chunk);
  WindowSpace s;
  s.delta = 0;
  s.dbias = al256(w.batch * w.heads * (int64_t)a.npad * 4);
  s.sinks = s.dbias + (bias_grad ? al256(w.batch * w.heads * a.tiles * (2 * (int64_t)a.r + 1) * 4) : 0);
  s.arrived = s.sinks + al256(w.batch * w.kv_heads * (int64_t)tiles * (1 + chunks) * 2 * kWRows * ((a.d + 15) & ~15) * 4);
  s.total = s.arrived + w.batch * w.kv_heads * (int64_t)tiles * 4;
  return s;
}

template <bool kF16, int kLanes>
static bool launch_window_delta(const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dout, const RowsOut& o, const RowsOut& rest, cudaStream_t st) {
  const int64_t blocks = (int64_t)a.heads * g.batches * (a.npad / delta_block(kLanes));
  return launch_pdl(window_delta_kernel<kF16, kLanes>, dim3((unsigned)blocks), 256, 0, st, a, g, dout, o, rest);
}
template <bool kF16, int kD, bool kBiasGrad>
static bool launch_window_dq(const CUtensorMap* m, const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dq, int64_t blocks, cudaStream_t st) {
  typedef WindowDqLayout<kD> L;
  static SmemLimit limit;
  const auto kernel = window_dq_kernel<kF16, kD, kBiasGrad>;
  if (!limit.set(kernel, L::bytes(kWMaxR, kBiasGrad) + 1024)) return false;
  return launch_pdl(kernel, dim3((unsigned)blocks), kWDqThreads, (size_t)L::bytes(a.r, kBiasGrad) + 1024, st, m[0], m[1], m[2], m[3], a, g, dq);
}
template <bool kF16, int kD>
static bool launch_window_dkv(const CUtensorMap* m, const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dk, const RowsOut& dv, int64_t blocks,
                              cudaStream_t st) {
  typedef WindowDkvLayout<kD> L;
  static SmemLimit limit;
  const auto kernel = window_dkv_kernel<kF16, kD>;
  if (!limit.set(kernel, L::bytes(kWMaxR) + 1024)) return false;
  return launch_pdl(kernel, dim3((unsigned)blocks), L::threads, (size_t)L::bytes(a.r) + 1024, st, m[0], m[1], m[2], m[3], a, g, dk, dv);
}

struct BwdRows {
  const px_rows *q, *k, *v, *o, *o_rest, *dout, *dq, *dk, *dv;
};
template <bool kF16>
static bool window_bwd(const px_window& w, const BwdRows& x, const WindowArgs& a, WindowBwdArgs g, void* dbias, cudaStream_t st) {
  const int64_t blocks = (int64_t)a.tiles * w.heads * w.batch;
  const RowsOut dout = rows_out(x.dout), o = rows_out(x.o), rest = rows_out(x.o_rest), dq = rows_out(x.dq), dk = rows_out(x.dk), dv = rows_out(x.dv);
  CUtensorMap m[4];
  if (!rows_map(&m[0], *x.q, w, w.heads) || !rows_map(&m[1], *x.dout, w, w.heads) || !rows_map(&m[2], *x.k, w, w.kv_heads) ||
      !rows_map(&m[3], *x.v, w, w.kv_heads))
    return false;
  g.own = dk.data || dv.data;
  const bool queries = dq.data || dbias;
  g.early = queries && g.own;
  if (!queries && !g.own) return true;
  const auto go_delta = w.d <= 32 ? launch_window_delta<kF16, 4> : w.d <= 64 ? launch_window_delta<kF16, 8> : launch_window_delta<kF16, 16>;
  if (!go_delta(a, g, dout, o, rest, st)) return false;
  const auto go_q = w.d <= 64 ? (dbias ? launch_window_dq<kF16, 64, true> : launch_window_dq<kF16, 64, false>)
                              : (dbias ? launch_window_dq<kF16, 128, true> : launch_window_dq<kF16, 128, false>);
  if (queries && !go_q(m, a, g, dq, blocks, st)) return false;
  const int64_t own = g.own ? (int64_t)(a.tiles + g.sink_tiles * g.chunks) * w.kv_heads * w.batch : 0;
  const int64_t buckets = dbias ? (int64_t)w.heads * g.bias_blocks : 0;
  if (own + buckets == 0) return true;
  const auto go_kv = w.d <= 32 ? launch_window_dkv<kF16, 32> : w.d <= 64 ? launch_window_dkv<kF16, 64> : launch_window_dkv<kF16, 128>;
  return go_kv(m, a, g, dk, dv, own + buckets, st);
}

}  // namespace px

extern "C" int64_t px_window_workspace_bytes(const px_window* w, int32_t bias_grad) {
  if (window_check(w) != PX_OK || w->batch == 0 || w->n == 0) return 0;
  return window_space(*w, window_args(*w), bias_grad && w->r_max >= 0).total;
}

extern "C" int32_t px_window_bwd(const px_window* w, const px_rows* q, const px_rows* k, const px_rows* v, const px_rows* o, const px_rows* o_rest,
                                 const px_rows* dout, const float* lse, const px_rows* dq, const px_rows* dk, const px_rows* dv, void* dbias, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const int32_t status = window_check(w);
  if (status != PX_OK) return status;
  const cudaStream_t st = (cudaStream_t)stream;
  if (w->batch == 0 || w->n == 0) {
    if (!dbias || w->r_max < 0) return PX_OK;
    const size_t bytes = (size_t)w->heads * (2 * w->r_max + 1) * (w->bias_dtype == PX_F32 ? 4 : 2);
    return cudaMemsetAsync(dbias, 0, bytes, st) == cudaSuccess ? PX_OK : PX_ERR_LAUNCH;
  }
  if (!rows_fit(q, *w, w->heads) || !rows_fit(k, *w, w->kv_heads) || !rows_fit(v, *w, w->kv_heads) || !rows_fit(o, *w, w->heads) ||
      (o_rest && !rows_fit(o_rest, *w, w->heads)) || !rows_fit(dout, *w, w->heads) || (dq && !rows_fit(dq, *w, w->heads)) || (dk && !rows_fit(dk, *w, w->kv_heads)) ||
      (dv && !rows_fit(dv, *w, w->kv_heads)) || !lse || ((uintptr_t)lse & 15) || !workspace || ((uintptr_t)workspace & 255) ||
      (dbias && w->r_max < 0))
    return PX_ERR_BAD_ARG;
  const WindowArgs a = window_args(*w);
  const WindowSpace space = window_space(*w, a, dbias != nullptr);
  if (workspace_bytes < space.total) return PX_ERR_WORKSPACE;
  if (!have_context()) return PX_ERR_LAUNCH;
  WindowBwdArgs g = {};
  unsigned char* const ws = (unsigned char*)workspace;
  g.nlse = lse;
  g.ndelta = (float*)(ws + space.delta);
  g.dbias = (float*)(ws + space.dbias);
  g.sinks = (float*)(ws + space.sinks);
  g.arrived = (unsigned int*)(ws + space.arrived);
  g.dbias_out = dbias;
  g.bias_blocks = dbias ? (2 * a.r + 1 + 31) / 32 : 0;
  g.batches = (int)w->batch;
  g.scale = w->scale;
  sink_chunks(a, &g.sink_tiles, &g.chunks, &g.chunk);
  if ((int64_t)(a.tiles + g.sink_tiles * g.chunks) * w->kv_heads * w->batch > 0x3fffffffll) return PX_ERR_UNSUPPORTED;
  const BwdRows rows = {q, k, v, o, o_rest, dout, dq, dk, dv};
  return (w->dtype == PX_F16 ? window_bwd<true>(*w, rows, a, g, dbias, st) : window_bwd<false>(*w, rows, a, g, dbias, st)) ? PX_OK : PX_ERR_LAUNCH;
}
