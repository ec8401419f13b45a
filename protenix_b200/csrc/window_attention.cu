// Attention with a sliding window, first tokens that stay visible and a learned bias by offset, on the 5th-generation tensor cores.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax over visible j of  scale q_i . k_j + bias[head][clip(j - i, -r, r) + r]
//   j is visible to i when mask[j] and j <= i + right and (j >= i - left or j < sinks);  a row that sees nothing gives 0.
//
// q, k, v: [batch][head][n][d], any strides along batch, head and row, bf16 or fp16, d a multiple of 8 up to 128; heads of k and v may serve a
// group of q's heads each.
//
// One CTA = 128 queries of a head, streamed over the 64-key tiles that they see.  Warps 0..3: one thread a query row.  Warp 4
// loads Q once and K, V tiles by TMA (panels of 64 elements, 128-byte swizzle, a ring of two each) and issues S = Q K^T and,
// once the rows have put P (16 bits) in S's place in tensor memory, O += P V with V read as it lies, along its rows.
// Softmax is online in base 2 with a reference maximum that moves (and O with it) only when a tile exceeds it by more than 8: P is 2^8 at most.
// Logits, statistics and O are fp32; P is rounded to the type of V, which the product needs (relative error of half a step, 2^-9 or 2^-12,
// with either sign); the denominators sum the fp32 values.
//
// Tiles that every query sees whole, the larger part of a wide window, take no per-element test; elsewhere a row's visible keys are a 64-bit
// word.  Where all offsets of a tile are clipped alike the bias is one number, elsewhere it is read from shared memory, where the head's row lies
// continued beyond its ends, so that a thread's 64 values lie side by side.
//
// TMEM: S / P (64 columns) | O.  d <= 64: 128 columns, four CTAs an SM hide one another's chain of product, softmax, product.
#include "px_window.cuh"

namespace px {

constexpr float kWRescaleGap = 8.0f;
constexpr int kWFwdThreads = 160;

struct WindowFwdBars {
  uint64_t q_full, k_full[2], v_full[2], s_full, p_ready, pv_done;
  uint32_t tmem_base;
};

template <int kPanels>
struct WindowFwdLayout {
  static constexpr int q = 0, tile = kPanels * kWCols * 128;
  static constexpr int k = kPanels * kWRows * 128, v = k + 2 * tile, bars = v + 2 * tile;
  static constexpr int bias = bars + 128;
  static constexpr int bytes(int r) { return bias + bias_floats(r) * 4; }
};
static_assert(sizeof(WindowFwdBars) <= 128, "room for the barriers");

template <bool kF16, int kPanels>
__global__ void __launch_bounds__(kWFwdThreads, kPanels == 1 ? 4 : 2)
window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const WindowArgs a, const RowsOut o, float* __restrict__ lse) {
  typedef WindowFwdLayout<kPanels> L;
  constexpr uint32_t kCols = kPanels == 1 ? 128 : 256;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  WindowFwdBars& bars = *reinterpret_cast<WindowFwdBars*>(sm + L::bars);
  float* const bias = reinterpret_cast<float*>(sm + L::bias);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int q0 = (int)(blockIdx.x % a.tiles) * kWRows, bh = blockIdx.x / a.tiles, head = bh % a.heads, batch = bh / a.heads;
  const KeyTiles tiles(a, q0);

  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    prefetch_maps(map_q, map_k, map_v);
    mbar_init(&bars.q_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.v_full[s], 1);
    }
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.p_ready, 4);
    mbar_init(&bars.pv_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 4) tmem_alloc(&bars.tmem_base, kCols);
  if (!cta_ready(skip, warp == 4, bars.tmem_base, kCols)) return;
  const uint32_t tmem = bars.tmem_base;
  if (a.r >= 0) bias_fill(a, head, bias);
  __syncthreads();

  if (warp == 4) {
    // ------------------------------------------------------------------ copies and products
    const int kv = head / a.group;
    const uint32_t q_at = smem_u32(sm), k_at = smem_u32(sm + L::k), v_at = smem_u32(sm + L::v);
    const uint32_t idesc_s = umma_idesc_16(128, kWCols, kF16, kF16), idesc_o = umma_idesc_16(128, (a.d + 15) & ~15, kF16, kF16, false, true);
    const auto load_k = [&](int t) {      // one lane
      mbar_expect_tx(&bars.k_full[t & 1], L::tile);
      load_rows<kPanels>(k_at + (t & 1) * L::tile, &map_k, &bars.k_full[t & 1], kWCols, tiles.key(t), kv, batch);
    };
    const auto load_v = [&](int t) {
      mbar_expect_tx(&bars.v_full[t & 1], L::tile);
      load_rows<kPanels>(v_at + (t & 1) * L::tile, &map_v, &bars.v_full[t & 1], kWCols, tiles.key(t), kv, batch);
    };
    const auto issue_s = [&](int t) {
      if (!mbar_wait_warp(&bars.k_full[t & 1], (t >> 1) & 1, 2u)) return false;
      tc_fence_after();
      if (elect_lane()) {
        mma_rows(tmem, q_at, k_at + (t & 1) * L::tile, kWCols, (a.d + 15) / 16, idesc_s);
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
      ok = mbar_wait_warp(&bars.p_ready, t & 1, 4u);          // S(t) is complete and read: its K tile is free
      if (!ok) break;
      if (t + 2 < tiles.count && elect_lane()) load_k(t + 2);
      __syncwarp();
      ok = mbar_wait_warp(&bars.v_full[t & 1], (t >> 1) & 1, 8u);
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        mma_streamed(tmem + kWCols, tmem, v_at + (t & 1) * L::tile, idesc_o, t == 0);
        umma_commit(&bars.pv_done);
      }
      __syncwarp();
      ok = mbar_wait_warp(&bars.pv_done, t & 1, 16u);         // P, which lies where the next S goes, has been read
      if (!ok) break;
      if (t + 2 < tiles.count && elect_lane()) load_v(t + 2);
      __syncwarp();
      if (t + 1 < tiles.count) ok = issue_s(t + 1);
    }
  } else {
    // ------------------------------------------------------------------ one query row a thread
    const int row = threadIdx.x, i = q0 + row;
    const uint32_t t_s = tmem + ((uint32_t)(32 * warp) << 16), t_o = t_s + kWCols;
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int t = 0; t < tiles.count; ++t) {
      const int k0 = tiles.key(t);
      const uint64_t keys = key_bits(a, batch, k0, lane);
      const bool whole = keys == ~0ull && window_covers(a, q0, k0);
      ok = mbar_wait(&bars.s_full, t & 1, 32u);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      float s[kWCols];
      tmem_ld32(t_s, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
      tmem_ld32(t_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
      tmem_wait_ld();
      // logits = s * mul + add, in base 2
      float mul = a.c, add = 0.f;
      if (a.r >= 0) {
        if (clipped_low(a, k0 + kWCols - 1 - q0)) {
          add = bias[0];
        } else if (clipped_high(a, k0 - q0 - (kWRows - 1))) {
          add = bias[bias_floats(a.r) - 1];
        } else {
          const float* b = bias + (k0 - i + a.r + kWBiasBeyond);
#pragma unroll
          for (int c = 0; c < kWCols; ++c) s[c] = fmaf(s[c], mul, b[c]);
          mul = 1.f;
        }
      }
      if (!whole) {
        const uint64_t seen = visible_bits(a, i, k0, keys);
        const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
        for (int c = 0; c < kWCols; ++c) s[c] = ((c < 32 ? lo : hi) >> (c & 31) & 1u) ? s[c] : -CUDART_INF_F;
      }
      float mq[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mq[k] = s[16 * k];
#pragma unroll
        for (int e = 1; e < 16; ++e) mq[k] = fmaxf(mq[k], s[16 * k + e]);
      }
      const float mt = fmaf(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])), mul, add);
      const bool up = mt > m + kWRescaleGap;
      const bool move = __any_sync(0xffffffffu, up) && t > 0;      // the first product overwrites O
      const float m_old = m;
      m = up ? mt : m;
      const float shift = add - (m == -CUDART_INF_F ? 0.f : m);
      if (move) {                                                   // O is at rest: S(t) was issued after P V (t - 1) was complete
        const float alpha = up ? fast_exp2(m_old - m) : 1.f;
        l *= alpha;
        for (int c = 0; c < a.d; c += 16) {
          uint32_t x[16];
          tmem_ld16(t_o + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
          tmem_st16(t_o + c, x);
        }
      }
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = fast_exp2(fmaf(s[32 * k + 2 * e], mul, shift)), p1 = fast_exp2(fmaf(s[32 * k + 2 * e + 1], mul, shift));
          add2(l0, l1, p0, p1);
          w[e] = pack16x2<kF16>(p0, p1);
        }
        tmem_st16(t_s + 16 * k, w);
      }
      l += l0 + l1;
      if (keys != bits_between(0, a.n - 1 - k0)) {                  // masked keys: their rows of V, by one thread of each half
        ok = mbar_wait_warp(&bars.v_full[t & 1], (t >> 1) & 1, 64u);
        if (!ok) break;
        if (!(keys >> (row & 63) & 1)) clear_row<kPanels>(sm + L::v + (t & 1) * L::tile, row & 63, row >> 6, 2);
        fence_async_shared();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_ready);
    }
    ok = ok && mbar_wait(&bars.pv_done, (tiles.count - 1) & 1, 128u);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      const bool empty = !(l > 0.f) && m == -CUDART_INF_F;
      const float inv = empty ? 0.f : 1.f / l;
      uint16_t* const out = o.at(batch, head, i);
      for (int c = 0; c < a.d; c += 16) {
        uint32_t x[16];
        tmem_ld16(t_o + c, x);
        tmem_wait_ld();
        if (i < a.n) {
          store8<kF16>(out + c, x, inv);
          if (c + 8 < a.d) store8<kF16>(out + c + 8, x + 8, inv);
        }
      }
      // Rows that see nothing, and those beyond the last, have weights of zero in the backward pass.
      if (lse) lse[(size_t)bh * a.npad + i] = i < a.n && !empty ? m + log2f(l) : CUDART_INF_F;
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

// A thread that has not used the device yet, as the one that runs a backward pass, has no context for the driver to encode a map in: naming the
// device that is current anyway gives it one.
static bool have_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

// [batch][head][n][d] 16-bit values: boxes of 64 elements x `rows`.
static bool rows_map(CUtensorMap* map, const px_rows& t, const px_window& w, int64_t heads, uint32_t rows) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  // the stride of an axis of length one is not used, but checked
  const auto stride = [&](int64_t s, int64_t len) { return (cuuint64_t)(len > 1 ? s * 2 : (w.d * 2 + 15) / 16 * 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)w.d, (cuuint64_t)w.n, (cuuint64_t)heads, (cuuint64_t)w.batch};
  const cuuint64_t strides[3] = {stride(t.row, w.n), stride(t.head, heads), stride(t.batch, w.batch)};
  const cuuint32_t box[4] = {64, rows, 1, 1}, one[4] = {1, 1, 1, 1};
  return enc(map, w.dtype == PX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.data), dims,
             strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int32_t window_check(const px_window* w) {
  if (!w || w->batch < 0 || w->n < 0 || w->heads <= 0 || w->kv_heads <= 0 || w->d <= 0 || w->left < 0 || w->right < 0 || w->sinks < 0 ||
      w->heads % w->kv_heads != 0 || !(w->scale > 0.f) || !(w->scale <= 3.0e38f))
    return PX_ERR_BAD_ARG;
  if ((w->dtype != PX_BF16 && w->dtype != PX_F16) || w->d % 8 != 0 || w->d > 128 || w->n > (1 << 24) || w->r_max > kWMaxR) return PX_ERR_UNSUPPORTED;
  if (w->batch * w->heads * ((w->n + kWRows - 1) / kWRows) > 0x3fffffffll || w->batch > 65535 || w->heads > 65535) return PX_ERR_UNSUPPORTED;
  if (w->r_max >= 0 && (!w->bias || (w->bias_dtype != PX_F32 && w->bias_dtype != PX_BF16 && w->bias_dtype != PX_F16))) return PX_ERR_BAD_ARG;
  return PX_OK;
}
// Rows that the kernels can address: 16-byte aligned, strides of the axes longer than one multiples of 8 elements, positive and below 2^40 bytes.
static bool rows_fit(const px_rows* t, const px_window& w, int64_t heads) {
  const auto fits = [](int64_t s, int64_t len) { return len <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
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

template <bool kF16, int kPanels>
static bool launch_window_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const WindowArgs& a, const RowsOut& o, float* lse,
                              int64_t blocks, cudaStream_t st) {
  typedef WindowFwdLayout<kPanels> L;
  static SmemLimit limit;
  if (!limit.set(window_fwd_kernel<kF16, kPanels>, L::bytes(kWMaxR) + 1024)) return false;
  return launch_pdl(window_fwd_kernel<kF16, kPanels>, dim3((unsigned)blocks), kWFwdThreads, (size_t)L::bytes(a.r) + 1024, st, mq, mk, mv, a, o, lse);
}

}  // namespace px

using namespace px;

extern "C" int64_t px_window_lse_floats(int64_t batch, int64_t heads, int64_t n) { return batch * heads * ((n + kWRows - 1) / kWRows * kWRows); }

extern "C" int32_t px_window_fwd(const px_window* w, const px_rows* q, const px_rows* k, const px_rows* v, const px_rows* o, float* lse,
                                 void* stream) {
  const int32_t status = window_check(w);
  if (status != PX_OK) return status;
  if (w->batch == 0 || w->n == 0) return PX_OK;
  if (!rows_fit(q, *w, w->heads) || !rows_fit(k, *w, w->kv_heads) || !rows_fit(v, *w, w->kv_heads) || !rows_fit(o, *w, w->heads))
    return PX_ERR_BAD_ARG;
  CUtensorMap mq, mk, mv;
  if (!have_context() || !rows_map(&mq, *q, *w, w->heads, kWRows) || !rows_map(&mk, *k, *w, w->kv_heads, kWCols) || !rows_map(&mv, *v, *w, w->kv_heads, kWCols))
    return PX_ERR_LAUNCH;
  const WindowArgs a = window_args(*w);
  const auto go = w->dtype == PX_F16 ? (w->d <= 64 ? launch_window_fwd<true, 1> : launch_window_fwd<true, 2>)
                                     : (w->d <= 64 ? launch_window_fwd<false, 1> : launch_window_fwd<false, 2>);
  return go(mq, mk, mv, a, rows_out(o), lse, (int64_t)a.tiles * w->heads * w->batch, (cudaStream_t)stream) ? PX_OK : PX_ERR_LAUNCH;
}

namespace px {

// How the queries beyond the window that see sinks are cut: key tiles that hold sinks, chunks each, streamed tiles a chunk.
static void sink_chunks(const WindowArgs& a, int* tiles, int* chunks, int* chunk) {
  *tiles = (a.sinks + kWRows - 1) / kWRows;
  const int window = ((kWRows + a.left + a.right) / kWCols + 2) * a.group;      // about what the other CTAs have
  *chunk = window > 64 ? window : 64;
  int most = 0;
  if (*tiles > 0) most = ((a.n - 1) / kWCols - last_of_window(a.n, a.left, 0)) * a.group;      // the first tile has the most
  *chunks = most > 0 ? (most + *chunk - 1) / *chunk : 0;
  if (*chunks == 0) *tiles = 0;
}
static int64_t al256(int64_t n) { return (n + 255) / 256 * 256; }
struct WindowSpace {
  int64_t delta, dbias, sinks, total;      // where they begin; bytes
};
static WindowSpace window_space(const px_window& w, const WindowArgs& a, bool bias_grad) {
  int tiles, chunks, chunk;
  sink_chunks(a, &tiles, &chunks, &chunk);
  WindowSpace s;
  s.delta = 0;
  s.dbias = al256(w.batch * w.heads * (int64_t)a.npad * 4);
  s.sinks = s.dbias + (bias_grad ? al256(w.batch * w.heads * a.tiles * (2 * (int64_t)a.r + 1) * 4) : 0);
  s.total = s.sinks + w.batch * w.kv_heads * (int64_t)tiles * (1 + chunks) * 2 * kWRows * ((a.d + 15) & ~15) * 4;
  return s;
}

template <bool kF16, int kPanels, bool kBiasGrad>
static bool launch_window_dq(const CUtensorMap* m, const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dout, const RowsOut& o,
                             const RowsOut& dq, int64_t blocks, cudaStream_t st) {
  typedef WindowDqLayout<kPanels> L;
  static SmemLimit limit;
  const auto kernel = window_dq_kernel<kF16, kPanels, kBiasGrad>;
  if (!limit.set(kernel, L::bytes(kWMaxR, kBiasGrad) + 1024)) return false;
  return launch_pdl(kernel, dim3((unsigned)blocks), kWBwdThreads, (size_t)L::bytes(a.r, kBiasGrad) + 1024, st, m[0], m[1], m[2], m[3], a, g, dout, o,
                    dq);
}
template <bool kF16, int kPanels>
static bool launch_window_dkv(const CUtensorMap* m, const WindowArgs& a, const WindowBwdArgs& g, const RowsOut& dk, const RowsOut& dv, int64_t blocks,
                              cudaStream_t st) {
  typedef WindowDkvLayout<kPanels> L;
  static SmemLimit limit;
  const auto kernel = window_dkv_kernel<kF16, kPanels>;
  if (!limit.set(kernel, L::bytes(kWMaxR) + 1024)) return false;
  return launch_pdl(kernel, dim3((unsigned)blocks), kWBwdThreads, (size_t)L::bytes(a.r) + 1024, st, m[0], m[1], m[2], m[3], a, g, dk, dv);
}

template <bool kF16, int kPanels>
static bool window_bwd(const px_window& w, const CUtensorMap* own_q, const CUtensorMap* own_k, const WindowArgs& a, const WindowBwdArgs& g,
                       const RowsOut& dout, const RowsOut& o, const RowsOut& dq, const RowsOut& dk, const RowsOut& dv, void* dbias, cudaStream_t st) {
  const int64_t blocks = (int64_t)a.tiles * w.heads * w.batch;
  if (!(dbias ? launch_window_dq<kF16, kPanels, true>(own_q, a, g, dout, o, dq, blocks, st)
              : launch_window_dq<kF16, kPanels, false>(own_q, a, g, dout, o, dq, blocks, st)))
    return false;
  if (dbias) {
    const int buckets = 2 * a.r + 1;
    window_dbias_kernel<<<dim3((unsigned)((buckets + 31) / 32), (unsigned)w.heads), 1024, 0, st>>>(g.dbias, dbias, a.bias_type, (int)w.batch, a.heads,
                                                                                                a.tiles, buckets);
    if (cudaGetLastError() != cudaSuccess) return false;
  }
  if (!dk.data && !dv.data) return true;
  if (!launch_window_dkv<kF16, kPanels>(own_k, a, g, dk, dv, (int64_t)(a.tiles + g.sink_tiles * g.chunks) * w.kv_heads * w.batch, st)) return false;
  if (g.chunks > 0) {
    const int rows = a.n < g.sink_tiles * kWRows ? a.n : g.sink_tiles * kWRows;
    const int64_t per = (2 * (int64_t)rows * (a.d / 8) + 255) / 256;
    window_sink_kernel<kF16><<<(unsigned)(per * w.batch * w.kv_heads), 256, 0, st>>>(a, g, dk, dv);
    if (cudaGetLastError() != cudaSuccess) return false;
  }
  return true;
}

}  // namespace px

extern "C" int64_t px_window_workspace_bytes(const px_window* w, int32_t bias_grad) {
  if (window_check(w) != PX_OK || w->batch == 0 || w->n == 0) return 0;
  return window_space(*w, window_args(*w), bias_grad && w->r_max >= 0).total;
}

extern "C" int32_t px_window_bwd(const px_window* w, const px_rows* q, const px_rows* k, const px_rows* v, const px_rows* o, const px_rows* dout,
                                 const float* lse, const px_rows* dq, const px_rows* dk, const px_rows* dv, void* dbias, void* workspace,
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
      !rows_fit(dout, *w, w->heads) || (dq && !rows_fit(dq, *w, w->heads)) || (dk && !rows_fit(dk, *w, w->kv_heads)) ||
      (dv && !rows_fit(dv, *w, w->kv_heads)) || !lse || ((uintptr_t)lse & 15) || !workspace || ((uintptr_t)workspace & 255) ||
      (dbias && w->r_max < 0))
    return PX_ERR_BAD_ARG;
  const WindowArgs a = window_args(*w);
  const WindowSpace space = window_space(*w, a, dbias != nullptr);
  if (workspace_bytes < space.total) return PX_ERR_WORKSPACE;
  CUtensorMap own_q[4], own_k[4];      // q, dO, k, v as the two kernels cut them
  if (!have_context() || !rows_map(&own_q[0], *q, *w, w->heads, kWRows) || !rows_map(&own_q[1], *dout, *w, w->heads, kWRows) ||
      !rows_map(&own_q[2], *k, *w, w->kv_heads, kWCols) || !rows_map(&own_q[3], *v, *w, w->kv_heads, kWCols) ||
      !rows_map(&own_k[0], *q, *w, w->heads, kWCols) || !rows_map(&own_k[1], *dout, *w, w->heads, kWCols) ||
      !rows_map(&own_k[2], *k, *w, w->kv_heads, kWRows) || !rows_map(&own_k[3], *v, *w, w->kv_heads, kWRows))
    return PX_ERR_LAUNCH;
  WindowBwdArgs g = {};
  unsigned char* const ws = (unsigned char*)workspace;
  g.lse = lse;
  g.delta = (float*)(ws + space.delta);
  g.dbias = (float*)(ws + space.dbias);
  g.sinks = (float*)(ws + space.sinks);
  g.scale = w->scale;
  sink_chunks(a, &g.sink_tiles, &g.chunks, &g.chunk);
  if ((int64_t)(a.tiles + g.sink_tiles * g.chunks) * w->kv_heads * w->batch > 0x3fffffffll) return PX_ERR_UNSUPPORTED;
  const auto go = w->dtype == PX_F16 ? (w->d <= 64 ? window_bwd<true, 1> : window_bwd<true, 2>) : (w->d <= 64 ? window_bwd<false, 1> : window_bwd<false, 2>);
  return go(*w, own_q, own_k, a, g, rows_out(dout), rows_out(o), rows_out(dq), rows_out(dk), rows_out(dv), dbias, st) ? PX_OK : PX_ERR_LAUNCH;
}
