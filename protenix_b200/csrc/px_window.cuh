// What the kernels of windowed attention share (window_attention.cu, px_window_bwd.cuh): the geometry of the window, the
// tiles, the learned bias.
#pragma once
#include <math_constants.h>

#include "px_tcgen05.cuh"

namespace px {

constexpr int kWRows = 128;      // rows a CTA owns: queries (forward, dQ) or keys (dK, dV)
constexpr int kWCols = 64;       // keys or queries of a streamed tile of the backward pass
constexpr int kWMaxR = 256;      // largest clipping distance of the learned bias

// A call, as the kernels see it.  left, right and sinks are at most n.
struct WindowArgs {
  int n, d, heads, kv_heads, group, tiles;     // group: heads / kv_heads; tiles of kWRows rows
  int left, right, sinks, r;                   // r < 0: no bias
  int npad;                                    // row statistics are [batch * heads][npad]
  float c;                                     // scale * log2(e)
  const uint8_t* mask;                         // [batch][n] or NULL
  const void* bias;                            // [heads][2 r + 1]
  int bias_type;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// A tile of `rows` rows (a multiple of 64, which is the box) as panels of 64 elements (128 bytes, 128-byte swizzle), one behind the other.  Elements
// beyond d and rows beyond n arrive as zeros.
template <int kPanels>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int rows, int row0, int head, int batch) {
#pragma unroll
  for (int p = 0; p < kPanels; ++p)
    for (int r = 0; r < rows; r += 64) tma_load_4d(dst + (p * rows + r) * 128, map, bar, 64 * p, row0 + r, head, batch);
}

// The products, by one lane.  What their descriptors have in common is formed once a call.
//
// D[128][kRows] = A B^T over d (`steps` of 16), A [128] and B [kRows] rows, both K-major panels of 64.
template <int kPanels, int kRows>
__device__ __forceinline__ void mma_rows(uint32_t d_tmem, uint32_t a, uint32_t b, int steps, uint32_t idesc) {
  const uint64_t da = umma_desc_sw128(a), db = umma_desc_sw128(b);
#pragma unroll
  for (int ks = 0; ks < 4 * kPanels; ++ks)
    if (ks < steps) umma_bf16(d_tmem, da + (ks >> 2) * (kWRows * 8) + 2 * (ks & 3), db + (ks >> 2) * (kRows * 8) + 2 * (ks & 3), idesc, ks > 0);
}
// D[128][d] += A[128][64] B with A in tensor memory and B a streamed tile [64][d], read along its rows.
__device__ __forceinline__ void mma_streamed(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool first) {
  const uint64_t db = umma_desc_mn_sw128(b, 64 * 128, 1024);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) umma_bf16_ts(d_tmem, a_tmem + 8 * ks, db + 128 * ks, idesc, !first || ks > 0);
}
// The same with A in shared memory, a panel of 64.
__device__ __forceinline__ void mma_streamed_ss(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, bool first) {
  const uint64_t da = umma_desc_sw128(a), db = umma_desc_mn_sw128(b, 64 * 128, 1024);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) umma_bf16(d_tmem, da + 2 * ks, db + 128 * ks, idesc, !first || ks > 0);
}
// 32 values (16 words) of row `row` into such a panel, columns 32 * half and up.
__device__ __forceinline__ void panel_store(unsigned char* panel, int row, int half, const uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    *reinterpret_cast<uint4*>(panel + row * 128 + (((4 * half + e) ^ (row & 7)) << 4)) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
}

// Streamed key tiles of the queries [q0, q0 + 128): the first tiles as far as they hold sinks, then those of the window.
template <int kKT>
struct KeyTiles {
  int sink, first, count;
  __device__ __forceinline__ KeyTiles(const WindowArgs& a, int q0) {
    const int lo = max(0, q0 - a.left), hi = min(a.n - 1, q0 + kWRows - 1 + a.right);
    first = lo / kKT;
    sink = min((a.sinks + kKT - 1) / kKT, first);
    count = sink + hi / kKT - first + 1;
  }
  __device__ __forceinline__ int key(int t) const { return (t < sink ? t : first + t - sink) * kKT; }
};

// Bits from .. to of a word, both cut to 0 .. 31.
__device__ __forceinline__ uint32_t bits_between(int from, int to) {
  from = max(from, 0), to = min(to, 31);
  return from > to ? 0u : (0xffffffffu << from) & (0xffffffffu >> (31 - to));
}
// Bit c: key k0 + c exists and is not masked (whole warp).
__device__ __forceinline__ uint32_t key_bits(const WindowArgs& a, int batch, int k0, int lane) {
  if (!a.mask) return bits_between(0, a.n - 1 - k0);
  return __ballot_sync(0xffffffffu, k0 + lane < a.n && __ldg(a.mask + (size_t)batch * a.n + min(k0 + lane, a.n - 1)) != 0);
}
// Bit c: query i sees key k0 + c.
__device__ __forceinline__ uint32_t visible_bits(const WindowArgs& a, int i, int k0, uint32_t keys) {
  const int hi = i + a.right - k0;
  return (bits_between(i - a.left - k0, hi) | bits_between(0, min(a.sinks - 1 - k0, hi))) & keys;
}
// What a block of 32 queries and 32 keys is, as far as the window goes: out of sight, or seen whole by all of the queries.
__device__ __forceinline__ bool block_dead(const WindowArgs& a, int q0, int k0) {
  return k0 > q0 + 31 + a.right || (k0 + 31 < q0 - a.left && k0 >= a.sinks);
}
__device__ __forceinline__ bool block_whole(const WindowArgs& a, int q0, int k0) {
  return k0 + 31 <= q0 + a.right && (k0 >= q0 + 31 - a.left || k0 + 32 <= a.sinks);
}
// For the 32 queries of a warp: which runs of keys are plain, that is seen whole, and with one bias for all.  Formed once, so that the tiles in the
// middle of a wide window cost four comparisons.
struct PlainKeys {
  int lo, hi, sink, low, high;
  bool none;
  float flat_low, flat_high;
  __device__ __forceinline__ PlainKeys(const WindowArgs& a, int q0, const float* bias, int bias_floats) {
    none = a.mask != nullptr;
    lo = q0 + 31 - a.left, hi = min(q0 + a.right, a.n - 1), sink = a.sinks - 1;      // first and last key of a run
    low = a.r < 0 ? 0x3fffffff : q0 - a.r, high = a.r < 0 ? 0x3fffffff : q0 + 31 + a.r;
    flat_low = a.r < 0 ? 0.f : bias[0], flat_high = a.r < 0 ? 0.f : bias[bias_floats - 1];
  }
  __device__ __forceinline__ bool plain(int first, int last) const {
    return !none && last <= hi && (first >= lo || last <= sink) && (last <= low || first >= high);
  }
  __device__ __forceinline__ float flat(int last) const { return last <= low ? flat_low : flat_high; }
};

// The learned bias of one head times log2(e), by offset j - i and continued beyond +-r far enough that every offset of a block of 32 x 32 that reaches
// into (-r, r) has its place.
constexpr int kWBiasBeyond = 64;
__host__ __device__ constexpr int bias_floats(int r) { return r < 0 ? 0 : 2 * r + 1 + 2 * kWBiasBeyond; }
__device__ __forceinline__ float bias_value(const WindowArgs& a, int head, int bucket) {
  const size_t at = (size_t)head * (2 * a.r + 1) + bucket;
  const float v = a.bias_type == PX_F32    ? __ldg((const float*)a.bias + at)
                  : a.bias_type == PX_BF16 ? __bfloat162float(__ldg((const bf16*)a.bias + at))
                                           : __half2float(__ldg((const __half*)a.bias + at));
  return v * kLog2e;
}
__device__ __forceinline__ void bias_fill(const WindowArgs& a, int head, float* to, int threads) {
  for (int k = threadIdx.x; k < bias_floats(a.r); k += threads) to[k] = bias_value(a, head, min(max(k - kWBiasBeyond, 0), 2 * a.r));
}
// How the bias meets a block of 32 queries from q0 and 32 keys from k0: `near`, by offset; otherwise one number, `flat` (the offsets are all clipped
// to the same side, or there is no bias).
struct BlockBias {
  bool near, low;
  float flat;
  __device__ __forceinline__ BlockBias(const WindowArgs& a, const float* bias, int q0, int k0) {
    low = k0 + 31 - q0 <= -a.r;
    const bool high = k0 - q0 - 31 >= a.r;
    near = a.r >= 0 && !low && !high;
    flat = a.r < 0 ? 0.f : low ? bias[0] : bias[2 * a.r + 2 * kWBiasBeyond];
  }
};
// The values of row i (query) from key k0 on: [0], [1], ...
__device__ __forceinline__ const float* bias_row(const WindowArgs& a, const float* bias, int i, int k0) {
  return bias + (k0 - i + a.r + kWBiasBeyond);
}

// Row `row` of a streamed tile of kKT rows in shared memory becomes zeros (part `part` of the 128 bytes of each panel).  What a product weights with
// zero must be finite: masked keys and rows that see nothing may hold anything.
template <int kPanels, int kKT>
__device__ __forceinline__ void clear_row(unsigned char* tile, int row, int part, int parts) {
#pragma unroll
  for (int p = 0; p < kPanels; ++p)
    for (int k = part * (8 / parts); k < (part + 1) * (8 / parts); ++k)
      *reinterpret_cast<uint4*>(tile + p * kKT * 128 + row * 128 + k * 16) = make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max32(const float* s) {
  float m[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    m[k] = max3f(s[8 * k], s[8 * k + 1], s[8 * k + 2]);
    m[k] = max3f(m[k], s[8 * k + 3], s[8 * k + 4]);
    m[k] = max3f(m[k], s[8 * k + 5], s[8 * k + 6]);
  }
  return max3f(max3f(m[0], m[1], s[7]), max3f(m[2], m[3], s[15]), fmaxf(s[23], s[31]));
}
// Barrier of `threads` threads that tells whether `ok` held for all: they leave a loop together after one of their waits ran out.
__device__ __forceinline__ bool barrier_all(int id, int threads, bool ok) {
  int all;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, %3, p;\n selp.b32 %0, 1, 0, q;\n}\n"
               : "=r"(all)
               : "r"((int)ok), "r"(id), "r"(threads)
               : "memory");
  return all != 0;
}
__device__ __forceinline__ void barrier_of(int id, int threads) { asm volatile("barrier.cta.sync %0, %1;\n" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool barrier_any(int id, int threads, bool p) {
  int any;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, %3, p;\n selp.b32 %0, 1, 0, q;\n}\n"
               : "=r"(any)
               : "r"((int)p), "r"(id), "r"(threads)
               : "memory");
  return any != 0;
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// 8 values of a gradient's row as 16 bytes; beyond the range of the type they are infinite, by which a loss scaler knows them.
template <bool kF16>
__device__ __forceinline__ void store8(void* to, const uint32_t* v, float scale) {
  uint4 w;
  uint32_t* o = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = pack16x2_inf<kF16>(__uint_as_float(v[2 * e]) * scale, __uint_as_float(v[2 * e + 1]) * scale);
  *reinterpret_cast<uint4*>(to) = w;
}

// A mean of fp16 values before it is rounded: infinite or NaN where one of them is, but never because the rounding of the weights has lifted it beyond 65504.
__device__ __forceinline__ float mean_of_f16(float v) { return fabsf(v) < CUDART_INF_F ? fminf(fmaxf(v, -65504.f), 65504.f) : v; }
// 8 values of an output's row as 16 bytes, and what the rounding has taken off each as 16 bits more, at `rest` unless that is NULL.
template <bool kF16>
__device__ __forceinline__ void store8(void* to, void* rest, const uint32_t* v, float scale) {
  uint4 w, r;
  uint32_t *o = reinterpret_cast<uint32_t*>(&w), *q = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a = __uint_as_float(v[2 * e]) * scale, b = __uint_as_float(v[2 * e + 1]) * scale;
    if constexpr (kF16) a = mean_of_f16(a), b = mean_of_f16(b);
    o[e] = pack16x2_inf<kF16>(a, b);
    const float2 back = unpack16x2<kF16>(o[e]);
    q[e] = pack16x2<kF16>(a - back.x, b - back.y);
  }
  *reinterpret_cast<uint4*>(to) = w;
  if (rest) *reinterpret_cast<uint4*>(rest) = r;
}

__device__ __forceinline__ void tmem_alloc(uint32_t* base, uint32_t cols) {      // whole warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(base)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(cols) : "memory");
}

// Rows of 16-bit values in global memory: strides in elements.
struct RowsOut {
  uint16_t* data;
  long long batch, head, row;
  __device__ __forceinline__ uint16_t* at(int b, int h, int i) const { return data + b * batch + h * head + i * row; }
};

}  // namespace px
