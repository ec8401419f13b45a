// What the kernels of the cross entropy share (cross_entropy.cu, px_head_small.cuh).
#pragma once
#include <math_constants.h>

#include "px_gemm.cuh"

namespace px {

constexpr float kDlScaleF16 = 16384.f;

// With a gradient for each row: the largest is made one where dl is rounded.
struct LossScale {
  float out;            // what dx and dW are multiplied by
  float each;           // what the gradient of a row's loss is multiplied by
};
// What dx, dW and db are multiplied by where they leave.
struct LossOut {
  const LossScale* scale;      // of gradients by row, or NULL
  const float* grad;           // of the mean or sum, with `inverse`
  const float* inverse;
  float by;                    // one over what dl is multiplied by
  __device__ __forceinline__ float operator()() const { return scale ? scale->out : *grad * *inverse * by; }
};

// What exponentials are taken relative to, in powers of two, for a maximum that may be that of nothing.
__device__ __forceinline__ float reference(float m) { return m == -CUDART_INF_F ? 0.f : m; }

// A row's part in the loss: its class, or a class that no column has.
__device__ __forceinline__ bool row_counts(int64_t target, int64_t ignore) { return target != ignore; }

// The loss of a row from its sum of exponentials, all logits relative to the same reference (in powers of two): nothing of its size is left in the
// difference.  valid: the row's class is one; hit: its logit; all: the sum of the logits (smooth > 0).
__device__ __forceinline__ float row_loss(float sum, float ref, float hit, bool valid, float smooth, float all, int classes) {
  float loss = CUDART_NAN_F;
  if (valid) loss = log2f(sum) - (1.f - smooth) * fmaf(hit, kLog2e, -ref);
  if (smooth > 0.f) loss -= smooth * fmaf(all / (float)classes, kLog2e, -ref);
  return loss < 0.f ? 0.f : loss * 0.6931471805599453f;
}

// The tensor core cuts an accumulator after each 16 channels, and what it aligns to it, towards zero: a logit comes out too small, in the mean, of rows that lean
// towards their class and of logits that are noise alike, by 1.5e-8 to 1.6e-8 (c / 16 + 1) of itself in bf16 and 1.7e-8 to 2.5e-8 in fp16, whose products are longer (512 to
// 4096 channels).  This puts the mean back, to within 0.4e-8.  Where all terms are of one sign 1e-8 (512 channels) to 4e-8 (4096) is missing in bf16 and 8e-8 to 1e-7 in
// fp16, of which it is a part; few channels whose sums are exact gain up to 1.2e-7.  Losses of 4096 rows of noise, 4096 channels: 1e-6 off in the mean, 6e-5 without (bf16).
static inline float uncut_logits(int64_t c, bool f16) { return 1.f + (f16 ? 2.1e-8f : 1.6e-8f) * (float)((c + 15) / 16 + 1); }
__device__ __forceinline__ void logits_of(const uint32_t (&r)[32], float uncut, float (&v)[32]) {
  const f32x2 u = pair2(uncut, uncut);
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 x = apart2(mul2(pair2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), u));
    v[j] = x.x, v[j + 1] = x.y;
  }
}

// v[at], 0 <= at < 32, by selection: written as a choice of elements the compiler makes it an indexed load and keeps v in local memory.
__device__ __forceinline__ float pick(const float (&v)[32], int at) {
  uint32_t u = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) u |= __float_as_uint(v[j]) & (at == j ? 0xffffffffu : 0u);
  return __uint_as_float(u);
}

// A bias in fp32 or 16 bits, 16-byte aligned.
struct HeadBias {
  const void* at;      // or NULL
  int type;
};
__device__ __forceinline__ float bias_value(const HeadBias& b, int i) {
  return b.type == PX_F32 ? __ldg((const float*)b.at + i) : b.type == PX_F16 ? __half2float(__ldg((const __half*)b.at + i)) : __bfloat162float(__ldg((const bf16*)b.at + i));
}
// Leaves the bias of an epilogue warp's classes in its shared memory, minus infinity for classes that are not there (no exponential); true where
// there is nothing to add.
template <class S>
__device__ __forceinline__ bool warp_bias(const GemmEpiTile& e, const HeadBias& b, int classes) {
  if (!b.at && e.n0 + S::kPartCols <= classes) return true;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < S::kPartCols; j += 32) {
    const int v = e.n0 + j + e.lane;
    e.own[j + e.lane] = v >= classes ? -CUDART_INF_F : b.at ? bias_value(b, v) : 0.f;
  }
  __syncwarp();
  return false;
}
__device__ __forceinline__ void add_bias(float (&v)[32], const float* b) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 x = *reinterpret_cast<const float4*>(b + j);
    v[j] += x.x, v[j + 1] += x.y, v[j + 2] += x.z, v[j + 3] += x.w;
  }
}
__device__ __forceinline__ void bias_store(void* to, int type, int i, float v) {
  if (type == PX_F32)
    ((float*)to)[i] = v;
  else if (type == PX_F16)
    ((__half*)to)[i] = __float2half_rn(v);
  else
    ((bf16*)to)[i] = __float2bfloat16_rn(v);
}

// v[0] of lane j = the sum of v[j] over the lanes: at each step half of the columns go to the other half of the lanes.
template <int kHalf = 16>
__device__ __forceinline__ void column_sums(float (&v)[32], int lane) {
  const bool up = (lane & kHalf) != 0;
#pragma unroll
  for (int j = 0; j < kHalf; ++j) {
    const float give = up ? v[j] : v[j + kHalf], keep = up ? v[j + kHalf] : v[j];
    v[j] = keep + __shfl_xor_sync(0xffffffffu, give, kHalf);
  }
  if constexpr (kHalf > 1) column_sums<kHalf / 2>(v, lane);
}

}  // namespace px
