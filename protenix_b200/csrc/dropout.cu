// Dropout whose mask is a function of (seed, offset, place), fused with the residual add:
//   out[o][s][i] = residual[o][s][i] + keep(o, i) * x[o][s][i] / (1 - p)
// for tensors [outer][shared][inner]: one truth value per (o, i), shared by all s (shared = 1: one per element).  With
// residual == NULL the product alone is written, which is also the gradient of x; nothing is stored between the two.
//
// keep(e) = [u(e) >= round(p 2^32)] for e = o * inner + i, where u(e) is word e mod 4 of Philox4x32-10 (Salmon, Moraes, Dror,
// Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) with counter (e / 4, offset) and key seed.  32 bits an element: p is met to
// 2^-33.  (16 bits would halve the generator's work and miss p = 0.1 by 6e-6.)  A dropped element gives the residual itself, whatever x
// holds.  Product and sum are fp32, rounded once.
//
// Bounds.  Unshared, a round is two 32 x 32 -> 64 products, which only the heavy half of the multiply pipe makes, and four bit operations for four
// elements: 768 x 768 x 128 in bf16 takes 74 us with the residual (453 MB) and 68 without (302 MB), the heavy multiply pipe busy for four fifths of it, so
// the generator bounds it and not memory (69 us and 46 at a copy's rate).  Shared, a thread keeps the mask of its 16 bytes in registers while it walks
// along the shared axis, and memory alone counts: 512 x 512 x 128 in fp32, 61 us for 403 MB, 41 for 268: a copy's rate.
#include <math.h>

#include "px_common.cuh"

namespace px {

// The keys of the ten rounds: made once a thread (made anew with every block of four they were a tenth of the kernel's instructions).
struct RoundKeys {
  uint32_t a[10], b[10];
  __device__ __forceinline__ explicit RoundKeys(unsigned long long seed) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      a[r] = (uint32_t)seed + r * 0x9E3779B9u;
      b[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
      asm volatile("" : "+r"(a[r]), "+r"(b[r]));      // values, no longer sums that the compiler would rather form again
    }
  }
};
__device__ __forceinline__ void philox4x32(uint32_t (&c)[4], const RoundKeys& k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c[0], b = (uint64_t)0xCD9E8D57u * c[2];
    c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k.a[r];
    c[1] = (uint32_t)b;
    c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k.b[r];
    c[3] = (uint32_t)a;
  }
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

struct DropoutArgs {
  long long outer, shared, inner;      // elements
  uint32_t threshold;                  // dropped below it
  bool none;                           // p = 1: nothing is kept
  float scale;                         // 1 / (1 - p)
  unsigned long long seed, offset;
  const long long* state;              // (seed, offset) in device memory in place of the two, or NULL
  long long* used;                     // receives the pair that the call used, or NULL
};

// Whether the elements at, at + 1, ... are kept.  `at` is a multiple of four unless VEC is 1.  kFew: there are fewer than 2^34 of them, so that the counter's
// second word is zero like the offset's are fixed, and two of the twenty products need not be made for each block of four.
template <int VEC, bool kFew>
__device__ __forceinline__ void kept(const DropoutArgs& a, const RoundKeys& keys, unsigned long long offset, long long at, bool (&keep)[VEC]) {
#pragma unroll
  for (int q = 0; q < (VEC + 3) / 4; ++q) {
    const unsigned long long block = ((unsigned long long)at >> 2) + q;
    uint32_t c[4] = {(uint32_t)block, kFew ? 0u : (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
    philox4x32(c, keys);
    if constexpr (VEC == 1) {
      const int w = (int)(at & 3);
      keep[0] = (w < 2 ? (w ? c[1] : c[0]) : (w == 2 ? c[2] : c[3])) >= a.threshold && !a.none;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) keep[4 * q + e] = c[e] >= a.threshold && !a.none;
    }
  }
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T>
__device__ __forceinline__ void round_pair(T* to, float a, float b);
template <>
__device__ __forceinline__ void round_pair<float>(float* to, float a, float b) { to[0] = a, to[1] = b; }
template <>
__device__ __forceinline__ void round_pair<bf16>(bf16* to, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(a, b); }
template <>
__device__ __forceinline__ void round_pair<__half>(__half* to, float a, float b) { *reinterpret_cast<__half2*>(to) = __floats2half2_rn(a, b); }

// A kept element's product and sum are fp32 and round once; a dropped one leaves the residual as it is.
template <typename T, int VEC, bool kResidual>
__device__ __forceinline__ Pack<T, VEC> dropped(const Pack<T, VEC>& x, const Pack<T, VEC>& r, const bool (&keep)[VEC], float scale) {
  Pack<T, VEC> o;
  float v[VEC];
  if constexpr (kResidual || VEC == 1) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = fmaf(keep[e] ? to_f32(x.v[e]) : 0.f, scale, kResidual ? to_f32(r.v[e]) : 0.f);
  } else {      // packed products: 70.9 -> 68.3 us at 768 x 768 x 128 in bf16; packed with the residual 73.7 -> 77.1
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float2 z = apart2(mul2(pair2(keep[e] ? to_f32(x.v[e]) : 0.f, keep[e + 1] ? to_f32(x.v[e + 1]) : 0.f), pair2(scale, scale)));
      v[e] = z.x, v[e + 1] = z.y;
    }
  }
  if constexpr (VEC == 1) {
    o.v[0] = from_f32<T>(v[0]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) round_pair(o.v + e, v[e], v[e + 1]);
  }
  return o;
}

// One value per element: thread = 16 bytes, the last of them element by element.
template <typename T, int VEC, bool kResidual, bool kFew>
__global__ void __launch_bounds__(256) dropout_kernel(const T* residual, const T* x, T* out, DropoutArgs a) {
  typedef Pack<T, VEC> V;
  const unsigned long long seed = a.state ? (unsigned long long)a.state[0] : a.seed;
  const unsigned long long offset = a.state ? (unsigned long long)a.state[1] : a.offset;
  if (a.used && blockIdx.x == 0 && threadIdx.x == 0) {
    a.used[0] = (long long)seed;
    a.used[1] = (long long)offset;
  }
  const RoundKeys keys(seed);
  const long long step = (long long)gridDim.x * blockDim.x * VEC, total = a.inner;
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * VEC; i < total; i += step) {
    if (i + VEC <= total) {
      const V xv = *reinterpret_cast<const V*>(x + i);
      V rv = xv;
      if (kResidual) rv = *reinterpret_cast<const V*>(residual + i);
      bool keep[VEC];
      kept<VEC, kFew>(a, keys, offset, i, keep);
      *reinterpret_cast<V*>(out + i) = dropped<T, VEC, kResidual>(xv, rv, keep, a.scale);
    } else {
      for (long long e = i; e < total; ++e) {
        const Pack<T, 1> x1 = {{x[e]}};
        Pack<T, 1> r1 = x1;
        if (kResidual) r1.v[0] = residual[e];
        bool keep[1];
        kept<1, false>(a, keys, offset, e, keep);
        out[e] = dropped<T, 1, kResidual>(x1, r1, keep, a.scale).v[0];
      }
    }
  }
}

constexpr int kSharedRows = 4;      // of the shared axis, a thread: what the generator costs is spread over them

// Shared along the middle axis: thread = 16 bytes of a row (o, i) and up to kSharedRows of the shared axis, all requested before the mask is made.
template <typename T, int VEC, bool kResidual>
__global__ void __launch_bounds__(256) dropout_shared_kernel(const T* residual, const T* x, T* out, DropoutArgs a, long long units) {
  typedef Pack<T, VEC> V;
  const unsigned long long seed = a.state ? (unsigned long long)a.state[0] : a.seed;
  const unsigned long long offset = a.state ? (unsigned long long)a.state[1] : a.offset;
  if (a.used && blockIdx.x == 0 && threadIdx.x == 0) {
    a.used[0] = (long long)seed;
    a.used[1] = (long long)offset;
  }
  const RoundKeys keys(seed);
  const long long vectors = a.outer * a.inner / VEC;       // of the mask
  for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < units; u += (long long)gridDim.x * blockDim.x) {
    const long long m = u % vectors * VEC, s0 = u / vectors * kSharedRows;
    const long long o = m / a.inner, i = m - o * a.inner;  // VEC divides inner: a vector never leaves its row
    const int count = (int)(a.shared - s0 < kSharedRows ? a.shared - s0 : kSharedRows);
    const long long at = (o * a.shared + s0) * a.inner + i;
    V xv[kSharedRows], rv[kSharedRows];
#pragma unroll
    for (int s = 0; s < kSharedRows; ++s) {
      if (s < count) {
        xv[s] = *reinterpret_cast<const V*>(x + at + s * a.inner);
        rv[s] = kResidual ? *reinterpret_cast<const V*>(residual + at + s * a.inner) : xv[s];
      }
    }
    bool keep[VEC];
    kept<VEC, false>(a, keys, offset, m, keep);
#pragma unroll
    for (int s = 0; s < kSharedRows; ++s)
      if (s < count) *reinterpret_cast<V*>(out + at + s * a.inner) = dropped<T, VEC, kResidual>(xv[s], rv[s], keep, a.scale);
  }
}

template <typename T, int VEC, bool kResidual>
static cudaError_t launch_dropout_as(const void* residual, const void* x, void* out, const DropoutArgs& a, cudaStream_t st) {
  const int64_t most = (int64_t)sm_count() * 32;           // blocks
  if (a.shared == 1) {
    const int64_t blocks = std::min<int64_t>((a.inner / VEC + 1 + 255) / 256, most);
    const auto kernel = a.inner < (1ll << 34) ? dropout_kernel<T, VEC, kResidual, true> : dropout_kernel<T, VEC, kResidual, false>;
    kernel<<<(unsigned)blocks, 256, 0, st>>>((const T*)residual, (const T*)x, (T*)out, a);
  } else {
    const int64_t units = a.outer * a.inner / VEC * ((a.shared + kSharedRows - 1) / kSharedRows);
    const int64_t blocks = std::min<int64_t>((units + 255) / 256, most);
    dropout_shared_kernel<T, VEC, kResidual><<<(unsigned)blocks, 256, 0, st>>>((const T*)residual, (const T*)x, (T*)out, a, units);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_dropout(const void* residual, const void* x, void* out, const DropoutArgs& a, cudaStream_t st) {
  constexpr int kWide = 16 / (int)sizeof(T);
  const bool wide = (a.shared == 1 || a.inner % kWide == 0) && (((uintptr_t)residual | (uintptr_t)x | (uintptr_t)out) & 15) == 0;
  if (wide)
    return residual ? launch_dropout_as<T, kWide, true>(residual, x, out, a, st) : launch_dropout_as<T, kWide, false>(residual, x, out, a, st);
  return residual ? launch_dropout_as<T, 1, true>(residual, x, out, a, st) : launch_dropout_as<T, 1, false>(residual, x, out, a, st);
}

}  // namespace px

extern "C" int32_t px_dropout_add(const void* residual, const void* x, void* out, int64_t outer, int64_t shared, int64_t inner, double p,
                                  int64_t seed, int64_t offset, const int64_t* state, int64_t* used, int32_t dtype, void* stream) {
  if (outer < 0 || shared < 0 || inner < 0 || !(p >= 0.0 && p <= 1.0)) return PX_ERR_BAD_ARG;
  if (dtype != PX_F32 && dtype != PX_BF16 && dtype != PX_F16) return PX_ERR_UNSUPPORTED;
  if (outer == 0 || shared == 0 || inner == 0) return PX_OK;
  if (!x || !out) return PX_ERR_BAD_ARG;
  px::DropoutArgs a;
  // one row after the other where nothing is shared
  a.outer = shared == 1 ? 1 : outer;
  a.shared = shared;
  a.inner = shared == 1 ? outer * inner : inner;
  const double t = rint(p * 4294967296.0);
  a.none = t >= 4294967296.0;
  a.threshold = a.none ? 0u : (uint32_t)t;
  a.scale = a.none ? 0.f : (float)(1.0 / (1.0 - p));
  a.seed = (unsigned long long)seed;
  a.offset = (unsigned long long)offset;
  a.state = (const long long*)state;
  a.used = (long long*)used;
  cudaError_t e;
  switch (dtype) {
    case PX_F32: e = px::launch_dropout<float>(residual, x, out, a, (cudaStream_t)stream); break;
    case PX_BF16: e = px::launch_dropout<px::bf16>(residual, x, out, a, (cudaStream_t)stream); break;
    default: e = px::launch_dropout<__half>(residual, x, out, a, (cudaStream_t)stream); break;
  }
  return e == cudaSuccess ? PX_OK : PX_ERR_LAUNCH;
}
