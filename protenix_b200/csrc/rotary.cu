// Rotary positions of several axes: pair j of a head (two channels) turns by the angle position[axis of j] * base^-e_j,
//   y = (u cos - v sin, v cos + u sin),   the gradient is the same with the angles negated.
//
// Memory bound: every element is read and written once, the angles are few.  Angles: a turn is 2^64, a pair's speed a 64-bit fraction of it, and
// position * speed modulo 2^64 is exact for any position, where fp32 angles are off by 0.06 at position 10^6; its top 32 bits go to
// sincospif.  A thread forms the sines of kVec pairs (16 bytes of each half) and uses them for all heads of its group; threads beside one another take
// neighbouring pairs, then neighbouring heads, so that heads inside the rows of a projection are read as whole lines.
#include <math.h>

#include "px_common.cuh"

namespace px {

constexpr int kRotaryPairs = 256, kRotaryThreads = 256;

struct RotaryTensor {
  const void* from;
  void* to;
  int64_t fb, fh, fr, tb, th, tr;      // strides of batch, head and row, in elements
};
struct RotaryArgs {
  RotaryTensor q, k;
  const int64_t* positions;
  int64_t pb, pr, pa;
  int64_t n;
  int heads, all_heads, head_groups;   // group g: heads g, g + head_groups, ..
  int pairs, chunks, d;                // chunks of kVec pairs, then of 2 kVec channels that stay as they are
  int tokens;                          // of a block
  int interleaved, inverse;
  uint64_t speed[kRotaryPairs];        // turns a position, times 2^64
  uint8_t axis[kRotaryPairs];
};

template <typename T>
__device__ __forceinline__ float rotary_float(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T rotary_round(float v);
template <>
__device__ __forceinline__ float rotary_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 rotary_round<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half rotary_round<__half>(float v) { return __float2half_rn(v); }

// a b + c d, in the same order in every form of the kernel
__device__ __forceinline__ float rotary_sum(float a, float b, float c, float d) { return fmaf(a, b, __fmul_rn(c, d)); }

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) RotaryVec {
  T v[kVec];
};

template <typename T, int kVec, int kHeads>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  typedef RotaryVec<T, kVec> Vec;
  __shared__ uint64_t speed[kRotaryPairs];
  __shared__ uint8_t axis[kRotaryPairs];
  for (int i = threadIdx.x; i < a.pairs; i += kRotaryThreads) speed[i] = a.speed[i], axis[i] = a.axis[i];
  __syncthreads();
  pdl_wait();
  const int per = a.chunks * a.head_groups, turning = a.pairs / kVec;
  const int64_t b = blockIdx.y, first = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.n - first);
  for (int i = threadIdx.x; i < tokens * per; i += kRotaryThreads) {
    const int token = i / per, in = i - token * per, group = in / a.chunks, chunk = in - group * a.chunks;
    const int64_t row = first + token;
    const bool turn = chunk < turning;
    int at0, at1;                      // the two vectors of a head: the halves of the pairs, or neighbours
    if (turn) {
      at0 = a.interleaved ? 2 * kVec * chunk : kVec * chunk;
      at1 = a.interleaved ? at0 + kVec : at0 + a.pairs;
    } else {
      at0 = 2 * a.pairs + 2 * kVec * (chunk - turning);
      at1 = at0 + kVec;
    }
    const bool second = at1 < a.d;     // the channels that stay may end with the first vector
    float c[kVec], s[kVec];
    if (turn) {
      const int64_t* p = a.positions + b * a.pb + row * a.pr;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int pair = kVec * chunk + j;
        const uint64_t turns = (uint64_t)__ldg(p + axis[pair] * a.pa) * speed[pair];
        sincospif((float)(int32_t)(turns >> 32) * 4.656612873077393e-10f, &s[j], &c[j]);      // 2^-31: half turns
        if (a.inverse) s[j] = -s[j];
      }
    }
#pragma unroll 1
    for (int head0 = group; head0 < a.all_heads; head0 += kHeads * a.head_groups) {
      Vec x[kHeads], y[kHeads];
      T* to[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const int head = head0 + h * a.head_groups;
        to[h] = nullptr;
        if (head < a.all_heads) {
          const bool is_k = head >= a.heads;
          const RotaryTensor& t = is_k ? a.k : a.q;
          const int64_t hh = is_k ? head - a.heads : head;
          const T* p = (const T*)t.from + b * t.fb + hh * t.fh + row * t.fr;
          x[h] = *reinterpret_cast<const Vec*>(p + at0);
          if (second) y[h] = *reinterpret_cast<const Vec*>(p + at1);
          to[h] = (T*)t.to + b * t.tb + hh * t.th + row * t.tr;
        }
      }
      if (turn) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            if (a.interleaved && kVec > 1) {
              // pair j: channels 2 j and 2 j + 1 of the two vectors as one
              Vec& w = 2 * j < kVec ? x[h] : y[h];
              const int e = 2 * j < kVec ? 2 * j : 2 * j - kVec;
              const float u = rotary_float(w.v[e]), v = rotary_float(w.v[(e + 1) % kVec]);
              w.v[e] = rotary_round<T>(rotary_sum(u, c[j], -v, s[j]));
              w.v[(e + 1) % kVec] = rotary_round<T>(rotary_sum(v, c[j], u, s[j]));
            } else {
              const float u = rotary_float(x[h].v[j]), v = rotary_float(y[h].v[j]);
              x[h].v[j] = rotary_round<T>(rotary_sum(u, c[j], -v, s[j]));
              y[h].v[j] = rotary_round<T>(rotary_sum(v, c[j], u, s[j]));
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        if (to[h]) {
          *reinterpret_cast<Vec*>(to[h] + at0) = x[h];
          if (second) *reinterpret_cast<Vec*>(to[h] + at1) = y[h];
        }
      }
    }
  }
}

template <typename T, int kVec, int kHeads>
static bool launch_rotary(RotaryArgs& a, int64_t batch, int groups, cudaStream_t st) {
  a.head_groups = groups;
  const int per = a.chunks * groups;
  a.tokens = (int)std::min<int64_t>(a.n, std::max(1, kRotaryThreads / per));
  const int64_t blocks = (a.n + a.tokens - 1) / a.tokens;
  return launch_pdl(rotary_kernel<T, kVec, kHeads>, dim3((unsigned)blocks, (unsigned)batch), kRotaryThreads, 0, st, a);
}

// The fewer groups the heads of a token are dealt to, the fewer threads form the same sines; as few as leave two rounds of threads on all SMs.  Four
// heads at a time are on their way then; where there are not that many threads, one.
template <typename T, int kVec>
static bool launch_rotary(RotaryArgs& a, int64_t batch, cudaStream_t st) {
  a.chunks = a.pairs / kVec + (a.d - 2 * a.pairs + 2 * kVec - 1) / (2 * kVec);
  const int64_t threads = batch * a.n * a.chunks, want = (int64_t)sm_count() * 2048;
  const int64_t groups = (want + threads - 1) / threads, most = (a.all_heads + 3) / 4;
  if (groups <= most) return launch_rotary<T, kVec, 4>(a, batch, (int)groups, st);
  return launch_rotary<T, kVec, 1>(a, batch, (int)std::min<int64_t>(groups, a.all_heads), st);
}
template <typename T>
static bool launch_rotary(RotaryArgs& a, int vec, int64_t batch, cudaStream_t st) {
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_rotary<T, 8>(a, batch, st);
    case 4: return launch_rotary<T, 4>(a, batch, st);
    case 2: return launch_rotary<T, 2>(a, batch, st);
    default: return launch_rotary<T, 1>(a, batch, st);
  }
}

}  // namespace px

using namespace px;

extern "C" int32_t px_rotary_turn(const px_rotary* r, const px_rows* q, const px_rows* q_out, const px_rows* k, const px_rows* k_out, int32_t inverse, void* stream) {
  if (!r || !q || !q_out || !k != !k_out || r->batch < 0 || r->heads < 1 || r->kv_heads < 0 || r->n < 0 || r->d < 2 || !r->sections || r->axes < 1)
    return PX_ERR_BAD_ARG;
  if ((r->kv_heads > 0) != (k != nullptr) || !(r->base >= 1.0) || !(r->base <= 1e30)) return PX_ERR_BAD_ARG;
  int64_t pairs = 0;
  for (int i = 0; i < r->axes; ++i) {
    if (r->sections[i] < 0) return PX_ERR_BAD_ARG;
    pairs += r->sections[i];
    if (pairs > kRotaryPairs) return PX_ERR_UNSUPPORTED;
  }
  if (pairs < 1 || 2 * pairs > r->d) return PX_ERR_BAD_ARG;
  if (r->axes > 255 || r->d > 65536 || r->batch > 65535 || r->n > (1 << 30) || r->heads + r->kv_heads > 65536) return PX_ERR_UNSUPPORTED;
  if (r->dtype != PX_F32 && r->dtype != PX_BF16 && r->dtype != PX_F16) return PX_ERR_UNSUPPORTED;
  if (r->batch == 0 || r->n == 0) return PX_OK;
  if (!r->positions || !q->data || !q_out->data || (k && (!k->data || !k_out->data))) return PX_ERR_BAD_ARG;

  const int size = r->dtype == PX_F32 ? 4 : 2;
  int vec = 16 / size;
  // strides of axes of length one are not looked at, here and in the kernel
  const auto fitted = [&](const px_rows* t, int64_t heads) {
    px_rows f = *t;
    if (r->batch == 1) f.batch = 0;
    if (heads == 1) f.head = 0;
    if (r->n == 1) f.row = 0;
    return f;
  };
  const px_rows qi = fitted(q, r->heads), qo = fitted(q_out, r->heads), ki = k ? fitted(k, r->kv_heads) : qi, ko = k ? fitted(k_out, r->kv_heads) : qo;
  const auto fits = [&](const px_rows& t, int v) { return (t.batch | t.head | t.row) % v == 0 && ((uintptr_t)t.data & (v * size - 1)) == 0; };
  while (vec > 1 && !(pairs % vec == 0 && r->d % vec == 0 && fits(qi, vec) && fits(qo, vec) && fits(ki, vec) && fits(ko, vec))) vec /= 2;
  if (!fits(qi, 1) || !fits(qo, 1) || !fits(ki, 1) || !fits(ko, 1)) return PX_ERR_BAD_ARG;

  RotaryArgs a = {};
  a.q = {qi.data, qo.data, qi.batch, qi.head, qi.row, qo.batch, qo.head, qo.row};
  a.k = {ki.data, ko.data, ki.batch, ki.head, ki.row, ko.batch, ko.head, ko.row};
  a.positions = r->positions;
  a.pb = r->position_batch, a.pr = r->position_row, a.pa = r->position_axis;
  a.n = r->n;
  a.heads = (int)r->heads, a.all_heads = (int)(r->heads + r->kv_heads);
  a.pairs = (int)pairs, a.d = (int)r->d;
  a.interleaved = r->interleaved != 0, a.inverse = inverse != 0;
  // one power an axis, or one in all; their products are off by 2^-63 a factor
  const long double turn = 0.159154943091895335768883763372514362034459645740L * 18446744073709551616.0L;      // 2^64 / 2 pi
  long double speed = turn, step = powl((long double)r->base, -1.0L / pairs);
  int j = 0;
  for (int i = 0; i < r->axes; ++i) {
    if (r->per_axis && r->sections[i]) speed = turn, step = powl((long double)r->base, -1.0L / r->sections[i]);
    for (int e = 0; e < r->sections[i]; ++e, ++j, speed *= step) a.speed[j] = (uint64_t)llrintl(speed), a.axis[j] = (uint8_t)i;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool ok = r->dtype == PX_F32    ? launch_rotary<float>(a, vec, r->batch, st)
                  : r->dtype == PX_BF16 ? launch_rotary<bf16>(a, vec, r->batch, st)
                                        : launch_rotary<__half>(a, vec, r->batch, st);
  return ok ? PX_OK : PX_ERR_LAUNCH;
}
