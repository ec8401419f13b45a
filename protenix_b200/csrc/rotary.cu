// Rotary positions of several axes: pair j of a head (two channels) turns by the angle position[axis of j] * base^-e_j,
//   y = (u cos - v sin, v cos + u sin),   the gradient is the same with the angles negated.
//
// Memory bound: every element is read and written once, the angles are few.  Angles: a turn is 2^64, a pair's speed a 64-bit fraction of it, and
// position * speed modulo 2^64 is exact for any position, where fp32 angles are off by 0.06 at position 10^6; its top 32 bits go to
// sincospif.  A thread forms the sines of kVec pairs (16 bytes of each half) and uses them for all heads of its group; threads beside one another take
// neighbouring pairs, then neighbouring heads, so that heads inside the rows of a projection are read as whole lines.
//
// 2 x 16384 tokens, 16 + 4 heads of 128, bf16, 336 MB: 60 us (5.6 TB/s; at once on their way 1, 2, 4 heads a thread 66, 60, 59); 5 x 31896, 8 heads of 32, fp32: 56
// (5.9 TB/s; 59, 56, 59).  With four heads, each vector converted by elements, 116 registers: 101 us.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "px_common.cuh"

namespace px {

constexpr int kRotaryPairs = 256, kRotaryThreads = 256;
constexpr int kHeadsAtOnce = 2, kWantThreads = 2048;      // a thread's heads on their way; threads that an SM shall have

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
  int heads, kv_heads, head_groups;   // group g: heads g, g + head_groups, ..
  int pairs, chunks, d;                // chunks of kVec pairs, then of 2 kVec channels that stay as they are
  int tokens;                          // of a block
  int inverse;
  uint64_t speed[kRotaryPairs];        // turns a position, times 2^64
  uint8_t axis[kRotaryPairs];
};

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) RotaryVec {
  T v[kVec];
};
// Two values at a time where there are two: one conversion for both.
template <typename T, int kVec>
__device__ __forceinline__ void rotary_read(const RotaryVec<T, kVec>& x, float* f) {
  if constexpr (sizeof(T) == 2 && kVec > 1) {
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
      uint32_t u;
      memcpy(&u, &x.v[j], 4);
      const float2 p = unpack16x2<std::is_same<T, __half>::value>(u);
      f[j] = p.x, f[j + 1] = p.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[j] = (float)x.v[j];
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void rotary_write(RotaryVec<T, kVec>& x, const float* f) {
  if constexpr (sizeof(T) == 2 && kVec > 1) {
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
      const uint32_t u = pack16x2_inf<std::is_same<T, __half>::value>(f[j], f[j + 1]);
      memcpy(&x.v[j], &u, 4);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) x.v[j] = (T)f[j];
  }
}
// a b + c d, in the same order in every form of the kernel
__device__ __forceinline__ float rotary_sum(float a, float b, float c, float d) { return fmaf(a, b, __fmul_rn(c, d)); }

// The heads first, first + step, .. of one tensor, at channels at0 and at1; kHeads of them are on their way at once.
template <typename T, int kVec, int kHeads, bool kNeighbours>
__device__ __forceinline__ void rotary_heads(const RotaryTensor& t, int64_t b, int64_t row, int first, int heads, int step, int at0, int at1, bool second, bool turn,
                                             const float (&c)[kVec], const float (&s)[kVec]) {
  typedef RotaryVec<T, kVec> Vec;
  const T* from = (const T*)t.from + b * t.fb + row * t.fr;
  T* to = (T*)t.to + b * t.tb + row * t.tr;
#pragma unroll 1
  for (int h0 = first; h0 < heads; h0 += kHeads * step) {
    Vec x[kHeads], y[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int64_t h = h0 + i * step;
      if (h < heads) {
        x[i] = *reinterpret_cast<const Vec*>(from + h * t.fh + at0);
        if (second) y[i] = *reinterpret_cast<const Vec*>(from + h * t.fh + at1);
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int64_t h = h0 + i * step;
      if (h >= heads) break;
      if (turn) {
        float f[2 * kVec], g[2 * kVec];
        rotary_read<T, kVec>(x[i], f);
        rotary_read<T, kVec>(y[i], f + kVec);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int u = kNeighbours ? 2 * j : j, v = kNeighbours ? 2 * j + 1 : j + kVec;
          g[u] = rotary_sum(f[u], c[j], -f[v], s[j]);
          g[v] = rotary_sum(f[v], c[j], f[u], s[j]);
        }
        rotary_write<T, kVec>(x[i], g);
        rotary_write<T, kVec>(y[i], g + kVec);
      }
      *reinterpret_cast<Vec*>(to + h * t.th + at0) = x[i];
      if (second) *reinterpret_cast<Vec*>(to + h * t.th + at1) = y[i];
    }
  }
}

template <typename T, int kVec, int kHeads, bool kNeighbours>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
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
      at0 = kNeighbours ? 2 * kVec * chunk : kVec * chunk;
      at1 = kNeighbours ? at0 + kVec : at0 + a.pairs;
    } else {
      at0 = 2 * a.pairs + 2 * kVec * (chunk - turning);
      at1 = at0 + kVec;
    }
    const bool second = at1 < a.d;     // the channels that stay may end with the first vector
    float c[kVec] = {}, s[kVec] = {};
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
    rotary_heads<T, kVec, kHeads, kNeighbours>(a.q, b, row, group, a.heads, a.head_groups, at0, at1, second, turn, c, s);
    rotary_heads<T, kVec, kHeads, kNeighbours>(a.k, b, row, group, a.kv_heads, a.head_groups, at0, at1, second, turn, c, s);
  }
}

template <typename T, int kVec, int kHeads, bool kNeighbours>
static bool launch_rotary(RotaryArgs& a, int64_t batch, int groups, cudaStream_t st) {
  a.head_groups = groups;
  const int per = a.chunks * groups;
  a.tokens = (int)std::min<int64_t>(a.n, std::max(1, kRotaryThreads / per));
  const int64_t blocks = (a.n + a.tokens - 1) / a.tokens;
  return launch_pdl(rotary_kernel<T, kVec, kHeads, kNeighbours>, dim3((unsigned)blocks, (unsigned)batch), kRotaryThreads, 0, st, a);
}

// The fewer groups the heads of a token are dealt to, the fewer threads form the same sines; as few as leave every SM kWantThreads.
template <typename T, int kVec, bool kNeighbours>
static bool launch_rotary(RotaryArgs& a, int64_t batch, cudaStream_t st) {
  a.chunks = a.pairs / kVec + (a.d - 2 * a.pairs + 2 * kVec - 1) / (2 * kVec);
  const int64_t threads = batch * a.n * a.chunks, want = (int64_t)sm_count() * kWantThreads, groups = (want + threads - 1) / threads;
  const int heads = std::max(a.heads, a.kv_heads);
  if (groups * kHeadsAtOnce <= heads) return launch_rotary<T, kVec, kHeadsAtOnce, kNeighbours>(a, batch, (int)groups, st);
  return launch_rotary<T, kVec, 1, kNeighbours>(a, batch, (int)std::min<int64_t>(groups, heads), st);
}
template <typename T, bool kNeighbours>
static bool launch_rotary(RotaryArgs& a, int vec, int64_t batch, cudaStream_t st) {
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_rotary<T, 8, kNeighbours>(a, batch, st);
    case 4: return launch_rotary<T, 4, kNeighbours>(a, batch, st);
    case 2: return launch_rotary<T, 2, kNeighbours>(a, batch, st);
    default: return launch_rotary<T, 1, kNeighbours>(a, batch, st);
  }
}
template <typename T>
static bool launch_rotary(RotaryArgs& a, int vec, bool neighbours, int64_t batch, cudaStream_t st) {
  return neighbours ? launch_rotary<T, true>(a, vec, batch, st) : launch_rotary<T, false>(a, vec, batch, st);
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
  a.heads = (int)r->heads, a.kv_heads = (int)r->kv_heads;
  a.pairs = (int)pairs, a.d = (int)r->d;
  a.inverse = inverse != 0;
  // one power an axis, or one in all; their products are off by 2^-63 a factor
  const long double turn = 0.159154943091895335768883763372514362034459645740L * 18446744073709551616.0L;      // 2^64 / 2 pi
  long double speed = turn, step = powl((long double)r->base, -1.0L / pairs);
  int j = 0;
  for (int i = 0; i < r->axes; ++i) {
    if (r->per_axis && r->sections[i]) speed = turn, step = powl((long double)r->base, -1.0L / r->sections[i]);
    for (int e = 0; e < r->sections[i]; ++e, ++j, speed *= step) a.speed[j] = (uint64_t)llrintl(speed), a.axis[j] = (uint8_t)i;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool ok = r->dtype == PX_F32    ? launch_rotary<float>(a, vec, r->interleaved != 0, r->batch, st)
                  : r->dtype == PX_BF16 ? launch_rotary<bf16>(a, vec, r->interleaved != 0, r->batch, st)
                                        : launch_rotary<__half>(a, vec, r->interleaved != 0, r->batch, st);
  return ok ? PX_OK : PX_ERR_LAUNCH;
}
