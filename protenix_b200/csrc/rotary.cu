// Rotary positions of several axes: pair j of a head (two channels) turns by the angle position[axis of j] * base^-e_j,
//   y = (u cos - v sin, v cos + u sin),   the gradient is the same with the angles negated.
//
// Memory bound: every element is read and written once, the angles are few.  Angles: a pair's speed is a fraction of a turn with 88 bits, so that position * speed
// modulo a turn is off by 2^-31 of a turn for positions up to 2^57 and by 2^-25 for any int64 (with 64 bits of the speed by 2^-24 at position 2^40 and by a tenth at
// 2^60; fp32 angles are off by 0.06 at position 10^6).  Its top 32 bits go to sincospif.  A thread forms the sines of kVec pairs (16 bytes of each half) and uses
// them for all heads of its group; threads beside one another take neighbouring pairs, then neighbouring heads, so that heads inside the rows of a projection are read as
// whole lines.
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
  uint64_t speed[kRotaryPairs];        // turns a position, times 2^64, to nearest
  int32_t rest[kRotaryPairs];          // what that leaves, times 2^96, in the first 24 bits; the axis in the last eight
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
// The fraction of a turn that a position turns by, times 2^32.  Of `rest` only the position's upper half counts: the lower one's part is below 2^-33 of a turn.  Against
// `speed` alone 2 x 16384 tokens, 16 + 4 heads of 128, bf16 take 59.9 us for 59.6, 20000 tokens of 4 + 4 heads of 256 26.4 for 26.0; with 128 bits of the speed 65 and
// 38, with a branch for positions beyond 32 bits 70 and 31.
__device__ __forceinline__ uint32_t rotary_turns(int64_t position, uint64_t speed, int32_t rest) {
  return (uint32_t)(((uint64_t)position * speed + (uint64_t)((int64_t)(int32_t)(position >> 32) * rest)) >> 32);
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
  __shared__ int32_t rest[kRotaryPairs];
  for (int i = threadIdx.x; i < a.pairs; i += kRotaryThreads) speed[i] = a.speed[i], rest[i] = a.rest[i];
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
        const int pair = kVec * chunk + j, more = rest[pair];
        const uint32_t turns = rotary_turns(__ldg(p + (more & 255) * a.pa), speed[pair], more & ~255);
        sincospif((float)(int32_t)turns * 4.656612873077393e-10f, &s[j], &c[j]);      // 2^-31: half turns
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
  // Lanes that read different arguments take turns, so a block brings the speeds in once for up to four turns of its threads, as long as every SM has 32 blocks:
  // one head of 64 channels, 3 000 000 tokens, bf16 311 us with one, 279 with four (with eight blocks 5 x 31896 tokens of 8 heads of 32, fp32 53 -> 58).
  const int once = std::max(1, kRotaryThreads / per);
  const int64_t turns = std::min<int64_t>(std::max<int64_t>(batch * a.n / once / (32 * sm_count()), 1), 4);
  a.tokens = (int)std::min<int64_t>(a.n, turns * once);
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

// ---- speeds ----------------------------------------------------------------------------------------------------------
typedef unsigned __int128 Bits128;
// m 2^(e - 128), the top bit of m set
struct Wide {
  Bits128 m;
  int e;
};
// the upper half of a b, one too small at most
static Bits128 upper(Bits128 a, Bits128 b) {
  const uint64_t a1 = (uint64_t)(a >> 64), a0 = (uint64_t)a, b1 = (uint64_t)(b >> 64), b0 = (uint64_t)b;
  const Bits128 x = (Bits128)a1 * b0, y = (Bits128)a0 * b1, low = ((Bits128)a0 * b0 >> 64) + (uint64_t)x + (uint64_t)y;
  return (Bits128)a1 * b1 + (x >> 64) + (y >> 64) + (low >> 64);
}
static Wide wide(long double v) {
  int e;
  const long double f = frexpl(v, &e);      // 64 bits
  return {(Bits128)(uint64_t)ldexpl(f, 64) << 64, e};
}
static Wide times(Wide a, Wide b) {
  Wide c = {upper(a.m, b.m), a.e + b.e};
  if (!(c.m >> 127)) c.m <<= 1, --c.e;
  return c;
}
// base^(-1/n): a step of Newton's iteration for r^n = 1 / base from long double's r, whose error e / n, 2^-61 or less of it, leaves its square
static Wide root_of_inverse(double base, int n) {
  Wide r = wide(powl((long double)base, -1.0L / n)), power = wide((long double)base), x = r;
  for (int k = n; k; k >>= 1, x = times(x, x))
    if (k & 1) power = times(power, x);
  // power = 1 + e
  const Bits128 one = (Bits128)1 << 127;
  const bool above = power.e == 1;
  const Bits128 e = above ? (power.m - one) << 1 : (Bits128)0 - power.m, change = upper(r.m, e / n);
  r.m = above ? r.m - change : r.m + change < r.m ? ~(Bits128)0 : r.m + change;
  return r;
}
// The speeds of the pairs, turns times 2^128: each the one before times the ladder's step, cut to 2^-128 of a turn (off by 2^-117 after 256 of them).
static void rotary_speeds(const px_rotary& r, int pairs, RotaryArgs& a) {
  const Bits128 turn = (Bits128)0x28be60db9391054aull << 64 | 0x7f09d5f47d4d3770ull;      // 1 / 2 pi
  Bits128 speed = turn;
  Wide step = {};
  int j = 0;
  for (int i = 0; i < r.axes; ++i) {
    if (r.per_axis ? r.sections[i] > 0 : i == 0) speed = turn, step = root_of_inverse(r.base, r.per_axis ? r.sections[i] : pairs);
    for (int e = 0; e < r.sections[i]; ++e, ++j) {
      const Bits128 near = speed + ((Bits128)1 << 39);                                  // to 88 bits
      a.speed[j] = (uint64_t)((near + ((Bits128)1 << 63)) >> 64), a.rest[j] = (int32_t)(((uint32_t)(near >> 32) & ~255u) | (uint32_t)i);
      if (step.e <= 0) speed = step.e > -128 ? upper(speed, step.m) >> -step.e : 0;      // a step of one otherwise
    }
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
  a.heads = (int)r->heads, a.kv_heads = (int)r->kv_heads;
  a.pairs = (int)pairs, a.d = (int)r->d;
  a.inverse = inverse != 0;
  rotary_speeds(*r, (int)pairs, a);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool ok = r->dtype == PX_F32    ? launch_rotary<float>(a, vec, r->interleaved != 0, r->batch, st)
                  : r->dtype == PX_BF16 ? launch_rotary<bf16>(a, vec, r->interleaved != 0, r->batch, st)
                                        : launch_rotary<__half>(a, vec, r->interleaved != 0, r->batch, st);
  return ok ? PX_OK : PX_ERR_LAUNCH;
}
