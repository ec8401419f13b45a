// Relative position encoding of token pairs (RelativePositionEncoding of the reference's input embedder; AlphaFold 3, algorithm 3):
//   z[i][j][:] = W_pos[bp] + W_tok[bt] + [same entity] W_ent + W_chain[bc]           rows of W^T, W = [c][4 r + 2 s + 7]
//   bp = same chain ? clip(residue_i - residue_j + r, 0, 2 r) : 2 r + 1
//   bt = same chain and residue ? clip(token_i - token_j + r, 0, 2 r) : 2 r + 1
//   bc = same entity ? clip(copy_i - copy_j + s, 0, 2 s) : 2 s + 1
// and the gradient of W: sums of dz over the pairs of a bucket.  The one-hot matrix never exists.
//
// Two table rows make a pair: bt differs from 2 r + 1 only where bp = r, and the entity's flag follows from bc, so there are
// 4 r + 3 sums W_pos + W_tok and 2 s + 2 sums W_chain + W_ent (both tables 35 KB of shared memory for r = 32, s = 2 and 64 channels).
//
// Forward: a warp takes 32 neighbouring pairs of a row; a lane finds one pair's two rows (a code, kept for the backward pass: 4 bytes beside the
// pair's 256 or 512), then the warp writes them, a few pairs side by side, 4 channels a lane, and looks the rows up again only where they
// change (most neighbours are far apart or in another chain: clipped alike).  Memory-bound writer: 1501 tokens x 128 channels in bf16, 91 us for
// 577 MB = 6.3 TB/s, 97 % of a copy's rate, and up to 104 with the 9 MB of codes between backward passes; 384 tokens in fp32 16 us for 76 MB = 4.7 TB/s.
// The smallest wait for W, from which every block makes its tables: 97 tokens 5 us for 4.8 MB.  So a block's tables are for 32 or 64 channels.
//
// Backward: memory-bound reader, two forms.  This one, for fp32 and for tables that the other has no room for: a block (a thread = one channel) reads
// strips of 32 pairs of a row through a ring of bulk copies and holds sums of its own for every table row in shared memory, so there are no atomics and
// a call gives the same bits every time.  Neighbours with the same rows are added up in registers; neighbours whose rows all differ, as near the
// diagonal, go to their sums eight at a time; the rest one by one.  What bounds it is the latency of a warp's
// chain of read, add and write: the sums leave shared memory for two blocks of four warps an SM, and no unit is full (issue slots 30 %, LSU 24 %, DRAM 33 %; 384 tokens
// x 128 channels in fp32, 29 us for 76 MB = 2.6 TB/s, 40 % of a copy's rate).
// The blocks' sums, folded to the columns of W, are added up in their order by a second kernel.
//
// What is not finite: a dz of one pair that is infinite or NaN stays so in its channel, in the columns of its own pair here; the form on the tensor cores
// makes all columns of the channel NaN (0 x inf).
#include "px_tcgen05.cuh"

namespace px {

constexpr int kRpChunk = 128;           // channels a block of the backward pass handles
constexpr int kRpMaxRows = 380;         // rows of both tables together: what shared memory holds beside the backward pass's ring
constexpr int kRpPairs = 32;            // pairs of a warp's step, and of a backward stage of 16-bit values
constexpr int kRpStages = 4;
constexpr int kRpStageBytes = 8192;

struct RelposArgs {
  const long long *asym, *residue, *entity, *token, *sym;      // [batch][n]
  long long n, pairs;                    // tokens; pairs of all batches
  int c, r, s;                           // channels and clipping distances
  __host__ __device__ int rows1() const { return 4 * r + 3; }
  __host__ __device__ int rows2() const { return 2 * s + 2; }
  __host__ __device__ int columns() const { return 4 * r + 2 * s + 7; }
};

__device__ __forceinline__ int clip_to(long long d, int r) {      // in 0 .. 2 r
  return d < -(long long)r ? 0 : d > (long long)r ? 2 * r : (int)d + r;
}
// The table rows of a pair: the first table's in the low half, the second's in the high half.  (Differences wrap as the tensor ones do.)
__device__ __forceinline__ uint32_t relpos_code(const RelposArgs& a, long long at_i, long long at_j) {
  const auto less = [&](const long long* v) { return (long long)((unsigned long long)__ldg(v + at_i) - (unsigned long long)__ldg(v + at_j)); };
  const bool chain = less(a.asym) == 0, entity = less(a.entity) == 0;
  const long long dr = less(a.residue);
  int first = 2 * a.r + 1;
  if (chain) first = dr == 0 ? 2 * a.r + 2 + clip_to(less(a.token), a.r) : clip_to(dr, a.r);
  const int second = entity ? clip_to(less(a.sym), a.s) : 2 * a.s + 1;
  return (uint32_t)first | (uint32_t)second << 16;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* p, float4 v) { __stcs(reinterpret_cast<float4*>(p), v); }
template <>
__device__ __forceinline__ void store4<bf16>(bf16* p, float4 v) {
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)));
}
template <>
__device__ __forceinline__ void store4<__half>(__half* p, float4 v) {
  const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi)));
}

constexpr int kRpFwdThreads = 1024;      // one block an SM
constexpr int kRpFwdBytes = 226 << 10;   // shared memory of one: the tables and, beside them, its channels of W
static_assert((kRpMaxRows + kRpMaxRows + 2) * 64 * 4 <= kRpFwdBytes, "room for 64 channels");      // W has two columns more than the tables have rows

// kW: channels of a block, whose table is made for all of them.  codes: what the backward pass reads, one a pair, or NULL.
template <typename T, int kW>
__global__ void __launch_bounds__(kRpFwdThreads) relpos_fwd_kernel(RelposArgs a, const float* __restrict__ w, T* __restrict__ z,
                                                                   uint32_t* __restrict__ codes) {
  constexpr int kLanes = kW / 4, kSide = 32 / kLanes;                   // lanes of a pair, pairs side by side in a warp
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full;
  const int c0 = blockIdx.y * kW, channels = min(kW, a.c - c0), t = a.columns();
  const int rows1 = a.rows1(), rows = rows1 + a.rows2(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tok = 2 * a.r + 2, ent = 4 * a.r + 4, chain = ent + 1;      // first columns of the parts of W behind the first
  float* const table = reinterpret_cast<float*>(smem_raw);              // [rows][kW]
  float* const part = table + rows * kW;                                // [kW][t]
  if (threadIdx.x == 0) {
    mbar_init(&full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    mbar_expect_tx(&full, (uint32_t)(channels * t * 4));
    bulk_load(part, w + (long long)c0 * t, (uint32_t)(channels * t * 4), &full);
  }
  const int strips = (int)((a.n + kRpPairs - 1) / kRpPairs);
  const long long units = a.pairs / a.n * strips, warps = (long long)gridDim.x * (kRpFwdThreads / 32);
  long long u = (long long)warp * gridDim.x + blockIdx.x;               // the blocks have equal shares, however few units there are
  const auto code_of = [&](long long unit) {                            // of this lane's pair
    const long long i = unit / strips;                                  // counts the rows of all batches
    const int j = (int)(unit - i * strips) * kRpPairs + lane;
    return relpos_code(a, i, i / a.n * a.n + min((long long)j, a.n - 1));
  };
  uint32_t code = u < units ? code_of(u) : 0u;                          // asked for while W is on its way
  __syncthreads();
  const bool ok = mbar_wait(&full, 0, 2u);
  // A lane = a channel: t is odd, so neither side of this transposition meets a bank twice.
  for (int v = threadIdx.x; v < rows * kW; v += kRpFwdThreads) {
    const int ch = v % kW, row = v / kW;
    if (ch < channels) {
      const float* const f = part + ch * t;
      const float x = row < tok     ? f[row] + f[tok + 2 * a.r + 1]
                      : row < rows1 ? f[a.r] + f[row]
                                    : f[chain + row - rows1] + (row - rows1 < 2 * a.s + 1 ? f[ent] : 0.f);
      table[row * kW + ch] = x;
    }
  }
  if (!__syncthreads_and(ok)) return;
  const int at = 4 * (lane % kLanes), side = lane / kLanes;
  const bool mine = at < channels;
  while (u < units) {
    const long long i = u / strips;
    const int j0 = (int)(u - i * strips) * kRpPairs, count = (int)min((long long)kRpPairs, a.n - j0);
    if (codes && blockIdx.y == 0 && lane < count) codes[i * a.n + j0 + lane] = code;
    T* out = z + (i * a.n + j0 + side) * a.c + c0 + at;
    uint32_t have = 0xffffffffu;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < count; k += kSide) {
      const uint32_t now = __shfl_sync(0xffffffffu, code, k + side);
      if (now != have) {
        have = now;
        const float4 p = *reinterpret_cast<const float4*>(table + (now & 0xffffu) * kW + at);
        const float4 q = *reinterpret_cast<const float4*>(table + (rows1 + (now >> 16)) * kW + at);
        v = make_float4(p.x + q.x, p.y + q.y, p.z + q.z, p.w + q.w);
      }
      if (mine && k + side < count) store4(out + (long long)k * a.c, v);
    }
    u += warps;
    if (u < units) code = code_of(u);
  }
}

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load1<__half>(const __half* p) { return __half2float(*p); }

constexpr int kRpBwdThreads = kRpChunk;      // a thread = one channel

// The columns of W from a thread's sums by table row (row k: mine[k * kRpChunk]): a row of the first table counts for its position and its token column, one of
// the second for its own and, unless the entities differ, the entity's.
__device__ __forceinline__ void relpos_fold(const RelposArgs& a, const float* mine, float* out) {
  const int t = a.columns(), tok = 2 * a.r + 2, ent = 4 * a.r + 4, rows1 = a.rows1();
  const auto range = [&](int from, int to) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = from; k < to; k += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += k + e < to ? mine[(k + e) * kRpChunk] : 0.f;
    return (v[0] + v[1]) + (v[2] + v[3]);
  };
#pragma unroll 8
  for (int k = 0; k < ent - 1; ++k) out[k * kRpChunk] = mine[k * kRpChunk];
  out[a.r * kRpChunk] = mine[a.r * kRpChunk] + range(tok, rows1);      // pairs of one residue, whatever their tokens
  out[(ent - 1) * kRpChunk] = range(0, tok);
  out[ent * kRpChunk] = range(rows1, rows1 + 2 * a.s + 1);
  for (int k = ent + 1; k < t; ++k) out[k * kRpChunk] = mine[(rows1 + k - ent - 1) * kRpChunk];
}

// Block b adds up the units [b * per, (b + 1) * per) of its channels; a unit is a row's strip of 32 pairs.  partial: [chunk][block][columns][kRpChunk].
template <typename T>
__global__ void __launch_bounds__(kRpBwdThreads, 2) relpos_bwd_kernel(RelposArgs a, const T* __restrict__ dz, const uint32_t* __restrict__ codes,
                                                                   float* __restrict__ partial, int per) {
  constexpr int kPairs = kRpStageBytes / (kRpChunk * (int)sizeof(T));      // of a stage: 16 (fp32) or 32
  constexpr int kParts = kRpPairs / kPairs;                                // stages of a unit
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full[kRpStages];
  T* stage = reinterpret_cast<T*>(smem_raw);
  float* const mine = reinterpret_cast<float*>(smem_raw + kRpStages * kRpStageBytes) + threadIdx.x;      // row k: mine[k * kRpChunk]
  const int c0 = blockIdx.y * kRpChunk, channels = min(kRpChunk, a.c - c0), lane = threadIdx.x & 31;
  const int rows1 = a.rows1(), rows = rows1 + a.rows2(), n = (int)a.n;
  const int strips = (n + kRpPairs - 1) / kRpPairs;
  const long long units = a.pairs / a.n * strips, begin = (long long)blockIdx.x * per;
  const int steps = (int)(min(begin + per, units) - begin) * kParts;
  if (threadIdx.x == 0) {
    for (int k = 0; k < kRpStages; ++k) mbar_init(&full[k], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  // the parts of a stage that no copy reaches (channels beyond the last) are added up as zeros
  if (channels < kRpChunk) {
    for (int k = threadIdx.x; k < kRpStages * kRpStageBytes / 16; k += kRpBwdThreads)
      reinterpret_cast<uint4*>(smem_raw)[k] = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  for (int k = 0; k < rows; ++k) mine[k * kRpChunk] = 0.f;
  __syncthreads();
  // Where a unit lies: its row of all batches, its first column; both kept up by additions.
  struct Place {
    long long i;
    int strip;
    __device__ __forceinline__ void next(int strips) {
      if (++strip == strips) strip = 0, ++i;
    }
  };
  const auto pairs_of = [&](const Place& p, int part) { return min(max(n - p.strip * kRpPairs - part * kPairs, 0), kPairs); };
  const auto fetch = [&](const Place& p, int step) {              // one thread
    const int part = step % kParts, count = pairs_of(p, part), b = step % kRpStages;
    const uint32_t bytes = (uint32_t)(channels * sizeof(T));
    T* const to = stage + b * (kRpStageBytes / (int)sizeof(T));
    const T* const from = dz + (p.i * n + p.strip * kRpPairs + part * kPairs) * a.c + c0;
    mbar_expect_tx(&full[b], bytes * count);
    if (a.c == kRpChunk) {
      if (count > 0) bulk_load(to, from, bytes * count, &full[b]);
    } else {
      for (int k = 0; k < count; ++k) bulk_load(to + k * kRpChunk, from + (long long)k * a.c, bytes, &full[b]);
    }
  };
  Place here = {begin / strips, (int)(begin % strips)}, ahead = here;
  if (threadIdx.x == 0) {
    for (int k = 0; k < kRpStages - 1 && k < steps; ++k) {
      fetch(ahead, k);
      if ((k + 1) % kParts == 0) ahead.next(strips);
    }
  }
  int row1 = -1, row2 = -1;                        // what the running sums belong to
  float run1 = 0.f, run2 = 0.f;
  const auto flush = [&](int row, float& run) {
    if (row >= 0) mine[row * kRpChunk] += run;
    run = 0.f;
  };
  const auto turn_to = [&](uint32_t now) {         // a code for the whole warp: what does not go on is put away
    if ((int)(now & 0xffffu) != row1) {
      flush(row1, run1);
      row1 = (int)(now & 0xffffu);
    }
    if ((int)(now >> 16) != row2) {
      flush(row2 >= 0 ? rows1 + row2 : -1, run2);
      row2 = (int)(now >> 16);
    }
  };
  const auto code_at = [&](const Place& p) { return __ldg(codes + p.i * n + min(p.strip * kRpPairs + lane, n - 1)); };
  Place then = here;
  uint32_t code = 0, next = steps > 0 ? code_at(then) : 0;
  bool ok = true;
  for (int step = 0; step < steps; ++step) {
    const int part = step % kParts, count = pairs_of(here, part), b = step % kRpStages;
    if (part == 0) {
      code = next;
      then.next(strips);
      if (step + kParts < steps) next = code_at(then);
    }
    ok = mbar_wait_warp(&full[b], (step / kRpStages) & 1, 1u);
    // All are through with the stage that is filled next.  (Barriers of the four warps' own, asked by a fifth warp or by the first, let them drift apart and
    // took 172 and 200 us at 1501 tokens where this takes 158.)
    ok = __syncthreads_and(ok) != 0;
    if (!ok) break;
    if (threadIdx.x == 0 && step + kRpStages - 1 < steps) {
      fetch(ahead, step + kRpStages - 1);
      if ((step + kRpStages) % kParts == 0) ahead.next(strips);
    }
    const T* const from = stage + b * (kRpStageBytes / (int)sizeof(T)) + threadIdx.x;
    const int l0 = part * kPairs;                  // the lane that has the code of the stage's first pair
    const uint32_t all = kPairs == 32 ? 0xffffffffu : 0xffffu << l0;
    const uint32_t lead = __shfl_sync(0xffffffffu, code, l0);
    if (count == kPairs && (__ballot_sync(0xffffffffu, code == lead) & all) == all) {
      turn_to(lead);
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPairs; ++k) t[k & 3] += load1(from + k * kRpChunk);
      const float sum = (t[0] + t[1]) + (t[2] + t[3]);
      run1 += sum, run2 += sum;
    } else {
      const uint32_t first = code & 0xffffu, second = code >> 16, mine8 = 0xffu << (lane & 24);      // the lanes of this lane's group of eight
      const uint32_t like = __match_any_sync(0xffffffffu, first) & mine8;
      const uint32_t distinct = __ballot_sync(0xffffffffu, like == 1u << lane), alike = __ballot_sync(0xffffffffu, like == mine8);
      const uint32_t copies = __ballot_sync(0xffffffffu, second == __shfl_sync(0xffffffffu, second, lane & 24));
#pragma unroll 1
      for (int g = 0; g < count; g += 8) {
        const uint32_t group = 0xffu << (l0 + g), now = __shfl_sync(0xffffffffu, code, l0 + g);
        if (g + 8 <= count && (copies & group) == group && ((distinct | alike) & group) == group) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = load1(from + (g + k) * kRpChunk);
          const float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
          if ((alike & group) == group) {
            turn_to(now);
            run1 += sum, run2 += sum;
          } else {
            // eight rows of the first table, side by side: their sums have no order among them
            turn_to((now & 0xffff0000u) | 0xffffu);
            row1 = -1;
            float* at[8];
            float u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) at[k] = mine + __shfl_sync(0xffffffffu, first, l0 + g + k) * kRpChunk;
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = *at[k];
#pragma unroll
            for (int k = 0; k < 8; ++k) *at[k] = u[k] + v[k];
            run1 = 0.f, run2 += sum;
          }
        } else {
          for (int k = g; k < min(g + 8, count); ++k) {
            const float v = load1(from + k * kRpChunk);
            turn_to(__shfl_sync(0xffffffffu, code, l0 + k));
            run1 += v, run2 += v;
          }
        }
      }
    }
    if (part == kParts - 1) here.next(strips);
  }
  flush(row1, run1);
  flush(row2 >= 0 ? rows1 + row2 : -1, run2);
  relpos_fold(a, mine, partial + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.columns() * kRpChunk + threadIdx.x);
}

// The same for 16-bit dz on the tensor cores: the sums by table row are dz^T times the pairs' two-hot rows, M = 128 channels, N = table rows, K = pairs.
// dz enters as it lies (its channels are the contiguous index: an MN-major operand), the two-hot operand [table row][64 pairs] lives in shared memory and costs
// a lane two stores a pair to set and two to clear (four warps of them: one took 1100 cycles a tile, where memory takes 700); the products with one are exact.
// 64 pairs are 288 cycles of the tensor pipe (N = 144), less than half of what their 16 KB take to arrive.  Memory bounds it: 1501 tokens x 128
// channels, 110 us for 577 MB + 9 MB of codes = 5.3 TB/s, 81 % of a copy's rate (six tiles on their way, or codes asked for two tiles ahead: the same).
// The tensor core truncates when it adds, so an accumulator takes eight tiles (32 additions) before four warps add it, rounding to nearest, to fp32
// sums in shared memory, while the next tiles go to the other accumulator.
// Warps 0..3 drain (a thread = one channel), 4 brings dz, 5 issues the products, 6..9 write the two-hot operands, 32 pairs of every other tile each.
constexpr int kRpTile = 64, kRpRing = 4, kRpGroup = 8;      // pairs of a tile, tiles on their way, tiles of an accumulator
constexpr int kRpTcThreads = 10 * 32, kRpTileBytes = kRpTile * kRpChunk * 2;
constexpr int kRpTcRows = 208;                              // what shared memory holds of sums and operands
struct RpTcBars {
  uint64_t full[kRpRing], empty[kRpRing], hot_full[2], hot_empty[2], acc_full[2], acc_free[2];
  uint32_t tmem_base;
};

template <bool kF16>
__global__ void __launch_bounds__(kRpTcThreads, 1) relpos_bwd_tc_kernel(const __grid_constant__ CUtensorMap map, RelposArgs a,
                                                                        const uint32_t* __restrict__ codes, float* __restrict__ partial, int n_cols,
                                                                        int per) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = smem_aligned(smem_raw);
  unsigned char* const hot = sm + kRpRing * kRpTileBytes;                                    // two operands [n_cols][64], 128-byte swizzle
  float* const sums = reinterpret_cast<float*>(hot + 2 * n_cols * 128);                      // [n_cols][128]
  RpTcBars& bars = *reinterpret_cast<RpTcBars*>(reinterpret_cast<unsigned char*>(sums) + n_cols * kRpChunk * 4);
  const int warp = warp_index(), lane = threadIdx.x & 31, c0 = blockIdx.y * kRpChunk;
  const long long all = (a.pairs + kRpTile - 1) / kRpTile, begin = (long long)blockIdx.x * per;
  const int tiles = (int)(min(begin + per, all) - begin), groups = (tiles + kRpGroup - 1) / kRpGroup;
  const bool skip = cta_begin();
  if (threadIdx.x == 0) {
    for (int k = 0; k < kRpRing; ++k) {
      mbar_init(&bars.full[k], 1);
      mbar_init(&bars.empty[k], 1);
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(&bars.hot_full[k], 2);
      mbar_init(&bars.hot_empty[k], 1);
      mbar_init(&bars.acc_full[k], 1);
      mbar_init(&bars.acc_free[k], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  for (int k = threadIdx.x; k < 2 * n_cols * 8; k += kRpTcThreads) reinterpret_cast<uint4*>(hot)[k] = make_uint4(0u, 0u, 0u, 0u);
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&bars.tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (!cta_ready(skip, warp == 5, bars.tmem_base, 512)) return;
  const uint32_t tmem = bars.tmem_base;
  if (warp == 4) {
    bool ok = true;
    for (int t = 0; t < tiles && ok; ++t) {
      const int s = t % kRpRing;
      if (t >= kRpRing) ok = mbar_wait_warp(&bars.empty[s], (t / kRpRing - 1) & 1, 1u);
      if (ok && elect_lane()) {
        const int p0 = (int)((begin + t) * kRpTile);
        const uint32_t dst = smem_u32(sm + s * kRpTileBytes);
        mbar_expect_tx(&bars.full[s], kRpTileBytes);
        tma_load_3d(dst, &map, &bars.full[s], c0, p0, 0);
        tma_load_3d(dst + kRpTile * 128, &map, &bars.full[s], c0 + 64, p0, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 6) {
    const int rows1 = a.rows1();
    const int b = warp & 1, k = 32 * ((warp - 6) >> 1) + lane;      // the operand, and this lane's pair of each of its tiles
    unsigned char* const operand = hot + b * n_cols * 128;
    const auto code_at = [&](int t) {
      const long long p = (begin + t) * kRpTile + k;
      return t < tiles && p < a.pairs ? __ldg(codes + p) : 0xffffffffu;
    };
    const auto put = [&](uint32_t code, uint16_t v) {
      if (code == 0xffffffffu) return;
      const int first = code & 0xffffu, second = rows1 + (code >> 16);
      *reinterpret_cast<uint16_t*>(operand + first * 128 + (((k >> 3) ^ (first & 7)) << 4) + 2 * (k & 7)) = v;
      *reinterpret_cast<uint16_t*>(operand + second * 128 + (((k >> 3) ^ (second & 7)) << 4) + 2 * (k & 7)) = v;
    };
    constexpr uint16_t kOne = kF16 ? 0x3c00 : 0x3f80;
    uint32_t was = 0xffffffffu, next = code_at(b);
    bool ok = true;
    for (int t = b; t < tiles && ok; t += 2) {
      const uint32_t now = next;
      next = code_at(t + 2);
      if (t >= 2) ok = mbar_wait_warp(&bars.hot_empty[b], (t / 2 - 1) & 1, 2u);
      if (now != was) {
        put(was, 0);
        put(now, kOne);
        was = now;
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.hot_full[b]);
    }
  } else if (warp == 5) {
    // the operands' first contents are zeros written by all threads
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    const uint32_t idesc = umma_idesc_16(128, n_cols, kF16, kF16, true, false);
    bool ok = true;
    for (int t = 0; t < tiles && ok; ++t) {
      const int s = t % kRpRing, b = t & 1, g = t / kRpGroup, in_group = t % kRpGroup;
      if (in_group == 0 && g >= 2) ok = mbar_wait_warp(&bars.acc_free[g & 1], (g / 2 - 1) & 1, 4u);
      ok = ok && mbar_wait_warp(&bars.hot_full[b], (t / 2) & 1, 8u) && mbar_wait_warp(&bars.full[s], (t / kRpRing) & 1, 16u);
      if (!ok) break;
      tc_fence_after();
      if (elect_lane()) {
        const uint64_t da = umma_desc_mn_sw128(smem_u32(sm + s * kRpTileBytes), kRpTile * 128, 1024), db = umma_desc_sw128(smem_u32(hot + b * n_cols * 128));
#pragma unroll
        for (int ks = 0; ks < kRpTile / 16; ++ks) umma_bf16(tmem + 256 * (g & 1), da + 128 * ks, db + 2 * ks, idesc, in_group > 0 || ks > 0);
        umma_commit(&bars.empty[s]);
        umma_commit(&bars.hot_empty[b]);
        if (in_group == kRpGroup - 1 || t == tiles - 1) umma_commit(&bars.acc_full[g & 1]);
      }
      __syncwarp();
    }
  } else {
    float* const mine = sums + threadIdx.x;       // a thread's channel: row k at mine[k * kRpChunk]
    const uint32_t t_lane = tmem + ((uint32_t)(32 * warp) << 16);
    bool ok = true;
    for (int g = 0; g < groups; ++g) {
      ok = mbar_wait_warp(&bars.acc_full[g & 1], (g >> 1) & 1, 32u);
      if (!ok) break;
      tc_fence_after();
      for (int k = 0; k < n_cols; k += 16) {
        uint32_t x[16];
        tmem_ld16(t_lane + 256 * (g & 1) + k, x);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = g > 0 ? mine[(k + e) * kRpChunk] : 0.f;
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(k + e) * kRpChunk] = v[e] + __uint_as_float(x[e]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.acc_free[g & 1]);
    }
    if (ok) relpos_fold(a, mine, partial + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.columns() * kRpChunk + threadIdx.x);
  }
  tc_fence_before();
  cta_teardown_sync();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
  }
}

// dw[c][t] = the blocks' sums, in their order: eight slices of the blocks, each added up by one thread a channel, then the slices.
__global__ void __launch_bounds__(8 * kRpChunk) relpos_reduce_kernel(const float* __restrict__ partial, float* __restrict__ dw, int blocks, int t,
                                                                     int c) {
  __shared__ float slice[8][kRpChunk];
  const int k = blockIdx.x, chunk = blockIdx.y, ch = threadIdx.x % kRpChunk, s = threadIdx.x / kRpChunk;
  const float* p = partial + ((long long)chunk * blocks * t + k) * kRpChunk + ch;
  float v = 0.f;
#pragma unroll 8
  for (int b = s; b < blocks; b += 8) v += p[(long long)b * t * kRpChunk];
  slice[s][ch] = v;
  __syncthreads();
  if (s == 0 && chunk * kRpChunk + ch < c) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += slice[e][ch];
    dw[(long long)(chunk * kRpChunk + ch) * t + k] = sum;
  }
}

PX_DEFINE_FAMILY_HOOKS(relpos)

static bool relpos_sizes(int64_t batch, int64_t n, int64_t c, int32_t r, int32_t s) {
  return batch >= 0 && n >= 0 && c > 0 && r >= 0 && s >= 0 && n < (1 << 17) && batch < (1 << 17) && c < (1 << 16);
}
static bool relpos_fits(int64_t c, int32_t r, int32_t s) {
  return c % 8 == 0 && r <= kRpMaxRows && s <= kRpMaxRows && 4 * r + 2 * s + 5 <= kRpMaxRows;
}
// Backward pass: units (strips of 32 pairs of a row), and blocks: two an SM, and no more than leave each two units, since each brings sums of its own
// (16 units and 2, both kernels, us: 33 tokens in fp32 32.2 / 10.8, 97 35.1 / 13.2, 200 31.9 / 18.3; bf16, 33 9.8 / 9.2, 97 11.1 / 10.5, 200 11.9 / 12.3).
static int64_t relpos_units(int64_t batch, int64_t n) { return batch * n * ((n + kRpPairs - 1) / kRpPairs); }
static int64_t relpos_blocks(int64_t units) { return std::max<int64_t>(1, std::min<int64_t>(2 * sm_count(), units / 2)); }

// Forward, channels of a block: 32 while each of its warps has one strip at most, for then the tables are what it waits for; otherwise 64.  With 32 / 64 / 128
// channels (128 in all, r = 32, s = 2), us: 97 tokens in fp32 5.0 / 6.1 / 8.8; 150 5.9 / 6.5 / 8.9; 200 8.2 / 7.7 / 9.5; 384 15.1 / 15.8 / 17.6;
// 1501 196 / 187 / 193; bf16, 200 7.3 / 6.6 / 9.1; 600 23.7 / 19.5 / 22.0; 1501 117 / 91 / 98.  (Two blocks an SM are slower at every size: 97 tokens 8.4.)
static bool relpos_narrow(int64_t batch, int64_t n, int64_t c) {
  return relpos_units(batch, n) <= kRpFwdThreads / 32 * std::max<int64_t>(sm_count() / ((c + 31) / 32), 1);
}

// 16-bit gradients with tables that fit, at every size: on the tensor cores / one by one (bf16, 128 channels, r = 32, s = 2), us: 33 tokens 7.6 / 23.3,
// 97 8.3 / 25.9, 200 8.8 / 22.7, 384 12.1 / 21.1, 600 27.7 / 38.4, 1000 61.6 / 85.1, 1501 110 / 158.  fp32 would need three 16-bit parts of dz, made on the way
// by warps of their own; it is not built.
static bool relpos_on_tensor_cores(int64_t pairs, int n_cols, int32_t dtype) {
  return dtype != PX_F32 && n_cols <= kRpTcRows && pairs < (int64_t)0x7fffff00;
}

}  // namespace px

using namespace px;

extern "C" int64_t px_relpos_workspace_bytes(int64_t batch, int64_t n, int64_t c, int32_t r_max, int32_t s_max) {
  if (!relpos_sizes(batch, n, c, r_max, s_max) || !relpos_fits(c, r_max, s_max)) return 0;
  const int64_t units = relpos_units(batch, n);
  return relpos_blocks(units) * ((c + kRpChunk - 1) / kRpChunk) * (4 * r_max + 2 * s_max + 7) * kRpChunk * 4;
}

extern "C" int64_t px_relpos_codes_bytes(int64_t batch, int64_t n) {
  return relpos_sizes(batch, n, 8, 0, 0) ? batch * n * n * 4 : 0;
}

extern "C" int32_t px_relpos_fwd(const int64_t* asym_id, const int64_t* residue_index, const int64_t* entity_id, const int64_t* token_index,
                                 const int64_t* sym_id, const float* w, void* z, uint32_t* codes, int64_t batch, int64_t n, int64_t c,
                                 int32_t r_max, int32_t s_max, int32_t dtype, void* stream) {
  if (!relpos_sizes(batch, n, c, r_max, s_max)) return PX_ERR_BAD_ARG;
  if (!relpos_fits(c, r_max, s_max) || (dtype != PX_F32 && dtype != PX_BF16 && dtype != PX_F16)) return PX_ERR_UNSUPPORTED;
  if (batch == 0 || n == 0) return PX_OK;
  if (!asym_id || !residue_index || !entity_id || !token_index || !sym_id || !w || !z || (((uintptr_t)z | (uintptr_t)w) & 15)) return PX_ERR_BAD_ARG;
  const RelposArgs a = {(const long long*)asym_id, (const long long*)residue_index, (const long long*)entity_id, (const long long*)token_index,
                        (const long long*)sym_id, n, batch * n * n, (int)c, r_max, s_max};
  const auto go = [&](auto* kernel, auto* out, int width, SmemLimit& limit) {
    const size_t smem = (size_t)(a.rows1() + a.rows2() + a.columns()) * width * 4;
    // a few strips a block at least, one block an SM at most
    const int64_t parts = (c + width - 1) / width;
    const dim3 grid((unsigned)std::min<int64_t>((relpos_units(batch, n) + 3) / 4, std::max<int64_t>(sm_count() / parts, 1)), (unsigned)parts);
    if (!limit.set(kernel, kRpFwdBytes)) return false;
    kernel<<<grid, kRpFwdThreads, smem, (cudaStream_t)stream>>>(a, w, out, codes);
    return cudaGetLastError() == cudaSuccess;
  };
  static SmemLimit limits[2][3];
  const auto as = [&](auto* out) {
    typedef std::remove_pointer_t<decltype(out)> T;
    return relpos_narrow(batch, n, c) ? go(relpos_fwd_kernel<T, 32>, out, 32, limits[0][dtype]) : go(relpos_fwd_kernel<T, 64>, out, 64, limits[1][dtype]);
  };
  const bool done = dtype == PX_F32 ? as((float*)z) : dtype == PX_BF16 ? as((bf16*)z) : as((__half*)z);
  return done ? PX_OK : PX_ERR_LAUNCH;
}

extern "C" int32_t px_relpos_bwd(const uint32_t* codes, const void* dz, float* dw, void* workspace, int64_t workspace_bytes, int64_t batch,
                                 int64_t n, int64_t c, int32_t r_max, int32_t s_max, int32_t dtype, void* stream) {
  if (!relpos_sizes(batch, n, c, r_max, s_max)) return PX_ERR_BAD_ARG;
  if (!relpos_fits(c, r_max, s_max) || (dtype != PX_F32 && dtype != PX_BF16 && dtype != PX_F16)) return PX_ERR_UNSUPPORTED;
  if (!dw) return PX_ERR_BAD_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  const RelposArgs a = {nullptr, nullptr, nullptr, nullptr, nullptr, n, batch * n * n, (int)c, r_max, s_max};
  if (batch == 0 || n == 0)
    return cudaMemsetAsync(dw, 0, (size_t)c * a.columns() * 4, st) == cudaSuccess ? PX_OK : PX_ERR_LAUNCH;
  if (!codes || !dz || !workspace || (((uintptr_t)dz | (uintptr_t)workspace) & 15)) return PX_ERR_BAD_ARG;
  if (workspace_bytes < px_relpos_workspace_bytes(batch, n, c, r_max, s_max)) return PX_ERR_WORKSPACE;
  const unsigned chunks = (unsigned)((c + kRpChunk - 1) / kRpChunk);
  float* const partial = (float*)workspace;
  const int rows = a.rows1() + a.rows2(), n_cols = (rows + 15) / 16 * 16;
  int blocks;
  bool done;
  if (relpos_on_tensor_cores(a.pairs, n_cols, dtype)) {
    const int64_t tiles = (a.pairs + kRpTile - 1) / kRpTile, most = std::min<int64_t>(relpos_blocks(relpos_units(batch, n)), sm_count());
    const int64_t per = (tiles + most - 1) / most;
    blocks = (int)((tiles + per - 1) / per);
    CUtensorMap map;
    if (!have_context() ||
        !make_map_3d(&map, dtype == PX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dz, (uint64_t)c, (uint64_t)a.pairs, 1,
                     (uint64_t)c * 2, (uint64_t)a.pairs * c * 2, 64, kRpTile, CU_TENSOR_MAP_SWIZZLE_128B))
      return PX_ERR_LAUNCH;
    const auto bytes = [](int cols) { return (size_t)kRpRing * kRpTileBytes + (size_t)cols * (2 * 128 + kRpChunk * 4) + sizeof(RpTcBars) + 1024; };
    static SmemLimit limit[2];
    const auto kernel = dtype == PX_F16 ? relpos_bwd_tc_kernel<true> : relpos_bwd_tc_kernel<false>;
    if (!limit[dtype == PX_F16].set(kernel, bytes(kRpTcRows))) return PX_ERR_LAUNCH;
    kernel<<<dim3((unsigned)blocks, chunks), kRpTcThreads, bytes(n_cols), st>>>(map, a, codes, partial, n_cols, (int)per);
    done = cudaGetLastError() == cudaSuccess;
  } else {
    const int64_t units = relpos_units(batch, n), most = relpos_blocks(units), per = (units + most - 1) / most;
    blocks = (int)((units + per - 1) / per);
    const size_t fixed = (size_t)kRpStages * kRpStageBytes, smem = fixed + (size_t)rows * kRpChunk * 4;
    static SmemLimit limit[3];
    const auto go = [&](auto* kernel, auto* in) {
      if (!limit[dtype].set(kernel, fixed + (size_t)kRpMaxRows * kRpChunk * 4)) return false;
      kernel<<<dim3((unsigned)blocks, chunks), kRpBwdThreads, smem, st>>>(a, in, codes, partial, (int)per);
      return cudaGetLastError() == cudaSuccess;
    };
    done = dtype == PX_F32    ? go(relpos_bwd_kernel<float>, (const float*)dz)
           : dtype == PX_BF16 ? go(relpos_bwd_kernel<bf16>, (const bf16*)dz)
                              : go(relpos_bwd_kernel<__half>, (const __half*)dz);
  }
  if (!done) return PX_ERR_LAUNCH;
  relpos_reduce_kernel<<<dim3((unsigned)a.columns(), chunks), 8 * kRpChunk, 0, st>>>(partial, dw, blocks, a.columns(), (int)c);
  return cudaGetLastError() == cudaSuccess ? PX_OK : PX_ERR_LAUNCH;
}
