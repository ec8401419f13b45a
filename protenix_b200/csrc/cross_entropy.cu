// Softmax cross entropy of a linear head, and its gradient, without the logits:
//   l_iv = x_i . w_v + b_v,   lse_i = log sum_v exp l_iv,   loss_i = lse_i - (1 - e) l_it - e / V sum_v l_iv
//   dl_iv = g_i (exp(l_iv - lse_i) - (1 - e) [v = t_i] - e / V),   dx = dl W,   dW = dl^T x,   db = sum_i dl_i
//
// Forward, one product whose epilogue keeps of a tile [128 rows][kN classes] each row's maximum, sum of exponentials and (smoothed
// labels) sum of logits, and the logit of the row's class where it lies in the tile; a second kernel joins the tiles of a row.
// Backward, for a piece of the classes at a time: the same product again, whose epilogue writes dl in 16 bits, then dx += dl W and
// dW = dl^T x from it.  What a piece leaves in memory is 16 bits a pair of row and class: kPieceBytes whatever the number of classes, or 512 bytes a row where
// that is more (a piece has 256 classes at least).
// Four products of 2 N V C where three are the least (the logits are formed twice).
//
// dl is formed without the scale of the loss, in [-2, 2] (fp16: times 2^14, so that probabilities down to 2^-28 stay normal numbers); the scale is
// applied in fp32 where dx and dW are rounded.  Logits, exponentials and their sums are fp32, the sum of the losses fp64; dx and dW fp32 accumulators of bounded length
// (longest_sum), added up in fp32; db fp32 over 32 rows and fp64 over these (small heads: fp32, px_head_small.cuh).
//
// Rows that are ignored take no part whatever they hold: their dl is zero by selection, and where one holds an infinity or a NaN (which a zero
// weight would not silence) dW takes a copy of x in which those rows are zero; the copy is made only then, where dx will be (dW is formed before it), or in the
// workspace of a call that wants no dx.  A row of x that is not finite has no
// finite logit, so the forward pass sees it in the row's sum; by a pass over the ignored rows and one for the verdict, two more launches, training on
// 384 rows took 104 us and on 3001 12 us more.
#include "px_head_small.cuh"

namespace px {

constexpr int64_t kPieceBytes = 512ll << 20;
constexpr int kScanBlocks = 592;
constexpr int kBiasGroups = 256;       // of 32 rows, whose sums the epilogue of dW adds up

// ---- forward ---------------------------------------------------------------------------------------------------------
struct EpiStats {
  const int64_t* target;
  HeadBias bias;
  float2* part;             // [tiles_n][rows]: maximum times log2(e), sum of exponentials relative to it
  float* part_sum;          // [tiles_n][rows]: sum of logits, or NULL
  float* hit;               // [rows]: logit of the row's class
  uint32_t* arrivals;
  uint32_t* dirty;
  int rows, classes;
  float uncut;
  static constexpr bool kMeets = true, kStores = false;
  __device__ __forceinline__ void begin() const { *arrivals = 0, *dirty = 0; }

  struct Row {
    int mine;                 // the column that is the row's class, or -1
    bool plain;               // all classes are there, without a bias
  };
  template <class S>
  __device__ __forceinline__ Row before(const GemmEpiTile& e) const {
    const int row = e.m0 + e.lane;
    const int64_t t = row < rows ? target[row] - e.n0 : -1;
    return {t >= 0 && t < S::kPartCols ? (int)t : -1, warp_bias<S>(e, bias, classes)};
  }
  template <class S, class F>
  __device__ __forceinline__ void tile(const GemmEpiTile& e, const Row& at, F release) const {
    constexpr int kCols = S::kPartCols;
    const int row = e.m0 + e.lane, base = e.n0, mine = at.mine;
    const bool there = row < rows;
    float m = -CUDART_INF_F, s = 0.f, sum = 0.f;
    if (base >= classes) release();
#pragma unroll 1
    for (int c = 0; c < kCols; c += 32) {
      const int left = classes - (base + c);
      if (left <= 0) break;
      uint32_t r[32];
      tmem_ld32(e.acc + c, r);
      tmem_wait_ld();
      if (c + 32 == kCols || left <= 32) release();
      float v[32];
      logits_of(r, uncut, v);
      if (!at.plain) add_bias(v, e.own + c);
      if (part_sum) {
        float a[4] = {};
#pragma unroll
        for (int j = 0; j < 32; ++j) a[j & 3] += j < left ? v[j] : 0.f;
        sum += (a[0] + a[1]) + (a[2] + a[3]);
      }
      if (mine >= c && mine < c + 32) {
        hit[row] = pick(v, mine - c);
      }
      float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int j = 4; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], v[j]);
      const float next = fmaxf(m, kLog2e * fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      const float ref = reference(next);
      float a[4] = {s * fast_exp2(m - ref), 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 32; ++j) a[j & 3] += fast_exp2(fmaf(v[j], kLog2e, -ref));
      s = (a[0] + a[1]) + (a[2] + a[3]);
      m = next;
    }
    // the parts of the columns
    float* const x = e.shared + 32 * e.quarter + e.lane;
    if (e.part) x[384 * (e.part - 1)] = m, x[384 * (e.part - 1) + 128] = s, x[384 * (e.part - 1) + 256] = sum;
    gemm_epi_sync<S>(e.set);
    if (!e.part) {
      float next = m;
#pragma unroll
      for (int p = 0; p < S::kParts - 1; ++p) next = fmaxf(next, x[384 * p]);
      const float ref = reference(next);
      s *= fast_exp2(m - ref);
#pragma unroll
      for (int p = 0; p < S::kParts - 1; ++p) s = fmaf(x[384 * p + 128], fast_exp2(x[384 * p] - ref), s), sum += x[384 * p + 256];
      if (there) {
        const int64_t at = (int64_t)e.at.nt * rows + row;
        part[at] = make_float2(next, s);
        if (part_sum) part_sum[at] = sum;
      }
    }
    gemm_epi_sync<S>(e.set);
  }
};

// Joins the tiles of each row: lse, loss, and (total) their mean or sum over the rows that count.  32 rows a block, the parts of a row over its
// warps; the last block to arrive adds up what the blocks have left, in their order.
constexpr int kJoinWarps = 16;
struct JoinArgs {
  const float2* part;
  const float* part_sum;
  const float* hit;
  const int64_t* target;
  float2* norm;             // [rows]: what exp(l - lse) is formed from, exp2(l log2(e) - x) / y
  float* losses;            // [rows], or NULL
  float* total;             // or NULL
  float* inverse;           // receives 1 / count
  double2* sums;            // [blocks]
  uint32_t* arrivals;
  uint32_t* dirty;          // becomes one where an ignored row of x may not be finite
  int64_t ignore;
  int rows, classes, parts, mean;
  float smooth;
};
__global__ void __launch_bounds__(32 * kJoinWarps) loss_join_kernel(const JoinArgs a) {
  __shared__ float xm[kJoinWarps][32], xs[kJoinWarps][32], xl[kJoinWarps][32];
  __shared__ double tl[32 * kJoinWarps], tc[32 * kJoinWarps];
  __shared__ bool last;
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float m = -CUDART_INF_F, s = 0.f, sum = 0.f;
  if (row < a.rows) {
    for (int p = w; p < a.parts; p += 4 * kJoinWarps) {      // four on their way at once
      float2 x[4];
      float t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = (int64_t)(p + j * kJoinWarps) * a.rows + row;
        const bool there = p + j * kJoinWarps < a.parts;
        x[j] = there ? a.part[at] : make_float2(-CUDART_INF_F, 0.f);
        t[j] = there && a.part_sum ? a.part_sum[at] : 0.f;
      }
      const float next = fmaxf(m, fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x))), ref = reference(next);
      s *= fast_exp2(m - ref);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fmaf(x[j].y, fast_exp2(x[j].x - ref), s), sum += t[j];
      m = next;
    }
  }
  xm[w][lane] = m, xs[w][lane] = s, xl[w][lane] = sum;
  __syncthreads();
  double l = 0.0, c = 0.0;
  if (w == 0 && row < a.rows) {
#pragma unroll 1
    for (int i = 1; i < kJoinWarps; ++i) m = fmaxf(m, xm[i][lane]);
    const float ref = reference(m);
    s = sum = 0.f;
#pragma unroll 1
    for (int i = 0; i < kJoinWarps; ++i) s += xs[i][lane] * fast_exp2(xm[i][lane] - ref), sum += xl[i][lane];
    const int64_t t = a.target[row];
    const bool counts = row_counts(t, a.ignore);
    float loss = 0.f;
    if (counts) {
      loss = row_loss(s, ref, a.hit[row], t >= 0 && t < a.classes, a.smooth, sum, a.classes);
      l = loss, c = 1.0;
    } else if (!(s > 0.f && s < CUDART_INF_F)) {
      *a.dirty = 1;
    }
    a.norm[row] = make_float2(ref, s);
    if (a.losses) a.losses[row] = loss;
  }
  if (!a.total) return;
  if (w == 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o), c += __shfl_xor_sync(0xffffffffu, c, o);
    if (lane == 0) {
      a.sums[blockIdx.x] = make_double2(l, c);
      __threadfence();
      last = atomicAdd(a.arrivals, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  l = c = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += 32 * kJoinWarps) {
    const double2 v = __ldcg(a.sums + i);
    l += v.x, c += v.y;
  }
  tl[threadIdx.x] = l, tc[threadIdx.x] = c;
  __syncthreads();
  for (int o = 16 * kJoinWarps; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) tl[threadIdx.x] += tl[threadIdx.x + o], tc[threadIdx.x] += tc[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *a.total = (float)(a.mean ? tl[0] / tc[0] : tl[0]);      // the mean of nothing is NaN
    *a.inverse = a.mean ? (float)(1.0 / fmax(tc[0], 1.0)) : 1.f;
  }
}

// ---- backward, with a gradient for each row --------------------------------------------------------------------------
// Bits of the largest finite |gradient| of the rows that count, by block.
__global__ void __launch_bounds__(256) loss_scan_kernel(const int64_t* __restrict__ target, const float* __restrict__ grad, uint32_t* __restrict__ found, int64_t ignore, int64_t rows) {
  __shared__ uint32_t big;
  if (threadIdx.x == 0) big = 0;
  __syncthreads();
  pdl_wait();
  uint32_t top = 0;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < rows; row += (int64_t)gridDim.x * 256) {
    const float g = fabsf(grad[row]);
    if (row_counts(target[row], ignore) && g < CUDART_INF_F) top = max(top, __float_as_uint(g));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) atomicMax(&big, top);
  __syncthreads();
  if (threadIdx.x == 0) found[blockIdx.x] = big;
}
__global__ void __launch_bounds__(256) loss_scale_kernel(const uint32_t* __restrict__ found, LossScale* __restrict__ scale, int blocks, float by) {
  __shared__ uint32_t big;
  if (threadIdx.x == 0) big = 0;
  __syncthreads();
  pdl_wait();
  uint32_t top = 0;
  for (int i = threadIdx.x; i < blocks; i += 256) top = max(top, found[i]);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) atomicMax(&big, top);
  __syncthreads();
  if (threadIdx.x == 0) {
    // a power of two, so that nothing is rounded; the smallest have no reciprocal that is finite
    const float power = fmaxf(__uint_as_float(big & 0x7f800000u), 1.17549435e-38f);
    *scale = {power * by, 1.f / power};
  }
}

// ---- backward: dl ----------------------------------------------------------------------------------------------------
struct EpiLogitGrad {
  CUtensorMap out;          // dl [rows][classes of the piece], boxes of 32 x 32
  const int64_t* target;
  HeadBias bias;            // of the piece
  const float2* norm;
  const float* grad;        // of each row's loss, with their scale, or NULL
  const LossScale* scale;
  const uint16_t* x;        // where a row of it may not be finite: receives the ignored rows as zeros in `clean`
  uint16_t* clean;          // or NULL
  const uint32_t* dirty;
  int64_t x_stride;
  int c;
  float* part_bias;         // [32-row groups][classes of the piece]: sums of dl, or NULL
  int64_t ignore;
  int rows, classes, first, all_classes;      // first: the piece's first class
  float smooth, uncut;
  int f16;
  static constexpr bool kMeets = false, kStores = true;
  __device__ __forceinline__ void begin() const {}

  struct Row {
    // dl = factor (p - smooth / V) - (mine) factor (1 - smooth), p = exp2(l log2(e) + ref) / sum
    float over, ref, less, less_hit;
    int mine;
    bool counts, plain;
  };
  __device__ __forceinline__ void copy(int row0, int lane) const {
    const int per = c / 8;
#pragma unroll 1
    for (int row = row0; row < min(row0 + 32, rows); ++row) {
      const bool there = row_counts(target[row], ignore);
      const uint4* const from = reinterpret_cast<const uint4*>(x + row * x_stride);
      uint4* const to = reinterpret_cast<uint4*>(clean) + (int64_t)row * per;
#pragma unroll 1
      for (int i = lane; i < per; i += 32) to[i] = there ? __ldg(from + i) : make_uint4(0, 0, 0, 0);
    }
  }
  template <class S>
  __device__ __forceinline__ Row before(const GemmEpiTile& e) const {
    if (clean && e.at.nt == 0 && e.part == 0 && *dirty) copy(e.m0, e.lane);      // the warps of the first classes see each row once
    Row at = {};
    const int row = e.m0 + e.lane;
    const int64_t t = row < rows ? target[row] : ignore;
    at.counts = row < rows && row_counts(t, ignore);
    const int64_t in_part = t - first - e.n0;
    const bool valid = t >= 0 && t < all_classes;
    at.mine = at.counts && valid && in_part >= 0 && in_part < S::kPartCols ? (int)in_part : -1;
    if (at.counts) {
      float factor = grad ? grad[row] * scale->each : 1.f;
      if (!valid) factor = CUDART_NAN_F;
      if (f16) factor *= kDlScaleF16;
      const float2 n = norm[row];
      at.ref = -n.x, at.over = factor / n.y;
      at.less = factor * smooth / (float)all_classes, at.less_hit = -at.less - factor * (1.f - smooth);
    }
    at.plain = warp_bias<S>(e, bias, classes);
    return at;
  }
  template <class S, class F>
  __device__ __forceinline__ void tile(const GemmEpiTile& e, const Row& at, F release) const {
    constexpr int kCols = S::kPartCols;
    const int base = e.n0, mine = at.mine;
    if (e.m0 >= rows || base >= classes) return release();
    const float over = at.over, ref = at.ref, less = at.less, less_hit = at.less_hit;
    const bool counts = at.counts;
#pragma unroll 1
    for (int c = 0; c < kCols; c += 32) {
      const int left = classes - (base + c);
      if (left <= 0) break;
      uint32_t r[32];
      tmem_ld32(e.acc + c, r);
      tmem_wait_ld();
      if (c + 32 == kCols || left <= 32) release();
      float v[32];
      logits_of(r, uncut, v);
      if (!at.plain) add_bias(v, e.own + c);
      const int own = mine - c;
      if (__any_sync(0xffffffffu, own >= 0 && own < 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = fmaf(over, fast_exp2(fmaf(v[j], kLog2e, ref)), own == j ? less_hit : -less);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = fmaf(over, fast_exp2(fmaf(v[j], kLog2e, ref)), -less);
      }
      if (!counts) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
      }
      if (e.lane == 0) tma_store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t o[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) o[w] = f16 ? pack_f16x2_inf(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]) : pack_bf16x2(v[8 * p + 2 * w], v[8 * p + 2 * w + 1]);
        *reinterpret_cast<uint4*>(e.stg + e.lane * 64 + ((p ^ (e.lane >> 1 & 3)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (e.lane == 0) {
        tma_store_3d(&out, smem_u32(e.stg), base + c, e.m0, 0);
        tma_store_commit();
      }
      if (part_bias) {
        column_sums(v, e.lane);
        if (e.lane < left) part_bias[(int64_t)(e.m0 / 32) * classes + base + c + e.lane] = v[0];
      }
    }
  }
};

// db of a piece: a warp's lanes along the classes, the groups of rows over the warps, in a fixed order.
__global__ void __launch_bounds__(512) loss_bias_kernel(const float* __restrict__ part, void* __restrict__ db, int type, const LossOut out, int classes, int groups) {
  __shared__ double x[16][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, v = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (v < classes)
    for (int g = w; g < groups; g += 16) s += part[(int64_t)g * classes + v];
  x[w][lane] = s;
  __syncthreads();
  if (w == 0 && v < classes) {
    double all = 0.0;
    for (int i = 0; i < 16; ++i) all += x[i][lane];
    bias_store(db, type, v, (float)all * out());
  }
}

// ---- backward: dx and dW ---------------------------------------------------------------------------------------------
// kF32: sums of one split, stored (or added to what the pieces before have left); otherwise the result in 16 bits.
template <bool kF32>
struct EpiGrad {
  CUtensorMap map;          // boxes of 32 rows of 128 bytes
  LossOut out;
  const int64_t* target;    // of the rows, those that are ignored get zeros; or NULL
  int64_t ignore;
  int rows, cols, add, f16;
  const float* part_bias;   // dW: sums of dl over 32 rows each, which become db here, or NULL
  void* db;
  int groups, db_type;
  static constexpr bool kMeets = false;
  __device__ __forceinline__ void begin() const {}

  struct Row {
    float by;
    bool zero;
  };
  template <class S>
  __device__ __forceinline__ Row before(const GemmEpiTile& e) const {
    const int row = e.m0 + e.lane;
    const float by = out();
    if (part_bias && e.at.nt == 0 && e.at.split == 0 && e.part == 0 && row < rows) {
      double s[4] = {};
      for (int g = 0; g < groups; g += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += g + j < groups ? part_bias[(int64_t)(g + j) * rows + row] : 0.f;
      }
      bias_store(db, db_type, row, (float)((s[0] + s[1]) + (s[2] + s[3])) * by);
    }
    return {by, !kF32 && target && row < rows && !row_counts(target[row], ignore)};
  }
  template <class S, class F>
  __device__ __forceinline__ void tile(const GemmEpiTile& e, const Row& at, F release) const {
    constexpr int kCols = S::kPartCols, kBlock = kF32 ? 32 : 64;
    const int base = e.n0;
    if (e.m0 >= rows || base >= cols) return release();
    const float by = at.by;
    const bool zero = at.zero;
#pragma unroll 1
    for (int c = 0; c < kCols; c += kBlock) {
      if (base + c >= cols) break;
      if (e.lane == 0) tma_store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int h = 0; h < kBlock; h += 32) {
        uint32_t r[32];
        tmem_ld32(e.acc + c + h, r);
        tmem_wait_ld();
        if (h + 32 == kBlock && (c + kBlock == kCols || base + c + kBlock >= cols)) release();
        if constexpr (kF32) {
#pragma unroll
          for (int p = 0; p < 8; ++p)
            *reinterpret_cast<uint4*>(e.stg + e.lane * 128 + ((p ^ (e.lane & 7)) << 4)) = make_uint4(r[4 * p], r[4 * p + 1], r[4 * p + 2], r[4 * p + 3]);
        } else {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = zero ? 0.f : by * __uint_as_float(r[8 * p + j]);
            uint4 o;
            if (f16)
              o = make_uint4(pack_f16x2_inf(v[0], v[1]), pack_f16x2_inf(v[2], v[3]), pack_f16x2_inf(v[4], v[5]), pack_f16x2_inf(v[6], v[7]));
            else
              o = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
            *reinterpret_cast<uint4*>(e.stg + e.lane * 128 + (((h / 8 + p) ^ (e.lane & 7)) << 4)) = o;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (e.lane == 0) {
        if (kF32 && add)
          asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];\n"
                       ::"l"(reinterpret_cast<uint64_t>(&map)), "r"(smem_u32(e.stg)), "r"(base + c), "r"(e.m0), "r"(e.at.split)
                       : "memory");
        else
          tma_store_3d(&map, smem_u32(e.stg), base + c, e.m0, e.at.split);
        tma_store_commit();
      }
    }
  }
};

// The splits' sums in their order, scaled and rounded.
__global__ void __launch_bounds__(256) loss_gather_kernel(const float* __restrict__ slots, uint16_t* __restrict__ to, const LossOut out,
                                                          const int64_t* __restrict__ target, int64_t ignore, int64_t rows, int c, int splits, bool f16) {
  pdl_wait();
  const int64_t all = rows * c / 4;
  const float by = out();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(slots + (int64_t)k * rows * c + 4 * i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    s.x *= by, s.y *= by, s.z *= by, s.w *= by;
    if (target && !row_counts(target[4 * i / c], ignore)) s = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<uint2*>(to)[i] = f16 ? make_uint2(pack_f16x2_inf(s.x, s.y), pack_f16x2_inf(s.z, s.w)) : make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
  }
}

PX_DEFINE_FAMILY_HOOKS(loss)

// ---- host ------------------------------------------------------------------------------------------------------------
static int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Shapes of the products: logits (both operands along k), dx (W across), dW (both across).
// The logits' epilogues: without anything to store (forward) or with blocks of 2 KB (backward).
template <bool kStore>
struct Logits {
  typedef GemmShape<1, 64, false, false, 6, 2, 4, kStore ? 2048 : 0, true> Narrow;
  typedef GemmShape<1, 256, false, false, kStore ? 3 : 4, 2, 8, kStore ? 2048 : 0, true> Single;
  typedef GemmShape<2, 256, false, false, kStore ? 5 : 6, 2, 8, kStore ? 2048 : 0, true> Pair;
};
typedef GemmShape<1, 128, false, true, 5> Dx128;
typedef GemmShape<1, 256, false, true, 4> Dx256;
typedef GemmShape<2, 256, false, true, 5> DxPair;
typedef GemmShape<1, 128, true, true, 5> Dw128;
typedef GemmShape<1, 256, true, true, 4> Dw256;
typedef GemmShape<2, 256, true, true, 5> DwPair;

// Steps of 64 terms that one accumulator of dx or dW takes.  The tensor core cuts it after each 16 terms: a sum of one sign loses 1.0e-7 (fp16) to 1.15e-7 (bf16) of itself
// a cut (dW of 131072 to 453000 rows in one accumulator), so what the cuts take off stays below a quarter of half a step of the result.
static int64_t longest_sum(bool f16) { return f16 ? 256 : 2048; }

// A product's tiles, and the parts that a long axis is cut into: as many as longest_sum() wants (0: not cut), more (of at least four steps each) where that shortens the
// rounds of its tiles, fewer than SMs or a last round with few.
struct HeadCut {
  int ctas, kn;
  GemmTiles t;
  int64_t cycles;
};
static HeadCut cut_for(int ctas, int kn, int64_t m, int64_t n, int64_t k, int64_t longest) {
  HeadCut c = {ctas, kn, {}, 0};
  const int64_t room = sm_count() / ctas;
  c.t.tiles_m = (int)(up(m, 128 * ctas) / (128 * ctas)), c.t.tiles_n = (int)(up(n, kn) / kn);
  c.t.batch = 1, c.t.splits = 1, c.t.group = 8;
  c.t.nk = c.t.nk_split = (int)(up(k, kGemmK) / kGemmK);
  const int64_t tiles = (int64_t)c.t.tiles_m * c.t.tiles_n, step = ctas == 2 ? 600 : 750;
  const int64_t least = longest ? (c.t.nk + longest - 1) / longest : 1, most = longest ? std::min<int64_t>(std::max<int64_t>(room / tiles, 4), c.t.nk / 4) : 1;
  for (int64_t s = least; s <= most || s == least; ++s) {
    const int64_t nk = (c.t.nk + s - 1) / s, parts = (c.t.nk + nk - 1) / nk;
    const int64_t cycles = (tiles * parts + room - 1) / room * (nk * step + 2000) + (parts > 1 ? 4000 + m * n * parts / 400 : 0);
    if (s == least || cycles < c.cycles) c.cycles = cycles, c.t.nk_split = (int)nk, c.t.splits = (int)parts;
  }
  return c;
}
// A pair of CTAs asks L2 for a third less and goes through a step in some 600 cycles, where one alone takes 750 (both measured with all SMs at work): dx of 8192
// rows, 32768 classes and 1024 channels, two rounds of either, 414 us alone.
static HeadCut cut(int64_t m, int64_t n, int64_t k, int64_t longest, int narrow) {
  if (n <= narrow || m <= 128) return cut_for(1, n <= narrow ? narrow : 256, m, n, k, longest);
  const HeadCut one = cut_for(1, 256, m, n, k, longest), two = cut_for(2, 256, m, n, k, longest);
  return two.cycles < one.cycles ? two : one;
}

struct HeadPlan {
  int64_t piece, pieces, ld;               // classes of a piece, row stride of dl
  HeadCut logits, dx, dw;
  bool dx_slots;
  int64_t scale, found, clean, dl, dx_at, dw_at, db_at, bytes;
};
static HeadPlan head_plan(const px_head& h, bool want_dx, bool want_dw, bool want_db) {
  HeadPlan p;
  int64_t most = std::max<int64_t>(256, kPieceBytes / (2 * h.rows) / 256 * 256);
  p.pieces = (h.classes + most - 1) / most;
  p.piece = p.pieces == 1 ? h.classes : up((h.classes + p.pieces - 1) / p.pieces, 256);
  p.pieces = (h.classes + p.piece - 1) / p.piece;
  p.ld = up(p.piece, 8);
  const int64_t longest = longest_sum(h.dtype == PX_F16);
  p.logits = cut(h.rows, p.piece, h.c, 0, 64);
  p.dx = cut(h.rows, h.c, p.piece, longest, 128);
  p.dw = cut(p.piece, h.c, h.rows, longest, 128);
  p.dx_slots = p.dx.t.splits > 1 || p.pieces > 1;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 1024);
    return here;
  };
  p.scale = take(sizeof(LossScale));
  p.found = take(kScanBlocks * 4);
  p.clean = take(want_dw && !want_dx ? h.rows * h.c * 2 : 0);
  p.dl = take(h.rows * p.ld * 2);
  p.dx_at = take(want_dx && p.dx_slots ? p.dx.t.splits * h.rows * h.c * 4 : 0);
  p.dw_at = take(want_dw && p.dw.t.splits > 1 ? p.dw.t.splits * p.piece * h.c * 4 : 0);
  p.db_at = take(want_db ? up(h.rows, 32) / 32 * p.piece * 4 : 0);
  p.bytes = at;
  return p;
}

static int32_t check_head(const px_head* h) {
  if (!h || h->rows < 0 || h->c <= 0 || h->classes <= 0) return PX_ERR_BAD_ARG;
  if (h->rows == 0) return PX_OK;
  if (!h->x || !h->w || !h->target || h->x_stride < h->c || h->w_stride < h->c || h->x_stride % 8 || h->w_stride % 8) return PX_ERR_BAD_ARG;
  if (((uintptr_t)h->x | (uintptr_t)h->w | (uintptr_t)h->bias) & 15) return PX_ERR_BAD_ARG;
  if (!(h->smoothing >= 0.f && h->smoothing <= 1.f)) return PX_ERR_BAD_ARG;
  if (h->bias_dtype != PX_F32 && h->bias_dtype != h->dtype) return PX_ERR_UNSUPPORTED;
  if ((h->dtype != PX_BF16 && h->dtype != PX_F16) || h->c % 8 || h->c > (1 << 20) || h->classes > (1 << 24) || h->rows > (1 << 26)) return PX_ERR_UNSUPPORTED;
  if (up(h->rows, 128) / 128 * (up(h->classes, 64) / 64) > (1ll << 30)) return PX_ERR_UNSUPPORTED;
  return PX_OK;
}
// boxes of 32 rows of 128 bytes of a result
static bool out_map(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, int64_t cols, int64_t rows, int64_t ld, int64_t slots) {
  return make_map_3d(map, type, base, (uint64_t)cols, (uint64_t)rows, (uint64_t)slots, (uint64_t)ld * size, (uint64_t)rows * ld * size, 128 / size, 32,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}
// boxes of 32 x 32 of a result in 16 bits
static bool dl_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t cols, int64_t rows, int64_t ld) {
  return make_map_3d(map, type, base, (uint64_t)cols, (uint64_t)rows, 1, (uint64_t)ld * 2, (uint64_t)rows * ld * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}
static CUtensorMapDataType type16(bool f16) { return f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

// rows of x against `classes` rows of w from class `first` on
template <class Epi>
static int32_t launch_logits(const px_head& h, int64_t first, int64_t classes, const HeadCut& c, const Epi& epi, cudaStream_t st) {
  const bool f16 = h.dtype == PX_F16;
  GemmOperands ops = {};
  if (!gemm_map(&ops.a, f16, h.x, h.c, h.rows, 1, h.x_stride, h.rows * h.x_stride, kGemmM) ||
      !gemm_map(&ops.b, f16, (const uint16_t*)h.w + first * h.w_stride, h.c, classes, 1, h.w_stride, classes * h.w_stride, c.kn / c.ctas))
    return PX_ERR_LAUNCH;
  GemmTiles t = c.t;
  t.tiles_n = (int)(up(classes, c.kn) / c.kn);
  typedef Logits<Epi::kStores> L;
  if (c.kn == 64) return ops.idesc = L::Narrow::idesc(f16), gemm_launch<typename L::Narrow>(ops, epi, t, st);
  if (c.ctas == 1) return ops.idesc = L::Single::idesc(f16), gemm_launch<typename L::Single>(ops, epi, t, st);
  return ops.idesc = L::Pair::idesc(f16), gemm_launch<typename L::Pair>(ops, epi, t, st);
}
template <class N, class W, class P, class Epi>
static int32_t launch_grad(GemmOperands& ops, bool f16, const HeadCut& c, const Epi& epi, const GemmTiles& t, cudaStream_t st) {
  if (c.kn == 128) return ops.idesc = N::idesc(f16), gemm_launch<N>(ops, epi, t, st);
  if (c.ctas == 1) return ops.idesc = W::idesc(f16), gemm_launch<W>(ops, epi, t, st);
  return ops.idesc = P::idesc(f16), gemm_launch<P>(ops, epi, t, st);
}
static int32_t gather(const float* slots, void* to, const LossOut& out, const int64_t* target, int64_t ignore, int64_t rows, int64_t c, int splits, bool f16, cudaStream_t st) {
  const int64_t blocks = std::min<int64_t>((rows * c / 4 + 255) / 256, 8 * sm_count());
  return launch_pdl(loss_gather_kernel, dim3((unsigned)blocks), 256, 0, st, slots, (uint16_t*)to, out, target, ignore, rows, (int)c, splits, f16) ? PX_OK : PX_ERR_LAUNCH;
}

// ---- heads that fit an SM --------------------------------------------------------------------------------------------
static bool small_head(int64_t c, int64_t classes) { return c <= kSmallC && classes <= kSmallV; }
static int64_t small_vp(int64_t classes) { return classes <= 64 ? 64 : 128; }

static bool small_args(SmallArgs* a, const px_head& h) {
  const bool f16 = h.dtype == PX_F16;
  const int vp = (int)small_vp(h.classes);
  *a = {};
  if (!gemm_map(&a->x, f16, h.x, h.c, h.rows, 1, h.x_stride, h.rows * h.x_stride, 128) || !gemm_map(&a->w, f16, h.w, h.c, h.classes, 1, h.w_stride, h.classes * h.w_stride, vp))
    return false;
  a->dx = a->x;
  a->target = h.target, a->bias = {h.bias, h.bias_dtype}, a->ignore = h.ignore, a->rows = (int)h.rows, a->classes = (int)h.classes;
  a->panels = (int)(up(h.c, 64) / 64), a->tiles = (int)(up(h.rows, 128) / 128), a->f16 = f16, a->smooth = h.smoothing, a->uncut = uncut_logits(h.c, h.dtype == PX_F16);
  a->idesc_logits = umma_idesc_16(128, vp, f16, f16);
  a->idesc_dx = umma_idesc_16(128, 64 * a->panels, f16, f16, false, true);
  a->idesc_dw = umma_idesc_16(128, vp, f16, f16, true, true);
  return true;
}
static int small_ctas(int64_t rows) { return even_grid(up(rows, 128) / 128, sm_count()); }
template <bool kBackward, int kVp>
static bool launch_small(const SmallArgs& a, cudaStream_t st) {
  typedef SmallShape<kBackward, kVp> S;
  static SmemLimit limit;
  return limit.set(small_head_kernel<kBackward, kVp>, S::kSmem) && launch_pdl(small_head_kernel<kBackward, kVp>, dim3(small_ctas(a.rows)), S::kThreads, S::kSmem, st, a);
}
template <bool kBackward>
static bool launch_small(const SmallArgs& a, cudaStream_t st) {
  return a.classes <= 64 ? launch_small<kBackward, 64>(a, st) : launch_small<kBackward, 128>(a, st);
}
// The rows of a launch are as many as its CTAs' accumulators of dW take; the launches' sums are joined in their order.
struct SmallPlan {
  int64_t rows, ctas;                      // of a launch; of all launches
  int64_t scale, found, w, b, bytes;
};
static SmallPlan small_plan(const px_head& h) {
  const int64_t vp = small_vp(h.classes), tiles = up(h.rows, 128) / 128, most = sm_count() * longest_sum(h.dtype == PX_F16) / 2, launches = (tiles + most - 1) / most;
  SmallPlan p;
  p.rows = (tiles + launches - 1) / launches * 128, p.ctas = 0;
  for (int64_t row = 0; row < h.rows; row += p.rows) p.ctas += small_ctas(std::min(p.rows, h.rows - row));
  const int64_t ctas = p.ctas;
  p.scale = 0, p.found = 1024, p.w = p.found + up(kScanBlocks * 4, 1024), p.b = p.w + ctas * 128 * vp * 4, p.bytes = p.b + ctas * 8 * vp * 4;
  return p;
}

}  // namespace px

using namespace px;

extern "C" int64_t px_head_loss_workspace_bytes(int64_t rows, int64_t classes) {
  if (rows <= 0 || classes <= 0) return 0;
  const int64_t tiles = up(classes, classes <= 64 ? 64 : 256) / (classes <= 64 ? 64 : 256);
  return 1024 + up(rows * 4, 1024) + up((rows + 31) / 32 * 16, 1024) + up(tiles * rows * 8, 1024) + up(tiles * rows * 4, 1024);
}

extern "C" int32_t px_head_loss_fwd(const px_head* head, float* norm, float* losses, float* total, float* inverse, int32_t mean, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  if (const int32_t status = check_head(head)) return status;
  const px_head& h = *head;
  if (!losses && !total) return PX_ERR_BAD_ARG;
  if (h.rows == 0) return PX_ERR_BAD_ARG;
  if (!norm || (total && !inverse) || !workspace || ((uintptr_t)workspace & 255) || ((uintptr_t)norm & 15)) return PX_ERR_BAD_ARG;
  if (workspace_bytes < px_head_loss_workspace_bytes(h.rows, h.classes)) return PX_ERR_WORKSPACE;
  if (!have_context()) return PX_ERR_LAUNCH;
  const cudaStream_t st = (cudaStream_t)stream;
  if (small_head(h.c, h.classes)) {
    SmallArgs a;
    if (!small_args(&a, h)) return PX_ERR_LAUNCH;
    a.norm = (float2*)norm, a.losses = losses, a.sums = total ? (double2*)workspace : nullptr;
    if (!launch_small<false>(a, st)) return PX_ERR_LAUNCH;
    return !total || launch_pdl(small_total_kernel, dim3(1), 32, 0, st, (const double2*)workspace, small_ctas(h.rows), total, inverse, (int)mean) ? PX_OK : PX_ERR_LAUNCH;
  }
  const HeadCut c = cut(h.rows, h.classes, h.c, 0, 64);
  char* at = (char*)workspace;
  uint32_t* arrivals = (uint32_t*)at;
  at += 1024;
  float* hit = (float*)at;
  at += up(h.rows * 4, 1024);
  double2* sums = (double2*)at;
  at += up((h.rows + 31) / 32 * 16, 1024);
  float2* part = (float2*)at;
  at += up(c.t.tiles_n * h.rows * 8, 1024);
  uint32_t* const dirty = (uint32_t*)(norm + 2 * h.rows);
  EpiStats epi = {h.target, {h.bias, h.bias_dtype}, part, h.smoothing > 0.f ? (float*)at : nullptr, hit, arrivals, dirty, (int)h.rows, (int)h.classes, uncut_logits(h.c, h.dtype == PX_F16)};
  if (const int32_t status = launch_logits(h, 0, h.classes, c, epi, st)) return status;
  JoinArgs j = {part, epi.part_sum, hit, h.target, (float2*)norm, losses, total, inverse, sums, arrivals, dirty, h.ignore, (int)h.rows, (int)h.classes, c.t.tiles_n, mean, h.smoothing};
  return launch_pdl(loss_join_kernel, dim3((unsigned)((h.rows + 31) / 32)), 32 * kJoinWarps, 0, st, j) ? PX_OK : PX_ERR_LAUNCH;
}

extern "C" int64_t px_head_loss_bwd_workspace_bytes(const px_head* head, int32_t dx, int32_t dw, int32_t dbias) {
  if (!head || head->rows <= 0 || head->c <= 0 || head->classes <= 0) return 0;
  return small_head(head->c, head->classes) ? small_plan(*head).bytes : head_plan(*head, dx, dw, dbias).bytes;
}

extern "C" int32_t px_head_loss_bwd(const px_head* head, const float* norm, const float* grad, int32_t each, const float* inverse, void* dx, void* dw,
                                    void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int32_t status = check_head(head)) return status;
  const px_head& h = *head;
  if (h.rows == 0 || !norm || !grad || (!each && !inverse) || !workspace || ((uintptr_t)workspace & 255)) return PX_ERR_BAD_ARG;
  if (((uintptr_t)dx | (uintptr_t)dw | (uintptr_t)norm) & 15) return PX_ERR_BAD_ARG;
  if (workspace_bytes < px_head_loss_bwd_workspace_bytes(head, dx != nullptr, dw != nullptr, dbias != nullptr)) return PX_ERR_WORKSPACE;
  if (!have_context()) return PX_ERR_LAUNCH;
  if (!dx && !dw && !dbias) return PX_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = h.dtype == PX_F16;
  const int64_t bias_size = h.bias_dtype == PX_F32 ? 4 : 2;
  char* const ws = (char*)workspace;
  LossOut out = {nullptr, grad, inverse, f16 ? 1.f / kDlScaleF16 : 1.f};
  const auto scales = [&](int64_t scale_at, int64_t found_at) {
    if (!each) return true;
    LossScale* const scale = (LossScale*)(ws + scale_at);
    uint32_t* const found = (uint32_t*)(ws + found_at);
    const int blocks = (int)std::min<int64_t>((h.rows + 255) / 256, kScanBlocks);
    out.scale = scale;
    return launch_pdl(loss_scan_kernel, dim3(blocks), 256, 0, st, h.target, grad, found, h.ignore, h.rows) &&
           launch_pdl(loss_scale_kernel, dim3(1), 256, 0, st, (const uint32_t*)found, scale, blocks, out.by);
  };
  if (small_head(h.c, h.classes)) {
    const SmallPlan p = small_plan(h);
    const int64_t vp = small_vp(h.classes);
    if (!scales(p.scale, p.found)) return PX_ERR_LAUNCH;
    int64_t slot = 0;
    for (int64_t row = 0; row < h.rows; row += p.rows) {
      px_head part = h;
      part.rows = std::min(p.rows, h.rows - row), part.x = (const uint16_t*)h.x + row * h.x_stride, part.target = h.target + row;
      SmallArgs a;
      if (!small_args(&a, part) || (dx && !out_map(&a.dx, type16(f16), 2, (uint16_t*)dx + row * h.c, h.c, part.rows, h.c, 1))) return PX_ERR_LAUNCH;
      a.norm = (float2*)const_cast<float*>(norm) + row, a.want_dx = dx != nullptr;
      a.part_w = dw ? (float*)(ws + p.w) + slot * 128 * vp : nullptr, a.part_b = dbias ? (float*)(ws + p.b) + slot * 8 * vp : nullptr;
      a.out = out;
      if (each) a.out.grad = grad + row;
      if (!launch_small<true>(a, st)) return PX_ERR_LAUNCH;
      slot += small_ctas(part.rows);
    }
    if (!dw && !dbias) return PX_OK;
    const int groups = (int)vp / 32;
    return launch_pdl(small_join_kernel, dim3((unsigned)(groups * (h.c + 1))), 256, 0, st, dw ? (const float*)(ws + p.w) : nullptr, dbias ? (const float*)(ws + p.b) : nullptr,
                      (uint16_t*)dw, dbias, (int)p.ctas, (int)vp, (int)h.c, (int)h.classes, (int)f16, (int)h.bias_dtype)
               ? PX_OK
               : PX_ERR_LAUNCH;
  }
  const HeadPlan p = head_plan(h, dx, dw, dbias);
  uint16_t* dl = (uint16_t*)(ws + p.dl);
  uint16_t* clean = dx ? (uint16_t*)dx : (uint16_t*)(ws + p.clean);      // dx is written after the last dW that reads them
  float* part_bias = (float*)(ws + p.db_at);
  const uint32_t* const dirty = (const uint32_t*)(norm + 2 * h.rows);
  const int bias_groups = (int)((h.rows + 31) / 32);
  if (!scales(p.scale, p.found)) return PX_ERR_LAUNCH;

  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t first = i * p.piece, vc = std::min(p.piece, h.classes - first);
    EpiLogitGrad el = {};
    if (!dl_map(&el.out, type16(f16), dl, vc, h.rows, p.ld)) return PX_ERR_LAUNCH;
    el.target = h.target, el.bias = {h.bias ? (const char*)h.bias + first * bias_size : nullptr, h.bias_dtype}, el.norm = (const float2*)norm, el.grad = each ? grad : nullptr, el.scale = out.scale;
    if (dw && i == 0) el.x = (const uint16_t*)h.x, el.x_stride = h.x_stride, el.c = (int)h.c, el.clean = clean, el.dirty = dirty;
    el.part_bias = dbias ? part_bias : nullptr, el.ignore = h.ignore, el.rows = (int)h.rows, el.classes = (int)vc, el.first = (int)first;
    el.all_classes = (int)h.classes, el.smooth = h.smoothing, el.uncut = uncut_logits(h.c, h.dtype == PX_F16), el.f16 = f16;
    if (const int32_t status = launch_logits(h, first, vc, p.logits, el, st)) return status;
    void* const db = dbias ? (char*)dbias + first * bias_size : nullptr;
    const bool bias_apart = dbias && (!dw || bias_groups > kBiasGroups);
    if (bias_apart && !launch_pdl(loss_bias_kernel, dim3((unsigned)((vc + 31) / 32)), 512, 0, st, (const float*)part_bias, db, (int)h.bias_dtype, out, (int)vc, bias_groups)) return PX_ERR_LAUNCH;
    if (dw) {
      uint16_t* to = (uint16_t*)dw + first * h.c;
      GemmOperands ops = {};
      if (!gemm_map(&ops.a, f16, dl, vc, h.rows, 1, p.ld, h.rows * p.ld, kGemmK) || !gemm_map(&ops.b, f16, h.x, h.c, h.rows, 1, h.x_stride, h.rows * h.x_stride, kGemmK) ||
          !gemm_map(&ops.b_other, f16, clean, h.c, h.rows, 1, h.c, h.rows * h.c, kGemmK))
        return PX_ERR_LAUNCH;
      ops.other = dirty;
      GemmTiles t = p.dw.t;
      t.tiles_m = (int)(up(vc, 128 * p.dw.ctas) / (128 * p.dw.ctas));
      const auto bias_here = [&](auto& ep) {
        if (dbias && !bias_apart) ep.part_bias = part_bias, ep.db = db, ep.groups = bias_groups, ep.db_type = (int)h.bias_dtype;
      };
      int32_t status;
      if (t.splits > 1) {
        EpiGrad<true> ep = {};
        bias_here(ep);
        if (!out_map(&ep.map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, ws + p.dw_at, h.c, vc, h.c, t.splits)) return PX_ERR_LAUNCH;
        ep.out = out, ep.rows = (int)vc, ep.cols = (int)h.c;
        status = launch_grad<Dw128, Dw256, DwPair>(ops, f16, p.dw, ep, t, st);
        if (!status) status = gather((const float*)(ws + p.dw_at), to, out, nullptr, 0, vc, h.c, t.splits, f16, st);
      } else {
        EpiGrad<false> ep = {};
        bias_here(ep);
        if (!out_map(&ep.map, type16(f16), 2, to, h.c, vc, h.c, 1)) return PX_ERR_LAUNCH;
        ep.out = out, ep.rows = (int)vc, ep.cols = (int)h.c, ep.f16 = f16;
        status = launch_grad<Dw128, Dw256, DwPair>(ops, f16, p.dw, ep, t, st);
      }
      if (status) return status;
    }
    if (dx) {
      GemmOperands ops = {};
      if (!gemm_map(&ops.a, f16, dl, vc, h.rows, 1, p.ld, h.rows * p.ld, kGemmM) ||
          !gemm_map(&ops.b, f16, (const uint16_t*)h.w + first * h.w_stride, h.c, vc, 1, h.w_stride, vc * h.w_stride, kGemmK))
        return PX_ERR_LAUNCH;
      GemmTiles t = p.dx.t;
      t.nk = (int)(up(vc, kGemmK) / kGemmK);
      if (t.splits == 1) t.nk_split = t.nk;
      // a last piece may be too short for all splits: the ones that it has leave the others' sums as they are
      t.splits = (t.nk + t.nk_split - 1) / t.nk_split;
      int32_t status;
      if (p.dx_slots) {
        EpiGrad<true> ep = {};
        if (!out_map(&ep.map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, ws + p.dx_at, h.c, h.rows, h.c, p.dx.t.splits)) return PX_ERR_LAUNCH;
        ep.out = out, ep.rows = (int)h.rows, ep.cols = (int)h.c, ep.add = i > 0;
        status = launch_grad<Dx128, Dx256, DxPair>(ops, f16, p.dx, ep, t, st);
      } else {
        EpiGrad<false> ep = {};
        if (!out_map(&ep.map, type16(f16), 2, dx, h.c, h.rows, h.c, 1)) return PX_ERR_LAUNCH;
        ep.out = out, ep.target = h.target, ep.ignore = h.ignore, ep.rows = (int)h.rows, ep.cols = (int)h.c, ep.f16 = f16;
        status = launch_grad<Dx128, Dx256, DxPair>(ops, f16, p.dx, ep, t, st);
      }
      if (status) return status;
    }
  }
  if (dx && p.dx_slots) return gather((const float*)(ws + p.dx_at), dx, out, h.target, h.ignore, h.rows, h.c, p.dx.t.splits, f16, st);
  return PX_OK;
}
