// Group norm with an activation over the rows of ragged samples, channels last; forward and backward.
//
//   m, v  = mean and variance over (rows of a sample) x (channels of a group),   r = 1 / sqrt(v + eps)
//   h     = (x - m) r,   z = h w + b,   y = act(z)
//   dz    = dy act'(z),  dw = sum dz h,  db = sum dz  (all rows),   q = dz w
//   dx    = r (q - mean(q) - h mean(q h))             (means as above)
//
// Short samples: one launch.  A team of threads -- a warp, a CTA, or a cluster of up to eight CTAs --
// takes a sample: sums, statistics and the apply pass one after the other, the second read out of L1.  The teams keep their
// own sums of the backward pass for dw and db, which a second launch adds up.  Else three launches a direction, chained:
//   1. sums: a CTA takes a block of consecutive rows and adds, channel by channel, the rows of each sample that it meets
//      there.  Forward it keeps mean and squared distance from the mean (not plain squares: a channel whose mean is far
//      from zero keeps its digits), backward dz and dz h.
//   2. join: one group of threads per (sample, channel group) joins the blocks' results in a fixed order;
//      backward also adds the columns up to dw and db.
//   3. apply: the blocks in reverse, so that what the first pass read last is still in L2.
// Results of (block j, sample s) go to slot j + s: walking along the rows either number grows by one from one result to
// the next, so slots are unique, those of a sample are consecutive, and nothing has to be planned ahead.
//
// Measured (B200): 166000 x 256 fp16 with SiLU, one sample, forward + backward 162 us (floor 65: x and y, x, dy and dx once each; with
// the second reads of x and dy 104), 39872 x 512 bf16 of four samples 95 us: sums 13, join 6, apply 19, backward 26, 7 and 27.
// Of the copy rate that is 57 and 77 % in the sums and apply of the first, 48 and 67 to 70 % of the second; a short sample is bound by its
// chain of latencies.
#include <algorithm>

#include "fgb_common.cuh"
#include "fgb_device.cuh"
#include "fgb_rows.cuh"
#include "fgb_umma.cuh"

namespace fgb {

constexpr int kNormThreads = 256;
constexpr int kNormCtas = 3;  // an SM; the backward kernels need some 80 registers a thread

// Two fp32 operations an instruction: these kernels are as near the issue rate as the memory's
struct F2 {
  float x, y;
};

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;             // y, or dx
  RowRanges ranges;
  int C, G, cpg;         // channels, groups, channels per group
  uint32_t R, blocks;    // rows per block
  uint32_t slots;        // backward: rows of `part` that make dw and db
  const void* w;
  const void* b;
  int param_dtype;
  int act;
  float eps;
  float* mean;           // [samples, G]
  float* rstd;
  F2* part;              // [blocks + samples - 1][C]: mean and squared distance from it, or the sums of dz and dz h
  float* joined;         // backward: [samples, G][2] mean(q), mean(q h)
  void* dw;
  void* db;
  int32_t* status;
  int32_t* mirror;
};

__device__ __forceinline__ uint64_t bits(F2 v) { return uint64_t(__float_as_uint(v.y)) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ F2 from_bits(uint64_t b) { return F2{__uint_as_float(static_cast<uint32_t>(b)), __uint_as_float(static_cast<uint32_t>(b >> 32))}; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return from_bits(d);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return from_bits(d);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return from_bits(d);
}
__device__ __forceinline__ F2 both(float v) { return F2{v, v}; }
__device__ __forceinline__ F2 neg2(F2 v) { return F2{-v.x, -v.y}; }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kExact>
__device__ __forceinline__ F2 sigmoid(F2 z) {
  if constexpr (kExact) return F2{1.f / (1.f + expf(-z.x)), 1.f / (1.f + expf(-z.y))};
  // 16-bit results: the fast exponential and reciprocal are exact to some 2^-21, far below the result's half step
  const F2 t = mul2(z, both(-1.44269504f));
  const F2 d = add2(F2{exp2_fast(t.x), exp2_fast(t.y)}, both(1.f));
  return F2{reciprocal_fast(d.x), reciprocal_fast(d.y)};
}
template <bool kExact, bool kSilu>
__device__ __forceinline__ F2 activate(F2 z) {
  if constexpr (!kSilu) return z;
  return mul2(z, sigmoid<kExact>(z));
}
// dy * act'(z).  Every rounding is named: the kernels that call it have to agree on the last bit, so that q - mean(q) is zero
// where a mean is of one value.
template <bool kExact, bool kSilu>
__device__ __forceinline__ F2 activate_grad(F2 dy, F2 z) {
  if constexpr (!kSilu) return dy;
  const F2 s = sigmoid<kExact>(z), y = mul2(z, s);
  return mul2(dy, add2(fma2(neg2(y), s, y), s));  // s + z s (1 - s)
}

// kVec channels as pairs (a single one leaves the second of its pair unused)
template <typename T, int kVec>
struct Pairs {
  static constexpr int kPairs = (kVec + 1) / 2;
  using Ch = Channels<T, kVec>;
  F2 v[kPairs];
  __device__ __forceinline__ void unpack(const typename Ch::Raw& raw) {
    float f[kVec];
    Ch::unpack(raw, f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) v[i] = F2{f[2 * i], kVec > 1 ? f[(2 * i + 1) % kVec] : 0.f};
  }
  __device__ __forceinline__ typename Ch::Raw pack() const {
    float f[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = i % 2 ? v[i / 2].y : v[i / 2].x;
    return Ch::pack(f);
  }
};

// What a thread keeps of its kVec channels: weight and bias, and the statistics of a sample -- one value where the channels
// lie in one group (kOne), which saves the registers of the others
template <int kVec, bool kOne>
struct ChannelParams {
  static constexpr int kPairs = (kVec + 1) / 2, kStats = kOne ? 1 : kPairs;
  F2 w[kPairs], b[kPairs], minus_mean[kStats], r[kStats];
  __device__ __forceinline__ void load(const NormArgs& p, int c0) {
    float fw[2 * kPairs], fb[2 * kPairs];
#pragma unroll
    for (int i = 0; i < 2 * kPairs; ++i) {
      fw[i] = p.w != nullptr && i < kVec ? load_param(p.w, p.param_dtype, c0 + i) : 1.f;
      fb[i] = p.b != nullptr && i < kVec ? load_param(p.b, p.param_dtype, c0 + i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) w[i] = F2{fw[2 * i], fw[2 * i + 1]}, b[i] = F2{fb[2 * i], fb[2 * i + 1]};
  }
  // statistic `of` of the channels' groups: stride values apart
  __device__ __forceinline__ static void gather(F2 (&to)[kStats], const float* of, int stride, const NormArgs& p, uint32_t s, int c0) {
    const float* row = of + size_t(s) * p.G * stride;
#pragma unroll
    for (int i = 0; i < kStats; ++i) {
      const float a = row[size_t((c0 + 2 * i) / p.cpg) * stride];
      to[i] = F2{a, kOne || kVec == 1 ? a : row[size_t((c0 + 2 * i + 1) / p.cpg) * stride]};
    }
  }
  __device__ __forceinline__ void load_stats(const NormArgs& p, uint32_t s, int c0) {
    gather(minus_mean, p.mean, 1, p, s, c0);
#pragma unroll
    for (int i = 0; i < kStats; ++i) minus_mean[i] = neg2(minus_mean[i]);
    gather(r, p.rstd, 1, p, s, c0);
  }
  __device__ __forceinline__ F2 h(F2 x, int i) const { return mul2(add2(x, minus_mean[kOne ? 0 : i]), r[kOne ? 0 : i]); }
  __device__ __forceinline__ F2 z(F2 h, int i) const { return fma2(h, w[i], b[i]); }
};

// Mean and squared distance from it of the rows r, r + lanes, ... below `end` (px: row r), channel by channel; returns their number.
// What cancels in sum d^2 - (sum d)^2 / n grows with n and with the distance of the pivot, from which d is taken, to the mean:
// with the first row as the pivot of all, an outlier there, or zeros in front of a large mean, cost the variance of 50000 rows 4e-3 of
// its value.  So the first row is the pivot of eight rows, and the mean so far, which an outlier among them moves by an eighth, that of
// the next kRunRows, and so on.  The squared distance of the rows before a run waits in shared memory (`park`, a place of the thread's own
// for each pair): 8 registers that the loop of 16-bit packs of eight does not have.
constexpr uint32_t kBatchRows = 8, kRunRows = 64;
template <typename T, int kVec>
__device__ __forceinline__ float moments_of_rows(const T* px, uint32_t r, uint32_t end, uint32_t lanes, size_t step, F2 (&mean)[Pairs<T, kVec>::kPairs],
                                                 F2 (&m2)[Pairs<T, kVec>::kPairs], F2* park) {
  using Ch = Channels<T, kVec>;
  using Raw = typename Ch::Raw;
  using P = Pairs<T, kVec>;
  constexpr int kPairs = P::kPairs;
  if (r >= end) return 0.f;
  uint32_t left = (end - r + lanes - 1u) / lanes;
  float n = 0.f;
  F2 minus_pivot[kPairs];
  {
    P pivot;
    pivot.unpack(Ch::load(px));
#pragma unroll
    for (int i = 0; i < kPairs; ++i) minus_pivot[i] = neg2(pivot.v[i]);
  }
  while (left > 0u) {
    const uint32_t rows = min(left, n == 0.f ? kBatchRows : kRunRows);
    F2 sum0[kPairs], sum1[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum0[i] = sum1[i] = both(0.f);
    auto add = [&](const Raw& raw) {
      P v;
      v.unpack(raw);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const F2 d = add2(v.v[i], minus_pivot[i]);
        sum0[i] = add2(sum0[i], d);
        sum1[i] = fma2(d, d, sum1[i]);
      }
    };
    uint32_t k = 0;
    for (; k + kBatchRows <= rows; k += kBatchRows, px += kBatchRows * step) {
      Raw raw[kBatchRows];
#pragma unroll
      for (uint32_t u = 0; u < kBatchRows; ++u) raw[u] = Ch::load(px + u * step);
#pragma unroll
      for (uint32_t u = 0; u < kBatchRows; ++u) add(raw[u]);
    }
#pragma unroll 4
    for (; k < rows; ++k, px += step) add(Ch::load(px));
    left -= rows;
    // the run's mean lies `d` from the pivot; its squared distance is not below zero (a NaN stays)
    const float count = static_cast<float>(rows), total = n + count, inv = __fdividef(1.f, count), share = n == 0.f ? 1.f : __fdividef(count, total);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const F2 d = mul2(sum0[i], both(inv)), w = fma2(neg2(sum0[i]), d, sum1[i]);
      F2 before = F2{w.x < 0.f ? 0.f : w.x, w.y < 0.f ? 0.f : w.y};
      if (n > 0.f) before = fma2(mul2(d, d), both(n * share), add2(park[i * kNormThreads], before));
      park[i * kNormThreads] = before;
      minus_pivot[i] = fma2(neg2(d), both(share), minus_pivot[i]);
    }
    n = total;
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) mean[i] = neg2(minus_pivot[i]), m2[i] = park[i * kNormThreads];
  return n;
}
// Joins the rows of (mean, m2, n) with those of (mean_b, m2_b, n_b), of which there are none where n_b is zero
__device__ __forceinline__ void join_moments(F2& mean, F2& m2, float n, F2 mean_b, F2 m2_b, float n_b) {
  const float share = __fdividef(n_b, n + n_b);  // exact to two last bits, as good as the products that follow
  const F2 d = add2(mean_b, neg2(mean));
  mean = fma2(d, both(share), mean);
  m2 = fma2(mul2(d, d), both(n * share), add2(m2, m2_b));
}

// ------------------------------------------------------------------ 1. sums
template <typename T, int kVec, bool kOne, bool kBackward, bool kSilu>
__global__ void __launch_bounds__(kNormThreads, kNormCtas) norm_sums_kernel(const NormArgs p) {
  using Ch = Channels<T, kVec>;
  using Raw = typename Ch::Raw;
  using P = Pairs<T, kVec>;
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kPairs = P::kPairs;
  __shared__ F2 s_sum[2 * kPairs][kNormThreads];
  __shared__ float s_rows[kNormThreads];
  chain_release();
  chain_wait();
  if constexpr (!kBackward) p.ranges.check(p.status, p.mirror);
  const uint32_t j = blockIdx.x;
  const int packs = p.C / kVec, pack0 = blockIdx.y * kNormThreads;
  const int width = min(kNormThreads, packs - pack0);  // packs of a row that this CTA takes
  const int lanes = kNormThreads / width;              // rows at a time
  const int cx = threadIdx.x % width, ry = threadIdx.x / width;
  const bool active = ry < lanes;
  const int c0 = (pack0 + cx) * kVec;
  const uint32_t row0 = j * p.R, row1 = min(p.ranges.n, row0 + p.R);
  ChannelParams<kVec, kOne> k;
  if (kBackward && active) k.load(p, c0);
  uint32_t first, last;
  p.ranges.of_block(row0, row0 + p.R, j + 1u >= p.blocks, first, last);
  const T* x = static_cast<const T*>(p.x) + c0;
  const T* dy = static_cast<const T*>(p.dy) + c0;
  for (uint32_t s = first; s <= last; ++s) {
    const uint32_t lo = max(p.ranges.at(s), row0), hi = min(p.ranges.at(s + 1u), row1);
    F2 sum0[kPairs], sum1[kPairs];  // forward: mean and squared distance from it
    float rows = 0.f;               // forward: that they are of
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum0[i] = sum1[i] = both(0.f);
    if (lo < hi && active) {
      const size_t step = size_t(lanes) * p.C;
      if constexpr (!kBackward) {
        rows = moments_of_rows<T, kVec>(x + size_t(lo + ry) * p.C, lo + ry, hi, lanes, step, sum0, sum1, &s_sum[0][threadIdx.x]);
      } else {
        k.load_stats(p, s, c0);
        auto add = [&](const Raw& raw, const Raw& raw_dy) {
          P v, g;
          v.unpack(raw);
          g.unpack(raw_dy);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const F2 h = k.h(v.v[i], i);
            const F2 dz = activate_grad<kExact, kSilu>(g.v[i], k.z(h, i));
            sum0[i] = add2(sum0[i], dz);
            sum1[i] = fma2(dz, h, sum1[i]);
          }
        };
        constexpr int kRows = 4;
        uint32_t r = lo + ry;
        const T* px = x + size_t(r) * p.C;
        const T* pg = dy + size_t(r) * p.C;
        for (; r + (kRows - 1u) * lanes < hi; r += kRows * lanes, px += kRows * step, pg += kRows * step) {
          Raw raw[kRows], raw_dy[kRows];
#pragma unroll
          for (int u = 0; u < kRows; ++u) raw[u] = Ch::load(px + u * step), raw_dy[u] = Ch::load(pg + u * step);
#pragma unroll
          for (int u = 0; u < kRows; ++u) add(raw[u], raw_dy[u]);
        }
        for (; r < hi; r += lanes, px += step, pg += step) add(Ch::load(px), Ch::load(pg));
      }
    }
    // the row lanes' sums: halved until one is left (always in the same order)
    for (int m = lanes; m > 1;) {
      const int half = (m + 1) / 2;
      if (active && ry >= half && ry < m) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) s_sum[i][threadIdx.x] = sum0[i], s_sum[kPairs + i][threadIdx.x] = sum1[i];
        if constexpr (!kBackward) s_rows[threadIdx.x] = rows;
      }
      __syncthreads();
      if (ry < m - half) {
        const int from = threadIdx.x + half * width;
        if constexpr (kBackward) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) sum0[i] = add2(sum0[i], s_sum[i][from]), sum1[i] = add2(sum1[i], s_sum[kPairs + i][from]);
        } else if (s_rows[from] > 0.f) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) join_moments(sum0[i], sum1[i], rows, s_sum[i][from], s_sum[kPairs + i][from], s_rows[from]);
          rows += s_rows[from];
        }
      }
      __syncthreads();
      m = half;
    }
    if (ry == 0) {
      F2* out = p.part + size_t(j + s) * p.C + c0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) out[i] = F2{i % 2 ? sum0[i / 2].y : sum0[i / 2].x, i % 2 ? sum1[i / 2].y : sum1[i / 2].x};
    }
  }
}

// ------------------------------------------------------------------ 2. join
template <int kThreads>
__device__ __forceinline__ void sum_of_threads(double& v0, double& v1, double (*s_red)[2]) {  // once a kernel
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v0 += __shfl_xor_sync(0xffffffffu, v0, d), v1 += __shfl_xor_sync(0xffffffffu, v1, d);
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5][0] = v0, s_red[threadIdx.x >> 5][1] = v1;
    __syncthreads();
    const int w = threadIdx.x & (kThreads / 32 - 1);
    v0 = s_red[w][0], v1 = s_red[w][1];
#pragma unroll
    for (int d = kThreads / 64; d > 0; d >>= 1) v0 += __shfl_xor_sync(0xffffffffu, v0, d), v1 += __shfl_xor_sync(0xffffffffu, v1, d);
  }
}

// Entries k0, k0 + step, ... below `end` of a column of the slots, zeros behind: all on their way at once.  (Whole batches and a
// remainder loop waited for each entry of the remainder, which is mostly all there is.)
constexpr int kJoinLoads = 8;
__device__ __forceinline__ void load_join(F2 (&v)[kJoinLoads], const F2* column, int C, uint32_t k0, uint32_t step, uint32_t end) {
#pragma unroll
  for (int u = 0; u < kJoinLoads; ++u) {
    const uint32_t k = k0 + u * step;
    v[u] = F2{0.f, 0.f};
    if (k < end) v[u] = column[size_t(k) * C];
  }
}

// kThreads threads of the CTA's 256 take one (sample, group); backward: the CTAs from `join_ctas` on add up eight columns each.
// A unit's entries are (block, channel of the group): a thread keeps to one channel and takes every few blocks.
template <int kThreads, bool kBackward>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const NormArgs p, uint32_t join_ctas) {
  __shared__ double s_red[kNormThreads / 32][2];
  __shared__ float s_col[2][32][8];
  chain_release();
  chain_wait();
  if (kBackward && blockIdx.x >= join_ctas) {
    const int c = (blockIdx.x - join_ctas) * 8 + (threadIdx.x & 7), w = threadIdx.x >> 3;
    const uint32_t slots = p.slots;
    float db = 0.f, dw = 0.f;
    if (c < p.C) {
      for (uint32_t k0 = w; k0 < slots; k0 += 32u * kJoinLoads) {
        F2 v[kJoinLoads];
        load_join(v, p.part + c, p.C, k0, 32u, slots);
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) db += v[u].x, dw += v[u].y;
      }
    }
    s_col[0][w][threadIdx.x & 7] = db;
    s_col[1][w][threadIdx.x & 7] = dw;
    __syncthreads();
    const int which = threadIdx.x >> 3;
    if (which < 2 && c < p.C) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) v += s_col[which][i][threadIdx.x & 7];
      if (which == 0 && p.db != nullptr) store_param(p.db, p.param_dtype, c, v);
      if (which == 1 && p.dw != nullptr) store_param(p.dw, p.param_dtype, c, v);
    }
    return;
  }
  const uint32_t unit = blockIdx.x * (kNormThreads / kThreads) + threadIdx.x / kThreads;  // samples * groups < 2^31
  if (unit >= p.ranges.count * static_cast<uint32_t>(p.G)) return;  // whole warps; with 256 threads a unit whole CTAs
  const uint32_t s = unit / p.G, g = unit - s * p.G, t = threadIdx.x % kThreads;
  const uint32_t lo = p.ranges.at(s), hi = max(lo, p.ranges.at(s + 1u));
  const uint32_t j0 = lo / p.R, blocks = lo < hi ? (hi - 1u) / p.R - j0 + 1u : 0u;
  const uint32_t cpg = p.cpg, across = min(cpg, static_cast<uint32_t>(kThreads)), down = kThreads / across;
  const uint32_t c_own = t % across, k_own = t / across;
  const double inv_count = 1.0 / (static_cast<double>(hi - lo) * cpg);  // unused where there are no rows
  const F2* part = p.part + size_t(j0 + s) * p.C + g * cpg;
  double v0 = 0, v1 = 0;
  if constexpr (!kBackward) {
    // with d = (a block's mean) - (the first block's): mean = first + sum n d / count, and the squared distances from it are
    // those within the blocks + sum n d^2 - (sum n d)^2 / count, all in 64 bits
    const double pivot = blocks > 0u ? part[0].x : 0.f;
    if (k_own < down) {
      for (uint32_t c = c_own; c < cpg; c += across) {
        for (uint32_t k0 = k_own; k0 < blocks; k0 += down * kJoinLoads) {
          F2 v[kJoinLoads];
          load_join(v, part + c, p.C, k0, down, blocks);
#pragma unroll
          for (int u = 0; u < kJoinLoads; ++u) {
            const uint32_t k = k0 + u * down;
            if (k >= blocks) break;
            const double rows = static_cast<double>(min(hi, (j0 + k + 1u) * p.R) - max(lo, (j0 + k) * p.R)), d = v[u].x - pivot;
            v0 += rows * d;
            v1 += v[u].y + rows * d * d;
          }
        }
      }
    }
    double mean = 0, var = 0;
    if (blocks > 0u) {
      sum_of_threads<kThreads>(v0, v1, s_red);
      v0 *= inv_count, v1 *= inv_count;
      mean = pivot + v0, var = v1 - v0 * v0;
      if (var < 0) var = 0;
    }
    if (t == 0) {
      p.mean[unit] = static_cast<float>(mean);
      p.rstd[unit] = static_cast<float>(rsqrt(var + static_cast<double>(p.eps)));
    }
  } else {
    if (k_own < down) {
      for (uint32_t c = c_own; c < cpg; c += across) {
        const double w = p.w != nullptr ? load_param(p.w, p.param_dtype, g * cpg + c) : 1.f;
        double q0 = 0, q1 = 0;
        for (uint32_t k0 = k_own; k0 < blocks; k0 += down * kJoinLoads) {
          F2 v[kJoinLoads];
          load_join(v, part + c, p.C, k0, down, blocks);
#pragma unroll
          for (int u = 0; u < kJoinLoads; ++u) q0 += v[u].x, q1 += v[u].y;
        }
        v0 += w * q0;
        v1 += w * q1;
      }
    }
    if (blocks > 0u) {
      sum_of_threads<kThreads>(v0, v1, s_red);
      v0 *= inv_count, v1 *= inv_count;
    }
    if (t == 0) {
      p.joined[size_t(unit) * 2] = static_cast<float>(v0);
      p.joined[size_t(unit) * 2 + 1] = static_cast<float>(v1);
    }
  }
}

// ------------------------------------------------------------------ 3. apply
template <typename T, int kVec, bool kOne, bool kBackward, bool kSilu>
__global__ void __launch_bounds__(kNormThreads, kNormCtas) norm_apply_kernel(const NormArgs p) {
  using Ch = Channels<T, kVec>;
  using Raw = typename Ch::Raw;
  using P = Pairs<T, kVec>;
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kPairs = P::kPairs;
  chain_release();
  chain_wait();
  const uint32_t j = p.blocks - 1u - blockIdx.x;
  const int packs = p.C / kVec, pack0 = blockIdx.y * kNormThreads;
  const int width = min(kNormThreads, packs - pack0), lanes = kNormThreads / width;
  const int cx = threadIdx.x % width, ry = threadIdx.x / width;
  const int c0 = (pack0 + cx) * kVec;
  const uint32_t row0 = j * p.R, row1 = min(p.ranges.n, row0 + p.R);
  ChannelParams<kVec, kOne> k;
  if (ry < lanes) k.load(p, c0);
  uint32_t first, last;
  p.ranges.of_block(row0, row0 + p.R, j + 1u >= p.blocks, first, last);  // whole warps take part
  if (ry >= lanes) return;
  const T* x = static_cast<const T*>(p.x) + c0;
  const T* dy = static_cast<const T*>(p.dy) + c0;
  T* out = static_cast<T*>(p.out) + c0;
  const size_t step = size_t(lanes) * p.C;
  for (uint32_t s = first; s <= last; ++s) {
    const uint32_t lo = max(p.ranges.at(s), row0), hi = min(p.ranges.at(s + 1u), row1);
    if (lo >= hi) continue;
    k.load_stats(p, s, c0);
    uint32_t r = lo + ry;
    size_t at = size_t(r) * p.C;
    constexpr int kRows = 4;
    if constexpr (!kBackward) {
      auto one = [&](const Raw& raw) {
        P v;
        v.unpack(raw);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v.v[i] = activate<kExact, kSilu>(k.z(k.h(v.v[i], i), i));
        return v.pack();
      };
      for (; r + (kRows - 1u) * lanes < hi; r += kRows * lanes, at += kRows * step) {
        Raw raw[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) raw[u] = Ch::load(x + at + u * step);
#pragma unroll
        for (int u = 0; u < kRows; ++u) Ch::store(out + at + u * step, one(raw[u]));
      }
      for (; r < hi; r += lanes, at += step) Ch::store(out + at, one(Ch::load(x + at)));
    } else {
      constexpr int kStats = ChannelParams<kVec, kOne>::kStats;
      F2 minus_m1[kStats], m2[kStats];
      ChannelParams<kVec, kOne>::gather(minus_m1, p.joined, 2, p, s, c0);
      ChannelParams<kVec, kOne>::gather(m2, p.joined + 1, 2, p, s, c0);
#pragma unroll
      for (int i = 0; i < kStats; ++i) minus_m1[i] = neg2(minus_m1[i]);
      auto one = [&](const Raw& raw, const Raw& raw_dy) {
        P v, g;
        v.unpack(raw);
        g.unpack(raw_dy);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const F2 h = k.h(v.v[i], i), dz = activate_grad<kExact, kSilu>(g.v[i], k.z(h, i));
          // not mul2: the compiler joins that with the subtraction of the mean to one operation with one rounding
          const F2 q = F2{__fmul_rn(dz.x, k.w[i].x), __fmul_rn(dz.y, k.w[i].y)};
          const int t = kOne ? 0 : i;
          v.v[i] = mul2(k.r[t], fma2(neg2(h), m2[t], add2(q, minus_m1[t])));
        }
        return v.pack();
      };
      for (; r + (kRows - 1u) * lanes < hi; r += kRows * lanes, at += kRows * step) {
        Raw raw[kRows], raw_dy[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) raw[u] = Ch::load(x + at + u * step), raw_dy[u] = Ch::load(dy + at + u * step);
#pragma unroll
        for (int u = 0; u < kRows; ++u) Ch::store(out + at + u * step, one(raw[u], raw_dy[u]));
      }
      for (; r < hi; r += lanes, at += step) Ch::store(out + at, one(Ch::load(x + at), Ch::load(dy + at)));
    }
  }
  // rows of no sample
  const uint32_t begin = p.ranges.at(0u), end = max(begin, p.ranges.at(p.ranges.count));
  if (row0 >= begin && row1 <= end) return;
  Raw zero{};
  for (uint32_t r = row0 + ry; r < row1; r += lanes)
    if (r < begin || r >= end) Ch::store(out + size_t(r) * p.C, zero);
}

// ------------------------------------------------------------------ short samples
// Ragged samples may be long ones in between, and a team would be at one long after all others are done.  Teams leave samples of
// more than long_rows rows out, and a second launch (kLong) takes them in clusters of kLongCtas CTAs; neighbours, which are often
// alike, go to different clusters.  us, in one launch / in two (bf16, 96 channels): 2000 samples of 7 rows around one of 50000, forward
// 2591 / 132, forward and backward 9965 / 378; 2000 samples of 20 rows 14.5 / 16.9 and 28.2 / 31.5.  Lengths that scatter like exp(N(0, 1)) (80000
// rows of fp32 in 2048 samples, forward + backward): 110 to 162 / 128.
constexpr int kLongCtas = 8, kLongClusters = 18;
struct SmallArgs {
  int team;            // threads of a CTA that take a sample: 32, 64, 128 or 256
  int cluster;         // CTAs that do (1 where a CTA has several teams)
  uint32_t teams;      // samples at a time; team t takes the samples t, t + teams, ...
  uint32_t long_rows;  // see above
  F2* columns;         // backward: [CTAs, or clusters][C] sums of dz and dz h
};

template <typename T, int kVec, bool kOne, bool kBackward, bool kSilu, bool kLong>
__global__ void __launch_bounds__(kNormThreads, kNormCtas) norm_small_kernel(const NormArgs p, const SmallArgs q) {
  using Ch = Channels<T, kVec>;
  using Raw = typename Ch::Raw;
  using P = Pairs<T, kVec>;
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kPairs = P::kPairs;
  extern __shared__ F2 s_mem[];  // of each team: sums [C] (forward: mean and squared distance from it), statistics [G], backward: columns [C]
  __shared__ F2 s_sum[2 * kPairs][kNormThreads];
  __shared__ float s_rows[kNormThreads];
  chain_release();
  chain_wait();
  p.ranges.check(p.status, p.mirror);
  const int size = q.team, t = threadIdx.x % size, here = threadIdx.x / size, teams_here = kNormThreads / size;
  const uint32_t rank = q.cluster > 1 ? cluster_ctarank() : 0u;
  const uint32_t team = q.cluster > 1 ? blockIdx.x / q.cluster : blockIdx.x * teams_here + here;
  F2* sums = s_mem + size_t(here) * ((kBackward ? 2 : 1) * p.C + p.G);
  F2* stats = sums + p.C;
  F2* columns = stats + p.G;
  auto sync = [&]() {
    if (size == 32) __syncwarp();
    else if (size == kNormThreads) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(here + 1), "r"(size) : "memory");  // a barrier of the team's own
  };
  const int packs = p.C / kVec;
  const double inv_cpg = 1.0 / p.cpg;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* out = static_cast<T*>(p.out);
  if constexpr (kBackward) {
    for (int c = t; c < p.C; c += size) columns[c] = both(0.f);
    sync();
  }
  auto sample = [&](uint32_t s, uint32_t lo, uint32_t hi) {
    const uint32_t len = hi - lo;
    const uint32_t share = (len + q.cluster - 1u) / q.cluster, from = min(hi, lo + rank * share), to = min(hi, from + share);
    // 1. sums of this CTA's rows, for each channel
    for (int pack0 = 0; pack0 < packs; pack0 += size) {
      const int width = min(size, packs - pack0), lanes = size / width;
      const int cx = t % width, ry = t / width, c0 = (pack0 + cx) * kVec;
      F2 sum0[kPairs], sum1[kPairs];
      float rows = 0.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sum0[i] = sum1[i] = both(0.f);
      if (ry < lanes && from < to) {
        const size_t step = size_t(lanes) * p.C;
        uint32_t r = from + ry;
        const T* px = x + size_t(r) * p.C + c0;
        if constexpr (!kBackward) {
          rows = moments_of_rows<T, kVec>(px, r, to, lanes, step, sum0, sum1, &s_sum[0][threadIdx.x]);
        } else {
          ChannelParams<kVec, kOne> k;
          k.load(p, c0);
          k.load_stats(p, s, c0);
          const T* pg = dy + size_t(r) * p.C + c0;
          auto add = [&](const Raw& raw, const Raw& raw_dy) {
            P v, g;
            v.unpack(raw);
            g.unpack(raw_dy);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const F2 h = k.h(v.v[i], i);
              const F2 dz = activate_grad<kExact, kSilu>(g.v[i], k.z(h, i));
              sum0[i] = add2(sum0[i], dz);
              sum1[i] = fma2(dz, h, sum1[i]);
            }
          };
          constexpr int kRows = 4;
          for (; r + (kRows - 1u) * lanes < to; r += kRows * lanes, px += kRows * step, pg += kRows * step) {
            Raw raw[kRows], raw_dy[kRows];
#pragma unroll
            for (int u = 0; u < kRows; ++u) raw[u] = Ch::load(px + u * step), raw_dy[u] = Ch::load(pg + u * step);
#pragma unroll
            for (int u = 0; u < kRows; ++u) add(raw[u], raw_dy[u]);
          }
#pragma unroll 2
          for (; r < to; r += lanes, px += step, pg += step) add(Ch::load(px), Ch::load(pg));
        }
      }
      for (int m = lanes; m > 1;) {
        const int half = (m + 1) / 2;
        if (ry >= half && ry < m) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) s_sum[i][threadIdx.x] = sum0[i], s_sum[kPairs + i][threadIdx.x] = sum1[i];
          if constexpr (!kBackward) s_rows[threadIdx.x] = rows;
        }
        sync();
        if (ry < m - half) {
          const int at = threadIdx.x + half * width;
          if constexpr (kBackward) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sum0[i] = add2(sum0[i], s_sum[i][at]), sum1[i] = add2(sum1[i], s_sum[kPairs + i][at]);
          } else if (s_rows[at] > 0.f) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) join_moments(sum0[i], sum1[i], rows, s_sum[i][at], s_sum[kPairs + i][at], s_rows[at]);
            rows += s_rows[at];
          }
        }
        sync();
        m = half;
      }
      if (ry == 0) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          sums[c0 + i] = F2{i % 2 ? sum0[i / 2].y : sum0[i / 2].x, i % 2 ? sum1[i / 2].y : sum1[i / 2].x};
      }
    }
    sync();
    if (q.cluster > 1) cluster_sync_all();
    // 2. the groups: a thread adds up a group, over the channels and the CTAs
    auto sum_of = [&](int c, int i) {  // CTA i's
      if (q.cluster == 1) return sums[c];
      F2 v;
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_map(smem_u32(&sums[c]), i)) : "memory");
      return v;
    };
    // lanes that share a group: as many as it has channels, up to a warp's
    int across = 1;
    while (across < 32 && across < p.cpg) across *= 2;
    for (int g0 = t / across; g0 < (p.G + size / across - 1) / (size / across) * (size / across); g0 += size / across) {  // whole warps
      const bool has = g0 < p.G && len > 0u;
      const int g = min(g0, p.G - 1);
      double v0 = 0, v1 = 0;
      if constexpr (!kBackward) {
        // as the joins of the longer way: the first channel's mean is the pivot of the means of channels and CTAs
        const double inv_n = inv_cpg / len;
        const double pivot = has ? sum_of(g * p.cpg, 0).x : 0.f;
        for (int i = t % across; i < p.cpg && has; i += across) {
#pragma unroll 4
          for (int k = 0; k < q.cluster; ++k) {  // all on their way at once: a CTA without rows has zeros
            const uint32_t begin = min(len, k * share), rows = min(len, begin + share) - begin;
            const F2 v = sum_of(g * p.cpg + i, k);
            const double d = v.x - pivot;
            v0 += rows * d;
            v1 += v.y + rows * d * d;
          }
        }
        for (int d = across / 2; d > 0; d >>= 1) v0 += __shfl_xor_sync(0xffffffffu, v0, d), v1 += __shfl_xor_sync(0xffffffffu, v1, d);
        v0 *= inv_n, v1 *= inv_n;
        const double var = v1 - v0 * v0 < 0 || !has ? 0.0 : v1 - v0 * v0;
        if (t % across == 0 && g0 < p.G) {
          const F2 st{has ? static_cast<float>(pivot + v0) : 0.f, 1.f / sqrtf(static_cast<float>(var + static_cast<double>(p.eps)))};
          stats[g] = st;
          if (rank == 0u) p.mean[size_t(s) * p.G + g] = st.x, p.rstd[size_t(s) * p.G + g] = st.y;
        }
      } else {
        for (int i = t % across; i < p.cpg && has; i += across) {
          const int c = g * p.cpg + i;
          F2 v = sum_of(c, 0);
          for (int k = 1; k < q.cluster; ++k) v = add2(v, sum_of(c, k));
          const double w = p.w != nullptr ? load_param(p.w, p.param_dtype, c) : 1.f;
          v0 += w * v.x;
          v1 += w * v.y;
          if (rank == 0u) columns[c] = add2(columns[c], v);
        }
        for (int d = across / 2; d > 0; d >>= 1) v0 += __shfl_xor_sync(0xffffffffu, v0, d), v1 += __shfl_xor_sync(0xffffffffu, v1, d);
        const double inv_n = inv_cpg / len;
        if (t % across == 0 && g0 < p.G) stats[g] = F2{static_cast<float>(v0 * inv_n), static_cast<float>(v1 * inv_n)};
      }
    }
    sync();
    if (q.cluster > 1) cluster_sync_all();  // the other CTAs have read this one's sums
    // 3. apply
    if (from < to && out != nullptr) {
      for (int pack0 = 0; pack0 < packs; pack0 += size) {
        const int width = min(size, packs - pack0), lanes = size / width;
        const int cx = t % width, ry = t / width, c0 = (pack0 + cx) * kVec;
        if (ry >= lanes) continue;
        constexpr int kStats = ChannelParams<kVec, kOne>::kStats;
        ChannelParams<kVec, kOne> k;
        k.load(p, c0);
        auto group_of = [&](int c) { return stats[(c0 + c) / p.cpg]; };
        F2 minus_m1[kStats], m2[kStats];
        if constexpr (kBackward) {
          k.load_stats(p, s, c0);
#pragma unroll
          for (int i = 0; i < kStats; ++i) {
            const F2 a = group_of(2 * i), b = kOne || kVec == 1 ? a : group_of(2 * i + 1);
            minus_m1[i] = F2{-a.x, -b.x}, m2[i] = F2{a.y, b.y};
          }
        } else {
#pragma unroll
          for (int i = 0; i < kStats; ++i) {
            const F2 a = group_of(2 * i), b = kOne || kVec == 1 ? a : group_of(2 * i + 1);
            k.minus_mean[i] = F2{-a.x, -b.x}, k.r[i] = F2{a.y, b.y};
          }
        }
        auto one = [&](const Raw& raw, const Raw& raw_dy) {
          P v;
          v.unpack(raw);
          if constexpr (!kBackward) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v.v[i] = activate<kExact, kSilu>(k.z(k.h(v.v[i], i), i));
          } else {
            P g;
            g.unpack(raw_dy);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const F2 h = k.h(v.v[i], i), dz = activate_grad<kExact, kSilu>(g.v[i], k.z(h, i));
              const F2 w = F2{__fmul_rn(dz.x, k.w[i].x), __fmul_rn(dz.y, k.w[i].y)};  // as in norm_apply_kernel
              const int j = kOne ? 0 : i;
              v.v[i] = mul2(k.r[j], fma2(neg2(h), m2[j], add2(w, minus_m1[j])));
            }
          }
          return v.pack();
        };
        const size_t step = size_t(lanes) * p.C;
        uint32_t r = from + ry;
        size_t at = size_t(r) * p.C + c0;
        constexpr int kRows = 4;
        for (; r + (kRows - 1u) * lanes < to; r += kRows * lanes, at += kRows * step) {
          Raw raw[kRows], raw_dy[kRows];
#pragma unroll
          for (int u = 0; u < kRows; ++u) {
            raw[u] = Ch::load(x + at + u * step);
            if (kBackward) raw_dy[u] = Ch::load(dy + at + u * step);
          }
#pragma unroll
          for (int u = 0; u < kRows; ++u) Ch::store(out + at + u * step, one(raw[u], raw_dy[u]));
        }
        for (; r < to; r += lanes, at += step) {
          const Raw raw = Ch::load(x + at);
          Ch::store(out + at, one(raw, kBackward ? Ch::load(dy + at) : raw));
        }
      }
    }
    sync();  // sums and statistics are written again
  };
  if constexpr (!kLong) {
    for (uint32_t s = team; s < p.ranges.count; s += q.teams) {
      const uint32_t lo = p.ranges.at(s), hi = max(lo, p.ranges.at(s + 1u));
      if (hi - lo <= q.long_rows) sample(s, lo, hi);
    }
  } else {
    // 256 of the cluster's samples are looked at at a time; all its CTAs find the same
    __shared__ uint32_t s_long[kNormThreads / 32];
    for (uint64_t s0 = team; s0 < p.ranges.count; s0 += uint64_t(kNormThreads) * q.teams) {
      const uint64_t k = s0 + uint64_t(threadIdx.x) * q.teams;
      bool is_long = false;
      if (k < p.ranges.count) {
        const uint32_t lo = p.ranges.at(static_cast<uint32_t>(k)), hi = p.ranges.at(static_cast<uint32_t>(k) + 1u);
        is_long = hi > lo && hi - lo > q.long_rows;
      }
      const uint32_t found = __ballot_sync(0xffffffffu, is_long);
      if ((threadIdx.x & 31u) == 0u) s_long[threadIdx.x / 32u] = found;
      __syncthreads();
      for (uint32_t word = 0; word < kNormThreads / 32; ++word)
        for (uint32_t left = s_long[word]; left != 0u; left &= left - 1u) {
          const uint32_t s = static_cast<uint32_t>(s0) + (word * 32u + __ffs(left) - 1u) * q.teams, lo = p.ranges.at(s);
          sample(s, lo, max(lo, p.ranges.at(s + 1u)));
        }
      __syncthreads();
    }
  }
  if constexpr (kBackward) {
    __syncthreads();
    if (rank == 0u && q.columns != nullptr) {
      // the CTA's teams in order
      F2* to = q.columns + size_t(blockIdx.x / q.cluster) * p.C;
      for (int c = threadIdx.x; c < p.C; c += kNormThreads) {
        F2 v = both(0.f);
        for (int i = 0; i < teams_here; ++i) v = add2(v, s_mem[size_t(i) * (2 * p.C + p.G) + p.C + p.G + c]);
        to[c] = v;
      }
    }
  }
  // rows of no sample
  if (!kLong && out != nullptr) {
    const uint32_t begin = p.ranges.at(0u), end = max(begin, p.ranges.at(p.ranges.count)), outside = begin + (p.ranges.n - end);
    Raw zero{};
    for (uint64_t i = uint64_t(blockIdx.x) * kNormThreads + threadIdx.x; i < uint64_t(outside) * packs; i += uint64_t(gridDim.x) * kNormThreads) {
      const uint32_t r = static_cast<uint32_t>(i / packs), row = r < begin ? r : r - begin + end;
      Ch::store(out + size_t(row) * p.C + (i - uint64_t(r) * packs) * kVec, zero);
    }
  }
}

// ------------------------------------------------------------------ host side
// A sample on average up to this size goes the short way (all passes in one launch).  Forward it is what eight CTAs hold in L1
// between the passes, with half of it to spare; backward there are two tensors to keep, and dw and db cost a launch anyway.
// us, short / long way (bf16): forward 16 samples of 2048 x 128 (512 KB): 16.2 / 21.2, 64 of 4096 x 128: 58.0 / 57.1; backward 2000
// of 30 x 256 (15 KB): 64 / 81, 64 of 300 x 128 (77 KB): 24.5 / 25.9, 300 of 256 x 256 (131 KB): 74 / 58, 16 of 2048 x 128: 30 / 22.
constexpr int64_t kSmallForward = 512 * 1024, kSmallBackward = 48 * 1024;
constexpr int kSmallChannels = 2048;

struct NormPlan {
  bool small;         // the short way:
  int team, cluster;  // threads of a CTA, and CTAs, for a sample
  unsigned grid;
  uint32_t long_rows;
  int long_clusters;  // of the second launch; 0: there is none
  size_t small_smem, long_smem;
  int vec;
  bool one;           // a pack lies in one group
  unsigned columns;   // CTAs along a row
  uint32_t R, blocks;
  size_t joined_off, bytes;
};
static NormPlan norm_plan(const fgb_group_norm_call& c) {
  NormPlan p;
  const bool backward = c.grad_out != nullptr || c.grad_weight != nullptr || c.grad_bias != nullptr;  // without rows there is no grad_out
  p.vec = row_pack(c.c, elem_bytes(c.dtype));
  if (p.vec == 8 && c.c / c.groups % 8 != 0) p.vec = 4;  // eight channels of several groups would take too many registers
  p.one = c.c / c.groups % p.vec == 0;
  const int packs = c.c / p.vec;
  const int64_t sms = device_sm_count(), mean_rows = c.n / c.samples, mean_bytes = mean_rows * c.c * elem_bytes(c.dtype);
  p.small = mean_bytes <= (backward ? kSmallBackward : kSmallForward) && c.c <= kSmallChannels;
  // Eight packs a thread: that many loads are on their way at a time, and a sample's chain of steps takes the same few
  // microseconds however many threads go through it, so small teams are more samples at a time.
  p.team = 32;
  auto team_smem = [&](int team) { return (kNormThreads / team) * (2 * size_t(c.c) + c.groups) * 8; };
  while (p.team < kNormThreads && (mean_rows * packs > 8 * p.team || team_smem(p.team) > 48 * 1024 || p.team * c.samples * 2 <= 32 * sms)) p.team *= 2;
  p.cluster = 1;
  // Clusters where samples are fewer than SMs, or for more than 64 KB a CTA.  A cluster's barriers cost more than its threads save
  // where there are samples for all SMs: 600 samples of 100 x 256 took 98 us in clusters of 16 KB a CTA, 31 in single CTAs.
  while (p.small && p.team == kNormThreads && p.cluster < 8 && (int64_t(p.cluster) * 65536 < mean_bytes || p.cluster * c.samples * 2 <= sms)) p.cluster *= 2;
  if (p.cluster > 1 && mean_bytes / p.cluster < 2048) p.cluster = 1;
  const int64_t ctas = ceil_div(c.samples, kNormThreads / p.team);
  p.grid = static_cast<unsigned>(std::min<int64_t>(ctas, std::max<int64_t>(sms * kNormCtas / p.cluster, 1)) * p.cluster);
  p.small_smem = team_smem(p.team), p.long_smem = team_smem(kNormThreads);
  // 128 packs a thread, some 10 us of a team
  p.long_rows = p.cluster == 1 && c.offsets_bits != 0 ? static_cast<uint32_t>(128 * p.team / packs) : 0xFFFFFFFFu;
  p.long_clusters = p.small && p.long_rows < c.n ? static_cast<int>(std::min<int64_t>(kLongClusters, c.samples)) : 0;
  p.columns = static_cast<unsigned>(ceil_div(packs, kNormThreads));
  const int width = packs < kNormThreads ? packs : kNormThreads, lanes = kNormThreads / width;
  // as many CTAs as run at a time, each thread at least eight rows
  const int64_t want = std::max<int64_t>(int64_t(device_sm_count()) * kNormCtas / p.columns, 1);
  const int64_t R = std::max<int64_t>(ceil_div(c.n, want), int64_t(lanes) * 8);
  p.R = static_cast<uint32_t>(R);
  p.blocks = static_cast<uint32_t>(std::max<int64_t>(ceil_div(c.n, R), 1));
  p.joined_off = p.small ? align256((int64_t(p.grid / p.cluster) + p.long_clusters) * c.c * 8) : align256((int64_t(p.blocks) + c.samples - 1) * 2 * c.c * 4);
  // one launch forward needs nothing between its passes
  p.bytes = p.small ? (backward ? p.joined_off : 0) : p.joined_off + align256(c.samples * c.groups * 8);
  return p;
}

static int norm_check(const fgb_group_norm_call* c) {
  if (c == nullptr) return FGB_E_NULL;
  if (c->dtype != FGB_F16 && c->dtype != FGB_BF16 && c->dtype != FGB_F32_TF32 && c->dtype != FGB_F32_IEEE) return FGB_E_DTYPE;
  if (c->param_dtype != c->dtype && c->param_dtype != FGB_F32_IEEE && c->param_dtype != FGB_F32_TF32) return FGB_E_DTYPE;
  if (c->act != FGB_ACT_NONE && c->act != FGB_ACT_SILU) return FGB_E_DTYPE;
  if (c->offsets_bits != 0 && c->offsets_bits != 32 && c->offsets_bits != 64) return FGB_E_DTYPE;
  if (c->n < 0 || c->n >= (int64_t(1) << 31) || c->samples < 1 || c->samples >= (int64_t(1) << 24)) return FGB_E_SIZE;
  if (c->c < 1 || c->c > 65536 || c->groups < 1 || c->c % c->groups != 0 || c->samples * c->groups >= (int64_t(1) << 31)) return FGB_E_SIZE;
  if (c->offsets_bits == 0 && c->n % c->samples != 0) return FGB_E_SIZE;
  return FGB_OK;
}

template <typename T, int kVec, bool kOne, bool kSilu>
static int norm_run_act(const NormArgs& a, const NormPlan& p, bool backward, bool want_out, bool want_param, cudaStream_t s) {
  const dim3 grid(p.blocks, p.columns);
  LaunchErrors chain;
  if (p.small) {
    const uint32_t slots = p.grid / p.cluster;
    const SmallArgs q{p.team, p.cluster, slots * (kNormThreads / p.team), p.long_rows, want_param ? a.part : nullptr};
    auto kernel = backward ? norm_small_kernel<T, kVec, kOne, true, kSilu, false> : norm_small_kernel<T, kVec, kOne, false, kSilu, false>;
    static PerDeviceTable configured[2], configured_long[2];
    int rc = ensure_dynamic_smem(configured[backward], kernel, p.small_smem);
    if (rc != FGB_OK) return rc;
    chain.add(launch_chained_clusters(kernel, dim3(p.grid), dim3(kNormThreads), p.small_smem, p.cluster, s, a, q));
    if (p.long_clusters > 0) {
      const unsigned clusters = static_cast<unsigned>(p.long_clusters);
      const SmallArgs l{kNormThreads, kLongCtas, clusters, p.long_rows, want_param ? a.part + size_t(slots) * a.C : nullptr};
      auto rest = backward ? norm_small_kernel<T, kVec, kOne, true, kSilu, true> : norm_small_kernel<T, kVec, kOne, false, kSilu, true>;
      rc = ensure_dynamic_smem(configured_long[backward], rest, p.long_smem);
      if (rc != FGB_OK) return rc;
      chain.add(launch_chained_clusters(rest, dim3(clusters * kLongCtas), dim3(kNormThreads), p.long_smem, kLongCtas, s, a, l));
    }
    if (want_param) {
      NormArgs cols = a;
      cols.slots = slots + static_cast<uint32_t>(p.long_clusters);
      chain.add(launch_chained(norm_join_kernel<32, true>, dim3(static_cast<unsigned>(ceil_div(a.C, 8))), dim3(kNormThreads), 0, s, cols, 0u));
    }
    return chain.first != cudaSuccess ? cuda_status(chain.first) : launch_status();
  }
  const int64_t units = int64_t(a.ranges.count) * a.G;
  // A CTA a (sample, group) where the samples cover many blocks, a warp where they are short: 166000 x 256 of 2 samples, forward,
  // 62 us by CTAs, 81 by warps; of 128 samples 73 and 66.
  const bool warps = int64_t(p.blocks) * a.cpg / a.ranges.count < 64;
  const uint32_t join = static_cast<uint32_t>(warps ? ceil_div(units, kNormThreads / 32) : units);
  if (!backward) {
    chain.add(launch_chained(norm_sums_kernel<T, kVec, kOne, false, false>, grid, dim3(kNormThreads), 0, s, a));
    chain.add(launch_chained(warps ? norm_join_kernel<32, false> : norm_join_kernel<kNormThreads, false>, dim3(join), dim3(kNormThreads), 0, s, a, join));
    chain.add(launch_chained(norm_apply_kernel<T, kVec, kOne, false, kSilu>, grid, dim3(kNormThreads), 0, s, a));
  } else {
    chain.add(launch_chained(norm_sums_kernel<T, kVec, kOne, true, kSilu>, grid, dim3(kNormThreads), 0, s, a));
    const unsigned cols = want_param ? static_cast<unsigned>(ceil_div(a.C, 8)) : 0u;
    chain.add(launch_chained(warps ? norm_join_kernel<32, true> : norm_join_kernel<kNormThreads, true>, dim3(join + cols), dim3(kNormThreads), 0, s, a, join));
    if (want_out) chain.add(launch_chained(norm_apply_kernel<T, kVec, kOne, true, kSilu>, grid, dim3(kNormThreads), 0, s, a));
  }
  return chain.first != cudaSuccess ? cuda_status(chain.first) : launch_status();
}

template <typename T, int kVec, bool kOne>
static int norm_run(const NormArgs& a, const NormPlan& p, bool backward, bool want_out, bool want_param, cudaStream_t s) {
  return a.act == FGB_ACT_SILU ? norm_run_act<T, kVec, kOne, true>(a, p, backward, want_out, want_param, s)
                               : norm_run_act<T, kVec, kOne, false>(a, p, backward, want_out, want_param, s);
}

static int norm_call(const fgb_group_norm_call* c, bool backward, cudaStream_t s) {
  const int rc = norm_check(c);
  if (rc != FGB_OK) return rc;
  if (c->offsets_bits != 0 && !c->offsets) return FGB_E_NULL;
  const bool want_param = backward && (c->grad_weight != nullptr || c->grad_bias != nullptr);
  if (!c->mean || !c->rstd) return FGB_E_NULL;
  if (c->n > 0 && (!c->x || (backward ? !c->grad_out : !c->out))) return FGB_E_NULL;
  if ((reinterpret_cast<uintptr_t>(c->x) | reinterpret_cast<uintptr_t>(c->grad_out) | reinterpret_cast<uintptr_t>(c->out)) & 15) return FGB_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(c->workspace) & 255) return FGB_E_ALIGN;
  const NormPlan p = norm_plan(*c);
  if (p.bytes > 0 && !c->workspace) return FGB_E_NULL;
  if (c->workspace_bytes < static_cast<int64_t>(p.bytes)) return FGB_E_WORKSPACE;
  NormArgs a{};
  a.x = c->x, a.dy = c->grad_out, a.out = c->out;
  a.ranges = RowRanges{c->offsets_bits ? c->offsets : nullptr, c->offsets_bits == 64, static_cast<uint32_t>(c->n), static_cast<uint32_t>(c->samples)};
  a.C = c->c, a.G = c->groups, a.cpg = c->c / c->groups;
  a.R = p.R, a.blocks = p.blocks, a.slots = p.blocks + static_cast<uint32_t>(c->samples) - 1u;
  a.w = c->weight, a.b = c->bias, a.param_dtype = c->param_dtype, a.act = c->act, a.eps = c->eps;
  a.mean = c->mean, a.rstd = c->rstd;
  a.part = static_cast<F2*>(c->workspace);
  a.joined = reinterpret_cast<float*>(static_cast<char*>(c->workspace) + p.joined_off);
  a.dw = c->grad_weight, a.db = c->grad_bias;
  a.status = c->status, a.mirror = status_mirror(c->status);
  const bool want_out = c->out != nullptr;
#define FGB_NORM(T, v, one) norm_run<T, v, one>(a, p, backward, want_out, want_param, s)
#define FGB_NORM_16(T)                                                   \
  (p.vec == 8   ? FGB_NORM(T, 8, true)                                   \
   : p.vec == 4 ? (p.one ? FGB_NORM(T, 4, true) : FGB_NORM(T, 4, false)) \
   : p.vec == 2 ? FGB_NORM(T, 2, false)                                  \
                : FGB_NORM(T, 1, true))
  if (c->dtype == FGB_F16) return FGB_NORM_16(__half);
  if (c->dtype == FGB_BF16) return FGB_NORM_16(__nv_bfloat16);
  return p.vec == 4 ? (p.one ? FGB_NORM(float, 4, true) : FGB_NORM(float, 4, false)) : p.vec == 2 ? FGB_NORM(float, 2, false) : FGB_NORM(float, 1, true);
#undef FGB_NORM_16
#undef FGB_NORM
}

// ------------------------------------------------------------------ row ranges of the samples
// A row whose batch index is larger than the one before begins the samples in between; the last row ends those behind it:
// entries behind index `before`, up to `upto`.  Both may be any number (padding often has the largest one): they are cut to the
// samples that there are before anything is added to them.
struct OffsetEntries {
  int first, last;
};
__host__ __device__ __forceinline__ OffsetEntries offset_entries(int before, int upto, int batch) {
  const int b = before < -1 ? -1 : before > batch ? batch : before;
  return OffsetEntries{b + 1, upto < batch ? upto : batch};
}
__host__ __device__ __forceinline__ bool batch_index_ok(int before, int b, int batch) { return b >= 0 && b < batch && b >= before; }

__global__ void __launch_bounds__(256) sample_offsets_kernel(const int4* __restrict__ coords, uint32_t n, uint32_t batch, int32_t* __restrict__ offsets,
                                                             int32_t* status, int32_t* mirror) {
  chain_release();
  chain_wait();
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= n) {
    if (n == 0u)
      for (uint32_t k = i; k <= batch; k += gridDim.x * 256u) offsets[k] = 0;
    return;
  }
  const int b = __ldg(&coords[i]).x, before = i > 0u ? __ldg(&coords[i - 1u]).x : -1, most = static_cast<int>(batch);
  if (!batch_index_ok(before, b, most)) {
    report(status, FGB_S_BAD_OFFSETS);
    mirror_code(mirror, FGB_S_BAD_OFFSETS);
  }
  const OffsetEntries begun = offset_entries(before, b, most);
  for (int k = begun.first; k <= begun.last; ++k) offsets[k] = static_cast<int32_t>(i);
  if (i == n - 1u) {
    const OffsetEntries rest = offset_entries(b, most, most);
    for (int k = rest.first; k <= rest.last; ++k) offsets[k] = static_cast<int32_t>(n);
  }
}

}  // namespace fgb

extern "C" int64_t fgb_group_norm_workspace_bytes(const fgb_group_norm_call* call) {
  const int rc = fgb::norm_check(call);
  return rc != FGB_OK ? rc : static_cast<int64_t>(fgb::norm_plan(*call).bytes);
}
extern "C" int fgb_group_norm_forward(const fgb_group_norm_call* call, void* stream) {
  return fgb::norm_call(call, false, static_cast<cudaStream_t>(stream));
}
extern "C" int fgb_group_norm_backward(const fgb_group_norm_call* call, void* stream) {
  return fgb::norm_call(call, true, static_cast<cudaStream_t>(stream));
}

extern "C" int fgb_sample_offsets(const int32_t* coords, int64_t n, int64_t batch, int32_t* offsets, int32_t* status, void* stream) {
  using namespace fgb;
  if (n < 0 || n >= (int64_t(1) << 31) || batch < 1 || batch >= (int64_t(1) << 24)) return FGB_E_SIZE;
  if (!offsets || (n > 0 && !coords)) return FGB_E_NULL;
  if (reinterpret_cast<uintptr_t>(coords) & 15) return FGB_E_ALIGN;
  const cudaError_t e = launch_chained(sample_offsets_kernel, dim3(static_cast<unsigned>(ceil_div(n > 0 ? n : 1, 256))), dim3(256), 0, static_cast<cudaStream_t>(stream),
                                       reinterpret_cast<const int4*>(coords), static_cast<uint32_t>(n), static_cast<uint32_t>(batch), offsets, status,
                                       status_mirror(status));
  return e != cudaSuccess ? cuda_status(e) : launch_status();
}

// The kernel's rows one after the other, on host memory
extern "C" int fgb_sample_offsets_host(const int32_t* coords, int64_t n, int64_t batch, int32_t* offsets) {
  using namespace fgb;
  if (n < 0 || n >= (int64_t(1) << 31) || batch < 1 || batch >= (int64_t(1) << 24)) return FGB_E_SIZE;
  if (!offsets || (n > 0 && !coords)) return FGB_E_NULL;
  const int most = static_cast<int>(batch);
  int status = 0, before = -1;
  for (int64_t i = 0; i <= n; ++i) {
    const int b = i < n ? coords[i * 4] : most;  // what is behind the last row ends the samples that are left
    if (i < n && !batch_index_ok(before, b, most)) status = FGB_S_BAD_OFFSETS;
    const OffsetEntries e = offset_entries(before, b, most);
    for (int k = e.first; k <= e.last; ++k) offsets[k] = static_cast<int32_t>(i);
    before = b;
  }
  return status;
}
