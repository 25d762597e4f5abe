// Group norm with an activation over the rows of ragged samples, channels last; forward and backward.
//
//   m, v  = mean and variance over (rows of a sample) x (channels of a group),   r = 1 / sqrt(v + eps)
//   h     = (x - m) r,   z = h w + b,   y = act(z)
//   dz    = dy act'(z),  dw = sum dz h,  db = sum dz  (all rows),   q = dz w
//   dx    = r (q - mean(q) - h mean(q h))             (means as above)
//
// Three launches a direction, chained:
//   1. sums: a CTA takes a block of consecutive rows and adds, channel by channel, the rows of each sample that it meets
//      there.  Forward it keeps mean and squared distance from the mean (not plain squares: a channel whose mean is far
//      from zero keeps its digits), backward dz and dz h.
//   2. join: one group of threads per (sample, channel group) joins the blocks' results in a fixed order;
//      backward also adds the columns up to dw and db.
//   3. apply: the blocks in reverse, so that what the first pass read last is still in L2.
// Results of (block j, sample s) go to slot j + s: walking along the rows either number grows by one from one result to
// the next, so slots are unique, those of a sample are consecutive, and nothing has to be planned ahead.
#include <algorithm>

#include "fgb_common.cuh"
#include "fgb_device.cuh"
#include "fgb_rows.cuh"

namespace fgb {

constexpr int kNormThreads = 256;

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;             // y, or dx
  RowRanges ranges;
  int C, G, cpg;         // channels, groups, channels per group
  uint32_t R, blocks;    // rows per block
  const void* w;
  const void* b;
  int param_dtype;
  int act;
  float eps;
  float* mean;           // [samples, G]
  float* rstd;
  float* part;           // [blocks + samples - 1][2][C]
  float* joined;         // backward: [samples, G][2] mean(q), mean(q h)
  void* dw;
  void* db;
  int32_t* status;
  int32_t* mirror;
};

// the samples a block of rows meets: first .. last; each block's first is the last of the one before
__device__ __forceinline__ void samples_of_block(const NormArgs& a, uint32_t j, uint32_t& first, uint32_t& last) {
  const uint32_t before = j == 0u ? 0u : a.ranges.begun_before(j * a.R);
  first = before > 0u ? before - 1u : 0u;
  if (j + 1u >= a.blocks) {
    last = a.ranges.count - 1u;
  } else {
    const uint32_t k = a.ranges.begun_before((j + 1u) * a.R);
    last = k > 0u ? k - 1u : 0u;
  }
}

template <bool kExact>
__device__ __forceinline__ float sigmoid(float z) {
  // 16-bit results: the fast exponential and reciprocal are exact to some 2^-21, far below the result's half step
  return kExact ? 1.f / (1.f + expf(-z)) : __fdividef(1.f, 1.f + __expf(-z));
}
template <bool kExact>
__device__ __forceinline__ float activate(float z, int act) {
  return act == FGB_ACT_SILU ? (z == -INFINITY ? 0.f : z * sigmoid<kExact>(z)) : z;
}
// dy * act'(z).  Every rounding is named: the kernels that call it have to agree on the last bit, so that q - mean(q) is zero
// where a mean is of one value.
template <bool kExact>
__device__ __forceinline__ float activate_grad(float dy, float z, int act) {
  if (act != FGB_ACT_SILU) return dy;
  const float s = sigmoid<kExact>(z);
  return __fmul_rn(dy, __fmul_rn(s, fmaf(z, __fsub_rn(1.f, s), 1.f)));
}

// What a thread keeps of its kVec channels for one sample
template <int kVec>
struct ChannelParams {
  float mean[kVec], r[kVec], w[kVec], b[kVec];
  __device__ __forceinline__ void load(const NormArgs& p, uint32_t s, int c0) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int c = c0 + i;
      const size_t g = size_t(s) * p.G + c / p.cpg;
      mean[i] = p.mean[g];
      r[i] = p.rstd[g];
      w[i] = p.w != nullptr ? load_param(p.w, p.param_dtype, c) : 1.f;
      b[i] = p.b != nullptr ? load_param(p.b, p.param_dtype, c) : 0.f;
    }
  }
  __device__ __forceinline__ float h(float x, int i) const { return __fmul_rn(__fsub_rn(x, mean[i]), r[i]); }
  __device__ __forceinline__ float z(float h, int i) const { return fmaf(h, w[i], b[i]); }
};

// ------------------------------------------------------------------ 1. sums
template <typename T, int kVec, bool kBackward>
__global__ void __launch_bounds__(kNormThreads) norm_sums_kernel(const NormArgs p) {
  using Ch = Channels<T, kVec>;
  constexpr bool kExact = sizeof(T) == 4;
  __shared__ float s_sum[kNormThreads * kVec * 2];
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
  uint32_t first, last;
  samples_of_block(p, j, first, last);
  const uint32_t row0 = j * p.R, row1 = min(p.ranges.n, row0 + p.R);
  const T* x = static_cast<const T*>(p.x) + c0;
  const T* dy = static_cast<const T*>(p.dy) + c0;
  for (uint32_t s = first; s <= last; ++s) {
    const uint32_t lo = max(p.ranges.at(s), row0), hi = min(p.ranges.at(s + 1u), row1);
    float sum0[kVec], sum1[kVec], pivot[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum0[i] = sum1[i] = pivot[i] = 0.f;
    if (lo < hi && active) {
      if constexpr (!kBackward) {
        // distances from the range's first row: what cancels in sum1 - sum0^2 / n is at most its share of the rows
        Ch::unpack(Ch::load(x + size_t(lo) * p.C), pivot);
        auto add = [&](const typename Ch::Raw& raw) {
          float v[kVec];
          Ch::unpack(raw, v);
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const float d = v[i] - pivot[i];
            sum0[i] += d;
            sum1[i] = fmaf(d, d, sum1[i]);
          }
        };
        uint32_t r = lo + ry;
        for (; r + 3u * lanes < hi; r += 4u * lanes) {
          typename Ch::Raw raw[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) raw[u] = Ch::load(x + size_t(r + u * lanes) * p.C);
#pragma unroll
          for (int u = 0; u < 4; ++u) add(raw[u]);
        }
        for (; r < hi; r += lanes) add(Ch::load(x + size_t(r) * p.C));
      } else {
        ChannelParams<kVec> k;
        k.load(p, s, c0);
        auto add = [&](const typename Ch::Raw& raw, const typename Ch::Raw& raw_dy) {
          float v[kVec], g[kVec];
          Ch::unpack(raw, v);
          Ch::unpack(raw_dy, g);
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const float h = k.h(v[i], i);
            const float dz = activate_grad<kExact>(g[i], k.z(h, i), p.act);
            sum0[i] += dz;
            sum1[i] = fmaf(dz, h, sum1[i]);
          }
        };
        uint32_t r = lo + ry;
        for (; r + lanes < hi; r += 2u * lanes) {
          const typename Ch::Raw x0 = Ch::load(x + size_t(r) * p.C), x1 = Ch::load(x + size_t(r + lanes) * p.C);
          const typename Ch::Raw g0 = Ch::load(dy + size_t(r) * p.C), g1 = Ch::load(dy + size_t(r + lanes) * p.C);
          add(x0, g0);
          add(x1, g1);
        }
        if (r < hi) add(Ch::load(x + size_t(r) * p.C), Ch::load(dy + size_t(r) * p.C));
      }
    }
    // the row lanes' sums: halved until one is left (always in the same order)
    for (int m = lanes; m > 1;) {
      const int half = (m + 1) / 2;
      if (active && ry >= half && ry < m) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          s_sum[i * kNormThreads + threadIdx.x] = sum0[i];
          s_sum[(kVec + i) * kNormThreads + threadIdx.x] = sum1[i];
        }
      }
      __syncthreads();
      if (ry < m - half) {
        const int from = threadIdx.x + half * width;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          sum0[i] += s_sum[i * kNormThreads + from];
          sum1[i] += s_sum[(kVec + i) * kNormThreads + from];
        }
      }
      __syncthreads();
      m = half;
    }
    if (ry == 0) {
      float* out = p.part + size_t(j + s) * 2 * p.C + c0;
      const float n = lo < hi ? static_cast<float>(hi - lo) : 1.f;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if constexpr (kBackward) {
          out[i] = sum0[i];
          out[p.C + i] = sum1[i];
        } else {
          const float d = sum0[i] / n;
          out[i] = pivot[i] + d;                              // mean
          out[p.C + i] = fmaxf(fmaf(-sum0[i], d, sum1[i]), 0.f);  // squared distance from it
          if (isnan(sum1[i])) out[p.C + i] = sum1[i];
        }
      }
    }
  }
}

// ------------------------------------------------------------------ 2. join
template <int kThreads>
__device__ __forceinline__ double sum_of_threads(double v, double* s_red) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kThreads > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) v += s_red[w];
  }
  return v;
}

// kThreads threads of the CTA's 256 take one (sample, group); backward: the CTAs from `join_ctas` on add up 32 columns each
template <int kThreads, bool kBackward>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const NormArgs p, uint32_t join_ctas) {
  __shared__ double s_red[kNormThreads / 32];
  __shared__ float s_col[2][8][32];
  chain_release();
  chain_wait();
  if (kBackward && blockIdx.x >= join_ctas) {
    const int c = (blockIdx.x - join_ctas) * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
    const uint32_t slots = p.blocks + p.ranges.count - 1u;
    double db = 0, dw = 0;  // some thousand terms of fp32 sums each
    if (c < p.C) {
#pragma unroll 4
      for (uint32_t k = w; k < slots; k += 8u) {
        db += p.part[size_t(k) * 2 * p.C + c];
        dw += p.part[size_t(k) * 2 * p.C + p.C + c];
      }
    }
    s_col[0][w][threadIdx.x & 31] = static_cast<float>(db);
    s_col[1][w][threadIdx.x & 31] = static_cast<float>(dw);
    __syncthreads();
    if (w < 2 && c < p.C) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += s_col[w][i][threadIdx.x & 31];
      if (w == 0 && p.db != nullptr) store_param(p.db, p.param_dtype, c, v);
      if (w == 1 && p.dw != nullptr) store_param(p.dw, p.param_dtype, c, v);
    }
    return;
  }
  const uint64_t unit = uint64_t(blockIdx.x) * (kNormThreads / kThreads) + threadIdx.x / kThreads;
  if (unit >= uint64_t(p.ranges.count) * p.G) return;  // whole warps; with 256 threads a unit whole CTAs
  const uint32_t s = static_cast<uint32_t>(unit / p.G), g = static_cast<uint32_t>(unit % p.G), t = threadIdx.x % kThreads;
  const uint32_t lo = p.ranges.at(s), hi = max(lo, p.ranges.at(s + 1u));
  const uint32_t j0 = lo / p.R, entries = lo < hi ? ((hi - 1u) / p.R - j0 + 1u) * p.cpg : 0u;
  const double count = static_cast<double>(hi - lo) * p.cpg;
  const float* part = p.part + size_t(j0 + s) * 2 * p.C + g * p.cpg;
  auto rows_of = [&](uint32_t k) { return min(hi, (j0 + k + 1u) * p.R) - max(lo, (j0 + k) * p.R); };
  double v0 = 0, v1 = 0;
  if constexpr (!kBackward) {
    for (uint32_t e = t; e < entries; e += kThreads) {
      const uint32_t k = e / p.cpg, c = e - k * p.cpg;
      v0 += static_cast<double>(rows_of(k)) * part[size_t(k) * 2 * p.C + c];
    }
    const double mean = entries > 0u ? sum_of_threads<kThreads>(v0, s_red) / count : 0.0;
    for (uint32_t e = t; e < entries; e += kThreads) {
      const uint32_t k = e / p.cpg, c = e - k * p.cpg;
      const double d = part[size_t(k) * 2 * p.C + c] - mean;
      v1 += part[size_t(k) * 2 * p.C + p.C + c] + rows_of(k) * d * d;
    }
    const double var = entries > 0u ? sum_of_threads<kThreads>(v1, s_red) / count : 0.0;
    if (t == 0) {
      p.mean[unit] = static_cast<float>(mean);
      p.rstd[unit] = static_cast<float>(1.0 / sqrt(var + static_cast<double>(p.eps)));
    }
  } else {
    for (uint32_t e = t; e < entries; e += kThreads) {
      const uint32_t k = e / p.cpg, c = e - k * p.cpg;
      const double w = p.w != nullptr ? load_param(p.w, p.param_dtype, g * p.cpg + c) : 1.f;
      v0 += w * part[size_t(k) * 2 * p.C + c];
      v1 += w * part[size_t(k) * 2 * p.C + p.C + c];
    }
    if (entries > 0u) {
      v0 = sum_of_threads<kThreads>(v0, s_red) / count;
      v1 = sum_of_threads<kThreads>(v1, s_red) / count;
    }
    if (t == 0) {
      p.joined[unit * 2] = static_cast<float>(v0);
      p.joined[unit * 2 + 1] = static_cast<float>(v1);
    }
  }
}

// ------------------------------------------------------------------ 3. apply
template <typename T, int kVec, bool kBackward>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const NormArgs p) {
  using Ch = Channels<T, kVec>;
  constexpr bool kExact = sizeof(T) == 4;
  chain_release();
  chain_wait();
  const uint32_t j = p.blocks - 1u - blockIdx.x;
  const int packs = p.C / kVec, pack0 = blockIdx.y * kNormThreads;
  const int width = min(kNormThreads, packs - pack0), lanes = kNormThreads / width;
  const int cx = threadIdx.x % width, ry = threadIdx.x / width;
  const int c0 = (pack0 + cx) * kVec;
  uint32_t first, last;
  samples_of_block(p, j, first, last);  // whole warps take part
  if (ry >= lanes) return;
  const uint32_t row0 = j * p.R, row1 = min(p.ranges.n, row0 + p.R);
  const T* x = static_cast<const T*>(p.x) + c0;
  const T* dy = static_cast<const T*>(p.dy) + c0;
  T* out = static_cast<T*>(p.out) + c0;
  for (uint32_t s = first; s <= last; ++s) {
    const uint32_t lo = max(p.ranges.at(s), row0), hi = min(p.ranges.at(s + 1u), row1);
    if (lo >= hi) continue;
    ChannelParams<kVec> k;
    k.load(p, s, c0);
    if constexpr (!kBackward) {
      auto one = [&](const typename Ch::Raw& raw, uint32_t r) {
        float v[kVec];
        Ch::unpack(raw, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = activate<kExact>(k.z(k.h(v[i], i), i), p.act);
        Ch::store(out + size_t(r) * p.C, Ch::pack(v));
      };
      uint32_t r = lo + ry;
      for (; r + 3u * lanes < hi; r += 4u * lanes) {
        typename Ch::Raw raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = Ch::load(x + size_t(r + u * lanes) * p.C);
#pragma unroll
        for (int u = 0; u < 4; ++u) one(raw[u], r + u * lanes);
      }
      for (; r < hi; r += lanes) one(Ch::load(x + size_t(r) * p.C), r);
    } else {
      float m1[kVec], m2[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const size_t g = size_t(s) * p.G + (c0 + i) / p.cpg;
        m1[i] = p.joined[g * 2], m2[i] = p.joined[g * 2 + 1];
      }
      auto one = [&](const typename Ch::Raw& raw, const typename Ch::Raw& raw_dy, uint32_t r) {
        float v[kVec], g[kVec];
        Ch::unpack(raw, v);
        Ch::unpack(raw_dy, g);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float h = k.h(v[i], i);
          const float q = __fmul_rn(activate_grad<kExact>(g[i], k.z(h, i), p.act), k.w[i]);
          v[i] = k.r[i] * fmaf(-h, m2[i], __fsub_rn(q, m1[i]));
        }
        Ch::store(out + size_t(r) * p.C, Ch::pack(v));
      };
      uint32_t r = lo + ry;
      for (; r + lanes < hi; r += 2u * lanes) {
        const typename Ch::Raw x0 = Ch::load(x + size_t(r) * p.C), x1 = Ch::load(x + size_t(r + lanes) * p.C);
        const typename Ch::Raw g0 = Ch::load(dy + size_t(r) * p.C), g1 = Ch::load(dy + size_t(r + lanes) * p.C);
        one(x0, g0, r);
        one(x1, g1, r + lanes);
      }
      if (r < hi) one(Ch::load(x + size_t(r) * p.C), Ch::load(dy + size_t(r) * p.C), r);
    }
  }
  // rows of no sample
  const uint32_t begin = p.ranges.at(0u), end = max(begin, p.ranges.at(p.ranges.count));
  if (row0 >= begin && row1 <= end) return;
  typename Ch::Raw zero{};
  for (uint32_t r = row0 + ry; r < row1; r += lanes)
    if (r < begin || r >= end) Ch::store(out + size_t(r) * p.C, zero);
}

// ------------------------------------------------------------------ host side
struct NormPlan {
  int vec;
  unsigned columns;   // CTAs along a row
  uint32_t R, blocks;
  size_t joined_off, bytes;
};
static NormPlan norm_plan(const fgb_group_norm_call& c) {
  NormPlan p;
  p.vec = row_pack(c.c, elem_bytes(c.dtype));
  const int packs = c.c / p.vec;
  p.columns = static_cast<unsigned>(ceil_div(packs, kNormThreads));
  const int width = packs < kNormThreads ? packs : kNormThreads, lanes = kNormThreads / width;
  // four CTAs on every SM, each thread at least eight rows
  const int64_t want = std::max<int64_t>(ceil_div(int64_t(device_sm_count()) * 4, p.columns), 1);
  const int64_t R = std::max<int64_t>(ceil_div(c.n, want), int64_t(lanes) * 8);
  p.R = static_cast<uint32_t>(R);
  p.blocks = static_cast<uint32_t>(std::max<int64_t>(ceil_div(c.n, R), 1));
  p.joined_off = align256((int64_t(p.blocks) + c.samples - 1) * 2 * c.c * 4);
  p.bytes = p.joined_off + align256(c.samples * c.groups * 8);
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

template <typename T, int kVec>
static int norm_run(const NormArgs& a, const NormPlan& p, bool backward, bool want_out, bool want_param, cudaStream_t s) {
  const dim3 grid(p.blocks, p.columns);
  LaunchErrors chain;
  const int64_t units = int64_t(a.ranges.count) * a.G;
  // a CTA a (sample, group) where the samples cover many blocks, a warp where they are short
  const bool warps = int64_t(p.blocks) * a.cpg / a.ranges.count < 64;
  const uint32_t join = static_cast<uint32_t>(warps ? ceil_div(units, kNormThreads / 32) : units);
  if (!backward) {
    chain.add(launch_chained(norm_sums_kernel<T, kVec, false>, grid, dim3(kNormThreads), 0, s, a));
    chain.add(launch_chained(warps ? norm_join_kernel<32, false> : norm_join_kernel<kNormThreads, false>, dim3(join), dim3(kNormThreads), 0, s, a, join));
    chain.add(launch_chained(norm_apply_kernel<T, kVec, false>, grid, dim3(kNormThreads), 0, s, a));
  } else {
    chain.add(launch_chained(norm_sums_kernel<T, kVec, true>, grid, dim3(kNormThreads), 0, s, a));
    const unsigned cols = want_param ? static_cast<unsigned>(ceil_div(a.C, 32)) : 0u;
    chain.add(launch_chained(warps ? norm_join_kernel<32, true> : norm_join_kernel<kNormThreads, true>, dim3(join + cols), dim3(kNormThreads), 0, s, a, join));
    if (want_out) chain.add(launch_chained(norm_apply_kernel<T, kVec, true>, grid, dim3(kNormThreads), 0, s, a));
  }
  return chain.first != cudaSuccess ? cuda_status(chain.first) : launch_status();
}

static int norm_call(const fgb_group_norm_call* c, bool backward, cudaStream_t s) {
  const int rc = norm_check(c);
  if (rc != FGB_OK) return rc;
  if (c->offsets_bits != 0 && !c->offsets) return FGB_E_NULL;
  const bool want_param = backward && (c->grad_weight != nullptr || c->grad_bias != nullptr);
  if (!c->mean || !c->rstd || !c->workspace) return FGB_E_NULL;
  if (c->n > 0 && (!c->x || (backward ? !c->grad_out : !c->out))) return FGB_E_NULL;
  if ((reinterpret_cast<uintptr_t>(c->x) | reinterpret_cast<uintptr_t>(c->grad_out) | reinterpret_cast<uintptr_t>(c->out)) & 15) return FGB_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(c->workspace) & 255) return FGB_E_ALIGN;
  const NormPlan p = norm_plan(*c);
  if (c->workspace_bytes < static_cast<int64_t>(p.bytes)) return FGB_E_WORKSPACE;
  NormArgs a{};
  a.x = c->x, a.dy = c->grad_out, a.out = c->out;
  a.ranges = RowRanges{c->offsets_bits ? c->offsets : nullptr, c->offsets_bits == 64, static_cast<uint32_t>(c->n), static_cast<uint32_t>(c->samples)};
  a.C = c->c, a.G = c->groups, a.cpg = c->c / c->groups;
  a.R = p.R, a.blocks = p.blocks;
  a.w = c->weight, a.b = c->bias, a.param_dtype = c->param_dtype, a.act = c->act, a.eps = c->eps;
  a.mean = c->mean, a.rstd = c->rstd;
  a.part = static_cast<float*>(c->workspace);
  a.joined = reinterpret_cast<float*>(static_cast<char*>(c->workspace) + p.joined_off);
  a.dw = c->grad_weight, a.db = c->grad_bias;
  a.status = c->status, a.mirror = status_mirror(c->status);
  const bool want_out = c->out != nullptr;
  switch (c->dtype) {
    case FGB_F16:
      return p.vec == 8   ? norm_run<__half, 8>(a, p, backward, want_out, want_param, s)
             : p.vec == 4 ? norm_run<__half, 4>(a, p, backward, want_out, want_param, s)
             : p.vec == 2 ? norm_run<__half, 2>(a, p, backward, want_out, want_param, s)
                          : norm_run<__half, 1>(a, p, backward, want_out, want_param, s);
    case FGB_BF16:
      return p.vec == 8   ? norm_run<__nv_bfloat16, 8>(a, p, backward, want_out, want_param, s)
             : p.vec == 4 ? norm_run<__nv_bfloat16, 4>(a, p, backward, want_out, want_param, s)
             : p.vec == 2 ? norm_run<__nv_bfloat16, 2>(a, p, backward, want_out, want_param, s)
                          : norm_run<__nv_bfloat16, 1>(a, p, backward, want_out, want_param, s);
    default:
      return p.vec == 4   ? norm_run<float, 4>(a, p, backward, want_out, want_param, s)
             : p.vec == 2 ? norm_run<float, 2>(a, p, backward, want_out, want_param, s)
                          : norm_run<float, 1>(a, p, backward, want_out, want_param, s);
  }
}

// ------------------------------------------------------------------ row ranges of the samples
// A row whose batch index is larger than the one before begins the samples in between; the last row ends those behind it.
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
  const int b = __ldg(&coords[i]).x, before = i > 0u ? __ldg(&coords[i - 1u]).x : -1;
  if (b < 0 || b >= static_cast<int>(batch) || b < before) {
    report(status, FGB_S_BAD_OFFSETS);
    mirror_code(mirror, FGB_S_BAD_OFFSETS);
  }
  const int most = static_cast<int>(batch);
  for (int k = max(before, -1) + 1; k <= min(b, most); ++k) offsets[k] = static_cast<int32_t>(i);
  if (i == n - 1u)
    for (int k = max(b, -1) + 1; k <= most; ++k) offsets[k] = static_cast<int32_t>(n);
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
