// Matrix products grouped by ragged row ranges: every group g multiplies its rows by a matrix of its own, W_g [co, ci].
//
//   forward           y_r  = W_g x_r + b_g            for the rows r of group g
//   input gradient    dx_r = W_g^T dy_r
//   weight gradient   dW_g = sum_r dy_r x_r^T,  db_g = sum_r dy_r
//
// One persistent tcgen05 kernel for all of them: D[m, n] = sum_k P[m, k] Q[n, k], tiles of 128 x BN, 64 k a stage.
//   kRows    m = rows, n = channels of the output.  The rows of a tile may reach into the next group: what they give is not
//            stored.  The gradient reads W_g as stored, with k along its rows (MN-major operand).
//   kFew     m = channels, n = rows (16 to 64 of them): where groups have few rows the matrices are what is read, and a tile
//            of 128 rows would be mostly empty.
//   kWeight  m = co, n = ci, k = rows: both operands MN-major.  The k blocks of a group end where its rows end: a block
//            that reaches further is cut in steps of 16 rows, and what its last step holds of other rows is cleared in
//            shared memory (both operands: another group's infinity times zero would be NaN).  db comes from the same
//            blocks, as one more product with a block of ones.
// Warps: 0-7 store tiles (two per quarter of the accumulator rows), 8 loads (TMA), 9 multiplies; two accumulators in TMEM
// where they fit, so that a tile is stored while the next is multiplied.
//
// Work is a line of iterations (one stage each): the tiles of group 0, then group 1, ..., a tile's iterations together.
// Where every CTA has several tiles to do, the line is cut at tiles; otherwise (the weight gradient; a few rows) into equal
// ranges, one for each CTA: a tile that lies in several ranges leaves fp32 pieces in a slab, which a second kernel adds up
// in their order.  What each CTA does follows from the sizes alone, so results do not depend on the run.
//
// fp32 operands are written as sums of bf16 planes (hi + mid + lo, 8 bits each) and multiplied plane by plane: six products
// (all whose weight is 2^-16 and more) for accurate fp32, three (2^-8 and more) where TF32 is allowed.  bf16 has
// fp32's range, so no scaling is needed, and six of them cost what three TF32 products do (half the rate, twice the bytes).
// The tensor cores cut what they add to an accumulator at its last bit instead of rounding: over a long k that is a bias
// (2e-8 of the sum for every 16 k; 1e-5 where k was 10^5).  So fp32 leaves the accumulator after each block of 64 k, the small
// products first, the large one last, and the storing warps add the blocks up in registers, rounding to nearest.
#include <algorithm>
#include <type_traits>

#include "fgb_common.cuh"
#include "fgb_device.cuh"
#include "fgb_rows.cuh"
#include "fgb_umma.cuh"

namespace fgb {

constexpr int kGrThreads = 320;
constexpr int kGrEpilogueWarps = 8;
constexpr int kGrMaxStages = 12;
constexpr int kGrMaxGroups = 2048;
constexpr int kGrCtrlBytes = 1024 + 2048 + 2048;  // barriers; a block of ones; bias of a pass for each warp
constexpr int kGrStoreBytes = kGrEpilogueWarps * 2048;
constexpr int kGrSmemLimit = 227 * 1024;
constexpr int kGrPBytes = 128 * 128;

enum { kRows = 0, kFew = 1, kWeight = 2 };

struct GroupedArgs {
  RowRanges ranges;
  int bn;               // columns of a tile
  int n_tiles;          // tiles along the channels that are not rows: kRows along n, kFew along m, kWeight along n
  int m_tiles;          // kWeight: tiles along co
  int k_blocks;         // kRows, kFew: blocks of 64 along k
  int k_extent;         // kRows, kFew: k
  int terms;            // products of planes
  uint32_t p_planes, q_planes;  // their planes, four bits a term
  int p_mn, q_mn;       // operand is MN-major
  int stages, q_bytes, acc_sets, acc_stride;
  uint32_t min_range;   // iterations that a range has at least; 0: a range is a tile
  uint32_t idesc, idesc_ones;
  uint32_t one_pair;    // two ones of the operand type
  const void* bias;     // [groups, nout] or null
  void* out;
  void* db;             // kWeight: [groups, co] or null
  float* slab;          // pieces of tiles that lie in several ranges
  int m_extent, n_extent;  // channels: kRows n; kFew m; kWeight m and n
  int out_ld;
  int vec_ok;           // rows of the output are whole 16-byte pieces
  int32_t* status;
  int32_t* mirror;
};

struct GroupedSmem {
  uint64_t full[kGrMaxStages], empty[kGrMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(GroupedSmem) <= 1024, "control block too large");

// iterations that group g has: tiles x blocks x terms
template <int kMode>
__device__ __forceinline__ uint32_t group_iterations(const GroupedArgs& p, uint32_t g) {
  const uint32_t lo = p.ranges.at(g), hi = p.ranges.at(g + 1u), len = hi > lo ? hi - lo : 0u;
  if constexpr (kMode == kRows) return (len + 127u) / 128u * p.n_tiles * p.k_blocks * p.terms;
  else if constexpr (kMode == kFew) return (len + p.bn - 1u) / p.bn * p.n_tiles * p.k_blocks * p.terms;
  else return (len + 63u) / 64u * p.terms * p.n_tiles * p.m_tiles;
}

// first[g] = iterations of the groups before g, first[groups] all of them; the whole CTA calls it (and waits at its end)
template <int kMode>
__device__ __forceinline__ void plan_groups(const GroupedArgs& p, uint32_t* first) {
  const uint32_t G = p.ranges.count;
  bool bad = false;
  for (uint32_t g = threadIdx.x; g < G; g += blockDim.x) {
    first[g + 1u] = group_iterations<kMode>(p, g);
    bad |= !p.ranges.good(g);
  }
  // ranges that overlap could ask for more tiles than there is room for: nothing is done
  if (__syncthreads_or(bad)) {
    for (uint32_t g = threadIdx.x; g < G; g += blockDim.x) first[g + 1u] = 0u;
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    const uint32_t lane = threadIdx.x;
    uint32_t run = 0;
    for (uint32_t g0 = 0; g0 < G; g0 += 32u) {
      uint32_t v = g0 + lane < G ? first[g0 + lane + 1u] : 0u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= static_cast<uint32_t>(d)) v += o;
      }
      if (g0 + lane < G) first[g0 + lane + 1u] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) first[0] = 0u;
  }
  __syncthreads();
}

// iterations of a range
template <int kMode>
__device__ __forceinline__ uint32_t range_length(const GroupedArgs& p, uint32_t total, uint32_t ctas) {
  if (p.min_range == 0u) return static_cast<uint32_t>(p.k_blocks * p.terms);  // a tile
  return max((total + ctas - 1u) / ctas, p.min_range);
}

// A tile, or the part of one that a range holds
struct GroupedItem {
  uint32_t group, tile;     // tile within the group
  uint32_t from, to, whole; // its iterations, of `whole`
  uint32_t lo, hi;          // rows of the group
  uint32_t range;
};

// walks the items of a CTA's ranges: every role goes through the same sequence
template <int kMode>
struct GroupedWalk {
  const GroupedArgs& p;
  const uint32_t* first;
  uint32_t total, length, range, at, end;
  __device__ __forceinline__ GroupedWalk(const GroupedArgs& p_, const uint32_t* first_, uint32_t ctas, uint32_t cta) : p(p_), first(first_) {
    total = first[p.ranges.count];
    length = range_length<kMode>(p, total, ctas);
    range = cta;
    at = 0, end = 0;
    step = ctas;
    begin_range();
  }
  __device__ __forceinline__ bool next(GroupedItem& it) {
    if (at >= end) {
      range += step;
      begin_range();
    }
    if (at >= end) return false;
    uint32_t lo = 0, hi = p.ranges.count - 1u;  // the last group that begins at or before `at` and is not empty
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1u) / 2u;
      if (first[mid] <= at) lo = mid;
      else hi = mid - 1u;
    }
    it.group = lo;
    const uint32_t begin = p.ranges.at(lo), stop = p.ranges.at(lo + 1u);
    it.lo = begin, it.hi = max(begin, stop);
    it.whole = kMode == kWeight ? (it.hi - it.lo + 63u) / 64u * p.terms : static_cast<uint32_t>(p.k_blocks * p.terms);
    const uint32_t local = at - first[lo];
    it.tile = local / it.whole;
    it.from = local - it.tile * it.whole;
    it.to = min(it.whole, it.from + (end - at));
    it.range = range;
    at += it.to - it.from;
    return true;
  }

 private:
  uint32_t step;
  __device__ __forceinline__ void begin_range() {
    // total and the number of ranges are below 2^31, checked on the host
    const uint64_t a = uint64_t(range) * length;
    at = a < total ? static_cast<uint32_t>(a) : total;
    end = min(total, at + length);
  }
};

template <typename T>
__device__ __forceinline__ void store_value(T* p, float v) {
  if constexpr (std::is_same<T, float>::value) *p = v;
  else *p = static_cast<T>(v);
}

// 32 columns of the warp's 32 accumulator rows to out[row * ld + c0 + i] (row < rows, c0 + i < cols).  64 bytes of each row
// at a time go through the warp's staging buffer (32 rows of 64 bytes, 16-byte pieces XORed with half the row), so that a
// store instruction writes whole sectors of eight rows.
template <typename T>
__device__ __forceinline__ void store_columns(uint32_t (&acc)[32], uint8_t* stage, float* s_bias, int lane, int c0, T* out, int64_t ld, int rows, int cols,
                                              int vec_ok, const void* bias, int bias_dtype) {
  constexpr int kPiece = 16 / sizeof(T), kCols = 4 * kPiece;  // columns of a piece, and of 64 bytes
  uint8_t* mine = stage + lane * 64;
  if (bias != nullptr) {
    s_bias[lane] = c0 + lane < cols ? load_param(bias, bias_dtype, c0 + lane) : 0.f;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4*>(s_bias)[i];
      acc[4 * i] = __float_as_uint(__uint_as_float(acc[4 * i]) + b.x), acc[4 * i + 1] = __float_as_uint(__uint_as_float(acc[4 * i + 1]) + b.y);
      acc[4 * i + 2] = __float_as_uint(__uint_as_float(acc[4 * i + 2]) + b.z), acc[4 * i + 3] = __float_as_uint(__uint_as_float(acc[4 * i + 3]) + b.w);
    }
  }
#pragma unroll
  for (int h = 0; h < 32 / kCols; ++h) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float f[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) f[i] = __uint_as_float(acc[h * kCols + g * kPiece + i]);
      *reinterpret_cast<uint4*>(mine + ((g ^ ((lane >> 1) & 3)) << 4)) = Channels<T, kPiece>::pack(f);
    }
    __syncwarp();
    const int piece = lane & 3, col = c0 + h * kCols + piece * kPiece;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + (lane >> 2);
      const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
      if (row < rows && col < cols) {
        T* to = out + int64_t(row) * ld + col;
        if (vec_ok) {
          *reinterpret_cast<uint4*>(to) = v;
        } else {
          const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (col + e < cols) to[e] = t[e];
        }
      }
    }
    __syncwarp();
  }
}

// whether the iterations [from, to) of a tile hold one whose second operand is the first plane
__device__ __forceinline__ bool meets_first_plane(const GroupedArgs& p, uint32_t from, uint32_t to) {
  uint32_t term = from % p.terms;
  for (uint32_t i = from; i < to && i < from + p.terms; ++i) {
    if (((p.q_planes >> (4 * term)) & 15u) == 0u) return true;
    if (++term == static_cast<uint32_t>(p.terms)) term = 0;
  }
  return false;
}

template <int kMode, typename T>
__global__ void __launch_bounds__(kGrThreads, 1) grouped_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                                                                const __grid_constant__ GroupedArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  GroupedSmem* ctl = reinterpret_cast<GroupedSmem*>(smem);
  uint8_t* ones = smem + 1024;
  float* s_bias = reinterpret_cast<float*>(smem + 3072);
  uint8_t* stages = smem + kGrCtrlBytes;  // multiples of 1024 from here on
  const int stage_bytes = kGrPBytes + p.q_bytes;
  uint8_t* store = stages + size_t(p.stages) * stage_bytes;
  uint32_t* first = reinterpret_cast<uint32_t*>(store + kGrStoreBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  constexpr int kParamDtype = std::is_same<T, __half>::value ? FGB_F16 : std::is_same<T, __nv_bfloat16>::value ? FGB_BF16 : FGB_F32_IEEE;
  constexpr bool kBlocks = std::is_same<T, float>::value;  // the accumulator is emptied after every block of 64 k
  constexpr int kSums = kMode == kFew ? 1 : 3;             // blocks of 32 columns that a storing warp adds up

  chain_release();
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&ctl->acc_full[a], 1);
      mbar_init(&ctl->acc_empty[a], kGrEpilogueWarps);
    }
    ctl->abort_flag = 0;
    mbar_init_fence();
  }
  if (kMode == kWeight) {
    for (int i = tid; i < 512; i += kGrThreads) reinterpret_cast<uint32_t*>(ones)[i] = p.one_pair;
    fence_proxy_async_smem();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
  }
  if (warp == 9) {
    tmem_alloc_dyn(&ctl->tmem_base, 512u);
    tmem_relinquish();
  }
  chain_wait();
  p.ranges.check(p.status, p.mirror);
  plan_groups<kMode>(p, first);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  GroupedWalk<kMode> walk(p, first, gridDim.x, blockIdx.x);
  GroupedItem it;

  // where the rows and columns of an item's tile begin
  auto m_tile_of = [&](const GroupedItem& t) { return kMode == kFew ? t.tile % p.n_tiles : t.tile / p.n_tiles; };
  auto n_tile_of = [&](const GroupedItem& t) { return kMode == kFew ? t.tile / p.n_tiles : t.tile % p.n_tiles; };

  if (warp == 8) {
    // ------------------------------------------------------------------ loads
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      while (walk.next(it)) {
        // first row (or channel) of the tile along m and n, first k
        const int m0 = static_cast<int>(m_tile_of(it)) * 128, n0 = static_cast<int>(n_tile_of(it)) * p.bn;
        const int lo = static_cast<int>(it.lo), g = static_cast<int>(it.group), G = static_cast<int>(p.ranges.count);
        uint32_t kb = it.from / p.terms, term = it.from - kb * p.terms;
        for (uint32_t i = it.from; i < it.to; ++i) {
          mbar_wait(&ctl->empty[s], ph ^ 1, abort_flag);
          mbar_arrive_expect_tx(&ctl->full[s], static_cast<uint32_t>(stage_bytes));
          const uint32_t pd = smem_u32(stages + size_t(s) * stage_bytes), qd = pd + kGrPBytes;
          const int pp = (p.p_planes >> (4 * term)) & 15, pq = (p.q_planes >> (4 * term)) & 15;
          const int k0 = static_cast<int>(kb) * 64;
          if constexpr (kMode == kRows) {
            tma_load_3d(pd, &tmap_p, &ctl->full[s], k0, lo + m0, pp);
            if (p.q_mn) {
              for (int c = 0; c * 64 < p.bn; ++c) tma_load_3d(qd + c * 8192, &tmap_q, &ctl->full[s], n0 + c * 64, k0, pq * G + g);
            } else {
              tma_load_3d(qd, &tmap_q, &ctl->full[s], k0, n0, pq * G + g);
            }
          } else if constexpr (kMode == kFew) {
            if (p.p_mn) {
              for (int c = 0; c < 2; ++c) tma_load_3d(pd + c * 8192, &tmap_p, &ctl->full[s], m0 + c * 64, k0, pp * G + g);
            } else {
              tma_load_3d(pd, &tmap_p, &ctl->full[s], k0, m0, pp * G + g);
            }
            tma_load_3d(qd, &tmap_q, &ctl->full[s], k0, lo + n0, pq);
          } else {
            for (int c = 0; c < 2; ++c) tma_load_3d(pd + c * 8192, &tmap_p, &ctl->full[s], m0 + c * 64, lo + k0, pp);
            for (int c = 0; c * 64 < p.bn; ++c) tma_load_3d(qd + c * 8192, &tmap_q, &ctl->full[s], n0 + c * 64, lo + k0, pq);
          }
          if (++term == static_cast<uint32_t>(p.terms)) term = 0, ++kb;
          if (++s == static_cast<uint32_t>(p.stages)) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ products
    uint32_t s = 0, ph = 0, set = 0, set_ph = 0;
    const uint64_t p_step = kMode == kWeight || p.p_mn ? 128u : 2u, q_step = kMode == kWeight || p.q_mn ? 128u : 2u;
    const uint32_t p_lbo = kMode == kWeight || p.p_mn ? 8192u : 16u, q_lbo = kMode == kWeight || p.q_mn ? 8192u : 16u;
    const uint64_t d_ones = make_smem_desc(smem_u32(ones), 16, 1024);
    while (walk.next(it)) {
      const bool with_ones = kMode == kWeight && p.db != nullptr && n_tile_of(it) == 0u;
      uint32_t kb = it.from / p.terms, term = it.from - kb * p.terms;
      uint32_t any = 0, any_ones = 0, acc = 0;
      for (uint32_t i = it.from; i < it.to; ++i) {
        if (any == 0u) {  // a new accumulator
          mbar_wait(&ctl->acc_empty[set], set_ph ^ 1, abort_flag);
          tc_fence_after_sync();
          acc = tmem_base + set * p.acc_stride;
        }
        mbar_wait(&ctl->full[s], ph, abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t base = smem_u32(stages + size_t(s) * stage_bytes);
        const uint32_t left = (kMode == kWeight ? it.hi - it.lo : static_cast<uint32_t>(p.k_extent)) - kb * 64u;
        const uint32_t valid = min(left, 64u), steps = (valid + 15u) / 16u;
        if (kMode == kWeight && (valid & 15u) != 0u) {
          // rows of other groups in the last step: cleared in both operands
          const uint32_t chunks = 2u + (p.bn + 63u) / 64u, rows = steps * 16u - valid;
          uint8_t* at = stages + size_t(s) * stage_bytes;
          for (uint32_t c = 0; c < chunks; ++c)
            for (uint32_t r = lane >> 3; r < rows; r += 4u)
              *reinterpret_cast<uint4*>(at + c * 8192u + (valid + r) * 128u + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        const bool ones_now = with_ones && ((p.q_planes >> (4 * term)) & 15u) == 0u;  // once for each plane of dy
        if (elect_one()) {
          const uint64_t dp = make_smem_desc(base, p_lbo, 1024), dq = make_smem_desc(base + kGrPBytes, q_lbo, 1024);
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            if (k < steps) {
              umma_ss<false>(acc, dp + k * p_step, dq + k * q_step, p.idesc, k == 0 ? any : 1u);
              if (ones_now) umma_ss<false>(acc + p.bn, dp + k * p_step, d_ones, p.idesc_ones, k == 0 ? any_ones : 1u);
            }
          }
          umma_commit(&ctl->empty[s]);
        }
        __syncwarp();
        any = 1u;
        any_ones |= ones_now ? 1u : 0u;
        if (++term == static_cast<uint32_t>(p.terms)) term = 0, ++kb;
        if (++s == static_cast<uint32_t>(p.stages)) s = 0, ph ^= 1;
        if (i + 1u == it.to || (kBlocks && term == 0u)) {  // the accumulator is done: the tile's last, or the block's
          if (elect_one()) umma_commit(&ctl->acc_full[set]);
          __syncwarp();
          if (++set == static_cast<uint32_t>(p.acc_sets)) set = 0, set_ph ^= 1;
          any = any_ones = 0u;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ stores
    const int quarter = warp & 3, group = warp >> 2;
    uint8_t* stage = store + warp * 2048;
    float* bias_buf = s_bias + warp * 64;
    uint32_t set = 0, set_ph = 0;
    // this warp's columns are [32 group, 32 group + 32) of every 64: at most 3 x 32 of them in fp32
    uint32_t sum[kBlocks ? kSums : 1][32];
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    auto wait_full = [&]() {
      mbar_wait(&ctl->acc_full[set], set_ph, abort_flag);
      tc_fence_after_sync();
      return tmem_base + set * p.acc_stride + lanes;
    };
    auto give_back = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->acc_empty[set]);
      if (++set == static_cast<uint32_t>(p.acc_sets)) set = 0, set_ph ^= 1;
    };
    while (walk.next(it)) {
      const int m0 = static_cast<int>(m_tile_of(it)) * 128 + quarter * 32, n0 = static_cast<int>(n_tile_of(it)) * p.bn;
      const bool whole = it.from == 0u && it.to == it.whole;
      const bool with_db = kMode == kWeight && p.db != nullptr && n0 == 0 && group == 0;
      float db = 0.f;
      uint32_t tmem = 0;
      if constexpr (kBlocks) {
#pragma unroll
        for (int b = 0; b < kSums; ++b)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[b][i] = 0u;
        for (uint32_t at = it.from; at < it.to;) {
          const uint32_t end = min(it.to, (at / p.terms + 1u) * p.terms);
          tmem = wait_full();
#pragma unroll
          for (int b = 0; b < kSums; ++b) {
            if (group * 32 + b * 64 < p.bn) {
              uint32_t acc[32];
              tmem_ld_32x32(tmem + group * 32 + b * 64, acc);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[b][i] = __float_as_uint(__uint_as_float(sum[b][i]) + __uint_as_float(acc[i]));
            }
          }
          if (with_db && meets_first_plane(p, at, end)) {
            uint32_t acc[32];
            tmem_ld_32x32(tmem + p.bn, acc);
            tmem_ld_wait();
            db += __uint_as_float(acc[0]);
          }
          give_back();
          at = end;
        }
      } else {
        tmem = wait_full();
        if (with_db) {
          uint32_t acc[32];
          tmem_ld_32x32(tmem + p.bn, acc);
          tmem_ld_wait();
          db = __uint_as_float(acc[0]);
        }
      }
      // a piece of a tile: the first slot of its range for one that began before it, else the second
      float* piece = whole ? nullptr : p.slab + (size_t(it.range) * 2 + (it.from == 0u ? 1 : 0)) * 128 * p.acc_stride;
      const int64_t row0 = kMode == kRows ? int64_t(it.lo) + m0 : int64_t(it.group) * p.m_extent + m0;
      const int rows = (kMode == kRows ? static_cast<int>(it.hi - it.lo) : p.m_extent) - m0;
      const void* bias = p.bias == nullptr ? nullptr
                         : static_cast<const char*>(p.bias) + (int64_t(it.group) * (kMode == kFew ? p.m_extent : p.n_extent) + (kMode == kFew ? 0 : n0)) *
                                                                  static_cast<int64_t>(sizeof(T));
      const float few_bias = kMode == kFew && whole && bias != nullptr && m0 + lane < p.m_extent ? load_param(bias, kParamDtype, m0 + lane) : 0.f;
      auto put = [&](uint32_t (&acc)[32], int c0) {
        if constexpr (kMode == kFew) {
          const int left = static_cast<int>(it.hi - it.lo) - n0;  // rows of the tile, and more
          T* out = static_cast<T*>(p.out) + int64_t(it.lo + n0) * p.out_ld + m0 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int r = c0 + i;
            if (r < p.bn) {
              if (piece != nullptr) piece[r * 128 + quarter * 32 + lane] = __uint_as_float(acc[i]);
              else if (r < left && m0 + lane < p.m_extent) store_value(out + int64_t(r) * p.out_ld, __uint_as_float(acc[i]) + few_bias);
            }
          }
        } else if (piece != nullptr) {
          store_columns<float>(acc, stage, bias_buf, lane, c0, piece + size_t(quarter * 32) * p.bn, p.bn, 32, p.bn, 1, nullptr, 0);
        } else {
          store_columns<T>(acc, stage, bias_buf, lane, c0, static_cast<T*>(p.out) + row0 * p.out_ld + n0, p.out_ld, rows, p.n_extent - n0, p.vec_ok, bias,
                           kParamDtype);
        }
      };
      if (*abort_flag == 0u) {  // else nothing that was waited for is there, and the status word says so
        if constexpr (kBlocks) {
#pragma unroll
          for (int b = 0; b < kSums; ++b)
            if (group * 32 + b * 64 < p.bn) put(sum[b], group * 32 + b * 64);
        } else {
          for (int c0 = group * 32; c0 < p.bn; c0 += 64) {
            uint32_t acc[32];
            tmem_ld_32x32(tmem + c0, acc);
            tmem_ld_wait();
            put(acc, c0);
          }
        }
        if (with_db) {
          const int m = m0 + lane;
          if (piece != nullptr) piece[128 * p.bn + quarter * 32 + lane] = db;
          else if (m < p.m_extent) store_value(static_cast<T*>(p.db) + int64_t(it.group) * p.m_extent + m, db);
        }
      }
      if constexpr (!kBlocks) give_back();
    }
    // rows of no group (forward and input gradient): zeros
    if constexpr (kMode != kWeight) {
      const uint32_t begin = p.ranges.at(0u), end = max(begin, p.ranges.at(p.ranges.count)), outside = begin + (p.ranges.n - end);
      const uint32_t t = blockIdx.x * (kGrEpilogueWarps * 32) + tid;
      const int channels = kMode == kRows ? p.n_extent : p.m_extent;
      for (uint64_t i = t; i < uint64_t(outside) * channels; i += uint64_t(gridDim.x) * (kGrEpilogueWarps * 32)) {
        const uint32_t r = static_cast<uint32_t>(i / channels), row = r < begin ? r : r - begin + end;
        store_value(static_cast<T*>(p.out) + int64_t(row) * p.out_ld + static_cast<int64_t>(i - uint64_t(r) * channels), 0.f);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512u);
  }
  if (tid == 0 && ctl->abort_flag) {
    report(p.status, FGB_S_WAIT_TIMEOUT);
    mirror_code(p.mirror, FGB_S_WAIT_TIMEOUT);
  }
}

// ------------------------------------------------------------------ pieces
// Tiles that lie in several ranges: their pieces added in order, and the tiles of empty groups (weight gradient), which no
// range holds: zeros.  gridDim.y CTAs a tile.
constexpr int kGrJoinThreads = 256;
template <int kMode, typename T>
__global__ void __launch_bounds__(kGrJoinThreads) grouped_join_kernel(const __grid_constant__ GroupedArgs p, uint32_t ctas, uint32_t tiles) {
  extern __shared__ uint32_t s_first[];
  constexpr int kParamDtype = std::is_same<T, __half>::value ? FGB_F16 : std::is_same<T, __nv_bfloat16>::value ? FGB_BF16 : FGB_F32_IEEE;
  chain_release();
  chain_wait();
  plan_groups<kMode>(p, s_first);
  const uint32_t G = p.ranges.count, total = s_first[G], length = range_length<kMode>(p, total, ctas);
  for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    uint32_t g, tile, whole;
    if constexpr (kMode == kWeight) {
      const uint32_t per = p.n_tiles * p.m_tiles;
      g = t / per, tile = t - g * per;
      whole = (s_first[g + 1u] - s_first[g]) / per;
    } else {
      whole = static_cast<uint32_t>(p.k_blocks * p.terms);
      if (uint64_t(t) * whole >= total) return;
      uint32_t lo = 0, hi = G - 1u;
      while (lo < hi) {
        const uint32_t mid = (lo + hi + 1u) / 2u;
        if (s_first[mid] <= t * whole) lo = mid;
        else hi = mid - 1u;
      }
      g = lo, tile = t - s_first[g] / whole;
    }
    const uint32_t begin = s_first[g] + tile * whole, end = begin + whole;
    const uint32_t r0 = begin / length, r1 = whole > 0u ? (end - 1u) / length : r0;
    if (whole > 0u && r0 == r1) continue;  // stored as a whole
    const uint32_t pieces = whole > 0u ? r1 - r0 + 1u : 0u;
    const size_t size = size_t(128) * p.acc_stride;
    const float* from = p.slab + (size_t(r0) * 2 + 1) * size;  // then (r0 + 1) * 2, (r0 + 2) * 2, ...
    auto sum_at = [&](uint32_t e) {
      float v = 0.f;
      if (pieces > 0u) {
        v = from[e];
#pragma unroll 8
        for (uint32_t k = 1; k < pieces; ++k) v += from[size * (2u * k - 1u) + e];
      }
      return v;
    };
    const uint32_t lo = p.ranges.at(g), hi = p.ranges.at(g + 1u);
    const uint32_t elements = 128u * p.bn, share = (elements + gridDim.y - 1u) / gridDim.y;
    const uint32_t e0 = blockIdx.y * share, e1 = min(elements, e0 + share);
    for (uint32_t e = e0 + threadIdx.x; e < e1; e += kGrJoinThreads) {
      if constexpr (kMode == kWeight) {
        const uint32_t a = e / p.bn, m = tile / p.n_tiles * 128u + a, n = tile % p.n_tiles * p.bn + (e - a * p.bn);
        if (m < static_cast<uint32_t>(p.m_extent) && n < static_cast<uint32_t>(p.n_extent))
          store_value(static_cast<T*>(p.out) + (int64_t(g) * p.m_extent + m) * p.out_ld + n, sum_at(e));
      } else {
        const uint32_t a = e / 128u, row = lo + tile / p.n_tiles * p.bn + a, m = tile % p.n_tiles * 128u + (e & 127u);
        if (row < hi && m < static_cast<uint32_t>(p.m_extent)) {
          const float b = p.bias != nullptr ? load_param(p.bias, kParamDtype, int64_t(g) * p.m_extent + m) : 0.f;
          store_value(static_cast<T*>(p.out) + int64_t(row) * p.out_ld + m, sum_at(e) + b);
        }
      }
    }
    if (kMode == kWeight && p.db != nullptr && tile % p.n_tiles == 0u && blockIdx.y == 0u && threadIdx.x < 128u) {
      const uint32_t m = tile / p.n_tiles * 128u + threadIdx.x;
      if (m < static_cast<uint32_t>(p.m_extent)) store_value(static_cast<T*>(p.db) + int64_t(g) * p.m_extent + m, sum_at(elements + threadIdx.x));
    }
  }
}

// ------------------------------------------------------------------ planes
// dst[plane][rows][cp] (16-bit) of src[rows][c]: fp32 as bf16 planes hi + mid + lo, 16-bit types as they are; columns from c
// on are zero.  A plane takes what the planes before it left, rounded to nearest; a value that would round to infinity is
// cut to the largest number instead, and nothing is left of an infinity or a NaN.
template <typename T>
__global__ void __launch_bounds__(256) grouped_planes_kernel(const T* __restrict__ src, uint16_t* __restrict__ dst, uint64_t rows, int c, int cp, int planes) {
  chain_release();
  chain_wait();
  const uint64_t total = rows * cp;
  for (uint64_t i = (uint64_t(blockIdx.x) * 256 + threadIdx.x) * 2; i < total; i += uint64_t(gridDim.x) * 512) {
    const uint64_t r = i / cp;
    const int col = static_cast<int>(i - r * cp);  // even, as cp is
    uint16_t q[3][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (sizeof(T) == 2) {
        q[0][j] = col + j < c ? reinterpret_cast<const uint16_t*>(src)[r * c + col + j] : uint16_t(0);
      } else {
        float v = col + j < c ? src[r * c + col + j] : 0.f;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          __nv_bfloat16 h = __float2bfloat16_rn(v);
          if (__hisinf(h) && !isinf(v)) h = __ushort_as_bfloat16(static_cast<unsigned short>(v < 0.f ? 0xFF7Fu : 0x7F7Fu));
          q[k][j] = __bfloat16_as_ushort(h);
          v = isfinite(v) ? v - __bfloat162float(h) : 0.f;
        }
      }
    }
    for (int k = 0; k < planes; ++k)
      *reinterpret_cast<uint32_t*>(dst + uint64_t(k) * total + i) = uint32_t(q[k][0]) | uint32_t(q[k][1]) << 16;
  }
}

// ------------------------------------------------------------------ host side
int make_rows_tmap_3d(CUtensorMap* map, const void* base, int dtype16, uint64_t d0, uint64_t d1, uint64_t d2, uint32_t b0, uint32_t b1);  // fgb_igemm.cu

static bool is_f32(int dtype) { return dtype == FGB_F32_TF32 || dtype == FGB_F32_IEEE; }

// operand [rows][c] as the kernel reads it
struct Operand {
  const void* base = nullptr;
  int cp = 0, planes = 1, dtype16 = FGB_F16;
};
static int planes_of(int dtype) { return dtype == FGB_F32_IEEE ? 3 : dtype == FGB_F32_TF32 ? 2 : 1; }
static bool needs_planes(int c, int dtype) { return is_f32(dtype) || c % 8 != 0; }
static int64_t plane_bytes(int64_t rows, int c, int dtype) {
  return needs_planes(c, dtype) ? align256(planes_of(dtype) * rows * ((c + 7) / 8 * 8) * 2) : 0;
}
// makes the planes at `at` (advanced) where they are needed
static cudaError_t make_operand(Operand& o, const void* src, int64_t rows, int c, int dtype, char*& at, cudaStream_t s) {
  o.planes = planes_of(dtype), o.dtype16 = is_f32(dtype) ? FGB_BF16 : dtype, o.cp = (c + 7) / 8 * 8;
  if (!needs_planes(c, dtype)) {
    o.base = src;
    return cudaSuccess;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(at);
  at += plane_bytes(rows, c, dtype);
  o.base = dst;
  const int64_t pairs = rows * o.cp / 2;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(pairs, 256), int64_t(device_sm_count()) * 16));
  if (is_f32(dtype))
    return launch_chained(grouped_planes_kernel<float>, dim3(grid), dim3(256), 0, s, static_cast<const float*>(src), dst, static_cast<uint64_t>(rows), c, o.cp, o.planes);
  return launch_chained(grouped_planes_kernel<__half>, dim3(grid), dim3(256), 0, s, static_cast<const __half*>(src), dst, static_cast<uint64_t>(rows), c, o.cp, 1);
}

// columns of a tile over `extent` channels: all of them in steps of 32 up to `most`, else equal tiles in steps of 64
static int tile_columns(int extent, int most) {
  if (extent <= most) return (extent + 31) / 32 * 32;
  const int whole = most / 64 * 64, tiles = (extent + whole - 1) / whole;
  return ((extent + tiles - 1) / tiles + 63) / 64 * 64;
}

struct GroupedPlan {
  int mode, bn, split;
  int64_t slots;        // pieces that the slab holds
  int64_t slab_bytes;
  uint32_t min_range;
  int acc_stride;
  int64_t tiles;        // most tiles (those that the join kernel looks at)
};

// A tile of few rows where a group has at most 64 on average: see the note on kFew above.
static bool few_rows(const fgb_grouped_linear_call& c) { return c.n <= 64 * c.groups; }

static int grouped_plan(const fgb_grouped_linear_call& c, int pass, GroupedPlan& p) {
  const int64_t sms = device_sm_count(), terms = c.dtype == FGB_F32_IEEE ? 6 : c.dtype == FGB_F32_TF32 ? 3 : 1;
  const int64_t N = c.n, G = c.groups;
  const int most = is_f32(c.dtype) ? 192 : 256;  // fp32: the blocks' sums of a tile are held in 3 x 32 registers
  int64_t iterations;
  p.split = 0, p.min_range = 0;
  if (pass == 2) {
    p.mode = kWeight;
    p.bn = tile_columns(c.ci, most);
    const int64_t per = ceil_div(c.ci, p.bn) * ceil_div(c.co, 128);
    p.tiles = G * per;
    iterations = (N / 64 + G) * per * terms;
    p.split = 1, p.min_range = 4;
  } else {
    const int nout = pass == 0 ? c.co : c.ci, k = pass == 0 ? c.ci : c.co;
    const int64_t kb = ceil_div(k, 64);
    if (few_rows(c)) {
      p.mode = kFew;
      // most groups in one tile, and no more columns than that takes
      p.bn = N <= 16 || N <= 4 * G ? 16 : N <= 16 * G ? 32 : 64;
      const int64_t m_tiles = ceil_div(nout, 128);
      p.tiles = std::min<int64_t>(N, N / p.bn + G) * m_tiles;
      iterations = p.tiles * kb * terms;
      if (p.tiles <= sms / 2 && kb * terms >= 8) p.split = 1, p.min_range = 4;
    } else {
      p.mode = kRows;
      p.bn = tile_columns(nout, most);
      p.tiles = (N / 128 + G) * ceil_div(nout, p.bn);
      iterations = p.tiles * kb * terms;
    }
  }
  if (iterations >= (int64_t(1) << 31) - 1) return FGB_E_SIZE;
  p.acc_stride = std::max(p.bn, 32) + (pass == 2 && c.grad_bias != nullptr ? 32 : 0);
  p.slots = p.split ? 2 * sms : 0;
  p.slab_bytes = align256(p.slots * 128 * p.acc_stride * 4);
  return FGB_OK;
}

static int grouped_check(const fgb_grouped_linear_call* c) {
  if (c == nullptr) return FGB_E_NULL;
  if (c->dtype != FGB_F16 && c->dtype != FGB_BF16 && !is_f32(c->dtype)) return FGB_E_DTYPE;
  if (c->offsets_bits != 32 && c->offsets_bits != 64) return FGB_E_DTYPE;
  if (c->n < 0 || c->n >= (int64_t(1) << 31) - 256 || c->groups < 1 || c->groups > kGrMaxGroups) return FGB_E_SIZE;
  if (c->ci < 1 || c->co < 1 || c->ci > 65536 || c->co > 65536) return FGB_E_SIZE;
  return FGB_OK;
}

static int64_t backward_planes(const fgb_grouped_linear_call& c) {
  return plane_bytes(c.n, c.co, c.dtype) + (c.grad_x != nullptr ? plane_bytes(c.groups * c.co, c.ci, c.dtype) : 0) +
         (c.grad_weight != nullptr ? plane_bytes(c.n, c.ci, c.dtype) : 0);
}

template <int kMode, typename T>
static int launch_grouped(const CUtensorMap& tp, const CUtensorMap& tq, GroupedArgs& a, const GroupedPlan& p, cudaStream_t s) {
  const int prefix = static_cast<int>(align256((int64_t(a.ranges.count) + 1) * 4));
  const int fixed = 1024 + kGrCtrlBytes + kGrStoreBytes + prefix;
  const int stage = kGrPBytes + a.q_bytes;
  a.stages = std::min(kGrMaxStages, (kGrSmemLimit - fixed) / stage);
  const size_t smem = size_t(fixed) + size_t(a.stages) * stage;
  static PerDeviceTable configured;
  const int rc = ensure_dynamic_smem(configured, grouped_kernel<kMode, T>, smem);
  if (rc != FGB_OK) return rc;
  const int ctas = device_sm_count();
  const unsigned grid = static_cast<unsigned>(p.split ? ctas : std::max<int64_t>(std::min<int64_t>(p.tiles, ctas), 1));
  cudaError_t e = launch_chained(grouped_kernel<kMode, T>, dim3(grid), dim3(kGrThreads), smem, s, tp, tq, a);
  if (e == cudaSuccess && p.split) {
    if constexpr (kMode != kRows) {
      const unsigned tiles = static_cast<unsigned>(p.tiles), x = std::min(tiles, 65535u * 8u);
      const unsigned y = static_cast<unsigned>(std::clamp<int64_t>(ceil_div(int64_t(ctas) * 8, tiles), 1, 64));
      e = launch_chained(grouped_join_kernel<kMode, T>, dim3(x, y), dim3(kGrJoinThreads), size_t(prefix), s, a, grid, tiles);
    }
  }
  return e != cudaSuccess ? cuda_status(e) : launch_status();
}

// one pass on operands that are ready; `features` has the rows, `other` the weight (passes 0, 1) or the second rows
static int grouped_pass(const fgb_grouped_linear_call& c, int pass, const Operand& features, const Operand& other, float* slab, cudaStream_t s) {
  GroupedPlan p{};
  int rc = grouped_plan(c, pass, p);
  if (rc != FGB_OK) return rc;
  GroupedArgs a{};
  a.ranges = RowRanges{c.offsets, c.offsets_bits == 64, static_cast<uint32_t>(c.n), static_cast<uint32_t>(c.groups)};
  a.bn = p.bn;
  a.terms = c.dtype == FGB_F32_IEEE ? 6 : c.dtype == FGB_F32_TF32 ? 3 : 1;
  // the small products first: (lo hi) (hi lo) (mid mid) (mid hi) (hi mid) (hi hi), or the last three of them
  a.p_planes = a.terms == 6 ? 0x001102u : a.terms == 3 ? 0x001u : 0u, a.q_planes = a.terms == 6 ? 0x010120u : a.terms == 3 ? 0x010u : 0u;
  a.min_range = p.min_range;
  a.acc_stride = p.acc_stride;
  a.acc_sets = 2 * p.acc_stride <= 512 ? 2 : 1;
  a.slab = slab;
  a.status = c.status, a.mirror = status_mirror(c.status);
  const uint32_t fmt = features.dtype16 == FGB_F16 ? kFmtF16 : kFmtBF16;
  a.one_pair = features.dtype16 == FGB_F16 ? 0x3C003C00u : 0x3F803F80u;
  const int eb = elem_bytes(c.dtype);
  CUtensorMap tp, tq;
  const uint64_t N = static_cast<uint64_t>(c.n), G = static_cast<uint64_t>(c.groups);
  if (pass == 2) {
    // features = dy, other = x
    a.m_extent = c.co, a.n_extent = c.ci, a.m_tiles = static_cast<int>(ceil_div(c.co, 128)), a.n_tiles = static_cast<int>(ceil_div(c.ci, p.bn));
    a.p_mn = a.q_mn = 1;
    a.q_bytes = (p.bn + 63) / 64 * 8192;
    a.out = c.grad_weight, a.out_ld = c.ci, a.db = c.grad_bias;
    rc = make_rows_tmap_3d(&tp, features.base, features.dtype16, features.cp, N, features.planes, 64, 64);
    if (rc == FGB_OK) rc = make_rows_tmap_3d(&tq, other.base, other.dtype16, other.cp, N, other.planes, 64, 64);
  } else {
    const int nout = pass == 0 ? c.co : c.ci;
    a.k_extent = pass == 0 ? features.cp : c.co;  // of the gradient, k runs over rows of the weight: as many as there are
    a.k_blocks = static_cast<int>(ceil_div(a.k_extent, 64));
    a.out = pass == 0 ? c.out : c.grad_x, a.out_ld = nout;
    a.bias = pass == 0 ? c.bias : nullptr;
    const uint64_t w_planes = G * other.planes, wc = other.cp, wr = static_cast<uint64_t>(c.co);
    const bool mn = pass == 1;
    if (p.mode == kFew) {
      a.m_extent = nout, a.n_tiles = static_cast<int>(ceil_div(nout, 128));
      a.p_mn = mn;
      a.q_bytes = (p.bn * 128 + 1023) / 1024 * 1024;
      rc = make_rows_tmap_3d(&tp, other.base, other.dtype16, wc, wr, w_planes, 64, mn ? 64 : 128);
      if (rc == FGB_OK) rc = make_rows_tmap_3d(&tq, features.base, features.dtype16, features.cp, N, features.planes, 64, p.bn);
      std::swap(a.p_planes, a.q_planes);  // the order of the terms stays: (x, W) planes
    } else {
      a.n_extent = nout, a.n_tiles = static_cast<int>(ceil_div(nout, p.bn));
      a.q_mn = mn;
      a.q_bytes = mn ? (p.bn + 63) / 64 * 8192 : p.bn * 128;
      rc = make_rows_tmap_3d(&tp, features.base, features.dtype16, features.cp, N, features.planes, 64, 128);
      if (rc == FGB_OK) rc = make_rows_tmap_3d(&tq, other.base, other.dtype16, wc, wr, w_planes, 64, mn ? 64 : p.bn);
    }
  }
  if (rc != FGB_OK) return rc;
  a.vec_ok = a.out_ld * eb % 16 == 0;
  a.idesc = make_idesc(fmt, 128, p.bn, a.p_mn, a.q_mn);
  a.idesc_ones = make_idesc(fmt, 128, 16, a.p_mn, 0);
#define FGB_GROUPED(mode)                                                              \
  (c.dtype == FGB_F16    ? launch_grouped<mode, __half>(tp, tq, a, p, s)               \
   : c.dtype == FGB_BF16 ? launch_grouped<mode, __nv_bfloat16>(tp, tq, a, p, s)        \
                         : launch_grouped<mode, float>(tp, tq, a, p, s))
  return p.mode == kRows ? FGB_GROUPED(kRows) : p.mode == kFew ? FGB_GROUPED(kFew) : FGB_GROUPED(kWeight);
#undef FGB_GROUPED
}

static bool misaligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return true;
  return false;
}

}  // namespace fgb

extern "C" int fgb_grouped_linear_max_groups(void) { return fgb::kGrMaxGroups; }

extern "C" int64_t fgb_grouped_linear_workspace_bytes(const fgb_grouped_linear_call* c, int backward) {
  using namespace fgb;
  int rc = grouped_check(c);
  if (rc != FGB_OK) return rc;
  GroupedPlan p{};
  int64_t bytes = 256;
  if (!backward) {
    rc = grouped_plan(*c, 0, p);
    bytes += p.slab_bytes + plane_bytes(c->n, c->ci, c->dtype) + plane_bytes(c->groups * c->co, c->ci, c->dtype);
    return rc != FGB_OK ? rc : bytes;
  }
  int64_t slab = 0;
  for (int pass : {1, 2}) {
    if (pass == 1 ? c->grad_x == nullptr : c->grad_weight == nullptr) continue;
    rc = grouped_plan(*c, pass, p);
    if (rc != FGB_OK) return rc;
    slab = std::max(slab, p.slab_bytes);
  }
  return bytes + slab + backward_planes(*c);
}

extern "C" int fgb_grouped_linear_forward(const fgb_grouped_linear_call* c, void* stream) {
  using namespace fgb;
  const int64_t bytes = fgb_grouped_linear_workspace_bytes(c, 0);
  if (bytes < 0) return static_cast<int>(bytes);
  if (c->n == 0) return FGB_OK;
  if (!c->x || !c->weight || !c->out || !c->offsets || !c->workspace) return FGB_E_NULL;
  if (misaligned({c->x, c->weight, c->out}) || (reinterpret_cast<uintptr_t>(c->workspace) & 255)) return FGB_E_ALIGN;
  if (c->workspace_bytes < bytes) return FGB_E_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  GroupedPlan p{};
  const int rc = grouped_plan(*c, 0, p);
  if (rc != FGB_OK) return rc;
  char* at = static_cast<char*>(c->workspace);
  float* slab = reinterpret_cast<float*>(at);
  at += p.slab_bytes;
  Operand x, w;
  cudaError_t e = make_operand(x, c->x, c->n, c->ci, c->dtype, at, s);
  if (e == cudaSuccess) e = make_operand(w, c->weight, c->groups * c->co, c->ci, c->dtype, at, s);
  return e != cudaSuccess ? cuda_status(e) : grouped_pass(*c, 0, x, w, slab, s);
}

extern "C" int fgb_grouped_linear_backward(const fgb_grouped_linear_call* c, void* stream) {
  using namespace fgb;
  const int64_t bytes = fgb_grouped_linear_workspace_bytes(c, 1);
  if (bytes < 0) return static_cast<int>(bytes);
  if (c->grad_bias != nullptr && c->grad_weight == nullptr) return FGB_E_NULL;
  if (c->grad_x == nullptr && c->grad_weight == nullptr) return FGB_OK;
  if (!c->offsets || !c->workspace || (c->grad_x != nullptr && !c->weight) || (c->n > 0 && (!c->grad_out || (c->grad_weight != nullptr && !c->x)))) return FGB_E_NULL;
  if (misaligned({c->x, c->weight, c->grad_out, c->grad_x, c->grad_weight}) || (reinterpret_cast<uintptr_t>(c->workspace) & 255)) return FGB_E_ALIGN;
  if (c->workspace_bytes < bytes) return FGB_E_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->n == 0) {
    cudaError_t e = c->grad_weight == nullptr ? cudaSuccess
                                              : cudaMemsetAsync(c->grad_weight, 0, size_t(c->groups) * c->co * c->ci * elem_bytes(c->dtype), s);
    if (e == cudaSuccess && c->grad_bias != nullptr) e = cudaMemsetAsync(c->grad_bias, 0, size_t(c->groups) * c->co * elem_bytes(c->dtype), s);
    return cuda_status(e);
  }
  const int64_t planes = backward_planes(*c);
  char* at = static_cast<char*>(c->workspace);
  float* slab = reinterpret_cast<float*>(at + planes);
  Operand g, w, x;
  cudaError_t e = make_operand(g, c->grad_out, c->n, c->co, c->dtype, at, s);
  if (e != cudaSuccess) return cuda_status(e);
  int rc = FGB_OK;
  if (c->grad_x != nullptr) {
    e = make_operand(w, c->weight, c->groups * c->co, c->ci, c->dtype, at, s);
    rc = e != cudaSuccess ? cuda_status(e) : grouped_pass(*c, 1, g, w, slab, s);
    if (rc != FGB_OK) return rc;
  }
  if (c->grad_weight != nullptr) {
    e = make_operand(x, c->x, c->n, c->ci, c->dtype, at, s);
    rc = e != cudaSuccess ? cuda_status(e) : grouped_pass(*c, 2, g, x, slab, s);
  }
  return rc;
}
