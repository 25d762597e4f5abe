// Matrix products grouped by ragged row ranges: every group g multiplies its rows by a matrix of its own, W_g [co, ci].
//
//   forward           y_r  = W_g x_r + b_g            for the rows r of group g
//   input gradient    dx_r = W_g^T dy_r
//   weight gradient   dW_g = sum_r dy_r x_r^T,  db_g = sum_r dy_r
//
// One persistent tcgen05 kernel for all of them: D[m, n] = sum_k P[m, k] Q[n, k], tiles of 128 (256 for a pair of CTAs) x BN,
// a block of 64 k a stage.
//   kRows    m = rows, n = channels of the output.  The rows of a tile may reach into the next group: what they give is not
//            stored.  The gradient reads W_g as stored, with k along its rows (MN-major operand).
//   kFew     m = channels, n = rows (16 or 32 of them): where groups have few rows the matrices are what is read, and a tile
//            of 128 rows would be mostly empty.
//   kWeight  m = co, n = ci, k = rows: both operands MN-major.  The k blocks of a group end where its rows end: a block
//            that reaches further is cut in steps of 16 rows, and what its last step holds of other rows is cleared in
//            shared memory (both operands: another group's infinity times zero would be NaN).  db comes from the same
//            blocks, as one more product with a block of ones.
// Warps: 0-7 store tiles (two per quarter of the accumulator rows), 8 loads (TMA), 9 multiplies; two accumulators in TMEM
// where they fit, so that a tile is stored while the next is multiplied.
//
// Work is dealt out in units, one after the other to the CTAs in turn: a tile, or where there are too few tiles to go round
// (the weight gradient; a few rows) one of the equal parts of its blocks of k.  The parts of a group's tiles that
// read the same k are neighbours, so that they find it in L2: equal ranges of one long line of blocks, which need no
// rounding up, read everything from memory once for each tile (16 groups of 8192 rows, 1024 x 1024: 422 us).  A tile in parts
// leaves fp32 pieces in a slab, which a second kernel adds up in their order.  Every CTA finds the number of parts from the
// sizes alone, so results do not depend on the run.
//
// fp32 operands are written as sums of bf16 planes (hi + mid + lo, 8 bits each) and multiplied plane by plane: six products
// (all whose weight is 2^-16 and more) for accurate fp32, three (2^-8 and more) where TF32 is allowed.  A plane leaves half a step of
// eight bits, 2^-8, of what it takes, so that four terms of 2^-24 of a product are left out, or three of 2^-16.  bf16 has
// fp32's range, so no scaling is needed, and six of them cost what three TF32 products do (half the rate, twice the bytes).
// The tensor cores cut what they add to an accumulator at its last bit instead of rounding: over a long k that is a bias, 5e-8 to 8e-8 of
// the sum for every 16 k where all terms have one sign (a weight gradient of 6400 / 25600 / 102400 rows that is not cut: 2e-5, 1.3e-4, 3.0e-4
// low).  16-bit results take that: half a step of fp16 is 4.9e-4, of bf16 3.9e-3, and where tiles are fewer than the CTAs have time for,
// their parts are added in fp32.  fp32 leaves the accumulator after each block of 64 k, the small
// products first, the large one last, and the storing warps add the blocks up in registers, rounding to nearest.  A stage has
// all planes of its block: each is loaded once for the two or three products that it is in.
#include <algorithm>
#include <type_traits>

#include "fgb_common.cuh"
#include "fgb_device.cuh"
#include "fgb_rows.cuh"
#include "fgb_umma.cuh"

namespace fgb {

// Measured (B200): 131072 rows of 16 groups, 1024 x 1024 bf16: forward 195 to 210 us, input gradient 211, weight gradient 254 and 21
// for the join (one cuBLAS product of that size 209, 209, 210; the clock is at the power cap); 166000 of 27, 256 x 256 fp16: 33, 33
// and 54 (33, 33, 45), forward at 80 % of the copy rate; 24 rows of 64 groups, 512 -> 1024: 8 us, a chain of plan, loads,
// products and stores (the touched matrices alone take 4).  40000 of 4, 256 x 256 fp32: forward 67 us.
constexpr int kGrThreads = 320;
constexpr int kGrEpilogueWarps = 8;
constexpr int kGrMaxStages = 12;
constexpr int kGrMaxGroups = 2048;
constexpr int kGrSmemLimit = 227 * 1024;  // all of it dynamic
constexpr int kGrOnesBytes = 2048;        // 16 columns of 64 k
constexpr int kGrPBytes = 128 * 128;

enum { kRows = 0, kFew = 1, kWeight = 2 };

struct GroupedArgs {
  RowRanges ranges;
  int bn;               // columns of a tile
  int tile_m;           // rows of it: 128, or 256 of a pair of CTAs
  int row_shift;        // kRows, kFew: log2 of the rows that a tile has of a group (tile_m; bn)
  int n_tiles;          // tiles along the channels that are not rows: kRows along n, kFew along m, kWeight along n
  int m_tiles;          // kWeight: tiles along co
  int k_blocks;         // kRows, kFew: blocks of 64 along k
  int k_extent;         // kRows, kFew: k
  int planes;           // of an operand
  int terms;            // products of planes
  uint32_t p_planes, q_planes;  // their planes, four bits a term
  int p_mn, q_mn;       // operand is MN-major
  int stages, q_bytes, acc_sets, acc_stride;
  uint32_t min_part;    // blocks of k that a part of a tile has at least; 0: tiles are not cut
  float piece_cost;     // what writing and adding up a piece takes, in blocks
  uint32_t* plan;       // where tiles are cut: the schedule, for the kernel that adds the pieces up
  uint32_t idesc, idesc_ones;
  uint32_t one_pair;    // two ones of the operand type
  const void* bias;     // [groups, nout] or null
  void* out;
  void* db;             // kWeight: [groups, co] or null
  float* slab;          // pieces of tiles: [tile_m][bn] each (kFew [bn][128])
  float* db_parts;      // kWeight: [units][tile_m], the unit's share of db
  int m_extent, n_extent;  // channels: kRows n; kFew m; kWeight m and n
  int out_ld;
  int vec_ok;           // rows of the output are whole 16-byte pieces
  int32_t* status;
  int32_t* mirror;
};

struct GroupedSmem {
  uint64_t full[kGrMaxStages], empty[kGrMaxStages];
  uint64_t peer_full[kGrMaxStages];  // pairs: the other CTA has cleared its operands of a stage
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drained;  // only after a wait that gave up: the products in flight
  uint32_t tmem_base, abort_flag;
};

// Shared memory: the stages (a multiple of 1024 bytes, as the ones behind them need it), the storing warps' buffers, a block of ones
// (kWeight) or those warps' bias (kRows), the barriers, the schedule.  Packed, so that a pair of CTAs has six stages of 32 KB:
// the products wait for loads half as long as with five.
template <int kMode, typename T>
__host__ __device__ constexpr int grouped_store_bytes() {  // of a storing warp: 32 rows of 64 or 128 bytes
  return sizeof(T) == 4 ? 2048 : 4096;
}
template <int kMode, typename T>
__host__ __device__ constexpr int grouped_extra_bytes() {
  return kMode == kWeight ? kGrOnesBytes : kMode == kRows ? kGrEpilogueWarps * 128 * static_cast<int>(sizeof(T)) : 0;
}
static_assert(sizeof(GroupedSmem) % 8 == 0, "the schedule follows the barriers");

// The rows and tiles of group g, and the blocks of k of a tile; `offsets` are those of the groups in shared memory
struct GroupSize {
  uint32_t lo, hi, tiles, whole;
};
template <int kMode>
__device__ __forceinline__ GroupSize group_size(const GroupedArgs& p, const uint32_t* offsets, uint32_t g) {  // tiles of tile_m rows, or of bn where n is rows
  GroupSize s;
  s.lo = offsets[g];
  s.hi = offsets[g + 1u];
  const uint32_t len = s.hi - s.lo;
  if constexpr (kMode != kWeight) s.tiles = ((len + (1u << p.row_shift) - 1u) >> p.row_shift) * p.n_tiles;
  else s.tiles = len > 0u ? p.n_tiles * p.m_tiles : 0u;
  s.whole = kMode == kWeight ? (len + 63u) / 64u : static_cast<uint32_t>(p.k_blocks);
  return s;
}
// length of the parts of a tile of `whole` blocks where `unit` are wanted: all parts but the last alike
__device__ __forceinline__ uint32_t part_length(const GroupedArgs& p, uint32_t whole, uint32_t unit) {
  if (p.min_part == 0u || whole <= unit) return whole;
  const uint32_t parts = min((whole + unit - 1u) / unit, max(whole / p.min_part, 1u));
  return (whole + parts - 1u) / parts;
}
__device__ __forceinline__ uint32_t parts_of(uint32_t whole, uint32_t length) {
  return length == 0u ? 0u : length == whole ? 1u : (whole + length - 1u) / length;
}

// What every CTA works out at its start: first[g] = units of the groups before g, piece[g] = pieces of tiles before g, the
// groups' offsets, and the length that parts should have.  The whole CTA calls it (and waits at its end).
//
// Cut tiles: 31 lengths between twice and a third of a CTA's share of the blocks (and none: whole tiles) are weighed by what
// the CTA with the most work then has -- rounds of equal units, or the share and half a unit where they differ -- and by
// the pieces.
constexpr int kGrMostUnits = 3;  // units of a CTA, on average, at the smallest length
struct GroupedSchedule {
  uint32_t* first;
  uint32_t* piece;
  uint32_t* offsets;
  uint32_t unit;
};
inline int64_t schedule_bytes(int64_t groups) { return (groups + 1) * 12 + 4; }
template <int kMode>
__device__ __forceinline__ GroupedSchedule plan_groups(const GroupedArgs& p, uint32_t* s_first, float* costs, uint32_t ctas) {
  const uint32_t G = p.ranges.count, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  GroupedSchedule plan{s_first, s_first + G + 1u, s_first + 2u * (G + 1u), 0xFFFFFFFFu};
  bool bad = false;
  for (uint32_t g = threadIdx.x; g <= G; g += blockDim.x) {
    plan.offsets[g] = p.ranges.at(g);
    bad |= g < G && !p.ranges.good(g);
  }
  // ranges that overlap could ask for more tiles than there is room for: nothing is done
  bad = __syncthreads_or(bad) != 0;
  if (bad && threadIdx.x == 0) {
    report(p.status, FGB_S_BAD_OFFSETS);
    mirror_code(p.mirror, FGB_S_BAD_OFFSETS);
  }
  if (p.min_part != 0u && !bad) {
    // every warp: all blocks of k
    unsigned long long total = 0;
    for (uint32_t g = lane; g < G; g += 32u) {
      const GroupSize z = group_size<kMode>(p, plan.offsets, g);
      total += static_cast<unsigned long long>(z.tiles) * z.whole;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float share = static_cast<float>(total) / static_cast<float>(ctas);
    auto unit_of = [&](uint32_t i) { return i == 31u ? 0xFFFFFFFFu : max(static_cast<uint32_t>(ceilf(share * 2.f * exp2f(-2.5849625f / 30.f * static_cast<float>(i)))), 1u); };
    for (uint32_t i = warp; i < 32u; i += blockDim.x / 32u) {
      const uint32_t unit = unit_of(i);
      uint32_t units = 0, pieces = 0, longest = 0, shortest = 0xFFFFFFFFu;
      for (uint32_t g = lane; g < G; g += 32u) {
        const GroupSize z = group_size<kMode>(p, plan.offsets, g);
        if (z.tiles == 0u) continue;
        const uint32_t len = part_length(p, z.whole, unit), parts = parts_of(z.whole, len);
        units += parts * z.tiles;
        if (parts > 1u) pieces += parts * z.tiles;
        longest = max(longest, len), shortest = min(shortest, len);
      }
      units = __reduce_add_sync(0xffffffffu, units), pieces = __reduce_add_sync(0xffffffffu, pieces);
      longest = __reduce_max_sync(0xffffffffu, longest), shortest = __reduce_min_sync(0xffffffffu, shortest);
      const float len = static_cast<float>(longest);
      const float most = longest == shortest ? static_cast<float>((units + ctas - 1u) / ctas) * len : fmaxf(share + 0.5f * len, len);
      if (lane == 0u) costs[i] = most + static_cast<float>(pieces) / static_cast<float>(ctas) * p.piece_cost;
    }
    __syncthreads();
    // the cheapest, of equally cheap ones the longest
    const uint32_t cost = __float_as_uint(costs[lane]), least = __reduce_min_sync(0xffffffffu, cost);
    plan.unit = unit_of(static_cast<uint32_t>(__ffs(__ballot_sync(0xffffffffu, cost == least)) - 1));
  }
  for (uint32_t g = threadIdx.x; g < G; g += blockDim.x) {
    const GroupSize z = group_size<kMode>(p, plan.offsets, g);
    const uint32_t parts = bad ? 0u : parts_of(z.whole, part_length(p, z.whole, plan.unit));
    plan.first[g + 1u] = parts * z.tiles;
    plan.piece[g + 1u] = parts > 1u ? parts * z.tiles : 0u;
  }
  __syncthreads();
  if (warp < 2) {
    uint32_t* v = warp == 0 ? plan.first : plan.piece;
    uint32_t run = 0;
    for (uint32_t g0 = 0; g0 < G; g0 += 32u) {
      uint32_t x = g0 + lane < G ? v[g0 + lane + 1u] : 0u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= static_cast<uint32_t>(d)) x += o;
      }
      if (g0 + lane < G) v[g0 + lane + 1u] = run + x;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) v[0] = 0u;
  }
  __syncthreads();
  if (p.min_part != 0u && blockIdx.x == 0) {
    for (uint32_t i = threadIdx.x; i < 3u * (G + 1u); i += blockDim.x) p.plan[i] = s_first[i];
    if (threadIdx.x == 0) p.plan[3u * (G + 1u)] = plan.unit;
  }
  return plan;
}

// A tile, or the part of one that is a unit
struct GroupedItem {
  uint32_t group, tile;     // tile within the group
  uint32_t from, to;        // its blocks of k
  uint32_t lo, hi;          // rows of the group
  uint32_t piece;           // its place in the slab, or kInvalid for a whole tile
  uint32_t unit;
};

// walks the units of a CTA: every role goes through the same sequence (whole warps)
template <int kMode>
struct GroupedWalk {
  const GroupedArgs& p;
  const GroupedSchedule& plan;
  uint32_t at, step, total, group = 0;
  __device__ __forceinline__ GroupedWalk(const GroupedArgs& p_, const GroupedSchedule& plan_, uint32_t ctas, uint32_t cta)
      : p(p_), plan(plan_), at(cta), step(ctas), total(plan_.first[p_.ranges.count]) {}
  __device__ __forceinline__ bool next(GroupedItem& it) {
    if (at >= total) return false;
    // the last group that begins at or before `at` (not an empty one): `at` only grows, and 32 groups are looked at at a time
    for (uint32_t passed = 32u; passed == 32u; group += passed) {
      const uint32_t ahead = group + 1u + (threadIdx.x & 31u);
      passed = __popc(__ballot_sync(0xffffffffu, ahead < p.ranges.count && plan.first[ahead] <= at));
    }
    const uint32_t lo = group;
    const GroupSize z = group_size<kMode>(p, plan.offsets, lo);
    const uint32_t length = part_length(p, z.whole, plan.unit), local = at - plan.first[lo], part = length < z.whole ? local / z.tiles : 0u;
    it.group = lo;
    it.tile = local - part * z.tiles;
    it.from = part * length, it.to = min(z.whole, it.from + length);
    it.lo = z.lo, it.hi = z.hi;
    it.piece = length < z.whole ? plan.piece[lo] + local : kInvalid;
    it.unit = at;
    at += step;
    return true;
  }
  // all that the products of kRows have to know of a unit: it is a whole tile
  __device__ __forceinline__ bool next_whole(GroupedItem& it) {
    if (at >= total) return false;
    it.from = 0u, it.to = static_cast<uint32_t>(p.k_blocks);
    at += step;
    return true;
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
__device__ __forceinline__ void store_columns(uint32_t (&acc)[32], uint8_t* stage, int lane, int c0, T* out, int64_t ld, int rows, int cols, int vec_ok) {
  constexpr int kPiece = 16 / sizeof(T), kCols = 4 * kPiece;  // columns of a piece, and of 64 bytes
  uint8_t* mine = stage + lane * 64;
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

// After a wait that gave up: what is in flight is waited for, with a limit of its own.  Not inlined: nothing comes here otherwise.
// The copies of the last blocks; those of a pair's second CTA count on the leader's barriers, and get a time in which copies end.
__noinline__ __device__ void drain_copies(GroupedSmem* ctl, uint32_t stages, uint32_t issued, uint32_t rank) {
  if (rank == 0u) {
    uint32_t late = 0;
    for (uint32_t b = issued - min(issued, stages); b != issued; ++b) mbar_wait(&ctl->full[b % stages], b / stages & 1u, &late);
  } else {
    for (const uint64_t t0 = global_timer_ns(); global_timer_ns() - t0 < 100000u;) __nanosleep(1000);
  }
}
template <bool kPair>
__noinline__ __device__ void drain_products(GroupedSmem* ctl) {
  uint32_t late = 0;
  const uint32_t bar = smem_u32(&ctl->drained);
  if constexpr (kPair) umma_commit_pair(cluster_map(bar, 0));
  else umma_commit(bar);
  mbar_wait(&ctl->drained, 0, &late);
}

// kPair: launched as clusters of two CTAs, which work on tiles of 256 rows together: each loads its 128 rows and half of the
// columns, the first CTA (the leader) issues products over both CTAs' operands, each gets its rows' accumulators.  A CTA loads
// 32 KB a stage instead of 48 for the same products: with one CTA a tile L2's rate to the SMs was the bound.
template <int kMode, typename T, bool kPair>
__global__ void __launch_bounds__(kGrThreads, 1) grouped_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                                                                const __grid_constant__ CUtensorMap tmap_o, const __grid_constant__ GroupedArgs p) {
  constexpr int kParamDtype = std::is_same<T, __half>::value ? FGB_F16 : std::is_same<T, __nv_bfloat16>::value ? FGB_BF16 : FGB_F32_IEEE;
  constexpr bool kBlocks = std::is_same<T, float>::value;  // the accumulator is emptied after every block of 64 k
  constexpr int kSums = kMode == kFew ? 1 : 3;             // blocks of 32 columns that a storing warp adds up
  constexpr int kStore = grouped_store_bytes<kMode, T>();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if ((smem_u32(smem_raw) & 1023u) != 0u) {  // the operands' swizzle needs it; no static shared memory is in the way
    if (threadIdx.x == 0) report(p.status, FGB_S_WAIT_TIMEOUT);
    return;
  }
  uint8_t* stages = smem_raw;
  const int planes = kBlocks ? p.planes : 1, terms = kBlocks ? p.terms : 1;
  const int plane_bytes = kGrPBytes + p.q_bytes, stage_bytes = planes * plane_bytes;  // of a plane: P, then Q
  uint8_t* store = stages + size_t(p.stages) * stage_bytes;
  uint8_t* ones = store + kGrEpilogueWarps * kStore;
  T* s_bias = reinterpret_cast<T*>(ones);  // of the storing warps' columns: 128 each
  GroupedSmem* ctl = reinterpret_cast<GroupedSmem*>(ones + grouped_extra_bytes<kMode, T>());
  uint32_t* first = reinterpret_cast<uint32_t*>(ctl + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = kPair ? cluster_ctarank() : 0u;
  const int half = kPair ? p.bn / 2 : p.bn;  // columns whose operand this CTA holds
  const uint32_t workers = kPair ? gridDim.x / 2u : gridDim.x, worker = kPair ? blockIdx.x / 2u : blockIdx.x;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  // A wait that gives up raises the CTA's abort flag: no load is issued after that, products run on what is there, nothing is
  // stored, and what is in flight is waited for (again with a limit).
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag); };

  chain_release();
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
      mbar_init(&ctl->peer_full[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&ctl->acc_full[a], 1);
      mbar_init(&ctl->acc_empty[a], kPair ? 2 * kGrEpilogueWarps : kGrEpilogueWarps);
    }
    mbar_init(&ctl->drained, 1);
    ctl->abort_flag = 0;
    mbar_init_fence();
  }
  if (kMode == kWeight) {
    for (int i = tid; i < kGrOnesBytes / 4; i += kGrThreads) reinterpret_cast<uint32_t*>(ones)[i] = p.one_pair;
    fence_proxy_async_smem();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
  }
  if (warp == 9) {
    if constexpr (kPair) {
      tmem_alloc_pair(&ctl->tmem_base, 512u);
    } else {
      tmem_alloc_dyn(&ctl->tmem_base, 512u);
      tmem_relinquish();
    }
  }
  // some 1000 cycles until the other CTA knows these barriers: the plan is made meanwhile
  if constexpr (kPair) cluster_arrive();
  chain_wait();
  const GroupedSchedule plan = plan_groups<kMode>(p, first, reinterpret_cast<float*>(store), workers);
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) cluster_wait();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  GroupedWalk<kMode> walk(p, plan, workers, worker);
  GroupedItem it;

  // where the rows and columns of an item's tile begin
  auto m_tile_of = [&](const GroupedItem& t) { return kMode == kFew ? t.tile % p.n_tiles : t.tile / p.n_tiles; };
  auto n_tile_of = [&](const GroupedItem& t) { return kMode == kFew ? t.tile / p.n_tiles : t.tile % p.n_tiles; };
  // the bias gradient's products: of a block of k in one of the tiles that read the same rows of dy, in turn
  auto ones_in = [&](const GroupedItem& t, uint32_t kb) { return kMode == kWeight && p.db != nullptr && kb % p.n_tiles == n_tile_of(t); };

  const uint32_t stage0 = smem_u32(stages);
  if (warp == 8) {
    // ------------------------------------------------------------------ loads
    // One elected lane goes through all blocks of a unit (elect picks the same lane each time).
    uint32_t s = 0, ph = 0, issued = 0;
    bool stopped = false;
    const int G = static_cast<int>(p.ranges.count);
    const uint32_t full_own = smem_u32(&ctl->full[0]), full_leader = kPair ? cluster_map(full_own, 0) : full_own;
    while (walk.next(it)) {
      if (elect_one()) {
        // first row (or channel) of the tile along m and n, first k
        const int m0 = static_cast<int>(m_tile_of(it) * p.tile_m + rank * 128u), n0 = static_cast<int>(n_tile_of(it) * p.bn + rank * half);
        const int lo = static_cast<int>(it.lo), g = static_cast<int>(it.group), len = static_cast<int>(it.hi - it.lo);
        const int k_end = static_cast<int>(it.to * 64u);
        for (int k0 = static_cast<int>(it.from * 64u); k0 < k_end; k0 += 64) {
          const bool cleared = kMode == kWeight && k0 + 64 > len && (len & 15) != 0;  // see the products
          if (stopped || !wait(&ctl->empty[s], ph ^ 1)) {
            stopped = true;
            break;
          }
          // Pairs: both CTAs' bytes count on the leader's barrier, so that it has one to wait for -- but for a block that
          // either has to clear rows of first.
          const bool shared = kPair && !cleared;
          const uint32_t full = shared ? full_leader + 8u * s : full_own + 8u * s;
          if (!shared || rank == 0u) mbar_arrive_expect_tx(&ctl->full[s], static_cast<uint32_t>(shared ? 2 * stage_bytes : stage_bytes));
          auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2) {
            if constexpr (kPair) tma_load_3d_pair(dst, map, full, c0, c1, c2);
            else tma_load_3d(dst, map, &ctl->full[s], c0, c1, c2);
          };
          uint32_t pd = stage0 + s * stage_bytes;
          for (int i = 0; i < planes; ++i, pd += plane_bytes) {
            const uint32_t qd = pd + kGrPBytes;
            if constexpr (kMode == kRows) {
              load(pd, &tmap_p, k0, lo + m0, i);
              if (p.q_mn) {
                for (int c = 0; c * 64 < half; ++c) load(qd + c * 8192, &tmap_q, n0 + c * 64, k0, i * G + g);
              } else {
                load(qd, &tmap_q, k0, n0, i * G + g);
              }
            } else if constexpr (kMode == kFew) {
              if (p.p_mn) {
                for (int c = 0; c < 2; ++c) load(pd + c * 8192, &tmap_p, m0 + c * 64, k0, i * G + g);
              } else {
                load(pd, &tmap_p, k0, m0, i * G + g);
              }
              load(qd, &tmap_q, k0, lo + n0, i);
            } else {
              for (int c = 0; c < 2; ++c) load(pd + c * 8192, &tmap_p, m0 + c * 64, lo + k0, i);
              for (int c = 0; c * 64 < half; ++c) load(qd + c * 8192, &tmap_q, n0 + c * 64, lo + k0, i);
            }
          }
          if (++s == static_cast<uint32_t>(p.stages)) s = 0, ph ^= 1;
          ++issued;
        }
      }
      __syncwarp();
    }
    if (elect_one() && *abort_flag != 0u) drain_copies(ctl, static_cast<uint32_t>(p.stages), issued, rank);
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------ products
    // One elected lane goes through all blocks of a unit and carries the ring's and the accumulators' state; the descriptors
    // move by one addition, and the next block's barrier is looked at behind the products.  With the whole warp in the loop and
    // a lane elected for each block the instructions around four products took 690 cycles, more than their 512: 131072 rows of
    // 16 groups, 1024 x 1024: 229 us, 217 with this loop, 210 with a sixth stage.  The whole warp clears rows, in the last block of a group (kWeight).
    const bool leader = rank == 0u;
    const uint32_t p_step = kMode == kWeight || p.p_mn ? 128u : 2u, q_step = kMode == kWeight || p.q_mn ? 128u : 2u;
    const uint32_t p_lbo = kMode == kWeight || p.p_mn ? 8192u : 16u, q_lbo = kMode == kWeight || p.q_mn ? 8192u : 16u;
    const uint64_t d_ones = make_smem_desc(smem_u32(ones), 16, 1024);
    // the low half of a descriptor holds the address: it moves, the high half stays
    const uint64_t dp0 = make_smem_desc(stage0, p_lbo, 1024), dq0 = make_smem_desc(stage0 + kGrPBytes, q_lbo, 1024);
    const uint64_t dp_high = dp0 >> 32 << 32, dq_high = dq0 >> 32 << 32;
    const uint32_t dp_low = static_cast<uint32_t>(dp0), dq_low = static_cast<uint32_t>(dq0);
    const uint32_t stage_step = static_cast<uint32_t>(stage_bytes) >> 4, plane_step = static_cast<uint32_t>(plane_bytes) >> 4;
    const uint32_t tmem0 = tmem_base, peer_full0 = kPair ? cluster_map(smem_u32(&ctl->peer_full[0]), 0) : 0u;
    const uint32_t empty0 = smem_u32(&ctl->empty[0]), acc_full0 = smem_u32(&ctl->acc_full[0]);
    const uint32_t empty1 = kPair ? cluster_map(empty0, 1) : 0u, acc_full1 = kPair ? cluster_map(acc_full0, 1) : 0u;
    auto product = [&](uint32_t acc, uint64_t dp, uint64_t dq, uint32_t idesc, uint32_t add) {
      if constexpr (kPair) umma_ss_pair(acc, dp, dq, idesc, add);
      else umma_ss<false>(acc, dp, dq, idesc, add);
    };
    auto commit = [&](uint32_t bar0, uint32_t bar1, uint32_t i) {  // barrier i, in both CTAs of a pair
      if constexpr (kPair) {
        umma_commit_pair(bar0 + 8u * i);
        umma_commit_pair(bar1 + 8u * i);
      } else {
        umma_commit(bar0 + 8u * i);
      }
    };
    // the elected lane's: stage, its phase and offset; accumulator set; whose turn it is to multiply with ones (0: ours)
    uint32_t s = 0, ph = 0, at = 0, set = 0, set_ph = 0, acc = 0, turn = 0, any_ones = 0;
    bool ready = false;  // the stage has been seen full
    auto block = [&](bool begins, bool ends, uint32_t steps, bool look_ahead) {
      if (begins) {  // a new accumulator
        wait(&ctl->acc_empty[set], set_ph ^ 1);
        tc_fence_after_sync();
        acc = tmem0 + set * p.acc_stride;
        any_ones = 0;
      }
      const bool with_ones = kMode == kWeight && p.db != nullptr && turn == 0u;
      for (int term = 0; term < terms; ++term) {
        const uint32_t pp = (p.p_planes >> (4 * term)) & 15u, pq = (p.q_planes >> (4 * term)) & 15u;
        const uint32_t da = dp_low + at + (kBlocks ? pp * plane_step : 0u), db = dq_low + at + (kBlocks ? pq * plane_step : 0u);
        const bool ones_now = with_ones && (!kBlocks || pq == 0u);  // once for each plane of dy
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if (kMode == kWeight && k >= steps) break;  // elsewhere what is behind the last k has been filled with zeros
          product(acc, dp_high | (da + k * p_step), dq_high | (db + k * q_step), p.idesc, k == 0 && term == 0 && begins ? 0u : 1u);
          if (ones_now) product(acc + p.bn, dp_high | (da + k * p_step), d_ones, p.idesc_ones, k == 0 ? any_ones : 1u);
        }
        if (ones_now) any_ones = 1u;
      }
      commit(empty0, empty1, s);
      if (ends) {  // the accumulator is done
        commit(acc_full0, acc_full1, set);
        if (++set == static_cast<uint32_t>(p.acc_sets)) set = 0, set_ph ^= 1;
      }
      at += stage_step;
      if (++s == static_cast<uint32_t>(p.stages)) s = 0, at = 0, ph ^= 1;
      if (kMode == kWeight && ++turn == static_cast<uint32_t>(p.n_tiles)) turn = 0u;
      ready = look_ahead && mbar_try_wait(&ctl->full[s], ph);
    };
    // the whole warp's: blocks before the unit; a bit for each stage: the phases of the barriers that only cleared blocks use
    uint32_t done = 0, own_ph = 0, peer_ph = 0;
    while (kMode == kRows ? walk.next_whole(it) : walk.next(it)) {
      const uint32_t n_blocks = it.to - it.from;
      const uint32_t valid = kMode == kWeight ? min(it.hi - it.lo - (it.to - 1u) * 64u, 64u) : 64u;  // k of the last block
      const uint32_t steps = (valid + 15u) / 16u;
      const bool cleared = kMode == kWeight && (valid & 15u) != 0u;
      const uint32_t plain = n_blocks - (cleared ? 1u : 0u);
      if (leader) {
        if (elect_one()) {
          turn = kMode == kWeight ? (it.from + p.n_tiles - n_tile_of(it)) % p.n_tiles : 0u;
          for (uint32_t kb = 0; kb < plain; ++kb) {
            if (!ready) wait(&ctl->full[s], ph);
            block(kBlocks || kb == 0u, kBlocks || kb + 1u == n_blocks, kb + 1u == n_blocks ? steps : 4u, kb + 1u < plain);
          }
        }
        __syncwarp();
      }
      if (cleared) {
        // rows of other groups in the last step: cleared in both operands
        const uint32_t stage = (done + plain) % static_cast<uint32_t>(p.stages);
        if (leader) {
          wait(&ctl->full[stage], (done + plain) / static_cast<uint32_t>(p.stages) & 1u);
        } else {
          wait(&ctl->full[stage], own_ph >> stage & 1u);
          own_ph ^= 1u << stage;
        }
        __syncwarp();
        const uint32_t chunks = static_cast<uint32_t>(stage_bytes) / 8192u, rows = steps * 16u - valid;
        uint8_t* from = stages + size_t(stage) * stage_bytes;
        for (uint32_t c = 0; c < chunks; ++c)
          for (uint32_t r = lane >> 3; r < rows; r += 4u)
            *reinterpret_cast<uint4*>(from + c * 8192u + (valid + r) * 128u + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if constexpr (kPair) {
          // the peer's ordinary stores: cluster scope on both sides, here only (a wait of that scope takes some 1000 cycles)
          if (leader) mbar_wait_cluster(&ctl->peer_full[stage], peer_ph >> stage & 1u, abort_flag);
          else if (lane == 0) mbar_arrive_cluster_release(peer_full0 + 8u * stage);
          peer_ph ^= 1u << stage;
          __syncwarp();
        }
        if (leader) {
          if (elect_one()) {
            if (plain == 0u) turn = (it.from + p.n_tiles - n_tile_of(it)) % p.n_tiles;
            block(kBlocks || plain == 0u, true, steps, false);
          }
          __syncwarp();
        }
      }
      done += n_blocks;
    }
    if (leader && elect_one() && *abort_flag != 0u) drain_products<kPair>(ctl);
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ stores
    const int quarter = warp & 3, group = warp >> 2;
    uint8_t* stage = store + warp * kStore;
    T* bias_buf = s_bias + warp * 128;
    uint32_t set = 0, set_ph = 0;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t acc_empty[2] = {kPair ? cluster_map(smem_u32(&ctl->acc_empty[0]), 0) : 0u, kPair ? cluster_map(smem_u32(&ctl->acc_empty[1]), 0) : 0u};
    auto wait_full = [&]() {
      wait(&ctl->acc_full[set], set_ph);
      tc_fence_after_sync();
      return tmem_base + set * p.acc_stride + lanes;
    };
    auto give_back = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_cluster(acc_empty[set]);
        else mbar_arrive(&ctl->acc_empty[set]);
      }
      if (++set == static_cast<uint32_t>(p.acc_sets)) set = 0, set_ph ^= 1;
    };
    // This warp's columns: the [kOwn group, kOwn group + kOwn) of every 2 kOwn.
    constexpr int kOwn = kBlocks || kMode == kFew ? 32 : 64;
    // The next unit, and the bias of its columns, are looked up while this one's accumulator is waited for and stored.
    const bool with_bias = kMode == kRows && p.bias != nullptr;
    float bias[4];
    GroupedItem next;
    auto look_up = [&]() {
      const bool more = walk.next(next);
      if (with_bias && more) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int in = kOwn == 32 ? group * 32 + b * 64 + lane : group * 64 + (b / 2) * 128 + (b % 2) * 32 + lane, c = static_cast<int>(n_tile_of(next)) * p.bn + in;
          bias[b] = in < p.bn && c < p.n_extent ? load_param(p.bias, kParamDtype, int64_t(next.group) * p.n_extent + c) : 0.f;
        }
      }
      return more;
    };
    for (bool more = look_up(); more;) {
      it = next;
      if (with_bias) {
        __syncwarp();
#pragma unroll
        for (int b = 0; b < 4; ++b) bias_buf[b * 32 + lane] = static_cast<T>(bias[b]);  // as it was given
        __syncwarp();
      }
      more = look_up();
      const int in_tile = static_cast<int>(rank) * 128 + quarter * 32;  // the warp's first row within the tile
      const int m0 = static_cast<int>(m_tile_of(it)) * p.tile_m + in_tile, n0 = static_cast<int>(n_tile_of(it)) * p.bn;
      const bool whole = it.piece == kInvalid;
      const bool with_db = kMode == kWeight && p.db != nullptr && group == 0;
      float* piece = whole ? nullptr : p.slab + size_t(it.piece) * p.tile_m * p.bn;
      const int64_t row0 = kMode == kRows ? int64_t(it.lo) + m0 : int64_t(it.group) * p.m_extent + m0;
      const int rows = (kMode == kRows ? static_cast<int>(it.hi - it.lo) : p.m_extent) - m0;
      constexpr int kBias = 16 / sizeof(T);
      auto add_bias = [&](uint32_t (&acc)[32], int b) {
        if (!with_bias) return;
#pragma unroll
        for (int i = 0; i < 32; i += kBias) {
          float v[kBias];
          Channels<T, kBias>::unpack(*reinterpret_cast<const typename Channels<T, kBias>::Raw*>(bias_buf + b * 32 + i), v);
#pragma unroll
          for (int j = 0; j < kBias; ++j) acc[i + j] = __float_as_uint(__uint_as_float(acc[i + j]) + v[j]);
        }
      };
      // 32 columns by ordinary stores; `b`: their place among the warp's columns
      auto put = [&](uint32_t (&acc)[32], int c0, int b) {
        if constexpr (kMode == kFew) {
          const int left = static_cast<int>(it.hi - it.lo) - n0;  // rows of the tile, and more
          const float few_bias =
              whole && p.bias != nullptr && m0 + lane < p.m_extent ? load_param(p.bias, kParamDtype, int64_t(it.group) * p.m_extent + m0 + lane) : 0.f;
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
          store_columns<float>(acc, stage, lane, c0, piece + size_t(in_tile) * p.bn, p.bn, 32, p.bn, 1);
        } else {
          add_bias(acc, b);
          store_columns<T>(acc, stage, lane, c0, static_cast<T*>(p.out) + row0 * p.out_ld + n0, p.out_ld, rows, p.n_extent - n0, p.vec_ok);
        }
      };
      if constexpr (kBlocks) {
        uint32_t sum[kSums][32];
        float db = 0.f;
#pragma unroll
        for (int b = 0; b < kSums; ++b)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[b][i] = 0u;
        for (uint32_t at = it.from; at < it.to; ++at) {
          const uint32_t tmem = wait_full();
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
          if (with_db && ones_in(it, at)) {
            uint32_t acc[32];
            tmem_ld_32x32(tmem + p.bn, acc);
            tmem_ld_wait();
            db += __uint_as_float(acc[0]);
          }
          give_back();
        }
        if (*abort_flag == 0u) {  // else nothing that was waited for is there, and the status word says so
#pragma unroll
          for (int b = 0; b < kSums; ++b)
            if (group * 32 + b * 64 < p.bn) put(sum[b], group * 32 + b * 64, b);
          if (with_db) p.db_parts[size_t(it.unit) * p.tile_m + in_tile + lane] = db;
        }
      } else {
        const uint32_t tmem = wait_full();
        const bool fine = *abort_flag == 0u;
        // the first of the unit's blocks whose turn it was, if there is one
        if (with_db) {
          float db = 0.f;
          if (it.from + (n_tile_of(it) + p.n_tiles - it.from % p.n_tiles) % p.n_tiles < it.to) {
            uint32_t acc[32];
            tmem_ld_32x32(tmem + p.bn, acc);
            tmem_ld_wait();
            db = __uint_as_float(acc[0]);
          }
          if (fine) p.db_parts[size_t(it.unit) * p.tile_m + in_tile + lane] = db;
        }
        // 16-bit results go out by TMA, 64 columns at a time (rows of other matrices are cut off by the map; rows of other groups
        // by nothing, so all 32 have to be the group's); else, and for pieces, by ordinary stores
        const bool by_tma = kMode != kFew && whole && p.vec_ok && (kMode == kWeight || rows >= 32);
        if (kMode != kFew) {  // the buffer may still be read
          if (elect_one()) bulk_wait_read<0>();
          __syncwarp();
        }
#pragma unroll
        for (int b = 0; b < (kMode == kFew ? 1 : 2); ++b) {
          const int c0 = group * kOwn + b * 128;
          if (c0 >= p.bn || !fine) continue;
          uint32_t acc[2][32];
          tmem_ld_32x32(tmem + c0, acc[0]);
          if (kMode != kFew) tmem_ld_32x32(tmem + c0 + 32, acc[1]);  // columns beyond the tile are cut off below
          tmem_ld_wait();
          if (by_tma) {
            // 32 rows of 128 bytes in the order that the map's swizzle says
            if (b > 0) {
              if (elect_one()) bulk_wait_read<0>();
              __syncwarp();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              add_bias(acc[h], b * 2 + h);
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(acc[h][g * 8 + i]);
                *reinterpret_cast<uint4*>(stage + lane * 128 + (((h * 4 + g) ^ (lane & 7)) << 4)) = Channels<T, 8>::pack(f);
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (elect_one()) {
              tma_store_3d(&tmap_o, smem_u32(stage), n0 + c0, kMode == kRows ? static_cast<int>(it.lo) + m0 : m0, kMode == kRows ? 0 : static_cast<int>(it.group));
              bulk_commit();
            }
          } else {
#pragma unroll
            for (int h = 0; h < (kMode == kFew ? 1 : 2); ++h)
              if (c0 + h * 32 < p.bn) put(acc[h], c0 + h * 32, b * 2 + h);
          }
        }
        give_back();
      }
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

  if (warp < kGrEpilogueWarps && elect_one()) bulk_wait_all();
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) cluster_sync_all();  // no CTA leaves while the other may still arrive on its barriers or read its operands
  if (warp == 9) {
    tc_fence_after_sync();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, 512u);
    else tmem_dealloc(tmem_base, 512u);
  }
  if (tid == 0 && ctl->abort_flag) {
    report(p.status, FGB_S_WAIT_TIMEOUT);
    mirror_code(p.mirror, FGB_S_WAIT_TIMEOUT);
  }
}

// ------------------------------------------------------------------ pieces
// Tiles in parts: their pieces added in order; and the tiles of empty groups (weight gradient), of which there are no units:
// zeros.  gridDim.y CTAs a tile.
constexpr int kGrJoinThreads = 256;
template <int kMode, typename T>
__global__ void __launch_bounds__(kGrJoinThreads) grouped_join_kernel(const __grid_constant__ GroupedArgs p, uint32_t tiles) {
  __shared__ uint32_t s_count;
  constexpr int kParamDtype = std::is_same<T, __half>::value ? FGB_F16 : std::is_same<T, __nv_bfloat16>::value ? FGB_BF16 : FGB_F32_IEEE;
  chain_release();
  chain_wait();
  const uint32_t G = p.ranges.count;
  const uint32_t *first = p.plan, *piece = p.plan + G + 1u, *offsets = p.plan + 2u * (G + 1u);
  const uint32_t unit = p.plan[3u * (G + 1u)];
  for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    uint32_t g, tile;
    if constexpr (kMode == kWeight) {
      const uint32_t per = p.n_tiles * p.m_tiles;
      g = t / per, tile = t - g * per;
    } else {
      // all tiles have equally many parts: that of tile t's first is t * parts
      const uint32_t whole = static_cast<uint32_t>(p.k_blocks), parts = parts_of(whole, part_length(p, whole, unit));
      if (uint64_t(t) * parts >= first[G]) return;
      if (threadIdx.x == 0) s_count = 0;
      __syncthreads();
      uint32_t before = 0;  // groups that begin at or before the tile, the last of which is not empty
      for (uint32_t i = threadIdx.x; i < G; i += kGrJoinThreads) before += first[i] <= t * parts ? 1u : 0u;
      atomicAdd(&s_count, before);
      __syncthreads();
      g = s_count - 1u, tile = t - first[g] / parts;
      __syncthreads();
    }
    const GroupSize z = group_size<kMode>(p, offsets, g);
    // none where the group is empty (or the offsets were bad)
    const uint32_t pieces = first[g] == first[g + 1u] ? 0u : parts_of(z.whole, part_length(p, z.whole, unit));
    const uint32_t elements = static_cast<uint32_t>(p.tile_m) * p.bn;
    if (kMode == kWeight && p.db != nullptr && tile % p.n_tiles == 0u && blockIdx.y == 0u && threadIdx.x < p.tile_m) {
      // the shares of db: of every part of the n tiles that read the same rows of dy
      const uint32_t m = tile / p.n_tiles * p.tile_m + threadIdx.x;
      if (m < static_cast<uint32_t>(p.m_extent)) {
        float v = 0.f;
        const float* share = p.db_parts + (size_t(first[g]) + tile) * p.tile_m + threadIdx.x;
        // eight at a time on their way
        const uint32_t n_tiles = static_cast<uint32_t>(p.n_tiles), shares = pieces * n_tiles;
        for (uint32_t i0 = 0; i0 < shares; i0 += 8u) {
          float x[8];
#pragma unroll
          for (uint32_t u = 0; u < 8u; ++u) {
            const uint32_t k = (i0 + u) / n_tiles, n = i0 + u - k * n_tiles;
            x[u] = i0 + u < shares ? share[(size_t(k) * z.tiles + n) * p.tile_m] : 0.f;
          }
#pragma unroll
          for (uint32_t u = 0; u < 8u; ++u) v += x[u];
        }
        store_value(static_cast<T*>(p.db) + int64_t(g) * p.m_extent + m, v);
      }
    }
    if (pieces == 1u) continue;  // stored as a whole
    const size_t apart = size_t(elements) * z.tiles;
    const float* from = p.slab + size_t(elements) * (piece[g] + tile);
    // four elements a thread: neighbours in the piece, and in the output
    const uint32_t quads = elements / 4u, share = (quads + gridDim.y - 1u) / gridDim.y;
    const uint32_t q0 = blockIdx.y * share, q1 = min(quads, q0 + share);
    for (uint32_t q = q0 + threadIdx.x; q < q1; q += kGrJoinThreads) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pieces > 0u) {
        // eight at a time on their way, also where there are fewer
        for (uint32_t k0 = 0; k0 < pieces; k0 += 8u) {
          float4 x[8];
#pragma unroll
          for (uint32_t u = 0; u < 8u; ++u) {
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + u < pieces) x[u] = __ldcg(reinterpret_cast<const float4*>(from + apart * (k0 + u)) + q);
          }
#pragma unroll
          for (uint32_t u = 0; u < 8u; ++u) v.x += x[u].x, v.y += x[u].y, v.z += x[u].z, v.w += x[u].w;
        }
      }
      const uint32_t e = q * 4u;
      float f[4] = {v.x, v.y, v.z, v.w};
      uint32_t col, cols;
      T* out;
      if constexpr (kMode == kWeight) {
        const uint32_t a = e / p.bn, m = tile / p.n_tiles * p.tile_m + a;
        if (m >= static_cast<uint32_t>(p.m_extent)) continue;
        col = tile % p.n_tiles * p.bn + (e - a * p.bn), cols = p.n_extent;
        out = static_cast<T*>(p.out) + (int64_t(g) * p.m_extent + m) * p.out_ld;
      } else {
        const uint32_t a = e / 128u, row = z.lo + tile / p.n_tiles * p.bn + a;
        if (row >= z.hi) continue;
        col = tile % p.n_tiles * 128u + (e & 127u), cols = p.m_extent;
        out = static_cast<T*>(p.out) + int64_t(row) * p.out_ld;
        if (p.bias != nullptr)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            if (col + i < cols) f[i] += load_param(p.bias, kParamDtype, int64_t(g) * p.m_extent + col + i);
      }
      if (p.vec_ok && col + 4u <= cols) {
        Channels<T, 4>::store(out + col, Channels<T, 4>::pack(f));
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (col + i < cols) store_value(out + col + i, f[i]);
      }
    }
  }
}

// ------------------------------------------------------------------ planes
// dst[plane][rows][cp] (16-bit) of src[rows][c]: fp32 as bf16 planes hi + mid + lo, 16-bit types as they are; columns from c
// on are zero.  A plane takes what the planes before it left, rounded to nearest; a value that would round to infinity is
// cut to the largest number instead, and nothing is left of an infinity or a NaN.
// A thread makes eight columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) grouped_planes_kernel(const T* __restrict__ src, uint16_t* __restrict__ dst, uint32_t rows, int c, int cp, int planes) {
  chain_release();
  chain_wait();
  const int packs = cp / 8, width = min(packs, 256), lanes = 256 / width;
  const int cx = threadIdx.x % width, ry = threadIdx.x / width;
  if (ry >= lanes) return;
  const size_t plane = size_t(rows) * cp;
  const bool whole = sizeof(T) == 4 && c % 4 == 0;
  for (uint32_t r = blockIdx.x * lanes + ry; r < rows; r += gridDim.x * lanes) {
    for (int q = cx; q < packs; q += width) {
      const T* from = src + size_t(r) * c + q * 8;
      uint16_t* to = dst + size_t(r) * cp + q * 8;
      const int have = min(8, c - q * 8);
      uint32_t out[3][4];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
          out[0][i / 2] = (i < have ? uint32_t(h[i]) : 0u) | (i + 1 < have ? uint32_t(h[i + 1]) << 16 : 0u);
        }
      } else {
        float v[8];
        if (whole) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(from)), b = have == 8 ? __ldg(reinterpret_cast<const float4*>(from) + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i < have ? from[i] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            uint32_t two = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = v[i + j];
              __nv_bfloat16 h = __float2bfloat16_rn(x);
              if (__hisinf(h) && !isinf(x)) h = __ushort_as_bfloat16(static_cast<unsigned short>(x < 0.f ? 0xFF7Fu : 0x7F7Fu));
              two |= uint32_t(__bfloat16_as_ushort(h)) << (16 * j);
              x = isfinite(x) ? x - __bfloat162float(h) : 0.f;
            }
            out[k][i / 2] = two;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < planes) *reinterpret_cast<uint4*>(to + k * plane) = make_uint4(out[k][0], out[k][1], out[k][2], out[k][3]);
    }
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
  const int64_t lanes = 256 / std::min(o.cp / 8, 256);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(rows, lanes), int64_t(device_sm_count()) * 16));
  if (is_f32(dtype))
    return launch_chained(grouped_planes_kernel<float>, dim3(grid), dim3(256), 0, s, static_cast<const float*>(src), dst, static_cast<uint32_t>(rows), c, o.cp, o.planes);
  return launch_chained(grouped_planes_kernel<__half>, dim3(grid), dim3(256), 0, s, static_cast<const __half*>(src), dst, static_cast<uint32_t>(rows), c, o.cp, 1);
}

// columns of a tile over `extent` channels: all of them in steps of 32 up to `most`, else equal tiles in steps of 64
static int tile_columns(int extent, int most) {
  if (extent <= most) return (extent + 31) / 32 * 32;
  const int whole = most / 64 * 64, tiles = (extent + whole - 1) / whole;
  return ((extent + tiles - 1) / tiles + 63) / 64 * 64;
}

struct GroupedPlan {
  int mode, bn, split, pair;
  int64_t pieces;       // that the slab holds
  int64_t slab_bytes, db_bytes, plan_bytes;
  int64_t bytes() const { return slab_bytes + db_bytes + plan_bytes; }
  uint32_t min_part;
  int acc_stride;
  int64_t tiles;        // most tiles (those that the join kernel looks at)
};

// A tile of few rows where a group has at most 16 on average: see the note on kFew above.  us of a forward call and an input
// gradient, few rows / tiles of 128 (bf16): 8 rows of 8 groups, 4096 -> 1024: 19.7 and 14.0 / 31.2 and 19.9; 1024 rows of
// 64 groups, 2048 -> 1024: 49.3 and 47.5 / 49.7 and 49.8; with 32 rows a group 256 of 8, 4096 -> 1024: 21.0 and 15.5 / 20.5 and 13.2.
static bool few_rows(const fgb_grouped_linear_call& c) { return c.n <= 16 * c.groups; }

static int grouped_plan(const fgb_grouped_linear_call& c, int pass, GroupedPlan& p) {
  const int64_t sms = device_sm_count();
  const int64_t N = c.n, G = c.groups;
  // fp32: the blocks' sums of a tile are held in 3 x 32 registers, and two stages of three planes in shared memory (a stage has 98304 bytes
  // at most; beyond some 1400 groups the schedule, 12 bytes each, leaves room for one of those, and loads and products take turns)
  auto most = [&](bool pair) { return !is_f32(c.dtype) ? 256 : pair ? 192 : 96; };
  int64_t blocks, db_units = 0;
  p = GroupedPlan{};
  if (pass == 2) {
    p.mode = kWeight;
    // A pair reads less for the same products, and has half as many tiles to deal out.  us, single / pair: 131072 rows of 16
    // groups, 1024 x 1024: 285 / 244; 39872 of 4, 512 x 512: 41.7 / 40.6; 4096 of 16, 1024 x 1024: 23.9 / 26.6.
    p.pair = c.co > 128 && c.ci > 64 && N >= 2048 * G;
    p.bn = tile_columns(c.ci, most(p.pair));
    const int64_t per = ceil_div(c.ci, p.bn) * ceil_div(c.co, p.pair ? 256 : 128);
    p.tiles = G * per;
    blocks = (N / 64 + G) * per;
    p.split = 1, p.min_part = 4;
    if (c.grad_bias != nullptr) db_units = p.tiles;
  } else {
    const int nout = pass == 0 ? c.co : c.ci, k = pass == 0 ? c.ci : c.co;
    const int64_t kb = ceil_div(k, 64);
    if (few_rows(c)) {
      p.mode = kFew;
      // most groups in one tile: tiles of 16 rows made 2048 rows of 64 groups, 1024 -> 1024, 51.8 us, tiles of 32 34.9
      p.bn = N <= 16 || N <= 4 * G ? 16 : 32;
      const int64_t m_tiles = ceil_div(nout, 128);
      p.tiles = std::min<int64_t>(N, N / p.bn + G) * m_tiles;
      blocks = p.tiles * kb;
      // A second launch that adds pieces up takes some 5 us.  24 rows of 2 groups to 512 channels, whole / cut: 1024 channels
      // 8.8 / 13.7 us, 4096 17.6 / 17.3 (16384 cut: 22.8).
      if (p.tiles <= sms / 2 && kb > 64) p.split = 1, p.min_part = 4;
    } else {
      p.mode = kRows;
      // tiles as they come out on average; the pairs' are twice as many rows
      auto tiles = [&](int rows, int64_t columns) { return (N / rows + (G + 1) / 2) * ceil_div(nout, columns); };
      // Pairs where there are two rounds of tiles and more.  us of a forward call, single / pair: 131072 rows of 16 groups,
      // 1024 -> 1024: 264 / 233; 166000 of 4, 256 -> 256: 41.7 / 39.1 (one lane a block, see the products); 20000 of 4: 10.7 /
      // 11.0; 10000 of 4: 7.8 / 8.6.
      p.pair = N >= 512 * G && nout > 64 && tiles(256, most(true)) >= sms;
      // Half as many columns where half of the SMs had no tile: 4096 rows of 2 groups, 512 -> 512, 9.2 us with 256, 7.6 with 128;
      // 8192 of 2: 10.1 / 11.0.
      p.bn = tile_columns(nout, !p.pair && !is_f32(c.dtype) && 2 * tiles(128, 256) <= sms ? 128 : most(p.pair));
      p.tiles = (N / (p.pair ? 256 : 128) + G) * ceil_div(nout, p.bn);
      blocks = p.tiles * kb;
    }
  }
  if (blocks >= (int64_t(1) << 31) - 1) return FGB_E_SIZE;
  // two accumulators a tile; the products with ones take 32 columns more
  p.acc_stride = std::max(p.bn, 32) + (pass == 2 && c.grad_bias != nullptr ? 32 : 0);
  const int64_t tile_m = p.pair ? 256 : 128, workers = p.pair ? sms / 2 : sms;
  // a part has half of the wanted length at least (a tile is cut only where it is longer), and min_part at least
  p.pieces = p.split ? std::min<int64_t>(2 * kGrMostUnits * workers + 2, blocks / p.min_part) : 0;
  p.plan_bytes = p.split ? align256(schedule_bytes(G)) : 0;
  p.slab_bytes = align256(p.pieces * tile_m * p.bn * 4);
  p.db_bytes = db_units > 0 ? align256((db_units + p.pieces) * tile_m * 4) : 0;
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

template <int kMode, typename T, bool kPair>
static int launch_grouped(const CUtensorMap& tp, const CUtensorMap& tq, const CUtensorMap& to, GroupedArgs& a, const GroupedPlan& p, cudaStream_t s) {
  const int prefix = static_cast<int>(schedule_bytes(a.ranges.count));
  const int fixed = kGrEpilogueWarps * grouped_store_bytes<kMode, T>() + grouped_extra_bytes<kMode, T>() + static_cast<int>(sizeof(GroupedSmem)) + prefix;
  const int stage = a.planes * (kGrPBytes + a.q_bytes);
  a.stages = std::min(kGrMaxStages, (kGrSmemLimit - fixed) / stage);
  const size_t smem = size_t(fixed) + size_t(a.stages) * stage;
  static PerDeviceTable configured;
  const int rc = ensure_dynamic_smem(configured, grouped_kernel<kMode, T, kPair>, smem);
  if (rc != FGB_OK) return rc;
  const int workers = kPair ? device_sm_count() / 2 : device_sm_count();
  const unsigned grid = static_cast<unsigned>(p.split ? workers : std::max<int64_t>(std::min<int64_t>(p.tiles, workers), 1));
  cudaError_t e = launch_chained_clusters(grouped_kernel<kMode, T, kPair>, dim3(grid * (kPair ? 2 : 1)), dim3(kGrThreads), smem, kPair ? 2 : 1, s, tp, tq, to, a);
  if (e == cudaSuccess && p.split) {
    if constexpr (kMode != kRows) {
      const unsigned tiles = static_cast<unsigned>(p.tiles), x = std::min(tiles, 65535u * 8u);
      const unsigned y = static_cast<unsigned>(std::clamp<int64_t>(ceil_div(int64_t(device_sm_count()) * 8, tiles), 1, 64));
      e = launch_chained(grouped_join_kernel<kMode, T>, dim3(x, y), dim3(kGrJoinThreads), 0, s, a, tiles);
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
  a.bn = p.bn, a.tile_m = p.pair ? 256 : 128;
  for (const int rows = p.mode == kFew ? a.bn : a.tile_m; (1 << a.row_shift) < rows;) ++a.row_shift;
  const int half = p.pair ? p.bn / 2 : p.bn;
  a.planes = planes_of(c.dtype);
  a.terms = c.dtype == FGB_F32_IEEE ? 6 : c.dtype == FGB_F32_TF32 ? 3 : 1;
  // the small products first: (lo hi) (hi lo) (mid mid) (mid hi) (hi mid) (hi hi), or the last three of them
  a.p_planes = a.terms == 6 ? 0x001102u : a.terms == 3 ? 0x001u : 0u, a.q_planes = a.terms == 6 ? 0x010120u : a.terms == 3 ? 0x010u : 0u;
  a.min_part = p.min_part;
  a.piece_cost = 10.f * static_cast<float>(p.bn) / 256.f / static_cast<float>(a.terms);  // 128 KB a CTA written, then read: some ten stages' time
  a.acc_stride = p.acc_stride;
  a.acc_sets = 2 * p.acc_stride <= 512 ? 2 : 1;
  a.slab = slab, a.db_parts = slab + p.slab_bytes / 4, a.plan = reinterpret_cast<uint32_t*>(slab + (p.slab_bytes + p.db_bytes) / 4);
  a.status = c.status, a.mirror = status_mirror(c.status);
  const uint32_t fmt = features.dtype16 == FGB_F16 ? kFmtF16 : kFmtBF16;
  a.one_pair = features.dtype16 == FGB_F16 ? 0x3C003C00u : 0x3F803F80u;
  const int eb = elem_bytes(c.dtype);
  CUtensorMap tp, tq, to{};
  const uint64_t N = static_cast<uint64_t>(c.n), G = static_cast<uint64_t>(c.groups);
  if (pass == 2) {
    // features = dy, other = x
    a.m_extent = c.co, a.n_extent = c.ci, a.m_tiles = static_cast<int>(ceil_div(c.co, a.tile_m)), a.n_tiles = static_cast<int>(ceil_div(c.ci, p.bn));
    a.p_mn = a.q_mn = 1;
    a.q_bytes = (half + 63) / 64 * 8192;
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
      a.q_bytes = mn ? (half + 63) / 64 * 8192 : half * 128;
      rc = make_rows_tmap_3d(&tp, features.base, features.dtype16, features.cp, N, features.planes, 64, 128);
      if (rc == FGB_OK) rc = make_rows_tmap_3d(&tq, other.base, other.dtype16, wc, wr, w_planes, 64, mn ? 64 : half);
    }
  }
  if (rc != FGB_OK) return rc;
  a.vec_ok = a.out_ld * eb % 16 == 0;
  if (a.vec_ok && eb == 2 && p.mode != kFew) {  // what is stored: 32 rows x 64 columns at a time
    rc = pass == 2 ? make_rows_tmap_3d(&to, a.out, c.dtype, c.ci, c.co, G, 64, 32) : make_rows_tmap_3d(&to, a.out, c.dtype, a.out_ld, N, 1, 64, 32);
    if (rc != FGB_OK) return rc;
  }
  a.idesc = make_idesc(fmt, a.tile_m, p.bn, a.p_mn, a.q_mn);
  a.idesc_ones = make_idesc(fmt, a.tile_m, p.pair ? 32 : 16, a.p_mn, 0);
#define FGB_GROUPED(mode, pair)                                                        \
  (c.dtype == FGB_F16    ? launch_grouped<mode, __half, pair>(tp, tq, to, a, p, s)         \
   : c.dtype == FGB_BF16 ? launch_grouped<mode, __nv_bfloat16, pair>(tp, tq, to, a, p, s)  \
                         : launch_grouped<mode, float, pair>(tp, tq, to, a, p, s))
  if (p.mode == kFew) return FGB_GROUPED(kFew, false);
  if (p.mode == kRows) return p.pair ? FGB_GROUPED(kRows, true) : FGB_GROUPED(kRows, false);
  return p.pair ? FGB_GROUPED(kWeight, true) : FGB_GROUPED(kWeight, false);
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
    bytes += p.bytes() + plane_bytes(c->n, c->ci, c->dtype) + plane_bytes(c->groups * c->co, c->ci, c->dtype);
    return rc != FGB_OK ? rc : bytes;
  }
  int64_t slab = 0;
  for (int pass : {1, 2}) {
    if (pass == 1 ? c->grad_x == nullptr : c->grad_weight == nullptr) continue;
    rc = grouped_plan(*c, pass, p);
    if (rc != FGB_OK) return rc;
    slab = std::max(slab, p.bytes());
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
  at += p.bytes();
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
