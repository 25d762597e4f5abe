// Embedding: rows of a table by index, scaled; the gradient of the table by sorted indices.
//
//   out[i] = scale * table[t_i]          grad[v] = scale * sum over i with t_i = v of g[i]
//
// The gradient sorts the positions by index (stable, fgb_sort.cu) and walks the sorted list in chunks of fixed length: a
// group of threads adds the rows of one chunk, one run of equal indices after the other, in fp32; the CTA's groups then add
// up the runs that lie in several of its chunks.  A run that lies in one CTA is final.  The two that may reach beyond its ends
// leave their sums in a slab, and a second kernel adds a run's pieces up.  Nothing is added atomically, so the order of every
// sum is fixed, and an index that every other position holds costs no more than a spread one.
//
// Measured (B200, int64 indices that repeat four times in a row): lookup 166000 x 256 fp16 from 4096 rows 19 us (5 TB/s; bound by
// the stores), 1.32 million x 64 bf16 from 50000 rows 43 us (4.2 TB/s); gradient 57 and 142 us, of which the two passes of the
// sort are 27 and 74 (scattered stores of 8 bytes) and the sums 22 and 50 (the rows of g in sorted order).  Up to 4096 positions take one
// launch, see embedding_few_kernel.
#include <algorithm>

#include "fgb_common.cuh"
#include "fgb_device.cuh"
#include "fgb_rows.cuh"
#include "fgb_sort.cuh"

namespace fgb {

constexpr int kEmbThreads = 256;
constexpr int kEmbRows = 4;      // rows in flight per thread of the lookup

__device__ __forceinline__ int64_t index_at(const void* p, int wide, uint32_t i) {
  return wide ? __ldg(static_cast<const int64_t*>(p) + i) : __ldg(static_cast<const int32_t*>(p) + i);
}

// ------------------------------------------------------------------ lookup
template <typename T, int kVec, bool kScaled>
__global__ void __launch_bounds__(kEmbThreads) embedding_kernel(const void* __restrict__ indices, int wide, const T* __restrict__ table, T* __restrict__ out,
                                                                uint32_t n, uint32_t rows, int C, float scale, int32_t* status, int32_t* mirror) {
  using Ch = Channels<T, kVec>;
  chain_release();
  chain_wait();
  const int packs = C / kVec, width = min(kEmbThreads, packs), lanes = kEmbThreads / width;
  const int cx = threadIdx.x % width, ry = threadIdx.x / width;
  if (ry >= lanes) return;
  // the next rows' indices are on their way while these are copied
  int64_t idx[kEmbRows], next[kEmbRows];
  auto look = [&](uint32_t r0) {
#pragma unroll
    for (int u = 0; u < kEmbRows; ++u) {
      const uint32_t r = r0 + u * lanes + ry;
      next[u] = r < n ? index_at(indices, wide, r) : 0;
    }
  };
  const uint32_t step = gridDim.x * (lanes * kEmbRows);
  look(blockIdx.x * (lanes * kEmbRows));
  for (uint32_t r0 = blockIdx.x * (lanes * kEmbRows); r0 < n; r0 += step) {  // n and step are below 2^30
#pragma unroll
    for (int u = 0; u < kEmbRows; ++u) idx[u] = next[u];
    look(r0 + step);
    for (int c = cx; c < packs; c += width) {
      typename Ch::Raw raw[kEmbRows];
#pragma unroll
      for (int u = 0; u < kEmbRows; ++u) {
        raw[u] = typename Ch::Raw{};
        if (idx[u] >= 0 && idx[u] < int64_t(rows)) raw[u] = Ch::load(table + size_t(idx[u]) * C + c * kVec);
      }
#pragma unroll
      for (int u = 0; u < kEmbRows; ++u) {
        const uint32_t r = r0 + u * lanes + ry;
        if (r >= n) continue;
        if constexpr (kScaled) {
          float f[kVec];
          Ch::unpack(raw[u], f);
#pragma unroll
          for (int i = 0; i < kVec; ++i) f[i] *= scale;
          raw[u] = Ch::pack(f);
        }
        // a result larger than L2 would push the table out of it: 166000 x 256 fp16 21.3 -> 18.4 us
        Ch::store_streaming(out + size_t(r) * C + c * kVec, raw[u]);
      }
    }
    if (cx == 0) {
#pragma unroll
      for (int u = 0; u < kEmbRows; ++u) {
        if (idx[u] < 0 || idx[u] >= int64_t(rows)) {
          report(status, FGB_S_BAD_INDEX);
          mirror_code(mirror, FGB_S_BAD_INDEX);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ gradient
// Sort keys: the index, or `rows` for a position that adds nothing (padding, out of range), which sorts behind all others.
// Also clears the gradient (rows of indices that no position holds stay zero).
__global__ void __launch_bounds__(kEmbThreads) embedding_keys_kernel(const void* __restrict__ indices, int wide, uint32_t n, uint32_t rows, int64_t padding,
                                                                     int32_t* __restrict__ keys, uint16_t* __restrict__ grad, uint64_t grad_halves,
                                                                     int32_t* status, int32_t* mirror) {
  chain_release();
  chain_wait();
  const uint32_t t = blockIdx.x * kEmbThreads + threadIdx.x, total = gridDim.x * kEmbThreads;
  for (uint32_t i = t; i < n; i += total) {
    const int64_t v = index_at(indices, wide, i);
    const bool in = v >= 0 && v < int64_t(rows);
    if (!in) {
      report(status, FGB_S_BAD_INDEX);
      mirror_code(mirror, FGB_S_BAD_INDEX);
    }
    keys[i] = static_cast<int32_t>(in && v != padding ? static_cast<uint32_t>(v) : rows);
  }
  const uint64_t whole = grad_halves / 8;
  for (uint64_t i = t; i < whole; i += total) reinterpret_cast<uint4*>(grad)[i] = make_uint4(0, 0, 0, 0);
  if (t < grad_halves - whole * 8) grad[whole * 8 + t] = 0;
}

// What a CTA of the sum kernel says of its positions
struct EmbInfo {
  uint32_t key;    // of its last position
  uint32_t flags;  // kGoesOn: the run of the last position goes on behind the CTA; kThrough: it began before the CTA, too
};
constexpr uint32_t kGoesOn = 1u, kThrough = 2u;
constexpr uint32_t kNoKey = 0xFFFFFFFFu;  // before the first position and behind the last one

struct EmbGrad {
  const void* g;
  void* grad;
  const int32_t* keys;      // by position
  const int64_t* order;     // positions by key
  float* slab;              // [ctas][2][C]: the sum of the CTA's run that began before it, and of the one that goes on behind it
  EmbInfo* info;            // [ctas]
  uint32_t n, rows, chunk, ctas;
  int C;
  float scale;
};

// Sums over `count` sorted positions, in shared memory with their keys (s_key[-1] and s_key[count]: the keys before and behind them), of the
// channels of the packs pack0 .. pack1 - 1: `lanes` groups of `width` threads take a chunk each.  s_head: of each group's chunk the sum of the run
// that began before it, s_through: whether that run goes on behind it.  slab: for the runs that leave the positions.  The whole CTA calls it.
template <typename T, int kVec, int kThreads, typename Pos>
__device__ __forceinline__ void embedding_runs(const EmbGrad& p, const uint32_t* s_key, const Pos* s_pos, float (*s_head)[kThreads], uint8_t* s_through,
                                               uint32_t count, uint32_t chunk, int pack0, int pack1, int width, float* slab) {
  using Ch = Channels<T, kVec>;
  const int lanes = kThreads / width, cx = threadIdx.x % width, ry = threadIdx.x / width;
  const uint32_t b = ry * chunk, e = min(b + chunk, count);
  const bool active = ry < lanes && b < e;
  const T* g = static_cast<const T*>(p.g);
  T* grad = static_cast<T*>(p.grad);
  auto open_at = [&](uint32_t i) { return s_key[int(i) - 1] == s_key[i]; };  // position i continues a run
  if (cx == 0 && ry < lanes) s_through[ry] = active && open_at(b) && s_key[b] == s_key[e - 1u] && s_key[e] == s_key[b];
  for (int c0 = pack0; c0 < pack1; c0 += width) {
    const int c = c0 + cx;
    const bool mine = active && c < pack1;
    float acc[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
    uint32_t key = 0;
    bool open = false;
    auto finish = [&](const float (&sum)[kVec], uint32_t k) {
      if (k >= p.rows) return;
      float f[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] = sum[i] * p.scale;
      Ch::store(grad + size_t(k) * p.C + c * kVec, Ch::pack(f));
    };
    auto head = [&]() {
#pragma unroll
      for (int i = 0; i < kVec; ++i) s_head[i][threadIdx.x] = acc[i];
    };
    if (mine) {
      key = s_key[b];
      open = open_at(b);
      auto add = [&](uint32_t i, const typename Ch::Raw& raw) {
        const uint32_t k = s_key[i];
        if (k != key) {
          if (open) head();
          else finish(acc, key);
          open = false;
          key = k;
#pragma unroll
          for (int v = 0; v < kVec; ++v) acc[v] = 0.f;
        }
        float f[kVec];
        Ch::unpack(raw, f);
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] += f[v];
      };
      uint32_t i = b;
      constexpr int kUnroll = 8;
      for (; i + kUnroll <= e; i += kUnroll) {
        typename Ch::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) raw[u] = Ch::load(g + size_t(s_pos[i + u]) * p.C + c * kVec);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) add(i + u, raw[u]);
      }
      for (; i < e; ++i) add(i, Ch::load(g + size_t(s_pos[i]) * p.C + c * kVec));
      if (open) head();  // the chunk's only run began before it
    }
    __syncthreads();
    // The last run of a chunk, where it began there, is its group's to finish, and the CTA's first, where it began before the
    // CTA, group 0's: the heads of the chunks that follow are added while the run goes on.
    if (mine) {
      const bool from_before = ry == 0 && open_at(0);
      auto collect = [&](float (&sum)[kVec], uint32_t k, int r, bool before) {
        for (bool more = true; more && r < lanes && r * chunk < count; ++r) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) sum[i] += s_head[i][r * width + cx];
          more = s_through[r] != 0;
          if (!more) {
            if (!before) {
              finish(sum, k);
              return;
            }
            break;
          }
        }
        // a run that began before the CTA, or goes on behind it
        if (k >= p.rows) return;
        float* to = slab + (before ? 0 : p.C) + c * kVec;
#pragma unroll
        for (int i = 0; i < kVec; ++i) to[i] = sum[i];
      };
      if (!open) {
        if (s_key[e] != key) finish(acc, key);
        else collect(acc, key, ry + 1, false);
      }
      if (from_before) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
        collect(acc, s_key[0], 0, true);
      }
    }
    __syncthreads();
  }
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kEmbThreads) embedding_sum_kernel(const EmbGrad p) {
  extern __shared__ uint32_t s_mem[];
  __shared__ float s_head[kVec][kEmbThreads];
  __shared__ uint8_t s_through[kEmbThreads];
  chain_release();
  const int packs = p.C / kVec, width = min(kEmbThreads, packs), lanes = kEmbThreads / width;
  const uint32_t per_cta = lanes * p.chunk;
  uint32_t* s_key = s_mem + 1;               // keys of the CTA's positions, one before and one behind them
  uint32_t* s_pos = s_mem + per_cta + 2;
  chain_wait();
  const uint32_t base = blockIdx.x * per_cta;  // < n
  for (uint32_t i = threadIdx.x; i < per_cta + 2u; i += kEmbThreads) {
    const uint32_t at = base + i - 1u;  // wraps to 2^32 - 1 ahead of the first
    uint32_t key = kNoKey, pos = 0;
    if (at < p.n) {
      pos = static_cast<uint32_t>(__ldg(&p.order[at]));
      pos = min(pos, p.n - 1u);  // the order is void after a sort that gave up
      key = static_cast<uint32_t>(__ldg(&p.keys[pos]));
    }
    s_mem[i] = key;
    if (i >= 1u && i <= per_cta) s_pos[i - 1u] = pos;
  }
  __syncthreads();
  const uint32_t count = min(per_cta, p.n - base);  // positions of the CTA
  if (threadIdx.x == 0) {
    const uint32_t last = s_key[count - 1u];
    p.info[blockIdx.x] = EmbInfo{last, (s_key[count] == last ? kGoesOn : 0u) | (s_key[-1] == s_key[0] && s_key[0] == last ? kThrough : 0u)};
  }
  embedding_runs<T, kVec, kEmbThreads>(p, s_key, s_pos, s_head, s_through, count, p.chunk, 0, packs, width, p.slab + size_t(blockIdx.x) * 2 * p.C);
}

// The runs that lie in more than one CTA of the sum kernel: CTA q takes the one that began in that kernel's CTA q and goes
// on behind it, if there is one, and 32 channels of it.  32 groups of eight threads add every 32nd piece, and their sums are
// added in order.
constexpr int kJoinCols = 32;
template <typename T>
__global__ void __launch_bounds__(kEmbThreads) embedding_join_kernel(const EmbGrad p) {
  __shared__ float s_sum[32][kJoinCols + 1];
  chain_release();
  chain_wait();
  const uint32_t q = blockIdx.x;
  const EmbInfo own = p.info[q];
  if (own.flags != kGoesOn || own.key >= p.rows) return;  // nothing goes on, or its beginning is another CTA's
  uint32_t last = q + 1u;  // the CTA in which the run ends: the first that it does not run through
  for (;;) {
    const uint32_t at = last + threadIdx.x;
    const bool through = at < p.ctas && p.info[at].flags == (kGoesOn | kThrough);
    const int run = __syncthreads_count(through);
    if (run == kEmbThreads) {
      last += kEmbThreads;
      continue;
    }
    // through holds for a run of threads from the first on: behind the end another run may fill a CTA
    __shared__ uint32_t s_end;
    if (threadIdx.x == 0) s_end = 0xFFFFFFFFu;
    __syncthreads();
    if (!through) atomicMin(&s_end, at);
    __syncthreads();
    last = min(s_end, p.ctas - 1u);
    break;
  }
  const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3;
  const int c0 = static_cast<int>(blockIdx.y) * kJoinCols + cx * 4;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t k0 = q + ry; k0 <= last; k0 += 4u * 32u) {
    float v[4][4];
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      const uint32_t k = k0 + u * 32u;
      const float* from = p.slab + (size_t(k) * 2 + (k == q ? 1 : 0)) * p.C + c0;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = k <= last && c0 + i < p.C ? from[i] : 0.f;
    }
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += v[u][i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s_sum[ry][cx * 4 + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < kJoinCols) {
    const int c = static_cast<int>(blockIdx.y) * kJoinCols + threadIdx.x;
    if (c < p.C) {
      float v = 0.f;
      for (int i = 0; i < 32; ++i) v += s_sum[i][threadIdx.x];
      static_cast<T*>(p.grad)[size_t(own.key) * p.C + c] = static_cast<T>(v * p.scale);
    }
  }
}

// ------------------------------------------------------------------ gradient of few positions
// One launch.  Every CTA sorts all positions by key in its shared memory (stable, 9 bits a pass, as fgb_sort.cu does over tiles).  The first
// ones take four packs of channels each and add up all runs, so that none leaves a CTA; the others clear the rows that no
// position holds.  Bound by the host: a call with gradient takes 45 us of its time, 37 of them autograd's, where it took 57 with seven launches
// (torch's plain operations 48).  On the device, forward and gradient, other way / this: 500 rows of 64 fp16 16.9 / 11.5 us, 4096 of 512
// fp32 and 60000 indices 47.5 / 34.5, 4096 of 2048 fp16 65.7 / 23.1; all of 4096 x 64 on one index 17.8 / 20.6.  Beyond 256 packs a row, or 4096
// positions, too many CTAs would sort, or one would add for too long.
constexpr int kFewThreads = 512, kFewItems = 8, kFewPositions = kFewThreads * kFewItems, kFewPacks = 4, kFewWarps = kFewThreads / 32;
constexpr int kFewBitWords = 2048;  // rows that a clearing CTA looks at at a time, in words of bits

struct FewArgs {
  const void* indices;
  int wide, passes;
  int64_t padding;
  unsigned sum_ctas;
  int32_t* status;
  int32_t* mirror;
};

template <typename T, int kVec>
__global__ void __launch_bounds__(kFewThreads) embedding_few_kernel(const EmbGrad p, const FewArgs q) {
  using Ch = Channels<T, kVec>;
  // counters of the sort [warps][digits]; then the heads of the sums, or the bits of the rows that positions hold
  __shared__ __align__(16) uint8_t s_shared[16384];
  __shared__ uint32_t s_mem[kFewPositions + 2];
  __shared__ uint16_t s_pos[kFewPositions];
  __shared__ uint32_t s_scan[kFewWarps];
  __shared__ uint8_t s_through[kFewThreads];
  static_assert(kFewWarps * kSortDigits * 2 <= 16384 && 8 * kFewThreads * 4 <= 16384 && kFewBitWords * 4 <= 16384 && kSortDigits == kFewThreads);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  chain_release();
  chain_wait();
  const int packs = p.C / kVec;
  const bool sums = blockIdx.x < q.sum_ctas;
  // item j of lane l of warp w: position w * 256 + j * 32 + l
  uint32_t key[kFewItems], pos[kFewItems];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kFewItems; ++j) {
    pos[j] = w * (32 * kFewItems) + j * 32 + lane;
    key[j] = kNoKey;
    if (pos[j] < p.n) {
      const int64_t v = index_at(q.indices, q.wide, pos[j]);
      const bool in = v >= 0 && v < int64_t(p.rows);
      bad |= !in;
      if (in && v != q.padding) key[j] = static_cast<uint32_t>(v);
    }
  }
  if (bad && blockIdx.x == 0u) {
    report(q.status, FGB_S_BAD_INDEX);
    mirror_code(q.mirror, FGB_S_BAD_INDEX);
  }
  if (!sums) {
    uint32_t* s_bits = reinterpret_cast<uint32_t*>(s_shared);
    T* grad = static_cast<T*>(p.grad);
    const int width = min(kFewThreads, packs), lanes = kFewThreads / width, cx = tid % width, ry = tid / width;
    const uint32_t ctas = gridDim.x - q.sum_ctas, per = min((p.rows + ctas - 1u) / ctas, kFewBitWords * 32u);
    for (uint64_t r0 = uint64_t(blockIdx.x - q.sum_ctas) * per; r0 < p.rows; r0 += uint64_t(ctas) * per) {
      const uint32_t first = static_cast<uint32_t>(r0), rows = min(per, p.rows - first);
      for (uint32_t i = tid; i < (rows + 31u) / 32u; i += kFewThreads) s_bits[i] = 0u;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kFewItems; ++j) {
        const uint32_t r = key[j] - first;  // no key: far beyond, first + rows is below 2^31
        if (key[j] != kNoKey && r < rows) atomicOr(&s_bits[r / 32u], 1u << (r & 31u));
      }
      __syncthreads();
      if (ry < lanes) {
        for (uint32_t r = ry; r < rows; r += lanes) {
          if (s_bits[r / 32u] >> (r & 31u) & 1u) continue;
          for (int c = cx; c < packs; c += width) Ch::store(grad + size_t(first + r) * p.C + c * kVec, typename Ch::Raw{});
        }
      }
      __syncthreads();
    }
    return;
  }
  uint32_t* s_key = s_mem + 1;
  uint16_t(*s_cnt)[kSortDigits] = reinterpret_cast<uint16_t(*)[kSortDigits]>(s_shared);
  uint32_t held = 0;  // positions that have a key
#pragma unroll
  for (int j = 0; j < kFewItems; ++j) held += __popc(__ballot_sync(0xffffffffu, key[j] != kNoKey));
  const uint32_t lt = (1u << lane) - 1u;
  for (int pass = 0; pass < q.passes; ++pass) {
    const int shift = pass * kSortDigitBits;
    for (int i = tid; i < kFewWarps * kSortDigits / 2; i += kFewThreads) reinterpret_cast<uint32_t*>(s_shared)[i] = 0u;
    __syncthreads();
    uint32_t rank[kFewItems];
#pragma unroll
    for (int j = 0; j < kFewItems; ++j) {  // positions without a key have the largest digit in every pass, and come last
      const uint32_t d = (key[j] >> shift) & (kSortDigits - 1);
      const unsigned peers = __match_any_sync(0xffffffffu, d);
      const int leader = __ffs(peers) - 1;
      uint32_t before = 0;
      if (lane == leader) {
        before = s_cnt[w][d];
        s_cnt[w][d] = static_cast<uint16_t>(before + __popc(peers));
      }
      rank[j] = __shfl_sync(0xffffffffu, before, leader) + __popc(peers & lt);
      __syncwarp();
    }
    __syncthreads();
    // thread t: digit t
    uint32_t count = 0;
#pragma unroll
    for (int ww = 0; ww < kFewWarps; ++ww) {
      const uint32_t c = s_cnt[ww][tid];
      s_cnt[ww][tid] = static_cast<uint16_t>(count);
      count += c;
    }
    uint32_t upto = count;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) s_scan[w] = upto;
    __syncthreads();
    uint32_t base = upto - count;
    for (int ww = 0; ww < w; ++ww) base += s_scan[ww];
#pragma unroll
    for (int ww = 0; ww < kFewWarps; ++ww) s_cnt[ww][tid] = static_cast<uint16_t>(s_cnt[ww][tid] + base);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kFewItems; ++j) {
      const uint32_t to = s_cnt[w][(key[j] >> shift) & (kSortDigits - 1)] + rank[j];
      s_key[to] = key[j], s_pos[to] = static_cast<uint16_t>(pos[j]);
    }
    __syncthreads();
    if (pass + 1 < q.passes) {
#pragma unroll
      for (int j = 0; j < kFewItems; ++j) {
        const uint32_t at = w * (32 * kFewItems) + j * 32 + lane;
        key[j] = s_key[at], pos[j] = s_pos[at];
      }
    }
  }
  if (tid == 0) s_key[-1] = kNoKey;
  if (lane == 0) s_scan[w] = held;
  __syncthreads();
  uint32_t count = 0;
#pragma unroll
  for (int ww = 0; ww < kFewWarps; ++ww) count += s_scan[ww];
  if (tid == 0) s_key[count] = kNoKey;  // behind the positions that have a key
  __syncthreads();
  const int pack0 = static_cast<int>(blockIdx.x) * kFewPacks, pack1 = min(packs, pack0 + kFewPacks), width = pack1 - pack0;
  // Long chunks are rows one after the other, short ones heads one after the other that a run through all of them collects
  const uint32_t lanes = kFewThreads / width;
  const uint32_t chunk = max(count <= 512u ? 8u : count <= 2048u ? 16u : 32u, (count + lanes - 1u) / lanes);
  embedding_runs<T, kVec, kFewThreads>(p, s_key, s_pos, reinterpret_cast<float(*)[kFewThreads]>(s_shared), s_through, count, chunk, pack0, pack1, width, nullptr);
}

// ------------------------------------------------------------------ host side
static bool emb_few(const fgb_embedding_call& c) { return c.n <= kFewPositions && c.c / row_pack(c.c, elem_bytes(c.dtype)) <= 256; }

template <typename T, int kVec>
static cudaError_t emb_few_launch(const EmbGrad& a, FewArgs q, cudaStream_t s) {
  q.sum_ctas = static_cast<unsigned>(ceil_div(a.C / kVec, kFewPacks));
  // rows are cleared some 16 KB a CTA, by two CTAs an SM at most
  const int64_t clear = std::min<int64_t>(ceil_div(int64_t(a.rows) * a.C * static_cast<int64_t>(sizeof(T)), 16384), int64_t(device_sm_count()) * 2);
  return launch_chained(embedding_few_kernel<T, kVec>, dim3(q.sum_ctas + static_cast<unsigned>(clear)), dim3(kFewThreads), 0, s, a, q);
}

struct EmbPlan {
  int vec, lanes;
  uint32_t chunk, ctas;
  size_t keys_off, order_off, sort_off, sort_bytes, slab_off, info_off, bytes;
};
static int emb_plan(const fgb_embedding_call& c, EmbPlan& p) {
  p.vec = row_pack(c.c, elem_bytes(c.dtype));
  const int packs = c.c / p.vec, width = std::min(packs, kEmbThreads);
  p.lanes = kEmbThreads / width;
  // long chunks leave less to be added up, short ones make more of them: some 500 threads for every SM before chunks grow.
  // us of a gradient with chunks of 8 / 32 / 64: 166000 x 256 fp16 82 / 63 / 57, 8000 x 256 22 / 23 / 28
  int64_t chunk = 8;
  while (chunk < 64 && c.n / (2 * chunk) * width >= int64_t(device_sm_count()) * 512) chunk *= 2;
  p.chunk = static_cast<uint32_t>(chunk);
  p.ctas = static_cast<uint32_t>(ceil_div(c.n, chunk * p.lanes));
  const int64_t sort = fgb_pp_sorted_idx_workspace_bytes(c.n);
  if (sort < 0) return static_cast<int>(sort);
  p.sort_bytes = static_cast<size_t>(sort);
  p.keys_off = 0;
  p.order_off = align256(c.n * 4);
  p.sort_off = p.order_off + align256(c.n * 8);
  p.slab_off = p.sort_off + align256(sort);
  p.info_off = p.slab_off + align256(int64_t(p.ctas) * 2 * c.c * 4);
  p.bytes = p.info_off + align256(int64_t(p.ctas) * static_cast<int64_t>(sizeof(EmbInfo)));
  return FGB_OK;
}

static int emb_check(const fgb_embedding_call* c) {
  if (c == nullptr) return FGB_E_NULL;
  if (c->dtype != FGB_F16 && c->dtype != FGB_BF16 && c->dtype != FGB_F32_TF32 && c->dtype != FGB_F32_IEEE) return FGB_E_DTYPE;
  if (c->index_bits != 32 && c->index_bits != 64) return FGB_E_DTYPE;
  if (c->n < 0 || c->n >= (int64_t(1) << 30) || c->rows < 1 || c->rows >= (int64_t(1) << 31) - 1 || c->c < 1 || c->c > 65536) return FGB_E_SIZE;
  return FGB_OK;
}

template <typename T, int kVec>
static cudaError_t emb_forward(const fgb_embedding_call& c, cudaStream_t s) {
  const int width = std::min(c.c / kVec, kEmbThreads), lanes = kEmbThreads / width;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(c.n, lanes * kEmbRows), int64_t(device_sm_count()) * 8));
  const uint32_t n = static_cast<uint32_t>(c.n), rows = static_cast<uint32_t>(c.rows);
  const T* table = static_cast<const T*>(c.table);
  T* out = static_cast<T*>(c.out);
  int32_t* mirror = status_mirror(c.status);
  const int wide = c.index_bits == 64;
  return c.scale == 1.f ? launch_chained(embedding_kernel<T, kVec, false>, dim3(grid), dim3(kEmbThreads), 0, s, c.indices, wide, table, out, n, rows, c.c,
                                         c.scale, c.status, mirror)
                        : launch_chained(embedding_kernel<T, kVec, true>, dim3(grid), dim3(kEmbThreads), 0, s, c.indices, wide, table, out, n, rows, c.c,
                                         c.scale, c.status, mirror);
}

template <typename T, int kVec>
static cudaError_t emb_sum(const EmbGrad& a, const EmbPlan& p, cudaStream_t s) {
  const uint32_t per_cta = p.lanes * p.chunk;
  const size_t smem = (2 * size_t(per_cta) + 2) * 4;
  static PerDeviceTable configured;
  if (ensure_dynamic_smem(configured, embedding_sum_kernel<T, kVec>, smem) != FGB_OK) return cudaErrorInvalidConfiguration;
  LaunchErrors chain;
  chain.add(launch_chained(embedding_sum_kernel<T, kVec>, dim3(p.ctas), dim3(kEmbThreads), smem, s, a));
  if (p.ctas > 1) chain.add(launch_chained(embedding_join_kernel<T>, dim3(p.ctas, static_cast<unsigned>(ceil_div(a.C, kJoinCols))), dim3(kEmbThreads), 0, s, a));
  return chain.first;
}

#define FGB_BY_PACK(T, vec, call)                                                       \
  ((vec) * sizeof(T) == 16  ? call<T, 16 / sizeof(T)>                                   \
   : (vec) * sizeof(T) == 8 ? call<T, 8 / sizeof(T)>                                    \
   : (vec) == 2             ? call<T, 2>                                                \
                            : call<T, 1>)

}  // namespace fgb

extern "C" int fgb_embedding_forward(const fgb_embedding_call* c, void* stream) {
  using namespace fgb;
  const int rc = emb_check(c);
  if (rc != FGB_OK) return rc;
  if (c->n == 0) return FGB_OK;
  if (!c->indices || !c->table || !c->out) return FGB_E_NULL;
  if ((reinterpret_cast<uintptr_t>(c->table) | reinterpret_cast<uintptr_t>(c->out)) & 15) return FGB_E_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int vec = row_pack(c->c, elem_bytes(c->dtype));
  cudaError_t e;
  if (c->dtype == FGB_F16) e = FGB_BY_PACK(__half, vec, emb_forward)(*c, s);
  else if (c->dtype == FGB_BF16) e = FGB_BY_PACK(__nv_bfloat16, vec, emb_forward)(*c, s);
  else e = FGB_BY_PACK(float, vec, emb_forward)(*c, s);
  return e != cudaSuccess ? cuda_status(e) : launch_status();
}

extern "C" int64_t fgb_embedding_workspace_bytes(const fgb_embedding_call* c) {
  using namespace fgb;
  int rc = emb_check(c);
  EmbPlan p;
  if (rc == FGB_OK) rc = emb_plan(*c, p);
  return rc != FGB_OK ? rc : static_cast<int64_t>(p.bytes);
}

extern "C" int fgb_embedding_backward(const fgb_embedding_call* c, void* stream) {
  using namespace fgb;
  int rc = emb_check(c);
  if (rc != FGB_OK) return rc;
  if (!c->grad_table || !c->workspace || (c->n > 0 && (!c->indices || !c->grad_out))) return FGB_E_NULL;
  if ((reinterpret_cast<uintptr_t>(c->grad_out) | reinterpret_cast<uintptr_t>(c->grad_table)) & 15) return FGB_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(c->workspace) & 255) return FGB_E_ALIGN;
  EmbPlan p;
  rc = emb_plan(*c, p);
  if (rc != FGB_OK) return rc;
  if (c->workspace_bytes < static_cast<int64_t>(p.bytes)) return FGB_E_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(c->workspace);
  int32_t* keys = reinterpret_cast<int32_t*>(ws + p.keys_off);
  int64_t* order = reinterpret_cast<int64_t*>(ws + p.order_off);
  const uint32_t n = static_cast<uint32_t>(c->n), rows = static_cast<uint32_t>(c->rows);
  int key_bits = 1;
  while (key_bits < 31 && (rows >> key_bits) != 0u) ++key_bits;  // the largest key is `rows`
  EmbGrad a{};
  a.g = c->grad_out, a.grad = c->grad_table, a.keys = keys, a.order = order;
  a.slab = reinterpret_cast<float*>(ws + p.slab_off), a.info = reinterpret_cast<EmbInfo*>(ws + p.info_off);
  a.n = n, a.rows = rows, a.chunk = p.chunk, a.ctas = p.ctas, a.C = c->c, a.scale = c->scale;
  if (n > 0 && emb_few(*c)) {
    const FewArgs q{c->indices, c->index_bits == 64, sort_passes_of(key_bits), c->padding_idx, 0u, c->status, status_mirror(c->status)};
    cudaError_t e;
    if (c->dtype == FGB_F16) e = FGB_BY_PACK(__half, p.vec, emb_few_launch)(a, q, s);
    else if (c->dtype == FGB_BF16) e = FGB_BY_PACK(__nv_bfloat16, p.vec, emb_few_launch)(a, q, s);
    else e = FGB_BY_PACK(float, p.vec, emb_few_launch)(a, q, s);
    return e != cudaSuccess ? cuda_status(e) : launch_status();
  }
  const uint64_t halves = uint64_t(c->rows) * c->c * (elem_bytes(c->dtype) / 2);
  const int64_t units = std::max<int64_t>(c->n, static_cast<int64_t>(halves / 8));
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(units, kEmbThreads), 1), int64_t(device_sm_count()) * 8));
  cudaError_t e = launch_chained(embedding_keys_kernel, dim3(grid), dim3(kEmbThreads), 0, s, c->indices, c->index_bits == 64, n, rows, c->padding_idx, keys,
                                 static_cast<uint16_t*>(c->grad_table), halves, c->status, status_mirror(c->status));
  if (e != cudaSuccess) return cuda_status(e);
  if (n == 0) return launch_status();
  rc = fgb_pp_sorted_idx(keys, c->n, key_bits, order, ws + p.sort_off, static_cast<int64_t>(p.sort_bytes), c->status, stream);
  if (rc != FGB_OK) return rc;
  if (c->dtype == FGB_F16) e = FGB_BY_PACK(__half, p.vec, emb_sum)(a, p, s);
  else if (c->dtype == FGB_BF16) e = FGB_BY_PACK(__nv_bfloat16, p.vec, emb_sum)(a, p, s);
  else e = FGB_BY_PACK(float, p.vec, emb_sum)(a, p, s);
  return e != cudaSuccess ? cuda_status(e) : launch_status();
}
