// Ragged rows: what the layers on [n, C] feature rows share -- row ranges of samples, and packs of channels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "fgb_common.cuh"

namespace fgb {

// Row ranges of `count` samples: offsets[s] .. offsets[s + 1], int32 or int64 on the device, or `count` equal ranges when
// there are none.  What is read is clamped to the rows that exist, so that ranges which do not ascend give wrong results
// (and a soft error, see check) but no access out of bounds.
struct RowRanges {
  const void* offsets;
  int wide;        // int64 offsets
  uint32_t n;      // rows
  uint32_t count;  // samples
  __device__ __forceinline__ uint32_t at(uint32_t s) const {
    if (offsets == nullptr) return static_cast<uint32_t>(uint64_t(n) * s / count);  // n is a multiple of count
    const int64_t v = wide ? __ldg(static_cast<const int64_t*>(offsets) + s) : __ldg(static_cast<const int32_t*>(offsets) + s);
    return v < 0 ? 0u : v > int64_t(n) ? n : static_cast<uint32_t>(v);
  }
  // whether entry s lies in [0, n] and not behind the next one
  __device__ __forceinline__ bool good(uint32_t s) const {
    if (offsets == nullptr) return true;
    const int64_t a = wide ? static_cast<const int64_t*>(offsets)[s] : static_cast<const int32_t*>(offsets)[s];
    const int64_t b = wide ? static_cast<const int64_t*>(offsets)[s + 1] : static_cast<const int32_t*>(offsets)[s + 1];
    return a >= 0 && a <= b && b <= int64_t(n);
  }
  // How many samples begin before `row`.  The whole warp calls it: 32 places are looked at per step.
  __device__ __forceinline__ uint32_t begun_before(uint32_t row) const {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0, hi = count;  // samples below lo begin before row, those from hi on do not
    while (hi > lo) {
      const uint32_t step = (hi - lo + 31u) / 32u, s = lo + lane * step;
      const unsigned yes = __ballot_sync(0xffffffffu, s < hi && at(s) < row);
      const uint32_t k = static_cast<uint32_t>(__popc(yes));
      if (k == 0u) return lo;
      const uint32_t top = lo + k * step;
      lo += (k - 1u) * step + 1u;
      if (top < hi) hi = top;
    }
    return lo;
  }
  // the samples that a block of rows [row0, row1) meets: first .. last; a block's first is the last of the block before.  The
  // whole warp calls it.
  __device__ __forceinline__ void of_block(uint32_t row0, uint32_t row1, bool last_block, uint32_t& first, uint32_t& last) const {
    uint32_t a, b;
    if (count <= 32u) {  // one load for both
      const uint32_t lane = threadIdx.x & 31u, v = lane < count ? at(lane) : 0xFFFFFFFFu;
      a = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, v < row0)));
      b = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, v < row1)));
    } else {
      a = row0 == 0u ? 0u : begun_before(row0);
      b = last_block ? count : begun_before(row1);
    }
    first = a > 0u ? a - 1u : 0u;
    last = last_block ? count - 1u : b > 0u ? b - 1u : 0u;
  }
  // every entry of the grid's share is looked at; threads of the whole grid call it
  __device__ __forceinline__ void check(int32_t* status, int32_t* mirror) const {
    if (offsets == nullptr) return;
    for (uint32_t s = (blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; s < count; s += gridDim.x * gridDim.y * blockDim.x) {
      if (!good(s)) {
        report(status, FGB_S_BAD_OFFSETS);
        mirror_code(mirror, FGB_S_BAD_OFFSETS);
      }
    }
  }
};

// kVec consecutive channels: 16 bytes where rows are whole 16-byte pieces, fewer otherwise
template <typename T, int kVec>
struct Channels;
template <int kBytes>
struct RawBytes;
template <>
struct RawBytes<16> {
  using type = uint4;
};
template <>
struct RawBytes<8> {
  using type = uint2;
};
template <>
struct RawBytes<4> {
  using type = uint32_t;
};
template <>
struct RawBytes<2> {
  using type = uint16_t;
};
template <typename T, int kVec>
struct Channels {
  using Raw = typename RawBytes<sizeof(T) * kVec>::type;
  static __device__ __forceinline__ Raw load(const T* p) { return __ldg(reinterpret_cast<const Raw*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& raw, float (&f)[kVec]) {
    if constexpr (std::is_same<T, float>::value) {
      const float* v = reinterpret_cast<const float*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] = v[i];
    } else if constexpr (kVec == 1) {
      f[0] = static_cast<float>(*reinterpret_cast<const T*>(&raw));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* v = reinterpret_cast<const T2*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) {
        float2 t;
        if constexpr (std::is_same<T, __half>::value) t = __half22float2(v[i]);
        else t = __bfloat1622float2(v[i]);
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[kVec]) {  // rounds to nearest
    Raw raw;
    if constexpr (std::is_same<T, float>::value) {
      float* v = reinterpret_cast<float*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = f[i];
    } else if constexpr (kVec == 1) {
      *reinterpret_cast<T*>(&raw) = static_cast<T>(f[0]);
    } else if constexpr (std::is_same<T, __half>::value) {
      __half2* v = reinterpret_cast<__half2*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) v[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    } else {
      __nv_bfloat162* v = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    }
    return raw;
  }
  static __device__ __forceinline__ void store(T* p, const Raw& raw) { *reinterpret_cast<Raw*>(p) = raw; }
  static __device__ __forceinline__ void store_streaming(T* p, const Raw& raw) { __stcs(reinterpret_cast<Raw*>(p), raw); }
};

// the widest pack that divides a row of C channels: 16 bytes, else 8 or 4, else one channel
inline int row_pack(int C, int elem) {
  for (int v = 16 / elem; v > 1; v /= 2)
    if (C % v == 0) return v;
  return 1;
}

// parameters of either the features' type or fp32.  The 16-bit types are loaded as integers: __ldg of __half and
// __nv_bfloat16 is an asm statement without side effects to the compiler, which may run it ahead of the test that guards it.
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t c) {
  if (dtype == FGB_F16) return __half2float(__ushort_as_half(__ldg(static_cast<const unsigned short*>(p) + c)));
  if (dtype == FGB_BF16) return __bfloat162float(__ushort_as_bfloat16(__ldg(static_cast<const unsigned short*>(p) + c)));
  return __ldg(static_cast<const float*>(p) + c);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t c, float v) {
  if (dtype == FGB_F16) static_cast<__half*>(p)[c] = __float2half_rn(v);
  else if (dtype == FGB_BF16) static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[c] = v;
}

}  // namespace fgb
