// Shared pieces of the token-model operators (embedding.hip, topk.hip, distill.hip): element types, 16-byte granules
// of a row, wave / workgroup reductions that leave the result in every lane, and the row loader.
//
// Element types: fp32, bf16, fp16 (tags BDE_F32 / BDE_BF16 / BDE_F16 of the C ABI).  Whatever the type, arithmetic is
// fp32; a value is rounded to its type once, when it is stored (round to nearest even, the hardware conversions).
#pragma once

#include "bde_common.hpp"

namespace bde {

using bf16_t = __bf16;
using f16_t = _Float16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
// v_exp_f32: 2^x to one ulp; results below 2^-126 are flushed to zero, 2^-inf = 0
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 16 bytes of a row, kept as raw words so that a row in registers costs its own size whatever its type
template <typename T>
struct Granule {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  union Bits {
    u32x4 raw;
    T v[N];
  };
};
template <typename T>
__device__ __forceinline__ float granule_get(const u32x4& g, int i);
template <>
__device__ __forceinline__ float granule_get<float>(const u32x4& g, int i) {
  return __uint_as_float(g[i]);
}
template <>
__device__ __forceinline__ float granule_get<bf16_t>(const u32x4& g, int i) {   // a bf16 is the upper half of an fp32
  return __uint_as_float((i & 1) ? (g[i >> 1] & 0xFFFF0000u) : (g[i >> 1] << 16));
}
template <>
__device__ __forceinline__ float granule_get<f16_t>(const u32x4& g, int i) {
  const uint16_t b = static_cast<uint16_t>((i & 1) ? (g[i >> 1] >> 16) : (g[i >> 1] & 0xFFFFu));
  return static_cast<float>(__builtin_bit_cast(f16_t, b));
}
template <typename T>
__device__ __forceinline__ void granule_set(u32x4& g, int i, T v) {
  if constexpr (sizeof(T) == 4) {
    g[i] = __builtin_bit_cast(uint32_t, v);
  } else {
    const uint32_t b = __builtin_bit_cast(uint16_t, v);
    g[i >> 1] = (i & 1) ? ((g[i >> 1] & 0xFFFFu) | (b << 16)) : ((g[i >> 1] & 0xFFFF0000u) | b);
  }
}
// A granule that stays packed between the phases of a kernel: without this the compiler unpacks a row once and keeps four (or
// two) times its registers alive -- into scratch memory.
__device__ __forceinline__ void stay_packed(u32x4& g) { asm volatile("" : "+v"(g)); }
// A running value that is brought up to date here, not after the branches that follow (which would keep its operands alive).
__device__ __forceinline__ void settle(float& x) { asm volatile("" : "+v"(x)); }
// fp32 values -> one granule of T, each rounded once
template <typename T>
__device__ __forceinline__ u32x4 granule_pack(const float* f) {
  typename Granule<T>::Bits b;
#pragma unroll
  for (int i = 0; i < Granule<T>::N; ++i) b.v[i] = static_cast<T>(f[i]);
  return b.raw;
}

// A row of V elements starting anywhere.  Granule g covers the elements [g * N - shift, g * N - shift + N) of the row, with
// `shift` = how far the row's first element lies behind a 16-byte border: whole granules are aligned 16-byte accesses, the
// one or two at the ends are read element by element (never a byte outside the row).
template <typename T>
struct RowView {
  const T* p;
  int V, shift, granules;
  __device__ __forceinline__ RowView(const T* row, int V_) : p(row), V(V_) {
    constexpr int N = Granule<T>::N;
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N);
    granules = (V + shift + N - 1) / N;
  }
  __device__ __forceinline__ int first(int g) const { return g * Granule<T>::N - shift; }
  __device__ __forceinline__ bool whole(int g) const { return first(g) >= 0 && first(g) + Granule<T>::N <= V; }
  // the granule's elements; places outside the row (and whole granules behind it) hold -inf
  __device__ __forceinline__ u32x4 load(int g) const {
    constexpr int N = Granule<T>::N;
    const int e0 = first(g);
    if (whole(g)) return *reinterpret_cast<const u32x4*>(p + e0);
    u32x4 r;
    constexpr uint32_t fill = sizeof(T) == 4 ? 0xFF800000u : __is_same(T, bf16_t) ? 0xFF80FF80u : 0xFC00FC00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fill;
    if (g < granules) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i >= 0 && e0 + i < V) granule_set<T>(r, i, p[e0 + i]);
    }
    return r;
  }
};

// ---- reductions whose result every lane holds: 4 DPP steps inside 16 lanes, then the four rows of the wave
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <typename F>
__device__ __forceinline__ float wave_all(float x, F f) {
  x = f(x, dpp_move<0xB1>(x));     // lane ^ 1
  x = f(x, dpp_move<0x4E>(x));     // lane ^ 2
  x = f(x, dpp_move<0x141>(x));    // the other four of eight
  x = f(x, dpp_move<0x140>(x));    // the other eight of sixteen
  const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 0));
  const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16));
  const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 32));
  const float d = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 48));
  return f(f(a, b), f(c, d));
}
__device__ __forceinline__ float wave_all_sum(float x) {
  return wave_all(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_all_max(float x) {
  return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
// A row is handled by NT threads: a workgroup of its own, or -- rows that fit one wave -- one of the four waves of a workgroup
// (a launch of one-wave workgroups is bound by their dispatch).  What the lanes of a wave exchange through LDS needs no barrier,
// only the wait for the LDS operations.
template <int NT>
constexpr int kRowsPerGroup = NT == 64 ? 4 : 1;
constexpr int64_t kRowsPerLaunch = 1 << 21;      // (a launch holds fewer than 2^32 threads)
template <int NT>
__device__ __forceinline__ void row_sync() {
  if constexpr (NT == 64) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}
// The reductions over a row's NT threads: one value per wave in `slots` (>= NT / 64 floats, not used by a reduction still being
// read), ONE barrier; every wave sums the slots in the same order.
template <int NT, typename F>
__device__ __forceinline__ float row_all(float x, float* slots, F f) {
  constexpr int W = NT / 64;
  x = wave_all(x, f);
  if constexpr (W == 1) {
    row_sync<NT>();                // what the caller wrote to LDS before is visible, whatever NT is
    return x;
  } else {
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = x;
    row_sync<NT>();
    float r = slots[0];
#pragma unroll
    for (int i = 1; i < W; ++i) r = f(r, slots[i]);
    return r;
  }
}
template <int NT>
__device__ __forceinline__ float row_all_sum(float x, float* slots) {
  return row_all<NT>(x, slots, [](float a, float b) { return a + b; });
}
template <int NT>
__device__ __forceinline__ float row_all_max(float x, float* slots) {
  return row_all<NT>(x, slots, [](float a, float b) { return fmaxf(a, b); });
}

// a token / class index of either width; -1 where it is outside [0, limit)
__device__ __forceinline__ int load_index(const void* p, int is64, int64_t i, int limit) {
  if (is64) {
    const int64_t t = static_cast<const int64_t*>(p)[i];
    return t >= 0 && t < limit ? static_cast<int>(t) : -1;
  }
  const int t = static_cast<const int*>(p)[i];
  return t >= 0 && t < limit ? t : -1;
}
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == BDE_F32) return static_cast<const float*>(p)[i];
  if (dtype == BDE_BF16) return static_cast<float>(static_cast<const bf16_t*>(p)[i]);
  return static_cast<float>(static_cast<const f16_t*>(p)[i]);
}
static inline size_t dtype_bytes(int dtype) { return dtype == BDE_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype == BDE_F32 || dtype == BDE_BF16 || dtype == BDE_F16; }

}  // namespace bde
