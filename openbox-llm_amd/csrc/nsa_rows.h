// Row-wise building blocks: runs of 8 elements at any element-aligned address,
// and sums / maxima over a wave or a workgroup.
//
// Rows of odd lengths start at addresses that are multiples of the element
// size only.  Global loads and stores of 16 bytes take such addresses on this
// GPU, so one form serves every length: whole runs of 8 elements as vectors
// of element alignment, the row's last run element by element.
#pragma once

#include <type_traits>

#include "nsa_common.h"

namespace nsa {

typedef bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void load_run8(const bf16* p, float (&f)[8]) {
  const bf16x8u v = *reinterpret_cast<const bf16x8u*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
}
__device__ __forceinline__ void load_run8(const float* p, float (&f)[8]) {
  const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = a[j], f[4 + j] = b[j];
}
__device__ __forceinline__ void store_run8(bf16* p, const float (&f)[8]) {
  bf16x8u v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (bf16)f[j];
  *reinterpret_cast<bf16x8u*>(p) = v;
}
__device__ __forceinline__ void store_run8(float* p, const float (&f)[8]) {
  *reinterpret_cast<f32x4u*>(p) = (f32x4u){f[0], f[1], f[2], f[3]};
  *reinterpret_cast<f32x4u*>(p + 4) = (f32x4u){f[4], f[5], f[6], f[7]};
}

// The same with only `n` elements in the row from here on (n may be <= 0 or
// more than 8); elements past the row's end read as `fill` and are not written.
template <typename T>
__device__ __forceinline__ void load_run8(const T* p, int n, float (&f)[8], float fill = 0.0f) {
  if (n >= 8) {
    load_run8(p, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = fill;
    if (n > 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) f[j] = (float)p[j];
    }
  }
}
template <typename T>
__device__ __forceinline__ void store_run8(T* p, int n, const float (&f)[8]) {
  if (n >= 8) {
    store_run8(p, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)f[j];
  }
}

// A run whose element type is known at run time only (uniform over the wave).
__device__ __forceinline__ void load_run8_of(const void* p, bool is_bf16, int64_t at, int n, float (&f)[8]) {
  if (is_bf16)
    load_run8(static_cast<const bf16*>(p) + at, n, f);
  else
    load_run8(static_cast<const float*>(p) + at, n, f);
}

// Combine each N = 8, 16, 32 or 64 neighbouring lanes of a wave by register
// moves alone (within rows of 16 by DPP, across rows by the row swaps); op is
// commutative, so that all of them end with the same bits.
template <int N, typename Op>
__device__ __forceinline__ uint32_t lanes_all(uint32_t v, Op op) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v = op(v, dpp(v, std::integral_constant<int, 0xB1>{}));     // quad_perm [1,0,3,2]
  v = op(v, dpp(v, std::integral_constant<int, 0x4E>{}));     // quad_perm [2,3,0,1]
  v = op(v, dpp(v, std::integral_constant<int, 0x141>{}));    // row_half_mirror: 8
  if (N >= 16) v = op(v, dpp(v, std::integral_constant<int, 0x140>{}));   // row_mirror: 16
  if (N >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(p[0], p[1]);
  }
  if (N >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(p[0], p[1]);
  }
  return v;
}
// (a 64-bit value moves as its halves)
template <int N>
__device__ __forceinline__ double wave_sum(double v) {
  auto dpp = [](double x, auto ctrl) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, decltype(ctrl)::value, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(u >> 32), decltype(ctrl)::value, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  auto rows = [](double x, auto swap) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
           __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});
  v += dpp(v, std::integral_constant<int, 0x4E>{});
  v += dpp(v, std::integral_constant<int, 0x141>{});
  if (N >= 16) v += dpp(v, std::integral_constant<int, 0x140>{});
  if (N >= 32) v = rows(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  if (N >= 64) v = rows(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}
template <int N = kWave>
__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(lanes_all<N>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(lanes_all<kWave>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}

// Sum over the N threads of a row: part of a wave, a wave, or a workgroup of
// several (`buf` then holds a float a wave in LDS and is free again after the
// next barrier that follows).
template <int N>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  v = wave_sum<(N < kWave ? N : kWave)>(v);
  if (N <= kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) buf[threadIdx.x / kWave] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N / kWave; ++i) s += buf[i];
  return s;
}

}  // namespace nsa
