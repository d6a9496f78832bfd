// Rows of a norm in the registers of the threads that share them: loads, stores
// and sums (add_norm.hip, gated_norm.hip).
#pragma once

#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

// The thread's values of a row: NV chunks of CH consecutive columns, chunk j
// at column (j * TPR + t) * CH.
template <class T, int CH>
__device__ __forceinline__ void load_chunk(const T* p, float* v) {
  if constexpr (CH == 8) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
  } else if constexpr (CH == 4) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = w[i];
  } else {
    v[0] = (float)p[0];
  }
}
template <class T, int CH>
__device__ __forceinline__ void store_chunk(T* p, const float* v) {
  if constexpr (CH == 8)
    *reinterpret_cast<u32x4*>(p) = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                         pack_bf16x2(v[6], v[7])};
  else if constexpr (CH == 4)
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  else
    p[0] = (T)v[0];
}
// A chunk as it was loaded (bf16 stays packed: half the registers), and its
// values.
template <class T, int CH>
using RawChunk = u32x4;
template <class T, int CH>
__device__ __forceinline__ RawChunk<T, CH> read_chunk(const T* p) {
  static_assert(CH * sizeof(T) == 16, "whole chunks");
  return *reinterpret_cast<const u32x4*>(p);
}
template <class T, int CH>
__device__ __forceinline__ float chunk_value(const RawChunk<T, CH>& r, int e) {
  if constexpr (CH == 8)
    return e & 1 ? bf16_hi(r[e / 2]) : bf16_lo(r[e / 2]);
  else
    return __uint_as_float(r[e]);
}
// The gain's columns: in the rows' type or fp32.
template <class T, int CH>
__device__ __forceinline__ void load_gain(const void* w, bool w32, int64_t col, float* v) {
  if constexpr (sizeof(T) == 4) {
    load_chunk<float, CH>(static_cast<const float*>(w) + col, v);
  } else if (!w32) {
    load_chunk<T, CH>(static_cast<const T*>(w) + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = static_cast<const float*>(w)[col + i];
  }
}
// Sum (or maximum) over the threads of a row: a wave (WAVE) or the workgroup,
// every thread of which calls it.  red: one float per wave.
template <bool WAVE, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = MAX ? fmaxf(v, __shfl_xor(v, off)) : v + __shfl_xor(v, off);
  if constexpr (!WAVE) {
    __syncthreads();  // the last reduction's values are read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < (int)blockDim.x / 64; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

}  // namespace

}  // namespace avattn
