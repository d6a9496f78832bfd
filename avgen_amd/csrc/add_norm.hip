// Residual addition and RMS norm over the model width, with the norm's output
// in the rows' type or in e4m3 with one scale per row, and its backward.
//
//   h = x + r (fp32; stored rounded to the rows' type)
//   rstd = 1 / sqrt(mean(h^2) + eps),  n = h * rstd * w      (from the fp32 h)
//   e4m3: scale = max|n| / 448 per row (1 for a row of zeros, at least 2^-126
//         so that its reciprocal stays finite), code = e4m3(n / scale)
// Backward, given dn (of n) and dh (of h, may be absent), from the stored h:
//   g = dn * w,  dx = dr = rstd * (g - h * rstd^2 * mean(g h)) + dh
//   dw = sum over rows of dn * h * rstd
// HBM-bound: the forward reads x and r and writes n and h (8 bytes an element
// in bf16), the backward reads dn, dh and h and writes dx.  A row stays in the
// registers of the threads that share it between its loads and its stores, so
// nothing is read twice; sums are fp32 and in a fixed order.
#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

constexpr int kMaxPartBlocks = 1024;  // dW partials of the backward

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
template <int CH>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* v) {
  if constexpr (CH == 8)
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_fp8x4(v[0], v[1], v[2], v[3]), pack_fp8x4(v[4], v[5], v[6], v[7])};
  else if constexpr (CH == 4)
    *reinterpret_cast<uint32_t*>(p) = pack_fp8x4(v[0], v[1], v[2], v[3]);
  else
    p[0] = (uint8_t)pack_fp8x4(v[0], 0.f, 0.f, 0.f);
}

// Sum (or maximum) over the TPR threads of a row; every thread of the
// workgroup calls it.  red: one float per wave.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = MAX ? fmaxf(v, __shfl_xor(v, off)) : v + __shfl_xor(v, off);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the last reduction's values are read
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

__device__ __forceinline__ float fp8_row_scale(float top) {
  return top > 0.f ? fmaxf(top / 448.f, 1.1754943508222875e-38f) : 1.f;
}

// Forward.  TPR threads per row: a wave for narrow rows (several rows per
// workgroup), a workgroup for wide ones.
template <class T, int CH, int TPR, int NV, bool FP8>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void add_norm_kernel(AddNormArgs a) {
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[TPR / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves (TPR 64) or nobody
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = static_cast<const T*>(a.r) + row * a.rs;
  float h[NV][CH], w[NV][CH];
  float y[NV][CH];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH;
    if (col < a.W) {
      load_chunk<T, CH>(x + col, h[j]);
      load_chunk<T, CH>(r + col, y[j]);
      load_gain<T, CH>(a.w, a.w32, col, w[j]);
    } else {
#pragma unroll
      for (int e = 0; e < CH; ++e) h[j][e] = y[j][e] = w[j][e] = 0.f;
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      h[j][e] += y[j][e];
      ss = fmaf(h[j][e], h[j][e], ss);
    }
  T* hp = static_cast<T*>(a.h) + row * a.W;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH;
    if (col < a.W) store_chunk<T, CH>(hp + col, h[j]);
  }
  ss = row_reduce<TPR, false>(ss, red);
  const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      h[j][e] = h[j][e] * rstd * w[j][e];
      if constexpr (FP8) top = fmaxf(top, fabsf(h[j][e]));
    }
  if constexpr (FP8) {
    top = row_reduce<TPR, true>(top, red);
    const float scale = fp8_row_scale(top), inv = 1.f / scale;
    if (t == 0) a.scale[row] = scale;
    uint8_t* np = static_cast<uint8_t*>(a.n) + row * a.W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * TPR + t) * CH;
#pragma unroll
      for (int e = 0; e < CH; ++e) h[j][e] *= inv;
      if (col < a.W) store_codes<CH>(np + col, h[j]);
    }
  } else {
    T* np = static_cast<T*>(a.n) + row * a.W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * TPR + t) * CH;
      if (col < a.W) store_chunk<T, CH>(np + col, h[j]);
    }
  }
}

// Rows of any width and alignment, one workgroup each, value by value; x and
// r are read again for the output (from L2 for all but the widest rows).
template <class T, bool FP8>
__global__ __launch_bounds__(256) void add_norm_any_kernel(AddNormArgs a) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = static_cast<const T*>(a.r) + row * a.rs;
  T* hp = static_cast<T*>(a.h) + row * a.W;
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < a.W; c += 256) {
    const float h = (float)x[c] + (float)r[c];
    hp[c] = (T)h;
    ss = fmaf(h, h, ss);
  }
  ss = row_reduce<256, false>(ss, red);
  const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
  auto norm = [&](int64_t c) {
    float w;
    load_gain<T, 1>(a.w, a.w32, c, &w);
    return ((float)x[c] + (float)r[c]) * rstd * w;
  };
  if constexpr (FP8) {
    float top = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) top = fmaxf(top, fabsf(norm(c)));
    top = row_reduce<256, true>(top, red);
    const float scale = fp8_row_scale(top), inv = 1.f / scale;
    if (threadIdx.x == 0) a.scale[row] = scale;
    uint8_t* np = static_cast<uint8_t*>(a.n) + row * a.W;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) {
      const float v = norm(c) * inv;
      store_codes<1>(np + c, &v);
    }
  } else {
    T* np = static_cast<T*>(a.n) + row * a.W;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) np[c] = (T)norm(c);
  }
}

// Backward.  Each row group walks over rows blockIdx, + gridDim, ...; its
// threads keep their columns of w and of the dW sum in registers.  Sum of h^2
// and of g h in one pass over the row.
template <class T, int CH, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void add_norm_bwd_kernel(AddNormArgs a) {
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[2][2][TPR / 64];
  const int t = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  float w[NV][CH], dw[NV][CH];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH;
#pragma unroll
    for (int e = 0; e < CH; ++e) w[j][e] = dw[j][e] = 0.f;
    if (col < a.W) load_gain<T, CH>(a.w, a.w32, col, w[j]);
  }
  const int64_t step = (int64_t)gridDim.x * RPB;
  int buf = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPB + rg; row < a.rows; row += step) {  // uniform over the row's threads
    const T* hp = static_cast<const T*>(a.x) + row * a.xs;
    const T* np = static_cast<const T*>(a.dn) + row * a.dns;
    float h[NV][CH], g[NV][CH], dh[NV][CH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * TPR + t) * CH;
#pragma unroll
      for (int e = 0; e < CH; ++e) h[j][e] = g[j][e] = dh[j][e] = 0.f;
      if (col < a.W) {
        load_chunk<T, CH>(hp + col, h[j]);
        load_chunk<T, CH>(np + col, g[j]);
        if (a.dh) load_chunk<T, CH>(static_cast<const T*>(a.dh) + row * a.dhs + col, dh[j]);
      }
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        ss = fmaf(h[j][e], h[j][e], ss);
        dot = fmaf(g[j][e] * w[j][e], h[j][e], dot);
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off), dot += __shfl_xor(dot, off);
    if constexpr (TPR > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) red[buf][0][wave] = ss, red[buf][1][wave] = dot;
      __syncthreads();
      ss = red[buf][0][0], dot = red[buf][1][0];
#pragma unroll
      for (int i = 1; i < TPR / 64; ++i) ss += red[buf][0][i], dot += red[buf][1][i];
      buf ^= 1;  // the next row's values go elsewhere: one barrier per row
    }
    const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
    const float m = dot / (float)a.W * rstd * rstd;
    T* op = static_cast<T*>(a.h) + row * a.W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * TPR + t) * CH;
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        dw[j][e] = fmaf(g[j][e], h[j][e] * rstd, dw[j][e]);
        dh[j][e] += rstd * (g[j][e] * w[j][e] - h[j][e] * m);
      }
      if (col < a.W) store_chunk<T, CH>(op + col, dh[j]);
    }
  }
  // The workgroup's row groups one after the other, then its partial.
  float* part = a.part + ((int64_t)blockIdx.x * RPB + rg) * a.W;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH;
    if (col < a.W) {
#pragma unroll
      for (int e = 0; e < CH; ++e) part[col + e] = dw[j][e];
    }
  }
}

// The backward for any width and alignment: two passes over each row, the dW
// partials of the workgroup's rows added in memory by the thread that owns the
// column.
template <class T>
__global__ __launch_bounds__(256) void add_norm_bwd_any_kernel(AddNormArgs a) {
  __shared__ float red[4];
  float* part = a.part + (int64_t)blockIdx.x * a.W;
  for (int64_t c = threadIdx.x; c < a.W; c += 256) part[c] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* hp = static_cast<const T*>(a.x) + row * a.xs;
    const T* np = static_cast<const T*>(a.dn) + row * a.dns;
    const T* dp = a.dh ? static_cast<const T*>(a.dh) + row * a.dhs : nullptr;
    float ss = 0.f, dot = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) {
      float w;
      load_gain<T, 1>(a.w, a.w32, c, &w);
      const float h = (float)hp[c];
      ss = fmaf(h, h, ss);
      dot = fmaf((float)np[c] * w, h, dot);
    }
    ss = row_reduce<256, false>(ss, red);
    dot = row_reduce<256, false>(dot, red);
    const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
    const float m = dot / (float)a.W * rstd * rstd;
    T* op = static_cast<T*>(a.h) + row * a.W;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) {
      float w;
      load_gain<T, 1>(a.w, a.w32, c, &w);
      const float h = (float)hp[c], g = (float)np[c];
      part[c] = fmaf(g, h * rstd, part[c]);
      op[c] = (T)((dp ? (float)dp[c] : 0.f) + rstd * (g * w - h * m));
    }
  }
}

// dW: the partials of 32 columns added in a fixed order by 8 groups of 32
// threads, then the groups.
__global__ __launch_bounds__(256) void add_norm_dw_kernel(const float* __restrict__ part, int nparts, int64_t W,
                                                          void* dw, bool dw32) {
  __shared__ float red[8][32];
  const int c = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < W) {
#pragma unroll 8
    for (int p = g; p < nparts; p += 8) s += part[p * W + col];
  }
  red[g][c] = s;
  __syncthreads();
  if (g == 0 && col < W) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][c];
    if (dw32)
      static_cast<float*>(dw)[col] = s;
    else
      static_cast<bf16*>(dw)[col] = (bf16)s;
  }
}

bool chunked(const AddNormArgs& a, int size, bool bwd) {
  const int64_t ch = 16 / size;
  uintptr_t p = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.w);
  bool ok = a.W % ch == 0 && a.xs % ch == 0;
  if (bwd) {
    p |= reinterpret_cast<uintptr_t>(a.dn) | reinterpret_cast<uintptr_t>(a.dh);
    ok = ok && a.dns % ch == 0 && a.dhs % ch == 0;
  } else {
    p |= reinterpret_cast<uintptr_t>(a.r) | reinterpret_cast<uintptr_t>(a.n);
    ok = ok && a.rs % ch == 0;
  }
  return ok && p % 16 == 0;
}

// Threads per row and chunks per thread for rows of `chunks` chunks: a wave
// up to 128 chunks, 256 threads up to 1,024, then 1,024.  Few rows leave the
// chip idle and wait for one row's latency: there a row takes 1,024 threads
// as soon as that shortens a thread's share.
struct RowShape {
  int tpr, nv;
};
// (A thread of 1,024 has 128 registers: at most 16 columns.)
RowShape row_shape(int64_t chunks, int64_t rows, int ch) {
  if (chunks <= 64) return {64, 1};
  if (chunks <= 128 && rows >= 1024) return {64, 2};
  if (chunks <= 256) return {256, 1};
  const int tpr = chunks > 1024 || rows <= 512 ? 1024 : 256;
  const int nv = (int)((chunks + tpr - 1) / tpr);
  if (tpr == 1024 && nv * ch > 16) return {0, 0};
  return {tpr, tpr == 1024 && nv == 3 ? 4 : nv};
}

template <class T, int TPR, int NV>
void launch_shape(const AddNormArgs& a, int mode, int blocks, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T), RPB = TPR < 256 ? 256 / TPR : 1;
  const dim3 block(TPR < 256 ? 256 : TPR);
  const dim3 grid(mode == 2 ? blocks : (unsigned)((a.rows + RPB - 1) / RPB));
  if (mode == 2)
    hipLaunchKernelGGL((add_norm_bwd_kernel<T, CH, TPR, NV>), grid, block, 0, stream, a);
  else if (mode == 1)
    hipLaunchKernelGGL((add_norm_kernel<T, CH, TPR, NV, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((add_norm_kernel<T, CH, TPR, NV, false>), grid, block, 0, stream, a);
}

// mode 0: forward, 1: forward with e4m3, 2: backward (`blocks` workgroups).
template <class T>
void launch_rows(const AddNormArgs& a, const RowShape& s, int mode, int blocks, hipStream_t stream) {
  if (s.tpr == 64 && s.nv == 1)
    launch_shape<T, 64, 1>(a, mode, blocks, stream);
  else if (s.tpr == 64)
    launch_shape<T, 64, 2>(a, mode, blocks, stream);
  else if (s.tpr == 256 && s.nv == 1)
    launch_shape<T, 256, 1>(a, mode, blocks, stream);
  else if (s.tpr == 256 && s.nv == 2)
    launch_shape<T, 256, 2>(a, mode, blocks, stream);
  else if (s.tpr == 256 && s.nv == 3)
    launch_shape<T, 256, 3>(a, mode, blocks, stream);
  else if (s.tpr == 256)
    launch_shape<T, 256, 4>(a, mode, blocks, stream);
  else if (s.nv == 1)
    launch_shape<T, 1024, 1>(a, mode, blocks, stream);
  else if (s.nv == 2)
    launch_shape<T, 1024, 2>(a, mode, blocks, stream);
  else if constexpr (sizeof(T) == 4)
    launch_shape<T, 1024, 4>(a, mode, blocks, stream);
}

// Workgroups of the backward and the dW partials they leave.
int bwd_blocks(int64_t rows, int rpb) {
  const int64_t want = (rows + rpb - 1) / rpb;
  return (int)(want < kMaxPartBlocks / rpb ? want : kMaxPartBlocks / rpb);
}

template <class T>
hipError_t forward(const AddNormArgs& a, bool fp8, hipStream_t stream) {
  if (a.rows > 2147483647) return hipErrorInvalidValue;
  constexpr int CH = 16 / (int)sizeof(T);
  LaunchTimer timer(kKidAddNorm, stream);
  const bool vec = chunked(a, sizeof(T), false);
  const RowShape s = vec ? row_shape(a.W / CH, a.rows, CH) : RowShape{0, 0};
  if (s.nv > 0) {
    launch_rows<T>(a, s, fp8 ? 1 : 0, 0, stream);
  } else {
    const dim3 grid((unsigned)a.rows);
    if (fp8)
      hipLaunchKernelGGL((add_norm_any_kernel<T, true>), grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((add_norm_any_kernel<T, false>), grid, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

template <class T>
hipError_t backward(const AddNormArgs& a, void* dw, bool dw32, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T);
  int nparts = 0;
  if (a.rows > 0) {
    LaunchTimer timer(kKidAddNormBwd, stream);
    const bool vec = chunked(a, sizeof(T), true);
    const RowShape s = vec ? row_shape(a.W / CH, a.rows, CH) : RowShape{0, 0};
    const int rpb = s.tpr == 64 ? 4 : 1, blocks = bwd_blocks(a.rows, rpb);
    nparts = blocks * rpb;
    if (s.nv > 0)
      launch_rows<T>(a, s, 2, blocks, stream);
    else
      hipLaunchKernelGGL(add_norm_bwd_any_kernel<T>, dim3(blocks), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(add_norm_dw_kernel, dim3((unsigned)((a.W + 31) / 32)), dim3(256), 0, stream, a.part, nparts, a.W,
                     dw, dw32);
  return hipGetLastError();
}

}  // namespace

size_t add_norm_bwd_workspace_bytes(int64_t rows, int64_t W) {
  const int64_t n = rows < kMaxPartBlocks ? (rows + 3) / 4 * 4 : kMaxPartBlocks;
  return (size_t)n * (size_t)W * sizeof(float);
}

hipError_t launch_add_norm(const AddNormArgs& a, bool f32, bool fp8, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  return f32 ? forward<float>(a, fp8, stream) : forward<bf16>(a, fp8, stream);
}

hipError_t launch_add_norm_bwd(const AddNormArgs& a, bool f32, void* dw, bool dw32, hipStream_t stream) {
  return f32 ? backward<float>(a, dw, dw32, stream) : backward<bf16>(a, dw, dw32, stream);
}

}  // namespace avattn
