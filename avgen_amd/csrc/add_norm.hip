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
// in bf16), the backward reads dn, dh and h and writes dx.  It starts from the
// stored h, in bf16 rounded (by up to 2^-8 of the value) where the forward
// normed the fp32 sum: h is what the next layer saw and the caller holds
// anyway, while x and r would be a quarter more bytes and two tensors kept.
// A row stays in the registers of the threads that share it between its loads
// and its stores, so nothing is read twice; sums are fp32 and in a fixed order.
// 18,900 rows of 5,120 bf16: forward 125 us (6.2 TB/s), backward 160 + 6 (4.8
// TB/s), 9,450 of float32 125 and 154 + 5; 37,800 rows of 2,560 to e4m3 120 us
// (5.6 TB/s); 8 rows of 5,120 4 us.
#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

// dW partials of the backward: one per row group in flight, four waves' rows
// per workgroup where rows are narrow.
constexpr int max_parts(int64_t W) { return W <= 1024 ? 4096 : 1024; }

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
template <int CH>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* v) {
  if constexpr (CH == 8)
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_fp8x4(v[0], v[1], v[2], v[3]), pack_fp8x4(v[4], v[5], v[6], v[7])};
  else if constexpr (CH == 4)
    *reinterpret_cast<uint32_t*>(p) = pack_fp8x4(v[0], v[1], v[2], v[3]);
  else
    p[0] = (uint8_t)pack_fp8x4(v[0], 0.f, 0.f, 0.f);
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

__device__ __forceinline__ float fp8_row_scale(float top) {
  return top > 0.f ? fmaxf(top / 448.f, 1.1754943508222875e-38f) : 1.f;
}

// Forward.  A row takes a wave (narrow rows, 4 per workgroup) or a workgroup of
// as many waves as its chunks fill (see row_shape).
template <class T, int CH, int NV, bool WAVE, bool FP8>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void add_norm_kernel(AddNormArgs a) {
  constexpr int RPB = WAVE ? 4 : 1;
  __shared__ float red[16];
  const int TPR = WAVE ? 64 : blockDim.x;
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves or nobody
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
  ss = row_reduce<WAVE, false>(ss, red);
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
    top = row_reduce<WAVE, true>(top, red);
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
// 18,900 rows of 5,123 bf16 319 us (5,120 above: 125), 9,450 of 5,121 float32
// 186 (125).
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
  ss = row_reduce<false, false>(ss, red);
  const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
  auto norm = [&](int64_t c) {
    float w;
    load_gain<T, 1>(a.w, a.w32, c, &w);
    return ((float)x[c] + (float)r[c]) * rstd * w;
  };
  if constexpr (FP8) {
    float top = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) top = fmaxf(top, fabsf(norm(c)));
    top = row_reduce<false, true>(top, red);
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
// AHEAD: the next row's values are loaded before this row's sums (more
// registers; with two chunks per thread up to 512 threads).
// DH: a gradient of h is given.  (The loads are unconditional: behind a branch
// the compiler would wait for them before it uses the row loaded earlier,
// 202 us in place of 161 for 18,900 rows of 5,120.)
template <class T, int CH, int NV, bool WAVE, bool AHEAD, bool DH>
__global__ __launch_bounds__(WAVE ? 256 : (AHEAD && NV > 1 ? 512 : 1024)) void add_norm_bwd_kernel(AddNormArgs a) {
  constexpr int RPB = WAVE ? 4 : 1;
  __shared__ float red[2][2][16];
  const int TPR = WAVE ? 64 : blockDim.x;
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
  struct Row {
    RawChunk<T, CH> h[NV], g[NV], d[NV];
  };
  int64_t at[NV];       // this thread's columns, 0 past the end of the row,
  uint32_t in[NV];      // where what is loaded is masked out
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH;
    at[j] = col < a.W ? col : 0;
    in[j] = col < a.W ? 0xffffffffu : 0u;
  }
  auto load = [&](int64_t row, Row& r) {
    row = row < a.rows ? row : a.rows - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      r.h[j] = read_chunk<T, CH>(static_cast<const T*>(a.x) + row * a.xs + at[j]);
      r.g[j] = read_chunk<T, CH>(static_cast<const T*>(a.dn) + row * a.dns + at[j]);
      if constexpr (DH) r.d[j] = read_chunk<T, CH>(static_cast<const T*>(a.dh) + row * a.dhs + at[j]);
    }
  };
  Row next;
  if constexpr (AHEAD) load((int64_t)blockIdx.x * RPB + rg, next);
  for (int64_t row = (int64_t)blockIdx.x * RPB + rg; row < a.rows; row += step) {  // uniform over the row's threads
    Row cur;
    if constexpr (AHEAD) {
      cur = next;
      load(row + step, next);
    } else {
      load(row, cur);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) cur.h[j] &= in[j], cur.g[j] &= in[j];
    const auto &rh = cur.h, &rg = cur.g, &rd = cur.d;
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = chunk_value<T, CH>(rh[j], e);
        ss = fmaf(h, h, ss);
        dot = fmaf(chunk_value<T, CH>(rg[j], e) * w[j][e], h, dot);
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off), dot += __shfl_xor(dot, off);
    if constexpr (!WAVE) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) red[buf][0][wave] = ss, red[buf][1][wave] = dot;
      __syncthreads();
      ss = red[buf][0][0], dot = red[buf][1][0];
      for (int i = 1; i < TPR / 64; ++i) ss += red[buf][0][i], dot += red[buf][1][i];
      buf ^= 1;  // the next row's values go elsewhere: one barrier per row
    }
    const float rstd = 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
    const float m = dot / (float)a.W * rstd * rstd;
    T* op = static_cast<T*>(a.h) + row * a.W;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * TPR + t) * CH;
      float dx[CH];
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = chunk_value<T, CH>(rh[j], e), g = chunk_value<T, CH>(rg[j], e);
        dw[j][e] = fmaf(g, h * rstd, dw[j][e]);
        dx[e] = rstd * (g * w[j][e] - h * m);
        if constexpr (DH) dx[e] += chunk_value<T, CH>(rd[j], e);
      }
      if (col < a.W) store_chunk<T, CH>(op + col, dx);
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
// column.  18,900 rows of 5,123 bf16 919 us (5,120 above: 160), 9,450 of 5,121
// float32 394 (154).
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
    ss = row_reduce<false, false>(ss, red);
    dot = row_reduce<false, false>(dot, red);
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
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < W; c0 += (int64_t)gridDim.x * 32) {
    const int64_t col = c0 + c;
    float s = 0.f;
    if (col < W) {
#pragma unroll 8
      for (int p = g; p < nparts; p += 8) s += part[p * W + col];
    }
    __syncthreads();  // the last columns' sums are read
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

// Threads per row and chunks per thread (nv 0: the value-by-value kernels).  A
// wave for up to 64 chunks (forward: up to 128 of many rows); else as many
// waves as one chunk per thread fills for few rows, whose latency counts, or up
// to 512 chunks, two chunks per thread beyond (four for float rows past 2,048).
// 18,900 rows of 5,120 bf16, backward: 5 waves of two chunks 161 us, 10 of one
// 179, 4 of three 168.
struct RowShape {
  int tpr, nv;
};
RowShape row_shape(int64_t chunks, int64_t rows, int ch, bool bwd) {
  if (chunks <= 64) return {64, 1};
  if (chunks <= 128 && rows >= 1024 && !bwd) return {64, 2};
  const int nv = chunks <= 512 || (chunks <= 1024 && rows <= 512) ? 1 : (chunks <= 2048 ? 2 : 4);
  if (chunks > 1024 * nv || nv * ch > 16) return {0, 0};
  return {(int)((chunks + 64 * nv - 1) / (64 * nv)) * 64, nv};
}

template <class T, int NV, bool WAVE>
void launch_shape(const AddNormArgs& a, int tpr, int mode, int blocks, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T), RPB = WAVE ? 4 : 1;
  const dim3 block(WAVE ? 256 : tpr);
  const dim3 grid(mode == 2 ? blocks : (unsigned)((a.rows + RPB - 1) / RPB));
  if (mode == 2) {
    if constexpr (!(WAVE && NV == 2)) {
      constexpr bool kAhead = NV <= 2;
      const bool ahead = NV == 1 || (kAhead && tpr <= 512);
      if (ahead && a.dh)
        hipLaunchKernelGGL((add_norm_bwd_kernel<T, CH, NV, WAVE, kAhead, true>), grid, block, 0, stream, a);
      else if (ahead)
        hipLaunchKernelGGL((add_norm_bwd_kernel<T, CH, NV, WAVE, kAhead, false>), grid, block, 0, stream, a);
      else if (a.dh)
        hipLaunchKernelGGL((add_norm_bwd_kernel<T, CH, NV, WAVE, NV == 1, true>), grid, block, 0, stream, a);
      else
        hipLaunchKernelGGL((add_norm_bwd_kernel<T, CH, NV, WAVE, NV == 1, false>), grid, block, 0, stream, a);
    }
  } else if (mode == 1)
    hipLaunchKernelGGL((add_norm_kernel<T, CH, NV, WAVE, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((add_norm_kernel<T, CH, NV, WAVE, false>), grid, block, 0, stream, a);
}

// mode 0: forward, 1: forward with e4m3, 2: backward (`blocks` workgroups).
template <class T>
void launch_rows(const AddNormArgs& a, const RowShape& s, int mode, int blocks, hipStream_t stream) {
  if (s.tpr == 64 && s.nv == 1)
    launch_shape<T, 1, true>(a, s.tpr, mode, blocks, stream);
  else if (s.tpr == 64)
    launch_shape<T, 2, true>(a, s.tpr, mode, blocks, stream);  // forward
  else if (s.nv == 1)
    launch_shape<T, 1, false>(a, s.tpr, mode, blocks, stream);
  else if (s.nv == 2)
    launch_shape<T, 2, false>(a, s.tpr, mode, blocks, stream);
  else if constexpr (sizeof(T) == 4)
    launch_shape<T, 4, false>(a, s.tpr, mode, blocks, stream);
}

// Workgroups of the backward: 16 waves on a CU with one chunk per thread, 12
// with two, all of them resident.  More gain nothing: 37,800 rows of 2,560 in 2
// / 3 / 4 workgroups of 5 waves per CU 157 / 155 / 186 us.
int bwd_blocks(int64_t rows, int64_t W, const RowShape& s) {
  const int rpb = s.tpr == 64 ? 4 : 1, waves = s.tpr <= 64 ? 4 : s.tpr / 64;
  const int64_t want = (rows + rpb - 1) / rpb;
  const int fit = (s.nv == 2 ? 12 : 16) / waves;
  int64_t most = 256 * (fit > 0 ? fit : 1);
  if (most > max_parts(W) / rpb) most = max_parts(W) / rpb;
  return (int)(want < most ? want : most);
}

template <class T>
hipError_t forward_rows(const AddNormArgs& a, bool fp8, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T);
  LaunchTimer timer(kKidAddNorm, stream);
  const bool vec = chunked(a, sizeof(T), false);
  const RowShape s = vec ? row_shape(a.W / CH, a.rows, CH, false) : RowShape{0, 0};
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

// Any number of rows: the threads of a grid (up to 1,024 a row) stay below 2^32.
template <class T>
hipError_t forward(const AddNormArgs& all, bool fp8, hipStream_t stream) {
  constexpr int64_t kMost = 1 << 21;
  AddNormArgs a = all;
  for (int64_t left = all.rows; left > 0; left -= kMost) {
    a.rows = left < kMost ? left : kMost;
    const hipError_t e = forward_rows<T>(a, fp8, stream);
    if (e != hipSuccess) return e;
    a.x = static_cast<const T*>(a.x) + kMost * a.xs;
    a.r = static_cast<const T*>(a.r) + kMost * a.rs;
    a.h = static_cast<T*>(a.h) + kMost * a.W;
    a.n = static_cast<char*>(a.n) + kMost * a.W * (fp8 ? 1 : (int)sizeof(T));
    if (fp8) a.scale += kMost;
  }
  return hipSuccess;
}

template <class T>
hipError_t backward(const AddNormArgs& a, void* dw, bool dw32, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T);
  int nparts = 0;
  if (a.rows > 0) {
    LaunchTimer timer(kKidAddNormBwd, stream);
    const bool vec = chunked(a, sizeof(T), true);
    const RowShape s = vec ? row_shape(a.W / CH, a.rows, CH, true) : RowShape{0, 0};
    const int rpb = s.tpr == 64 ? 4 : 1, blocks = bwd_blocks(a.rows, a.W, s);
    nparts = blocks * rpb;
    if (s.nv > 0)
      launch_rows<T>(a, s, 2, blocks, stream);
    else
      hipLaunchKernelGGL(add_norm_bwd_any_kernel<T>, dim3(blocks), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t groups = (a.W + 31) / 32;
  hipLaunchKernelGGL(add_norm_dw_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(256), 0, stream,
                     a.part, nparts, a.W, dw, dw32);
  return hipGetLastError();
}

}  // namespace

size_t add_norm_bwd_workspace_bytes(int64_t rows, int64_t W) {
  const int64_t n = rows < max_parts(W) ? (rows + 3) / 4 * 4 : max_parts(W);
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
