// The step between two sections of a block: the norm behind a section, its gate,
// the residual addition, and the modulated norm in front of the next section.
//
//   y = x * rx * p           rx = 1 / sqrt(mean(x^2) + eps)    (without p: y = x)
//   h = alpha r + g y        (fp32; stored rounded to the rows' type)
//   n = h * rh * w (1 + s) + t,  rh = 1 / sqrt(mean(h^2) + eps), the fp32 h
// Without w, g, s or t: 1, 1, 0, 0.  g, s and t have a row for each group of R
// consecutive rows (R = all of them: one row; R = 1: one per token).
// Backward, given dn and dh (may be absent), from x and r, which give h again
// without its rounding, and the forward's rx and rh:
//   A = w (1 + s),  d = dh + rh (dn A - h rh^2 m),  m = mean(dn A h),  dr = alpha d
//   b = g p,        dx = d b                            without p
//                   dx = rx (d b - x rx^2 mean(d b x))  with it, where
//   sum(d b x) = sum(b x (dh + rh dn A)) - rh^3 m sum(b x h): one pass of sums
// and per column, over the rows of a group, the sums N = dn h rh, T = dn and
// C = d x rx (without p: d x), from which ds = w N, dt = T, dg = p C, and over
// the groups dw = sum (1 + s) N, dp = sum g C.
// HBM-bound: the forward reads x and r and writes h and n, the backward reads x,
// r, dn and dh and writes dx and dr (one tensor where they are alike).  A row
// stays in the registers of the threads that share it (8 to 64 lanes of a wave, or a
// workgroup), which keep their columns of A, b and t, and of the sums, over the rows of a
// group that they take one after the other.  Sums are fp32, in a fixed order.
#include "norm_parts.h"

namespace avattn {

namespace {

// A per-column vector of the rows' type or fp32 (null: `otherwise`), CH columns
// from `at` on; CH > 1: whole 16-byte chunks.
template <class T, int CH>
__device__ __forceinline__ void load_vector(const void* p, bool f32, int64_t at, float otherwise, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < CH; ++e) v[e] = otherwise;
  } else if (sizeof(T) == 2 && !f32) {
    load_chunk<T, CH>(static_cast<const T*>(p) + at, v);
  } else {
    constexpr int C4 = CH > 1 ? 4 : 1;
#pragma unroll
    for (int e = 0; e < CH; e += C4) load_chunk<float, C4>(static_cast<const float*>(p) + at + e, v + e);
  }
}
template <class T, int CH>
__device__ __forceinline__ void store_vector(void* p, bool f32, int64_t at, const float* v) {
  if (sizeof(T) == 2 && !f32) {
    store_chunk<T, CH>(static_cast<T*>(p) + at, v);
  } else {
    constexpr int C4 = CH > 1 ? 4 : 1;
#pragma unroll
    for (int e = 0; e < CH; e += C4) store_chunk<float, C4>(static_cast<float*>(p) + at + e, v + e);
  }
}

// CH columns as loaded: 16 bytes of them, or one value (its fp32 bits).
template <int CH>
struct RawOf {
  typedef u32x4 type;
};
template <>
struct RawOf<1> {
  typedef uint32_t type;
};
template <int CH>
using Raw = typename RawOf<CH>::type;
template <class T, int CH>
__device__ __forceinline__ float raw_value(const Raw<CH>& r, int e) {
  if constexpr (CH == 1)
    return __uint_as_float(r);
  else
    return chunk_value<T, CH>(r, e);
}
// Those at a byte offset of a row.
template <class T, int CH>
__device__ __forceinline__ Raw<CH> read_at(const void* base, int64_t row, int64_t stride, uint32_t off) {
  const char* p = static_cast<const char*>(base) + row * stride * (int64_t)sizeof(T) + off;
  if constexpr (CH == 1 && sizeof(T) == 2)
    return (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16;
  else
    return *reinterpret_cast<const Raw<CH>*>(p);
}
template <class T, int CH>
__device__ __forceinline__ void write_at(void* base, int64_t row, int64_t stride, uint32_t off, const float* v) {
  store_chunk<T, CH>(reinterpret_cast<T*>(static_cast<char*>(base) + row * stride * (int64_t)sizeof(T) + off), v);
}

// What a thread knows of its columns for the rows of a group: a = w (1 + s),
// b = g p.
template <class T, int CH>
__device__ __forceinline__ void group_vectors(const GatedNormArgs& a, int64_t group, int64_t col, float* av, float* bv,
                                              float* tv) {
  float y[CH];
  load_vector<T, CH>(a.w, a.w32, col, 1.f, av);
  load_vector<T, CH>(a.s, a.m32, group * a.ss + col, 0.f, y);
#pragma unroll
  for (int e = 0; e < CH; ++e) av[e] *= 1.f + y[e];
  load_vector<T, CH>(a.g, a.m32, group * a.gs + col, 1.f, bv);
  load_vector<T, CH>(a.p, a.p32, col, 1.f, y);
#pragma unroll
  for (int e = 0; e < CH; ++e) bv[e] *= y[e];
  if (tv) load_vector<T, CH>(a.t, a.m32, group * a.ts + col, 0.f, tv);
}

// The same of chunk j, zeros past the end of the row (in 0), where an infinite or
// NaN entry of column 0 would reach the row's sums through 0 * inf.
template <int CH>
__device__ __forceinline__ void mask_vectors(uint32_t in, float* av, float* bv) {
#pragma unroll
  for (int e = 0; e < CH; ++e) {
    av[e] = __uint_as_float(__float_as_uint(av[e]) & in);
    bv[e] = __uint_as_float(__float_as_uint(bv[e]) & in);
  }
}

__device__ __forceinline__ float row_rstd(float ss, const GatedNormArgs& a) {
  return 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
}

// How rows are shared: SIZE 0: a row by tpr lanes of a wave, 256 / tpr rows in a
// workgroup; 1, 2, 3: by a workgroup of up to 512, 768 or 1,024 threads.  Waves per
// SIMD that a kernel is compiled for: as many as its registers allow without
// spills.
template <int SIZE>
struct Threads {
  static constexpr int most = SIZE == 0 ? 256 : (SIZE == 1 ? 512 : (SIZE == 2 ? 768 : 1024));
  static constexpr int fwd = SIZE == 3 ? 4 : 5, bwd = SIZE == 3 ? 4 : 3;
};

// N sums over the threads of a row; red: a float per sum and wave, another one for
// the next sums (so that one barrier does).
template <bool WAVE, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[16], int tpr) {
  if constexpr (WAVE) {
    for (int off = tpr >> 1; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], off);
  } else {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], off);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = red[k][0];
      for (int i = 1; i < tpr / 64; ++i) v[k] += red[k][i];
    }
  }
}

// Forward.  A worker, tpr lanes or a workgroup, takes every per_group-th row of a
// group, the next row loaded before this one's sums.
template <class T, int CH, int NV, int SIZE, bool POST>
__global__ __launch_bounds__(Threads<SIZE>::most, Threads<SIZE>::fwd) void gated_norm_kernel(GatedNormArgs a) {
  constexpr bool WAVE = SIZE == 0;
  constexpr bool AHEAD = NV * CH * sizeof(T) <= 32;  // (else registers spill)
  __shared__ float red[2][1][16];
  const int TPR = WAVE ? a.tpr : (int)blockDim.x, RPB = WAVE ? 256 / TPR : 1;
  const int t = WAVE ? threadIdx.x & (TPR - 1) : threadIdx.x;
  const int64_t worker = a.first + (int64_t)blockIdx.x * RPB + (WAVE ? threadIdx.x / TPR : 0);
  const int64_t group = worker / a.per_group, end = min((group + 1) * a.R, a.rows);
  int64_t row = group * a.R + worker % a.per_group;
  if (row >= end) return;  // all threads of a row
  float av[NV][CH], bv[NV][CH], tv[NV][CH];
  uint32_t off[NV];  // this thread's columns, 0 past the end of the row,
  uint32_t in[NV];   // where what is loaded is masked out
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH, at = col < a.W ? col : 0;
    in[j] = col < a.W ? 0xffffffffu : 0u;
    off[j] = (uint32_t)at * sizeof(T);
    group_vectors<T, CH>(a, group, at, av[j], bv[j], tv[j]);
    mask_vectors<CH>(in[j], av[j], bv[j]);
  }
  struct Row {
    Raw<CH> x[NV], r[NV];
  };
  auto load = [&](int64_t row, Row& q) {
    row = row < end ? row : end - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = read_at<T, CH>(a.x, row, a.xs, off[j]);
      q.r[j] = read_at<T, CH>(a.r, row, a.rs, off[j]);
    }
  };
  auto value = [](const Raw<CH>& r, int e) { return raw_value<T, CH>(r, e); };
  Row next;
  if (AHEAD) load(row, next);
  int buf = 0;
  for (; row < end; row += a.per_group) {
    Row cur;
    if (AHEAD) {
      cur = next;
      load(row + a.per_group, next);
    } else {
      load(row, cur);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) cur.x[j] &= in[j], cur.r[j] &= in[j];
    float rx = 1.f;
    if constexpr (POST) {
      float ss[1] = {0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < CH; ++e) ss[0] = fmaf(value(cur.x[j], e), value(cur.x[j], e), ss[0]);
      row_sums<WAVE, 1>(ss, red[0], TPR);
      rx = row_rstd(ss[0], a);
    }
    float ss[1] = {0.f};
    float h[NV][CH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        h[j][e] = fmaf(value(cur.x[j], e) * rx, bv[j][e], a.alpha * value(cur.r[j], e));
        ss[0] = fmaf(h[j][e], h[j][e], ss[0]);
      }
      if (in[j]) write_at<T, CH>(a.h, row, a.W, off[j], h[j]);
    }
    row_sums<WAVE, 1>(ss, red[POST ? 1 : buf], TPR);
    buf ^= 1;
    const float rh = row_rstd(ss[0], a);
    if (a.stats != nullptr && t == 0) *reinterpret_cast<f32x2*>(a.stats + 2 * row) = f32x2{rx, rh};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) h[j][e] = fmaf(h[j][e] * rh, av[j][e], tv[j][e]);
      if (in[j]) write_at<T, CH>(a.n, row, a.W, off[j], h[j]);
    }
  }
}

constexpr int kAny = 1024;  // threads of the kernels that take any row

// Rows of any width and alignment, one workgroup each, value by value; x and r
// are read again for the sum's norm and for the output.
template <class T>
__global__ __launch_bounds__(kAny) void gated_norm_any_kernel(GatedNormArgs a) {
  __shared__ float red[16];
  const int64_t row = a.first + blockIdx.x, group = row / a.R;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = static_cast<const T*>(a.r) + row * a.rs;
  float rx = 1.f;
  if (a.p != nullptr) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += kAny) ss = fmaf((float)x[c], (float)x[c], ss);
    rx = row_rstd(row_reduce<false, false>(ss, red), a);
  }
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < a.W; c += kAny) {
    float av, bv;
    group_vectors<T, 1>(a, group, c, &av, &bv, nullptr);
    const float h = fmaf((float)x[c] * rx, bv, a.alpha * (float)r[c]);
    static_cast<T*>(a.h)[row * a.W + c] = (T)h;
    ss = fmaf(h, h, ss);
  }
  const float rh = row_rstd(row_reduce<false, false>(ss, red), a);
  if (a.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<f32x2*>(a.stats + 2 * row) = f32x2{rx, rh};
  for (int64_t c = threadIdx.x; c < a.W; c += kAny) {
    float av, bv, tv;
    group_vectors<T, 1>(a, group, c, &av, &bv, &tv);
    const float h = fmaf((float)x[c] * rx, bv, a.alpha * (float)r[c]);
    static_cast<T*>(a.n)[row * a.W + c] = (T)fmaf(h * rh, av, tv);
  }
}

// Backward.  Workgroups take rows of a group in turn, as many at once as they
// have workers, and leave a part of the sums each; with a row of g, s and t per token
// (TOKEN) they take all rows, write that token's ds, dt and dg and keep the sums of
// dw and dp.  A row is loaded ahead of the last one's sums ((18,900, 5,120) bf16 233
// us; two ahead are no faster, nor with p: 244).  Rows of up to a workgroup of 1,024
// threads leave room for 128 registers a thread: two of the three sums are in LDS then,
// and of two or more chunks a thread, A and b are read again for each row and none is
// loaded ahead (2,000 rows of 16,384, bf16 148 us, float32 367, where their bytes take 77
// and 155).
template <class T, int CH, int NV, int SIZE, bool POST, bool TOKEN>
__global__ __launch_bounds__(Threads<SIZE>::most, Threads<SIZE>::bwd) void gated_norm_bwd_kernel(GatedNormArgs a) {
  constexpr bool WAVE = SIZE == 0, LDS = SIZE == 3, HOLD = !TOKEN && NV * CH <= 8;
  constexpr bool AHEAD = SIZE != 3 || NV == 1;
  constexpr int NS = POST ? 3 : 1, MOST = Threads<SIZE>::most;
  __shared__ float red[2][NS][16];
  __shared__ __attribute__((aligned(16))) float acc[LDS ? 2 * NV * MOST * CH : (WAVE ? 256 * NV * CH : 4)];
  const int TPR = WAVE ? a.tpr : (int)blockDim.x, RPB = WAVE ? 256 / TPR : 1;
  const int t = WAVE ? threadIdx.x & (TPR - 1) : threadIdx.x, sub = WAVE ? threadIdx.x / TPR : 0;
  const int64_t wg = a.first + blockIdx.x, group = TOKEN ? 0 : wg / a.per_group;
  const int64_t end = TOKEN ? a.rows : min((group + 1) * a.R, a.rows);
  const int64_t step = a.per_group * RPB;
  const int64_t row0 = (TOKEN ? 0 : group * a.R) + (wg - group * a.per_group) * RPB + sub;
  float held_a[HOLD ? NV : 1][CH], held_b[HOLD ? NV : 1][CH];
  float sn[NV][CH], st[NV][CH], sc[NV][CH];
  uint32_t off[NV];  // this thread's columns, 0 past the end of the row,
  uint32_t in[NV];   // where what is loaded is masked out
  auto sums_of = [&](int which, int j) { return acc + ((which * NV + j) * MOST + t) * CH; };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH, at = col < a.W ? col : 0;
    in[j] = col < a.W ? 0xffffffffu : 0u;
    off[j] = (uint32_t)at * sizeof(T);
    if constexpr (HOLD) {
      group_vectors<T, CH>(a, group, at, held_a[j], held_b[j], nullptr);
      mask_vectors<CH>(in[j], held_a[j], held_b[j]);
    }
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      sn[j][e] = st[j][e] = sc[j][e] = 0.f;
      if constexpr (LDS) sums_of(0, j)[e] = sums_of(1, j)[e] = 0.f;
    }
  }
  struct Row {
    Raw<CH> x[NV], r[NV], g[NV], d[NV];
  };
  auto load = [&](int64_t row, Row& q) {
    row = row < end ? row : end - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = read_at<T, CH>(a.x, row, a.xs, off[j]);
      q.r[j] = read_at<T, CH>(a.r, row, a.rs, off[j]);
      q.g[j] = read_at<T, CH>(a.dn, row, a.dns, off[j]);
      q.d[j] = Raw<CH>{};
      if (a.dh != nullptr) q.d[j] = read_at<T, CH>(a.dh, row, a.dhs, off[j]);
    }
  };
  Row next;
  if (AHEAD) load(row0, next);
  int buf = 0;
  for (int64_t row = row0; row < end; row += step) {  // the same for a row's threads
    Row cur;
    if constexpr (AHEAD) {
      cur = next;
      load(row + step, next);
    } else {
      load(row, cur);
    }
    // A and B of chunk j (opaque: read again rather than kept over the sums).
    auto vectors = [&](int j, float* av, float* bv) {
      if constexpr (HOLD) {
#pragma unroll
        for (int e = 0; e < CH; ++e) av[e] = held_a[j][e], bv[e] = held_b[j][e];
      } else {
        group_vectors<T, CH>(a, TOKEN ? row : group, opaque(off[j]) / sizeof(T), av, bv, nullptr);
        mask_vectors<CH>(in[j], av, bv);
      }
    };
    const f32x2 stats = *reinterpret_cast<const f32x2*>(a.stats + 2 * row);
    const float rx = POST ? stats[0] : 1.f, rh = stats[1];
#pragma unroll
    for (int j = 0; j < NV; ++j) cur.x[j] &= in[j], cur.r[j] &= in[j], cur.g[j] &= in[j], cur.d[j] &= in[j];
    auto value = [](const Raw<CH>& r, int e) { return raw_value<T, CH>(r, e); };
    auto sum_h = [&](int j, int e, float b) {
      return fmaf(value(cur.x[j], e) * rx, b, a.alpha * value(cur.r[j], e));
    };
    float sums[NS] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float av[CH], bv[CH];
      vectors(j, av, bv);
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = sum_h(j, e, bv[e]), ga = value(cur.g[j], e) * av[e];
        sums[0] = fmaf(ga, h, sums[0]);
        if constexpr (POST) {
          const float bx = bv[e] * value(cur.x[j], e);
          sums[1] = fmaf(bx, fmaf(rh, ga, value(cur.d[j], e)), sums[1]);
          sums[2] = fmaf(bx, h, sums[2]);
        }
      }
    }
    row_sums<WAVE, NS>(sums, red[buf], TPR);
    buf ^= 1;  // the next row's sums go elsewhere: one barrier a row
    const float m = sums[0] / (float)a.W * rh * rh;
    float mx = 0.f;
    if constexpr (POST) mx = fmaf(-rh * m, sums[2], sums[1]) / (float)a.W * rx * rx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float av[CH], bv[CH], d[CH], out[CH];
      vectors(j, av, bv);
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = sum_h(j, e, bv[e]), g = value(cur.g[j], e);
        d[e] = rh * (g * av[e] - h * m) + value(cur.d[j], e);
        out[e] = d[e] * bv[e];
        if constexpr (POST) out[e] = rx * (out[e] - value(cur.x[j], e) * mx);
      }
      if (in[j]) write_at<T, CH>(a.dx, row, a.W, off[j], out);
      if (a.dr != nullptr) {
#pragma unroll
        for (int e = 0; e < CH; ++e) out[e] = a.alpha * d[e];
        if (in[j]) write_at<T, CH>(a.dr, row, a.W, off[j], out);
      }
      float tn[CH], tc[CH];
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        tn[e] = value(cur.g[j], e) * (sum_h(j, e, bv[e]) * rh);
        tc[e] = d[e] * (value(cur.x[j], e) * rx);
      }
      if constexpr (TOKEN) {
        const int64_t at = off[j] / sizeof(T);
        float v[CH], dn[CH], dc[CH];
        load_vector<T, CH>(a.s, a.m32, row * a.ss + at, 0.f, v);
#pragma unroll
        for (int e = 0; e < CH; ++e) dn[e] = tn[e], tn[e] *= 1.f + v[e];
        load_vector<T, CH>(a.g, a.m32, row * a.gs + at, 1.f, v);
#pragma unroll
        for (int e = 0; e < CH; ++e) dc[e] = tc[e], tc[e] *= v[e];
        if (in[j]) {
          if (a.ds) {
            load_vector<T, CH>(a.w, a.w32, at, 1.f, v);
#pragma unroll
            for (int e = 0; e < CH; ++e) dn[e] *= v[e];
            store_vector<T, CH>(a.ds, a.m32, row * a.W + at, dn);
          }
          if (a.dt) {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[e] = value(cur.g[j], e);
            store_vector<T, CH>(a.dt, a.m32, row * a.W + at, v);
          }
          if (a.dg) {
            load_vector<T, CH>(a.p, a.p32, at, 1.f, v);
#pragma unroll
            for (int e = 0; e < CH; ++e) dc[e] *= v[e];
            store_vector<T, CH>(a.dg, a.m32, row * a.W + at, dc);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        if constexpr (LDS) {
          sums_of(0, j)[e] += tn[e];
          sums_of(1, j)[e] += tc[e];
        } else {
          sn[j][e] += tn[e];
          sc[j][e] += tc[e];
        }
        if constexpr (!TOKEN) st[j][e] += value(cur.g[j], e);
      }
    }
  }
  float* part = a.part + wg * 3 * a.W;
  if constexpr (WAVE) {
    // The workers' sums, in order.
    const int width = TPR * NV * CH;
#pragma unroll
    for (int which = 0; which < 3; ++which) {
      if (TOKEN && which == 1) continue;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < CH; ++e)
          acc[sub * width + (j * TPR + t) * CH + e] = which == 0 ? sn[j][e] : (which == 1 ? st[j][e] : sc[j][e]);
      __syncthreads();
      for (int c = threadIdx.x; c < a.W; c += 256) {
        float s = acc[c];
        for (int i = 1; i < RPB; ++i) s += acc[i * width + c];
        part[which * a.W + c] = s;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!in[j]) continue;
      const int64_t col = off[j] / sizeof(T);
      store_vector<float, CH>(part, true, col, LDS ? sums_of(0, j) : sn[j]);
      if (!TOKEN) store_vector<float, CH>(part, true, a.W + col, st[j]);
      store_vector<float, CH>(part, true, 2 * a.W + col, LDS ? sums_of(1, j) : sc[j]);
    }
  }
}

// The backward for any width and alignment: passes over each row, the sums of
// the worker's rows added in memory by the thread that owns the column.
template <class T, bool TOKEN>
__global__ __launch_bounds__(kAny) void gated_norm_bwd_any_kernel(GatedNormArgs a) {
  __shared__ float red[16];
  const int64_t worker = a.first + blockIdx.x;
  const int64_t group = TOKEN ? 0 : worker / a.per_group;
  const int64_t end = TOKEN ? a.rows : min((group + 1) * a.R, a.rows);
  float* part = a.part + worker * 3 * a.W;
  for (int64_t c = threadIdx.x; c < a.W; c += kAny) part[c] = part[a.W + c] = part[2 * a.W + c] = 0.f;
  for (int64_t row = TOKEN ? worker : group * a.R + worker % a.per_group; row < end; row += a.per_group) {
    const int64_t mine = TOKEN ? row : group;
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const T* r = static_cast<const T*>(a.r) + row * a.rs;
    const T* gr = static_cast<const T*>(a.dn) + row * a.dns;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * a.dhs : nullptr;
    const float rx = a.p ? a.stats[2 * row] : 1.f, rh = a.stats[2 * row + 1];
    float dot = 0.f, s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += kAny) {
      float av, bv;
      group_vectors<T, 1>(a, mine, c, &av, &bv, nullptr);
      const float h = fmaf((float)x[c] * rx, bv, a.alpha * (float)r[c]), ga = (float)gr[c] * av;
      const float bx = bv * (float)x[c];
      dot = fmaf(ga, h, dot);
      s1 = fmaf(bx, (dh ? (float)dh[c] : 0.f) + rh * ga, s1);
      s2 = fmaf(bx, h, s2);
    }
    dot = row_reduce<false, false>(dot, red);
    const float m = dot / (float)a.W * rh * rh;
    float mx = 0.f;
    if (a.p) {
      s1 = row_reduce<false, false>(s1, red);
      s2 = row_reduce<false, false>(s2, red);
      mx = fmaf(-rh * m, s2, s1) / (float)a.W * rx * rx;
    }
    for (int64_t c = threadIdx.x; c < a.W; c += kAny) {
      float av, bv;
      group_vectors<T, 1>(a, mine, c, &av, &bv, nullptr);
      const float xv = (float)x[c], g = (float)gr[c], h = fmaf(xv * rx, bv, a.alpha * (float)r[c]);
      const float d = rh * (g * av - h * m) + (dh ? (float)dh[c] : 0.f);
      const float tn = g * (h * rh), tc = d * (xv * rx);
      float dx = d * bv;
      if (a.p) dx = rx * (dx - xv * mx);
      static_cast<T*>(a.dx)[row * a.W + c] = (T)dx;
      if (a.dr) static_cast<T*>(a.dr)[row * a.W + c] = (T)(a.alpha * d);
      if constexpr (TOKEN) {
        float w, s, p, gt;
        load_vector<T, 1>(a.w, a.w32, c, 1.f, &w);
        load_vector<T, 1>(a.s, a.m32, row * a.ss + c, 0.f, &s);
        load_vector<T, 1>(a.p, a.p32, c, 1.f, &p);
        load_vector<T, 1>(a.g, a.m32, row * a.gs + c, 1.f, &gt);
        part[c] = fmaf(tn, 1.f + s, part[c]);
        part[2 * a.W + c] = fmaf(tc, gt, part[2 * a.W + c]);
        const float ds = tn * w, dg = tc * p;
        if (a.ds) store_vector<T, 1>(a.ds, a.m32, row * a.W + c, &ds);
        if (a.dt) store_vector<T, 1>(a.dt, a.m32, row * a.W + c, &g);
        if (a.dg) store_vector<T, 1>(a.dg, a.m32, row * a.W + c, &dg);
      } else {
        part[c] += tn;
        part[a.W + c] += g;
        part[2 * a.W + c] += tc;
      }
    }
  }
}

// The sums of the parts, by 16 threads for V columns in a fixed order: a group's
// ds, dt and dg (blockIdx.z 0, 1, 2) and over all groups dw and dp (3, 4; each part
// weighted by its group's row of s and g, which with a row per token (TOKEN) it is
// already).
template <class T, bool TOKEN, int V>
__global__ __launch_bounds__(256) void gated_norm_sums_kernel(GatedNormArgs a, int64_t groups) {
  __shared__ float red[16][16][V];
  const int c = threadIdx.x % 16, g = threadIdx.x / 16, z = blockIdx.z;
  const int64_t col = ((int64_t)blockIdx.x * 16 + c) * V, stride = 3 * a.W;
  const bool in = col < a.W, all = z > 2;
  void* out = z == 0 ? a.ds : (z == 1 ? a.dt : (z == 2 ? a.dg : (z == 3 ? a.dw : a.dp)));
  if (out == nullptr || (all && blockIdx.y > 0)) return;
  const float* part = a.part + (z == 3 ? 0 : (z == 4 ? 2 : z)) * a.W + col;
  const uint32_t per = (uint32_t)a.per_group;  // (of a grid's workgroups)
  auto vec = [&](const void* p, bool f32, int64_t at, float otherwise, float* v) {
#pragma unroll
    for (int e = 0; e < V; ++e) load_vector<T, 1>(p, f32, at + e, otherwise, v + e);
  };
  for (int64_t i = blockIdx.y; i < (all ? 1 : groups); i += gridDim.y) {
    const uint32_t n = all ? (uint32_t)groups * per : per;
    const float* p = part + (all ? 0 : i * per * stride);
    float s[V] = {}, f[V];
    auto add_part = [&](uint32_t k, auto&& weight) {
      float x[V];
      load_chunk<float, V>(p + k * stride, x);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = fmaf(x[e], weight(e), s[e]);
    };
    if (in) {
      if (all && !TOKEN && groups > 1 && (z == 3 ? a.s : a.g) != nullptr) {
        auto weighted = [&](auto* w, int64_t ws, float add) {
#pragma unroll 8
          for (uint32_t k = g; k < n; k += 16)
            add_part(k, [&](int e) { return add + (float)w[k / per * ws + col + e]; });
        };
        const void* w = z == 3 ? a.s : a.g;
        const int64_t ws = z == 3 ? a.ss : a.gs;
        const float add = z == 3 ? 1.f : 0.f;
        if (a.m32)
          weighted(static_cast<const float*>(w), ws, add);
        else
          weighted(static_cast<const T*>(w), ws, add);
      } else {
#pragma unroll 8
        for (uint32_t k = g; k < n; k += 16) add_part(k, [](int) { return 1.f; });
      }
    }
    __syncthreads();  // the last sums are read
#pragma unroll
    for (int e = 0; e < V; ++e) red[g][c][e] = s[e];
    __syncthreads();
    if (g == 0 && in) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        for (int k = 1; k < 16; ++k) s[e] += red[k][c][e];
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = 1.f;
      if (all && !TOKEN && groups == 1) {
        vec(z == 3 ? a.s : a.g, a.m32, col, z == 3 ? 0.f : 1.f, f);
        if (z == 3)
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] += 1.f;
      }
      if (z == 0) vec(a.w, a.w32, col, 1.f, f);
      if (z == 2) vec(a.p, a.p32, col, 1.f, f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s[e] *= f[e];
        store_vector<T, 1>(out, all ? (z == 3 ? a.w32 : a.p32) : a.m32, (all ? 0 : i * a.W) + col + e, s + e);
      }
    }
  }
}

// Whole 16-byte chunks everywhere.
bool chunked(const GatedNormArgs& a, int size) {
  const int64_t ch = 16 / size;
  uintptr_t p = 0;
  for (const void* q : {a.x, a.r, a.dn, a.dh, (const void*)a.h, (const void*)a.n, (const void*)a.dx,
                        (const void*)a.dr, a.w, a.p, a.g, a.s, a.t, (const void*)a.dg, (const void*)a.ds,
                        (const void*)a.dt})
    p |= reinterpret_cast<uintptr_t>(q);
  bool ok = p % 16 == 0 && a.W % ch == 0;
  for (int64_t s : {a.xs, a.rs, a.dns, a.dhs, a.gs, a.ss, a.ts}) ok = ok && s % ch == 0;
  return ok;
}

// Threads per row, columns of a chunk, chunks per thread (nv 0: none of these
// kernels) and the Threads to compile for.
struct RowShape {
  int tpr, ch, nv, size;
};
// chunk: columns of 16 bytes, 1 where not all is aligned.  rows: of a group, which
// a workgroup of several rows should not have more of.
RowShape row_shape(int64_t W, int chunk, int64_t rows) {
  const int64_t n = (W + chunk - 1) / chunk;  // chunks of a row
  if (n <= 64) {
    int tpr = 8;
    while (tpr < n || (tpr < 64 && 256 / tpr > rows)) tpr *= 2;
    return {tpr, chunk, 1, 0};
  }
  if (chunk == 1) {
    if (n <= 512) return {64, 1, n <= 128 ? 2 : (n <= 256 ? 4 : 8), 0};
    const int tpr = (int)((n + 511) / 512) * 64;
    if (tpr > 1024) return {0, 1, 0, 0};
    return {tpr, 1, 8, tpr <= 512 ? 1 : 3};
  }
  const int nv = n <= 1024 ? 1 : (n <= 2048 ? 2 : 4);
  if (n > 1024 * nv || nv * chunk > 16) return {0, 1, 0, 0};
  const int tpr = (int)((n + 64 * nv - 1) / (64 * nv)) * 64;
  return {tpr, chunk, nv, nv > 1 ? 3 : (tpr <= 512 ? 1 : (tpr <= 768 ? 2 : 3))};
}

// Workgroups of a launch: the threads of a grid (up to 1,024 a row) stay below 2^32.
constexpr int64_t kMostGrid = 1 << 21;

// f(columns of a chunk, chunks per thread, size) as compile-time constants.
template <class T, class F>
void with_shape(const RowShape& s, F&& f) {
  constexpr int CH = 16 / (int)sizeof(T);
  auto call = [&](auto ch, auto nv, auto size) {
    if (s.ch == decltype(ch)::value && s.nv == decltype(nv)::value && s.size == decltype(size)::value) f(ch, nv, size);
  };
  using std::integral_constant;
  integral_constant<int, 0> c0;
  integral_constant<int, 1> c1;
  integral_constant<int, 2> c2;
  integral_constant<int, 3> c3;
  integral_constant<int, 4> c4;
  integral_constant<int, 8> c8;
  integral_constant<int, CH> ch;
  call(ch, c1, c0), call(ch, c1, c1), call(ch, c1, c2), call(ch, c1, c3), call(ch, c2, c3);
  if constexpr (CH == 4) call(ch, c4, c3);
  call(c1, c1, c0), call(c1, c2, c0), call(c1, c4, c0), call(c1, c8, c0), call(c1, c8, c1), call(c1, c8, c3);
}

template <class T>
hipError_t forward(const GatedNormArgs& all, hipStream_t stream) {
  GatedNormArgs a = all;
  LaunchTimer timer(kKidGatedNorm, stream);
  const RowShape s = row_shape(a.W, chunked(a, sizeof(T)) ? 16 / (int)sizeof(T) : 1, a.rows);
  const int64_t groups = (a.rows + a.R - 1) / a.R;
  const int rpb = s.nv > 0 && s.size == 0 ? 256 / s.tpr : 1;
  a.tpr = s.tpr;
  // Rows of a worker: up to 8 while there are 512 workgroups ((2,048, 5,120) bf16
  // 23.6 us with 1, 16.0 with 4, 16.9 with 8; (8,000, 2,560) 45.2, 34.1, 30.1; (500,
  // 5,120) 7.7, 9.7, 14.1), 16 of narrow rows.
  int64_t mine = a.rows / (512 * (int64_t)rpb);
  const int64_t most = s.size == 0 ? 16 : 8;
  mine = mine < 1 || s.nv == 0 ? 1 : (mine > most ? most : mine);
  a.per_group = (a.R + mine - 1) / mine;
  const int64_t blocks = (groups * a.per_group + rpb - 1) / rpb;
  for (int64_t done = 0; done < blocks; done += kMostGrid) {
    a.first = done * rpb;
    const unsigned grid = (unsigned)(blocks - done < kMostGrid ? blocks - done : kMostGrid);
    if (s.nv == 0)
      hipLaunchKernelGGL(gated_norm_any_kernel<T>, dim3(grid), dim3(kAny), 0, stream, a);
    else
      with_shape<T>(s, [&](auto ch, auto nv, auto size) {
        constexpr int CH = decltype(ch)::value, NV = decltype(nv)::value, S = decltype(size)::value;
        const dim3 block(S == 0 ? 256 : s.tpr);
        if (a.p)
          hipLaunchKernelGGL((gated_norm_kernel<T, CH, NV, S, true>), dim3(grid), block, 0, stream, a);
        else
          hipLaunchKernelGGL((gated_norm_kernel<T, CH, NV, S, false>), dim3(grid), block, 0, stream, a);
      });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Workgroups of the backward: of a group (TOKEN: in all).  A round of them: more
// leave more parts of the sums ((18,900, 5,120) bf16 402 us forward and backward
// with two rounds, 393 with one; (8,000, 2,560) with both norms 130, 123), and no fewer than two rows for each worker.
struct Workgroups {
  int64_t groups, per_group;
  bool token;
};
Workgroups bwd_workgroups(int64_t rows, int64_t R, int rpb, int waves, bool modulated) {
  const int64_t groups = (rows + R - 1) / R;
  int64_t most = 256 * (waves < 12 ? 12 / waves : 1);
  const bool token = R == 1 && modulated && rows > 1;
  const int64_t of = token ? rows : R;  // rows that they share
  int64_t per = token ? most : most / groups;
  if (rpb > 1 && per > (of + 2 * rpb - 1) / (2 * rpb)) per = (of + 2 * rpb - 1) / (2 * rpb);
  if (per < 1) per = 1;
  if (per > of) per = of;
  return {token ? 1 : groups, per, token};
}

template <class T, bool TOKEN>
hipError_t backward_rows(const GatedNormArgs& all, const RowShape& s, int64_t workgroups, hipStream_t stream) {
  GatedNormArgs a = all;
  for (int64_t done = 0; done < workgroups; done += kMostGrid) {
    a.first = done;
    const dim3 grid((unsigned)(workgroups - done < kMostGrid ? workgroups - done : kMostGrid));
    if (s.nv == 0)
      hipLaunchKernelGGL((gated_norm_bwd_any_kernel<T, TOKEN>), grid, dim3(kAny), 0, stream, a);
    else
      with_shape<T>(s, [&](auto ch, auto nv, auto size) {
        constexpr int CH = decltype(ch)::value, NV = decltype(nv)::value, S = decltype(size)::value;
        const dim3 block(S == 0 ? 256 : s.tpr);
        if (a.p)
          hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, true, TOKEN>), grid, block, 0, stream, a);
        else
          hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, false, TOKEN>), grid, block, 0, stream, a);
      });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T>
hipError_t backward(const GatedNormArgs& all, hipStream_t stream) {
  GatedNormArgs a = all;
  const bool modulated = a.g || a.s || a.t;
  const RowShape s = row_shape(a.W, chunked(a, sizeof(T)) ? 16 / (int)sizeof(T) : 1,
                               a.R == 1 && modulated ? a.rows : a.R);
  const int rpb = s.nv > 0 && s.size == 0 ? 256 / s.tpr : 1;
  const int waves = s.nv == 0 ? kAny / 64 : (s.size == 0 ? 4 : s.tpr / 64);
  const Workgroups w = bwd_workgroups(a.rows, a.R, rpb, waves, modulated);
  a.per_group = w.per_group;
  a.tpr = s.tpr;
  hipError_t e;
  {
    LaunchTimer timer(kKidGatedNormBwd, stream);
    e = w.token ? backward_rows<T, true>(a, s, w.per_group, stream)
                : backward_rows<T, false>(a, s, w.groups * w.per_group, stream);
  }
  if (e != hipSuccess) return e;
  GatedNormArgs b = a;
  if (w.token) b.ds = b.dt = b.dg = nullptr;  // written
  if (b.ds || b.dt || b.dg || b.dw || b.dp) {
    const unsigned y = b.ds || b.dt || b.dg ? (unsigned)(w.groups < 16384 ? w.groups : 16384) : 1;
    auto sum = [&](auto v) {
      constexpr int V = decltype(v)::value;
      const dim3 grid((unsigned)((a.W + 16 * V - 1) / (16 * V)), y, 5);
      if (w.token)
        hipLaunchKernelGGL((gated_norm_sums_kernel<T, true, V>), grid, dim3(256), 0, stream, b, w.groups);
      else
        hipLaunchKernelGGL((gated_norm_sums_kernel<T, false, V>), grid, dim3(256), 0, stream, b, w.groups);
    };
    if (a.W % 4 == 0)
      sum(std::integral_constant<int, 4>());
    else
      sum(std::integral_constant<int, 1>());
  }
  return hipGetLastError();
}

}  // namespace

size_t gated_norm_bwd_workspace_bytes(int64_t rows, int64_t R, int64_t W, bool modulated) {
  if (rows == 0) return 0;
  // Of any type and alignment: float32 chunks have more waves a row than the others,
  // and so no more workgroups.
  const int64_t waves = W <= 512 ? 2 : (W <= 8192 ? (W + 511) / 512 : 16);
  const Workgroups w = bwd_workgroups(rows, R, 1, (int)waves, modulated);
  return (size_t)(w.groups * w.per_group) * 3 * (size_t)W * sizeof(float);
}

hipError_t launch_gated_norm(const GatedNormArgs& a, bool f32, hipStream_t stream) {
  return f32 ? forward<float>(a, stream) : forward<bf16>(a, stream);
}

hipError_t launch_gated_norm_bwd(const GatedNormArgs& a, bool f32, hipStream_t stream) {
  return f32 ? backward<float>(a, stream) : backward<bf16>(a, stream);
}

}  // namespace avattn
