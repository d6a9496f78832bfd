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
// stays in the registers of the threads that share it (a wave, or a workgroup),
// which keep their columns of A, b and t, and of the sums, over the rows of a
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

// A row's chunk at a byte offset, from the row's (uniform) address.
template <class T, int CH>
__device__ __forceinline__ RawChunk<T, CH> read_at(const void* base, int64_t row, int64_t stride, uint32_t off) {
  return *reinterpret_cast<const RawChunk<T, CH>*>(static_cast<const char*>(base) + row * stride * (int64_t)sizeof(T) +
                                                   off);
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

__device__ __forceinline__ float row_rstd(float ss, const GatedNormArgs& a) {
  return 1.f / __builtin_sqrtf(ss / (float)a.W + a.eps);
}

// Threads of a workgroup up to which a kernel is compiled, and its waves per SIMD.
template <int SIZE>
struct Threads;  // 0: four waves, a row each; 1, 2, 3: a row per workgroup
template <>
struct Threads<0> {
  static constexpr int most = 256, fwd = 5, bwd = 3;
};
template <>
struct Threads<1> {
  static constexpr int most = 512, fwd = 5, bwd = 4;
};
template <>
struct Threads<2> {
  static constexpr int most = 768, fwd = 5, bwd = 3;
};
template <>
struct Threads<3> {
  static constexpr int most = 1024, fwd = 4, bwd = 4;
};

// Forward.  A worker, a wave (narrow rows, 4 per workgroup) or a workgroup, takes
// every per_group-th row of a group, the next row loaded before this one's sums.
template <class T, int CH, int NV, int SIZE, bool POST>
__global__ __launch_bounds__(Threads<SIZE>::most, Threads<SIZE>::fwd) void gated_norm_kernel(GatedNormArgs a) {
  constexpr bool WAVE = SIZE == 0;
  constexpr int RPB = WAVE ? 4 : 1;
  __shared__ float red[16];
  const int TPR = WAVE ? 64 : blockDim.x;
  const int t = threadIdx.x % TPR;
  const int64_t worker = a.first + (int64_t)blockIdx.x * RPB + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const int64_t group = worker / a.per_group, end = min((group + 1) * a.R, a.rows);
  int64_t row = group * a.R + worker % a.per_group;
  if (row >= end) return;  // whole waves or nobody
  float av[NV][CH], bv[NV][CH], tv[NV][CH];
  uint32_t off[NV];  // this thread's columns, 0 past the end of the row,
  uint32_t in[NV];   // where what is loaded is masked out
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH, at = col < a.W ? col : 0;
    in[j] = col < a.W ? 0xffffffffu : 0u;
    off[j] = (uint32_t)at * sizeof(T);
    group_vectors<T, CH>(a, group, at, av[j], bv[j], tv[j]);
  }
  struct Row {
    RawChunk<T, CH> x[NV], r[NV];
  };
  auto load = [&](int64_t row, Row& q) {
    row = row < end ? row : end - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = read_at<T, CH>(a.x, row, a.xs, off[j]);
      q.r[j] = read_at<T, CH>(a.r, row, a.rs, off[j]);
    }
  };
  Row next;
  load(row, next);
  for (; row < end; row += a.per_group) {
    Row cur = next;
    load(row + a.per_group, next);
#pragma unroll
    for (int j = 0; j < NV; ++j) cur.x[j] &= in[j], cur.r[j] &= in[j];
    float rx = 1.f;
    if constexpr (POST) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < CH; ++e) ss = fmaf(chunk_value<T, CH>(cur.x[j], e), chunk_value<T, CH>(cur.x[j], e), ss);
      rx = row_rstd(row_reduce<WAVE, false>(ss, red), a);
    }
    float ss = 0.f;
    float h[NV][CH];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        h[j][e] = fmaf(chunk_value<T, CH>(cur.x[j], e) * rx, bv[j][e], a.alpha * chunk_value<T, CH>(cur.r[j], e));
        ss = fmaf(h[j][e], h[j][e], ss);
      }
      if (in[j]) write_at<T, CH>(a.h, row, a.W, off[j], h[j]);
    }
    const float rh = row_rstd(row_reduce<WAVE, false>(ss, red), a);
    if (a.stats != nullptr && t == 0) *reinterpret_cast<f32x2*>(a.stats + 2 * row) = f32x2{rx, rh};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < CH; ++e) h[j][e] = fmaf(h[j][e] * rh, av[j][e], tv[j][e]);
      if (in[j]) write_at<T, CH>(a.n, row, a.W, off[j], h[j]);
    }
  }
}

// Rows of any width and alignment, one workgroup each, value by value; x and r
// are read again for the sum's norm and for the output.
template <class T>
__global__ __launch_bounds__(256) void gated_norm_any_kernel(GatedNormArgs a) {
  __shared__ float red[4];
  const int64_t row = a.first + blockIdx.x, group = row / a.R;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = static_cast<const T*>(a.r) + row * a.rs;
  float rx = 1.f;
  if (a.p != nullptr) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) ss = fmaf((float)x[c], (float)x[c], ss);
    rx = row_rstd(row_reduce<false, false>(ss, red), a);
  }
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < a.W; c += 256) {
    float av, bv;
    group_vectors<T, 1>(a, group, c, &av, &bv, nullptr);
    const float h = fmaf((float)x[c] * rx, bv, a.alpha * (float)r[c]);
    static_cast<T*>(a.h)[row * a.W + c] = (T)h;
    ss = fmaf(h, h, ss);
  }
  const float rh = row_rstd(row_reduce<false, false>(ss, red), a);
  if (a.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<f32x2*>(a.stats + 2 * row) = f32x2{rx, rh};
  for (int64_t c = threadIdx.x; c < a.W; c += 256) {
    float av, bv, tv;
    group_vectors<T, 1>(a, group, c, &av, &bv, &tv);
    const float h = fmaf((float)x[c] * rx, bv, a.alpha * (float)r[c]);
    static_cast<T*>(a.n)[row * a.W + c] = (T)fmaf(h * rh, av, tv);
  }
}

// N sums over the threads of a row; red: a float per sum and wave.
template <bool WAVE, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[16], int waves) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], off);
  if constexpr (!WAVE) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = red[k][0];
      for (int i = 1; i < waves; ++i) v[k] += red[k][i];
    }
  }
}

// Backward.  Workers take rows as in the forward; with a row of g, s and t per
// token (TOKEN) every worker takes all rows in turn, writes that token's ds, dt
// and dg and keeps the sums of dw and dp.  DH: a gradient of h is given.  The
// next row is loaded before this one's sums.
template <class T, int CH, int NV, int SIZE, bool POST, bool DH, bool TOKEN>
__global__ __launch_bounds__(Threads<SIZE>::most, Threads<SIZE>::bwd) void gated_norm_bwd_kernel(GatedNormArgs a) {
  constexpr bool WAVE = SIZE == 0;
  constexpr int RPB = WAVE ? 4 : 1, NS = POST ? 3 : 1;
  __shared__ float red[2][NS][16];
  const int TPR = WAVE ? 64 : blockDim.x, waves = TPR / 64;
  const int t = threadIdx.x % TPR;
  const int64_t worker = (int64_t)blockIdx.x * RPB + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const int64_t group = TOKEN ? 0 : worker / a.per_group;
  const int64_t end = TOKEN ? a.rows : min((group + 1) * a.R, a.rows);
  const int64_t step = a.per_group;
  const int64_t row0 = TOKEN ? worker : group * a.R + worker % a.per_group;
  if (!TOKEN && group * a.R >= a.rows) return;  // whole waves or nobody
  float av[NV][CH], bv[NV][CH];
  float sn[NV][CH], st[NV][CH], sc[NV][CH];
  uint32_t off[NV];  // this thread's columns, 0 past the end of the row,
  uint32_t in[NV];   // where what is loaded is masked out
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t col = (int64_t)(j * TPR + t) * CH, at = col < a.W ? col : 0;
    in[j] = col < a.W ? 0xffffffffu : 0u;
    off[j] = (uint32_t)at * sizeof(T);
    if constexpr (!TOKEN) group_vectors<T, CH>(a, group, at, av[j], bv[j], nullptr);
#pragma unroll
    for (int e = 0; e < CH; ++e) sn[j][e] = st[j][e] = sc[j][e] = 0.f;
  }
  struct Row {
    RawChunk<T, CH> x[NV], r[NV], g[NV], d[NV];
  };
  auto load = [&](int64_t row, Row& q) {
    row = row < end ? row : end - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = read_at<T, CH>(a.x, row, a.xs, off[j]);
      q.r[j] = read_at<T, CH>(a.r, row, a.rs, off[j]);
      q.g[j] = read_at<T, CH>(a.dn, row, a.dns, off[j]);
      if constexpr (DH) q.d[j] = read_at<T, CH>(a.dh, row, a.dhs, off[j]);
    }
  };
  Row next;
  if (row0 < end) load(row0, next);
  int buf = 0;
  for (int64_t row = row0; row < end; row += step) {  // uniform over the row's threads
    Row cur = next;
    load(row + step, next);
    if constexpr (TOKEN) {
#pragma unroll
      for (int j = 0; j < NV; ++j) group_vectors<T, CH>(a, row, off[j] / sizeof(T), av[j], bv[j], nullptr);
    }
    const f32x2 stats = *reinterpret_cast<const f32x2*>(a.stats + 2 * row);
    const float rx = POST ? stats[0] : 1.f, rh = stats[1];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur.x[j] &= in[j], cur.r[j] &= in[j], cur.g[j] &= in[j];
      if constexpr (DH) cur.d[j] &= in[j];
    }
    auto value = [](const RawChunk<T, CH>& r, int e) { return chunk_value<T, CH>(r, e); };
    auto sum_h = [&](int j, int e) { return fmaf(value(cur.x[j], e) * rx, bv[j][e], a.alpha * value(cur.r[j], e)); };
    float sums[NS] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = sum_h(j, e), ga = value(cur.g[j], e) * av[j][e];
        sums[0] = fmaf(ga, h, sums[0]);
        if constexpr (POST) {
          const float bx = bv[j][e] * value(cur.x[j], e);
          float u = rh * ga;
          if constexpr (DH) u += value(cur.d[j], e);
          sums[1] = fmaf(bx, u, sums[1]);
          sums[2] = fmaf(bx, h, sums[2]);
        }
      }
    row_sums<WAVE, NS>(sums, red[buf], waves);
    buf ^= 1;  // the next row's sums go elsewhere: one barrier a row
    const float m = sums[0] / (float)a.W * rh * rh;
    float mx = 0.f;
    if constexpr (POST) mx = fmaf(-rh * m, sums[2], sums[1]) / (float)a.W * rx * rx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float d[CH], out[CH];
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float h = sum_h(j, e), g = value(cur.g[j], e);
        d[e] = rh * (g * av[j][e] - h * m);
        if constexpr (DH) d[e] += value(cur.d[j], e);
        out[e] = d[e] * bv[j][e];
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
        tn[e] = value(cur.g[j], e) * (sum_h(j, e) * rh);
        tc[e] = d[e] * (value(cur.x[j], e) * rx);
      }
      if constexpr (TOKEN) {
        const int64_t at = off[j] / sizeof(T);
        float v[CH];
        load_vector<T, CH>(a.s, a.m32, row * a.ss + at, 0.f, v);
#pragma unroll
        for (int e = 0; e < CH; ++e) sn[j][e] = fmaf(tn[e], 1.f + v[e], sn[j][e]);
        load_vector<T, CH>(a.g, a.m32, row * a.gs + at, 1.f, v);
#pragma unroll
        for (int e = 0; e < CH; ++e) sc[j][e] = fmaf(tc[e], v[e], sc[j][e]);
        if (in[j]) {
          if (a.ds) {
            load_vector<T, CH>(a.w, a.w32, at, 1.f, v);
#pragma unroll
            for (int e = 0; e < CH; ++e) tn[e] *= v[e];
            store_vector<T, CH>(a.ds, a.m32, row * a.W + at, tn);
          }
          if (a.dt) {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[e] = value(cur.g[j], e);
            store_vector<T, CH>(a.dt, a.m32, row * a.W + at, v);
          }
          if (a.dg) {
            load_vector<T, CH>(a.p, a.p32, at, 1.f, v);
#pragma unroll
            for (int e = 0; e < CH; ++e) tc[e] *= v[e];
            store_vector<T, CH>(a.dg, a.m32, row * a.W + at, tc);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          sn[j][e] += tn[e];
          st[j][e] += value(cur.g[j], e);
          sc[j][e] += tc[e];
        }
      }
    }
  }
  float* part = a.part + worker * 3 * a.W;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!in[j]) continue;
    const int64_t col = off[j] / sizeof(T);
    store_vector<float, CH>(part, true, col, sn[j]);
    if (!TOKEN) store_vector<float, CH>(part, true, a.W + col, st[j]);
    store_vector<float, CH>(part, true, 2 * a.W + col, sc[j]);
  }
}

// The backward for any width and alignment: passes over each row, the sums of
// the worker's rows added in memory by the thread that owns the column.
template <class T, bool TOKEN>
__global__ __launch_bounds__(256) void gated_norm_bwd_any_kernel(GatedNormArgs a) {
  __shared__ float red[4];
  const int64_t worker = blockIdx.x;
  const int64_t group = TOKEN ? 0 : worker / a.per_group;
  const int64_t end = TOKEN ? a.rows : min((group + 1) * a.R, a.rows);
  float* part = a.part + worker * 3 * a.W;
  for (int64_t c = threadIdx.x; c < a.W; c += 256) part[c] = part[a.W + c] = part[2 * a.W + c] = 0.f;
  for (int64_t row = TOKEN ? worker : group * a.R + worker % a.per_group; row < end; row += a.per_group) {
    const int64_t mine = TOKEN ? row : group;
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const T* r = static_cast<const T*>(a.r) + row * a.rs;
    const T* gr = static_cast<const T*>(a.dn) + row * a.dns;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * a.dhs : nullptr;
    const float rx = a.p ? a.stats[2 * row] : 1.f, rh = a.stats[2 * row + 1];
    float dot = 0.f, s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < a.W; c += 256) {
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
    for (int64_t c = threadIdx.x; c < a.W; c += 256) {
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

// The sums of 32 columns over n parts, `stride` floats apart, by 8 groups of 32
// threads in a fixed order; the first group has the result.
__device__ __forceinline__ float part_sum(const float* p, int64_t stride, int64_t n, bool in, float (*red)[32]) {
  const int c = threadIdx.x % 32, g = threadIdx.x / 32;
  float s = 0.f;
  if (in) {
#pragma unroll 8
    for (int64_t i = g; i < n; i += 8) s += p[i * stride];
  }
  __syncthreads();  // the last sums are read
  red[g][c] = s;
  __syncthreads();
  if (g == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][c];
  }
  return s;
}

// A group's ds, dt and dg; of a single group also dw and dp.  Its N and C stay in
// its first worker's part.
template <class T>
__global__ __launch_bounds__(256) void gated_norm_groups_kernel(GatedNormArgs a, int64_t groups) {
  __shared__ float red[8][32];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const bool in = col < a.W, writes = in && threadIdx.x < 32;
  for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    float* part = a.part + g * a.per_group * 3 * a.W + col;
    const int64_t stride = 3 * a.W;
    auto vec = [&](const void* p, bool f32, int64_t at, float otherwise) {
      float v;
      load_vector<T, 1>(p, f32, at, otherwise, &v);
      return v;
    };
    if (a.ds || a.dw) {
      const float n = part_sum(part, stride, a.per_group, in, red);
      if (writes) {
        const float ds = n * vec(a.w, a.w32, col, 1.f), dw = n * (1.f + vec(a.s, a.m32, g * a.ss + col, 0.f));
        if (a.ds) store_vector<T, 1>(a.ds, a.m32, g * a.W + col, &ds);
        if (a.dw && groups == 1) store_vector<T, 1>(a.dw, a.w32, col, &dw);
        part[0] = n;
      }
    }
    if (a.dt) {
      const float v = part_sum(part + a.W, stride, a.per_group, in, red);
      if (writes) store_vector<T, 1>(a.dt, a.m32, g * a.W + col, &v);
    }
    if (a.dg || a.dp) {
      const float c = part_sum(part + 2 * a.W, stride, a.per_group, in, red);
      if (writes) {
        const float dg = c * vec(a.p, a.p32, col, 1.f), dp = c * vec(a.g, a.m32, g * a.gs + col, 1.f);
        if (a.dg) store_vector<T, 1>(a.dg, a.m32, g * a.W + col, &dg);
        if (a.dp && groups == 1) store_vector<T, 1>(a.dp, a.p32, col, &dp);
        part[2 * a.W] = c;
      }
    }
  }
}

// dw and dp over n parts `stride` floats apart, each weighted by its group's row
// of s and g (TOKEN: they are in the sums already).
template <class T, bool TOKEN>
__global__ __launch_bounds__(256) void gated_norm_gains_kernel(GatedNormArgs a, int64_t n, int64_t stride) {
  __shared__ float red[8][32];
  const int c = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  for (int which = 0; which < 2; ++which) {
    void* out = which ? a.dp : a.dw;
    if (out == nullptr) continue;
    const float* p = a.part + (which ? 2 * a.W : 0) + col;
    float s = 0.f;
    if (col < a.W) {
      for (int64_t i = g; i < n; i += 8) {
        float f = 1.f;
        if constexpr (!TOKEN) {
          if (which)
            load_vector<T, 1>(a.g, a.m32, i * a.gs + col, 1.f, &f);
          else
            load_vector<T, 1>(a.s, a.m32, i * a.ss + col, 0.f, &f), f += 1.f;
        }
        s = fmaf(p[i * stride], f, s);
      }
    }
    __syncthreads();
    red[g][c] = s;
    __syncthreads();
    if (g == 0 && col < a.W) {
#pragma unroll
      for (int i = 1; i < 8; ++i) s += red[i][c];
      store_vector<T, 1>(out, which ? a.p32 : a.w32, col, &s);
    }
  }
}

// Whole 16-byte chunks everywhere.
bool chunked(const GatedNormArgs& a, int size) {
  const int64_t ch = 16 / size;
  uintptr_t p = 0;
  for (const void* q : {a.x, a.r, a.dn, a.dh, (const void*)a.h, (const void*)a.n, (const void*)a.dx,
                        (const void*)a.dr, a.w, a.p, a.g, a.s, a.t})
    p |= reinterpret_cast<uintptr_t>(q);
  bool ok = p % 16 == 0 && a.W % ch == 0;
  for (int64_t s : {a.xs, a.rs, a.dns, a.dhs, a.gs, a.ss, a.ts}) ok = ok && s % ch == 0;
  return ok;
}

// Threads per row and chunks per thread (nv 0: value by value), and the Threads
// to compile for.
struct RowShape {
  int tpr, nv, size;
};
RowShape row_shape(int64_t chunks, int ch) {
  if (chunks <= 64) return {64, 1, 0};
  const int nv = chunks <= 1024 ? 1 : (chunks <= 2048 ? 2 : 4);
  if (chunks > 1024 * nv || nv * ch > 16) return {0, 0, 0};
  const int tpr = (int)((chunks + 64 * nv - 1) / (64 * nv)) * 64;
  return {tpr, nv, tpr <= 512 ? 1 : (tpr <= 768 ? 2 : 3)};
}

// f(chunks per thread, size) as compile-time constants.
template <class T, class F>
void with_shape(const RowShape& s, F&& f) {
  using std::integral_constant;
  if (s.size == 0)
    f(integral_constant<int, 1>(), integral_constant<int, 0>());
  else if (s.nv == 1 && s.size == 1)
    f(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (s.nv == 1 && s.size == 2)
    f(integral_constant<int, 1>(), integral_constant<int, 2>());
  else if (s.nv == 1)
    f(integral_constant<int, 1>(), integral_constant<int, 3>());
  else if (s.nv == 2)
    f(integral_constant<int, 2>(), integral_constant<int, 3>());
  else if constexpr (sizeof(T) == 4)
    f(integral_constant<int, 4>(), integral_constant<int, 3>());
}

template <class T>
hipError_t forward(const GatedNormArgs& all, hipStream_t stream) {
  GatedNormArgs a = all;
  LaunchTimer timer(kKidGatedNorm, stream);
  constexpr int CH = 16 / (int)sizeof(T);
  const RowShape s = chunked(a, sizeof(T)) ? row_shape(a.W / CH, CH) : RowShape{0, 0, 0};
  const int64_t groups = (a.rows + a.R - 1) / a.R;
  // Workers: 4 rows each where that leaves enough of them.
  a.per_group = a.rows <= 16384 || s.nv == 0 ? a.R : (a.R + 3) / 4;
  const int rpb = s.nv > 0 && s.size == 0 ? 4 : 1;
  // Any number of rows: the threads of a grid (up to 1,024 a row) stay below 2^32.
  constexpr int64_t kMost = 1 << 21;
  const int64_t blocks = (groups * a.per_group + rpb - 1) / rpb;
  for (int64_t done = 0; done < blocks; done += kMost) {
    a.first = done * rpb;
    const unsigned grid = (unsigned)(blocks - done < kMost ? blocks - done : kMost);
    if (s.nv == 0)
      hipLaunchKernelGGL(gated_norm_any_kernel<T>, dim3(grid), dim3(256), 0, stream, a);
    else
      with_shape<T>(s, [&](auto nv, auto size) {
        const dim3 block(size == 0 ? 256 : s.tpr);
        if (a.p)
          hipLaunchKernelGGL((gated_norm_kernel<T, CH, decltype(nv)::value, decltype(size)::value, true>), dim3(grid),
                             block, 0, stream, a);
        else
          hipLaunchKernelGGL((gated_norm_kernel<T, CH, decltype(nv)::value, decltype(size)::value, false>), dim3(grid),
                             block, 0, stream, a);
      });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Workers of the backward: in all, and per group (TOKEN: all).
struct Workers {
  int64_t groups, per_group;
  bool token;
};
constexpr int64_t kMostWorkers = 512, kMostNarrow = 4096;
Workers bwd_workers(int64_t rows, int64_t R, int64_t W, bool modulated) {
  const int64_t most = W <= 1024 ? kMostNarrow : kMostWorkers, groups = (rows + R - 1) / R;
  if (R == 1 && modulated && rows > 1) return {1, rows < most ? (rows + 3) / 4 * 4 : most, true};
  int64_t per = most / groups;
  if (per < 1) per = 1;
  if (per > R) per = R;
  return {groups, per, false};
}

template <class T, bool TOKEN>
void backward_rows(const GatedNormArgs& a, const RowShape& s, int64_t workers, hipStream_t stream) {
  constexpr int CH = 16 / (int)sizeof(T);
  if (s.nv == 0) {
    hipLaunchKernelGGL((gated_norm_bwd_any_kernel<T, TOKEN>), dim3((unsigned)workers), dim3(256), 0, stream, a);
    return;
  }
  with_shape<T>(s, [&](auto nv, auto size) {
    constexpr int NV = decltype(nv)::value, S = decltype(size)::value;
    const dim3 grid((unsigned)(S == 0 ? (workers + 3) / 4 : workers)), block(S == 0 ? 256 : s.tpr);
    if (a.p && a.dh)
      hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, true, true, TOKEN>), grid, block, 0, stream, a);
    else if (a.p)
      hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, true, false, TOKEN>), grid, block, 0, stream, a);
    else if (a.dh)
      hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, false, true, TOKEN>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((gated_norm_bwd_kernel<T, CH, NV, S, false, false, TOKEN>), grid, block, 0, stream, a);
  });
}

template <class T>
hipError_t backward(const GatedNormArgs& all, hipStream_t stream) {
  GatedNormArgs a = all;
  constexpr int CH = 16 / (int)sizeof(T);
  const RowShape s = chunked(a, sizeof(T)) ? row_shape(a.W / CH, CH) : RowShape{0, 0, 0};
  const Workers w = bwd_workers(a.rows, a.R, a.W, a.g || a.s || a.t);
  a.per_group = w.per_group;
  {
    LaunchTimer timer(kKidGatedNormBwd, stream);
    if (w.token)
      backward_rows<T, true>(a, s, w.per_group, stream);
    else
      backward_rows<T, false>(a, s, w.groups * w.per_group, stream);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const unsigned columns = (unsigned)((a.W + 31) / 32);
  if (w.token) {
    if (a.dw || a.dp)
      hipLaunchKernelGGL((gated_norm_gains_kernel<T, true>), dim3(columns), dim3(256), 0, stream, a, w.per_group,
                         3 * a.W);
    return hipGetLastError();
  }
  if (a.ds || a.dt || a.dg || a.dw || a.dp)
    hipLaunchKernelGGL(gated_norm_groups_kernel<T>, dim3(columns, (unsigned)(w.groups < 32768 ? w.groups : 32768)),
                       dim3(256), 0, stream, a, w.groups);
  if (w.groups > 1 && (a.dw || a.dp))
    hipLaunchKernelGGL((gated_norm_gains_kernel<T, false>), dim3(columns), dim3(256), 0, stream, a, w.groups,
                       w.per_group * 3 * a.W);
  return hipGetLastError();
}

}  // namespace

size_t gated_norm_bwd_workspace_bytes(int64_t rows, int64_t R, int64_t W, bool modulated) {
  if (rows == 0) return 0;
  const Workers w = bwd_workers(rows, R, W, modulated);
  // (Whole workgroups of four narrow rows.)
  return (size_t)((w.groups * w.per_group + 3) / 4 * 4) * 3 * (size_t)W * sizeof(float);
}

hipError_t launch_gated_norm(const GatedNormArgs& a, bool f32, hipStream_t stream) {
  return f32 ? forward<float>(a, stream) : forward<bf16>(a, stream);
}

hipError_t launch_gated_norm_bwd(const GatedNormArgs& a, bool f32, hipStream_t stream) {
  return f32 ? backward<float>(a, stream) : backward<bf16>(a, stream);
}

}  // namespace avattn
