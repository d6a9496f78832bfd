// Rotation of token sequences by their positions: tables of cos and sin for
// integer positions (the 1D counterpart of rope.hip's coordinate tables) and
// the rotation of part of each head in either pair layout, query and key in
// one launch.
//
//   tables   cos[b, i, p] = A cos(pos[b, i] f_p),  sin likewise
//   rotation of channels [start, start + 2P) of a head, pair p = (x0, x1):
//            y0 = x0 c - x1 s,  y1 = x0 s + x1 c     (s -> -s: the transpose)
//            interleaved: x0, x1 at start + 2p, + 1; half: at start + p,
//            start + P + p; the other channels are copied.
// The rotation is HBM-bound: it reads and writes every value once; the tables
// are read once per token, not once per head.  2 x 4,096 tokens of 80
// heads of 128 bf16, half of each rotated: 73 us (4.6 TB/s); 65,537 tokens of
// 20 heads, all of it: 150 us (4.5 TB/s), their tables 20 us (1.7 TB/s: the
// vector ALUs are busy in every cycle, with about 119 instructions an entry,
// 31 of them in double and 36 of the two index divisions); 16 tokens of 40
// heads 4 us.  Value by value (VEC false), 2 x 4,096 tokens of 80 heads of 80,
// 20 pairs in half layout, 97 us, where the interleaved layout's chunks take 33.
#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

constexpr int kThreads = 256;

// sin and cos of x in double, to 1e-11: x is reduced to [-pi/4, pi/4] by a
// two-term pi/2 and both Taylor series are summed to their 13th and 12th
// power.  (The library's double sincos, after a reduction to [-pi, pi], took
// 65,537 x 64 entries from 25 us.)
__device__ __forceinline__ void sincos_f64(double x, double& s, double& c) {
  constexpr double k2OverPi = 0.63661977236758134308, kPi2Hi = 1.57079632679489661923, kPi2Lo = 6.123233995736766e-17;
  const double n = rint(x * k2OverPi);
  const double r = fma(-n, kPi2Lo, fma(-n, kPi2Hi, x)), z = r * r;
  const double sp = fma(fma(fma(fma(fma(fma(z, 1. / 6227020800., -1. / 39916800.), z, 1. / 362880.), z, -1. / 5040.),
                                z, 1. / 120.),
                            z, -1. / 6.),
                        z * r, r);
  const double cp =
      fma(fma(fma(fma(fma(fma(z, 1. / 479001600., -1. / 3628800.), z, 1. / 40320.), z, -1. / 720.), z, 1. / 24.), z,
              -0.5),
          z, 1.);
  const int q = (int)fma(-4., floor(n * 0.25), n);  // n mod 4
  const double a = q & 1 ? cp : sp, b = q & 1 ? sp : cp;
  s = q & 2 ? -a : a;
  c = (q + 1) & 2 ? -b : b;
}

// The angle pos * f in double (a position of a million turns a pair of
// frequency 1 by a million radians, which float rounds by 0.06), its cos and
// sin rounded to float once.
template <class P>
__global__ __launch_bounds__(kThreads) void position_tables_kernel(PositionTableArgs a, const P* __restrict__ pos) {
  const int64_t n = (int64_t)a.B * a.L * a.P;
  for (int64_t u = blockIdx.x * (int64_t)kThreads + threadIdx.x; u < n; u += (int64_t)gridDim.x * kThreads) {
    const int64_t bi = u / a.P;
    const int p = (int)(u - bi * a.P);
    const int64_t b = bi / a.L, i = bi - b * a.L;
    const double ang = (double)pos[b * a.psb + i] * a.freq[p];
    double s, c;
    sincos_f64(ang, s, c);
    a.cos_out[u] = (float)(c * a.amplitude);
    a.sin_out[u] = (float)(s * a.amplitude);
  }
}

// CH consecutive values of T as floats and back (rounded once).
template <class T, int CH>
struct Chunk {
  struct Values {
    T e[CH];
  };
  using Raw = std::conditional_t<(CH >= 4), u32x4, Values>;
  float v[CH];
  static __device__ __forceinline__ Raw read(const T* p) {
    if constexpr (CH >= 4) {
      return *reinterpret_cast<const u32x4*>(p);
    } else {
      Raw r;
#pragma unroll
      for (int i = 0; i < CH; ++i) r.e[i] = p[i];
      return r;
    }
  }
  __device__ __forceinline__ explicit Chunk(const Raw& w) {
    if constexpr (CH == 8) {  // bf16
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else if constexpr (CH == 4) {  // float
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) v[i] = (float)w.e[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (CH == 8) {
      *reinterpret_cast<u32x4*>(p) = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                           pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    } else if constexpr (CH == 4) {
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) p[i] = (T)v[i];
    }
  }
};

// A unit is what one thread does to one row of one head: half layout, a chunk
// of x0 and the chunk of x1 that goes with it, or a chunk to copy;
// interleaved, a chunk of whole pairs or one to copy.  A thread keeps its unit
// (so its table values) and walks over heads.  A workgroup takes one token
// with its heads spread over 256 / units thread groups, or several tokens when
// one token's heads do not fill it.  CH 16-byte chunks (VEC), or single values
// and pairs for widths, starts or strides that are no multiple of them.
template <class T, bool HALF, bool VEC>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
  // Every product rounded separately (no FMA), as the full-head rotation of
  // rope.hip computes it.
#pragma clang fp contract(off)
  constexpr int CH = VEC ? 16 / (int)sizeof(T) : (HALF ? 1 : 2);
  constexpr int NC = HALF ? CH : CH / 2;  // table values per unit
  const int dims = 2 * a.P;
  const int rot = HALF ? a.P / CH : dims / CH;                   // rotating units per row
  const int CP = VEC ? CH : 1;                                   // channels of a copying unit
  const int units = rot + (a.D - dims) / CP;
  const int cu = min(units, kThreads), groups = kThreads / cu;
  const int c0 = threadIdx.x % cu, g = threadIdx.x / cu;
  if (g >= groups) return;
  const int heads = a.H[0] + a.H[1];
  const int tpb = max(1, groups / heads);
  const int64_t tok = a.first + (int64_t)blockIdx.x * tpb + (tpb > 1 ? g / heads : 0);
  if (tok >= (int64_t)a.B * a.L || (tpb > 1 && g >= tpb * heads)) return;
  const int h0 = tpb > 1 ? g % heads : g, hstep = tpb > 1 ? heads : groups;
  const int b = (int)(tok / a.L), i = (int)(tok - (int64_t)b * a.L);
  for (int c = c0; c < units; c += cu) {
    const bool turn = c < rot;
    // First channel of the unit, and of its partner chunk (half layout).
    int ch;
    if (turn) {
      ch = a.start + c * CH;
    } else {
      ch = (c - rot) * CP;
      if (ch >= a.start) ch += dims;
    }
    float cs[NC], sn[NC];
    if (turn) {
      const int64_t t = b * a.tsb + (int64_t)i * a.P + (HALF ? c * CH : c * CH / 2);
      if constexpr (VEC && NC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < NC; j += 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(a.ct + t + j), y = *reinterpret_cast<const f32x4*>(a.st + t + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) cs[j + e] = x[e], sn[j + e] = y[e];
        }
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j) cs[j] = a.ct[t + j], sn[j] = a.st[t + j];
      }
      if (a.inverse) {
#pragma unroll
        for (int j = 0; j < NC; ++j) sn[j] = -sn[j];
      }
    }
    // Heads in batches of four: their loads are in flight together.
    const T* xt[2];
    T* ot[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      xt[w] = reinterpret_cast<const T*>(a.x[w]) + b * a.xs[w][0] + (int64_t)i * a.xs[w][2] + ch;
      ot[w] = reinterpret_cast<T*>(a.o[w]) + b * a.os[w][0] + (int64_t)i * a.os[w][2] + ch;
    }
    auto row = [&](int h, const T*& x, T*& o) {
      const int w = h >= a.H[0], hw = h - (w ? a.H[0] : 0);
      x = (w ? xt[1] : xt[0]) + hw * (w ? a.xs[1][1] : a.xs[0][1]);
      o = (w ? ot[1] : ot[0]) + hw * (w ? a.os[1][1] : a.os[0][1]);
    };
    constexpr int U = 4;
    using Raw = typename Chunk<T, CH>::Raw;
    for (int hb = h0; hb < heads; hb += U * hstep) {
      const T* x[U];
      T* o[U];
      Raw p[U], q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = hb + u * hstep;
        row(h < heads ? h : hb, x[u], o[u]);
        if (h < heads) {
          if (VEC || turn) p[u] = Chunk<T, CH>::read(x[u]);
          if (HALF && turn) q[u] = Chunk<T, CH>::read(x[u] + a.P);
          if constexpr (!VEC) {
            if (!turn) *o[u] = *x[u];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (hb + u * hstep >= heads) break;
        if (!turn) {
          if constexpr (VEC) *reinterpret_cast<Raw*>(o[u]) = p[u];
          continue;
        }
        Chunk<T, CH> y(p[u]);
        if constexpr (HALF) {
          Chunk<T, CH> z(q[u]);
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const float e = y.v[j], f = z.v[j];
            y.v[j] = e * cs[j] - f * sn[j];
            z.v[j] = e * sn[j] + f * cs[j];
          }
          z.store(o[u] + a.P);
        } else {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const float e = y.v[2 * j], f = y.v[2 * j + 1];
            y.v[2 * j] = e * cs[j] - f * sn[j];
            y.v[2 * j + 1] = e * sn[j] + f * cs[j];
          }
        }
        y.store(o[u]);
      }
    }
  }
}

bool chunked(const RotateArgs& a, int size, bool half) {
  const int ch = 16 / size;
  auto whole = [&](int64_t n) { return n % ch == 0; };
  bool ok = whole(a.D) && whole(a.start) && whole(half ? a.P : 2 * a.P) && a.P % 4 == 0 && a.tsb % 4 == 0 &&
            (reinterpret_cast<uintptr_t>(a.ct) | reinterpret_cast<uintptr_t>(a.st)) % 16 == 0;
  for (int w = 0; w < 2; ++w) {
    if (a.H[w] == 0) continue;
    ok = ok && (reinterpret_cast<uintptr_t>(a.x[w]) | reinterpret_cast<uintptr_t>(a.o[w])) % 16 == 0;
    for (int d = 0; d < 3; ++d) ok = ok && whole(a.xs[w][d]) && whole(a.os[w][d]);
  }
  return ok;
}

template <class T>
hipError_t rotate(const RotateArgs& a, bool half, hipStream_t stream) {
  const bool vec = chunked(a, sizeof(T), half);
  const int ch = vec ? 16 / (int)sizeof(T) : (half ? 1 : 2);
  const int units = (half ? a.P : 2 * a.P) / ch + (a.D - 2 * a.P) / (vec ? ch : 1);
  const int groups = kThreads / (units < kThreads ? units : kThreads);
  const int heads = a.H[0] + a.H[1];
  const int tpb = groups / heads > 1 ? groups / heads : 1;
  const int64_t blocks = ((int64_t)a.B * a.L + tpb - 1) / tpb;
  LaunchTimer timer(kKidRopeApply, stream);
  // Any number of tokens: the threads of a grid stay below 2^32.
  constexpr int64_t kMost = 1 << 23;
  for (int64_t done = 0; done < blocks; done += kMost) {
    RotateArgs r = a;
    r.first = done * tpb;
    const dim3 grid((unsigned)(blocks - done < kMost ? blocks - done : kMost)), block(kThreads);
    if (half && vec)
      hipLaunchKernelGGL((rotate_kernel<T, true, true>), grid, block, 0, stream, r);
    else if (half)
      hipLaunchKernelGGL((rotate_kernel<T, true, false>), grid, block, 0, stream, r);
    else if (vec)
      hipLaunchKernelGGL((rotate_kernel<T, false, true>), grid, block, 0, stream, r);
    else
      hipLaunchKernelGGL((rotate_kernel<T, false, false>), grid, block, 0, stream, r);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_position_tables(const PositionTableArgs& a, const void* pos, bool wide, hipStream_t stream) {
  const int64_t n = (int64_t)a.B * a.L * a.P;
  if (n == 0) return hipSuccess;
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  LaunchTimer timer(kKidRopeTables, stream);
  if (wide)
    hipLaunchKernelGGL(position_tables_kernel<int64_t>, grid, dim3(kThreads), 0, stream, a,
                       static_cast<const int64_t*>(pos));
  else
    hipLaunchKernelGGL(position_tables_kernel<int32_t>, grid, dim3(kThreads), 0, stream, a,
                       static_cast<const int32_t*>(pos));
  return hipGetLastError();
}

hipError_t launch_rotate(const RotateArgs& a, bool half, bool f32, hipStream_t stream) {
  if ((int64_t)a.B * a.L * (a.H[0] + a.H[1]) == 0) return hipSuccess;
  return f32 ? rotate<float>(a, half, stream) : rotate<bf16>(a, half, stream);
}

}  // namespace avattn
