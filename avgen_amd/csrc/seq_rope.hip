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
// Both are HBM-bound: the rotation reads and writes every value once; the
// tables are read once per token, not once per head.
#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

constexpr int kThreads = 256;

// The angle pos * f in double (a position of a million turns a pair of
// frequency 1 by a million radians, which float rounds by 0.06), reduced to
// [-pi, pi] by a two-term 2 pi before the library's double sincos, whose slow
// path for large arguments is then never taken; rounded to float once.
template <class P>
__global__ __launch_bounds__(kThreads) void position_tables_kernel(PositionTableArgs a, const P* __restrict__ pos) {
  constexpr double kInv2Pi = 0.15915494309189533577, k2PiHi = 6.28318530717958647693,
                   k2PiLo = 2.4492935982947064e-16;
  const int64_t n = (int64_t)a.B * a.L * a.P;
  for (int64_t u = blockIdx.x * (int64_t)kThreads + threadIdx.x; u < n; u += (int64_t)gridDim.x * kThreads) {
    const int64_t bi = u / a.P;
    const int p = (int)(u - bi * a.P);
    const int64_t b = bi / a.L, i = bi - b * a.L;
    const double ang = (double)pos[b * a.psb + i] * a.freq[p];
    const double turns = rint(ang * kInv2Pi);
    const double r = fma(-turns, k2PiLo, fma(-turns, k2PiHi, ang));
    double s, c;
    sincos(r, &s, &c);
    a.cos_out[u] = (float)(c * a.amplitude);
    a.sin_out[u] = (float)(s * a.amplitude);
  }
}

// CH consecutive values of T as floats and back (rounded once).
template <class T, int CH>
struct Chunk {
  float v[CH];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (CH == 8) {  // bf16
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else if constexpr (CH == 4) {  // float
      const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) v[i] = (float)p[i];
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
  const int64_t tok = (int64_t)blockIdx.x * tpb + (tpb > 1 ? g / heads : 0);
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
    for (int h = h0; h < heads; h += hstep) {
      const int w = h >= a.H[0];
      const int64_t xo = b * a.xs[w][0] + (int64_t)(h - (w ? a.H[0] : 0)) * a.xs[w][1] + (int64_t)i * a.xs[w][2] + ch;
      const int64_t oo = b * a.os[w][0] + (int64_t)(h - (w ? a.H[0] : 0)) * a.os[w][1] + (int64_t)i * a.os[w][2] + ch;
      const T* x = reinterpret_cast<const T*>(a.x[w]) + xo;
      T* o = reinterpret_cast<T*>(a.o[w]) + oo;
      if (!turn) {
        if constexpr (VEC)
          *reinterpret_cast<u32x4*>(o) = *reinterpret_cast<const u32x4*>(x);
        else
          *o = *x;
        continue;
      }
      if constexpr (HALF) {
        Chunk<T, CH> p, q;
        p.load(x);
        q.load(x + a.P);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const float e = p.v[j], f = q.v[j];
          p.v[j] = e * cs[j] - f * sn[j];
          q.v[j] = e * sn[j] + f * cs[j];
        }
        p.store(o);
        q.store(o + a.P);
      } else {
        Chunk<T, CH> p;
        p.load(x);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const float e = p.v[2 * j], f = p.v[2 * j + 1];
          p.v[2 * j] = e * cs[j] - f * sn[j];
          p.v[2 * j + 1] = e * sn[j] + f * cs[j];
        }
        p.store(o);
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
  if (blocks > 2147483647) return hipErrorInvalidValue;
  LaunchTimer timer(kKidRopeApply, stream);
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (half && vec)
    hipLaunchKernelGGL((rotate_kernel<T, true, true>), grid, block, 0, stream, a);
  else if (half)
    hipLaunchKernelGGL((rotate_kernel<T, true, false>), grid, block, 0, stream, a);
  else if (vec)
    hipLaunchKernelGGL((rotate_kernel<T, false, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((rotate_kernel<T, false, false>), grid, block, 0, stream, a);
  return hipGetLastError();
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
