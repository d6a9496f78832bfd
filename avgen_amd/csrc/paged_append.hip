// Appending keys and values to a cache of pages, the keys (and a query)
// rotated on the way, and reading back what pages hold.
//
// Token i of the new ones of sequence b is at position p = length - count + i
// and goes to slot p % P of page table[b][p / P].  bf16 pages hold the rounded
// values; e4m3 pages codes c = e4m3(x / 2^e) with one exponent e for the
// slots of a page and head:
//   e = least integer with 448 2^e >= max |x| over the new tokens of the page,
//       and not below the page's exponent where earlier tokens are in it;
//   if that raises the exponent, the page's other codes become e4m3(c 2^(e' - e)),
//   those behind the new tokens too: what they stand for stays.
// A power of two costs e4m3 nothing (its own steps are relative) and makes
// c 2^e a bf16 value exactly, so readers convert without rounding, and a raised
// exponent moves codes without rounding them, subnormal ones apart.
// HBM-bound: k, v and q are read once and written once.  A workgroup takes the
// slots of one page and one head (their maximum is needed before the first is
// written), its values in registers in between.
#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

constexpr int kItem = 16;  // channels a thread rotates at once: two chunks of 8

__device__ __forceinline__ void unpack8(const u32x4& w, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
}
__device__ __forceinline__ void store8(bf16* p, const float* v) {
  *reinterpret_cast<u32x4*>(p) =
      u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// The two 8-channel chunks of item u of a row.  Half layout: a chunk of the
// pairs' first channels and the one of their second channels, then the channels
// that are not rotated; else consecutive chunks.
struct ItemPlace {
  int c0, c1;
  bool pair;  // c0 and c1 turn together
};
__device__ __forceinline__ ItemPlace item_place(const AppendRotation& r, int u) {
  if (!r.half || r.cos == nullptr) return {kItem * u, kItem * u + 8, false};
  const int rot = r.pairs / 8;
  if (u < rot) return {r.start + 8 * u, r.start + r.pairs + 8 * u, true};
  int c0 = kItem * (u - rot), c1 = c0 + 8;
  if (c0 >= r.start) c0 += 2 * r.pairs;
  if (c1 >= r.start) c1 += 2 * r.pairs;
  return {c0, c1, false};
}

// The factors of an item of whole chunks, the same for all heads: of a pair of
// chunks all eight, else four for each chunk that is rotated.
struct Turn {
  float c[8] = {}, s[8] = {};
  bool on0 = false, on1 = false;
  __device__ __forceinline__ void load4(const AppendRotation& r, int64_t at, int j) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(r.cos + at), y = *reinterpret_cast<const f32x4*>(r.sin + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j + i] = x[i], s[j + i] = y[i];
  }
  // t: the row's place in the tables.
  __device__ __forceinline__ void load(const AppendRotation& r, int64_t t, int u, const ItemPlace& at) {
    on0 = on1 = at.pair;
    if (r.cos == nullptr) return;
    if (at.pair) {
      load4(r, t + 8 * u, 0);
      load4(r, t + 8 * u + 4, 4);
    } else if (!r.half) {
      auto in = [&](int ch) { return ch >= r.start && ch < r.start + 2 * r.pairs; };
      on0 = in(at.c0), on1 = in(at.c1);
      if (on0) load4(r, t + (at.c0 - r.start) / 2, 0);
      if (on1) load4(r, t + (at.c1 - r.start) / 2, 4);
    }
  }
  // Every product rounded separately, as rotate_kernel does.
  __device__ __forceinline__ void apply(const ItemPlace& at, float* v) const {
#pragma clang fp contract(off)
    if (at.pair) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = v[i], f = v[8 + i];
        v[i] = e * c[i] - f * s[i];
        v[8 + i] = e * s[i] + f * c[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = v[2 * i], f = v[2 * i + 1];
        const bool on = i < 4 ? on0 : on1;
        v[2 * i] = on ? e * c[i] - f * s[i] : e;
        v[2 * i + 1] = on ? e * s[i] + f * c[i] : f;
      }
    }
  }
};

// Item u of the rows of HB heads, `hs` apart from x on (those below `heads`), rotated
// (ROT) by the table row at t.  VEC: whole 16-byte chunks; else channel by channel,
// any pairs, start and strides.
template <bool VEC, bool ROT, int HB>
__device__ __forceinline__ void load_items(const AppendRotation& r, const bf16* x, int64_t hs, int heads, int64_t t,
                                           int u, float (*v)[kItem]) {
#pragma clang fp contract(off)
  if constexpr (VEC) {
    ItemPlace at{kItem * u, kItem * u + 8, false};
    if (ROT) at = item_place(r, u);
    Turn turn;
    if (ROT) turn.load(r, t, u, at);
    u32x4 r0[HB], r1[HB];
#pragma unroll
    for (int e = 0; e < HB; ++e) {
      const bf16* row = x + (e < heads ? e : 0) * hs;  // (past the last head: the first one again)
      r0[e] = *reinterpret_cast<const u32x4*>(row + at.c0);
      r1[e] = *reinterpret_cast<const u32x4*>(row + at.c1);
    }
#pragma unroll
    for (int e = 0; e < HB; ++e) {
      unpack8(r0[e], v[e]);
      unpack8(r1[e], v[e] + 8);
      if (ROT) turn.apply(at, v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < HB; ++e) {
      if (e >= heads) continue;
#pragma unroll
      for (int j = 0; j < kItem; ++j) {
        const int ch = kItem * u + j, at = ch - r.start;
        const bf16* row = x + e * hs;
        float y = (float)row[ch];
        if (ROT && r.cos != nullptr && at >= 0 && at < 2 * r.pairs) {
          const int p = r.half ? at % r.pairs : at / 2;
          const bool second = r.half ? at >= r.pairs : at & 1;
          const int mate = r.half ? (second ? ch - r.pairs : ch + r.pairs) : (second ? ch - 1 : ch + 1);
          const float o = (float)row[mate], c = r.cos[t + p], s = r.sin[t + p];
          y = second ? o * s + y * c : y * c - o * s;
        }
        v[e][j] = y;
      }
    }
  }
}

template <bool VEC, bool ROT>
__device__ __forceinline__ ItemPlace stored_place(const AppendRotation& r, int u) {
  if (VEC && ROT) return item_place(r, u);
  return {kItem * u, kItem * u + 8, false};
}

// Least e with 448 2^e >= m, in the range in which code * 2^e stays a normal
// bf16 number.  448 = 1.75 * 2^8.
__device__ __forceinline__ int code_exponent(float m) {
  const uint32_t bits = __float_as_uint(m);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kMinCodeExponent), kMaxCodeExponent);
}

// e4m3(x): values past the largest code (of an exponent at its limit) saturate,
// what is not finite becomes NaN.
__device__ __forceinline__ float code_value(float x) {
  return fabsf(x) < kPosInf ? fminf(fmaxf(x, -448.f), 448.f) : __builtin_nanf("");
}
__device__ __forceinline__ u32x2 codes8(const float* v, float unit) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = code_value(v[i] * unit);
  return u32x2{pack_fp8x4(y[0], y[1], y[2], y[3]), pack_fp8x4(y[4], y[5], y[6], y[7])};
}

// Four codes times 2^shift, as codes again (shift <= 0).
__device__ __forceinline__ uint32_t moved_codes(uint32_t w, int shift) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = w >> (8 * i) & 0xffu;
    y[i] = ldexpf(__builtin_amdgcn_cvt_f32_fp8((int)c, 0), shift);
  }
  return pack_fp8x4(y[0], y[1], y[2], y[3]);
}

// The page, the tokens and their place of one workgroup of the k and v part.
struct PagePlace {
  int64_t page;  // -1: none
  int lo, hi;    // slots of new tokens
  int i0;        // token of slot 0 (negative where earlier ones precede)
};
__device__ __forceinline__ PagePlace page_place(const AppendArgs& a, int b, int j) {
  const int count = a.counts ? min(max(a.counts[b], 0), a.L) : a.L;
  const int64_t first = (int64_t)a.lengths[b] - count;  // may be negative: such tokens have no slot
  const int64_t block = (first > 0 ? first >> a.pages.shift : 0) + j, slot0 = block << a.pages.shift;
  PagePlace p{-1, 0, 0, 0};
  const int64_t lo = first > slot0 ? first - slot0 : 0, hi = first + count - slot0;
  if (hi <= lo || block >= a.pages.blocks) return p;
  p.lo = (int)lo;
  p.hi = (int)(hi < (1 << a.pages.shift) ? hi : (1 << a.pages.shift));
  p.i0 = (int)(slot0 - first);
  p.page = a.pages.page(b, block);
  return p;
}

// Heads that a thread takes together (the factors of the rotation are read once
// for them, and their rows are in flight together): of the query, and of bf16 pages
// as far as registers allow (two prompts of 8,192 tokens, 32 heads of 128: 187 ->
// 151 us).  A page and head of codes needs its maximum before the first is written;
// beside it more of the query's heads cost waves (four of 4,133 tokens, 32 query
// heads: 80 us, with 4 together 93).
template <bool FP8>
constexpr int kQueryHeads = FP8 ? 1 : 4;
template <bool FP8, int NI>
constexpr int kPageHeads = FP8 ? 1 : (NI == 1 ? 4 : (NI == 2 ? 2 : 1));

// Workgroups [0, nkv): (b, block, kv heads, key or value); then the query's rows.
template <int D, bool FP8, bool VEC, int NI>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int nkv) {
  constexpr int IPR = D / kItem;  // items of a row
  constexpr int HB = kPageHeads<FP8, NI>, HQ = kQueryHeads<FP8>;
  const int tid = threadIdx.x, n = blockDim.x;
  if ((int)blockIdx.x >= nkv) {
    const int64_t u0 = ((int64_t)blockIdx.x - nkv) * n + tid;
    const int u = (int)(u0 % IPR);
    const int nh = (a.Hq + HQ - 1) / HQ;
    const int64_t bi = u0 / IPR / nh;
    if (bi >= (int64_t)a.B * a.L) return;
    const int h0 = (int)(u0 / IPR - bi * nh);  // heads h0, h0 + nh, ..
    const int b = (int)(bi / a.L), i = (int)(bi - (int64_t)b * a.L);
    const int heads = (a.Hq - h0 + nh - 1) / nh;
    float v[HQ][kItem];
    load_items<VEC, true, HQ>(a.rot, a.q + b * a.qsb + h0 * a.qsh + i * a.qsl, nh * a.qsh, heads,
                                       b * a.rot.tsb + (int64_t)i * a.rot.pairs, u, v);
    const ItemPlace at = stored_place<VEC, true>(a.rot, u);
#pragma unroll
    for (int e = 0; e < HQ; ++e) {
      if (e >= heads) continue;
      bf16* o = a.q_out + b * a.osb + (h0 + e * nh) * a.osh + i * a.osl;
      if constexpr (VEC) {
        store8(o + at.c0, v[e]);
        store8(o + at.c1, v[e] + 8);
      } else {
#pragma unroll
        for (int j = 0; j < kItem; ++j) o[kItem * u + j] = (bf16)v[e][j];
      }
    }
    return;
  }
  __shared__ float red[4];
  int w = blockIdx.x;
  const int which = w & 1;
  w >>= 1;
  const int nh = (a.Hkv + HB - 1) / HB;
  const int h = w % nh * HB;
  w /= nh;
  const int j = w % a.nblocks, b = w / a.nblocks;
  const PagePlace pp = page_place(a, b, j);
  if (pp.page < 0) return;  // the whole workgroup
  const bool key = which == 0;
  const bf16* x = (key ? a.k + b * a.ksb + h * a.ksh : a.v + b * a.vsb + h * a.vsh);
  const int64_t sl = key ? a.ksl : a.vsl, sh = key ? a.ksh : a.vsh;
  const int heads = min(HB, a.Hkv - h);
  float v[NI][HB][kItem];
#pragma unroll
  for (int m = 0; m < NI; ++m) {
    const int it = m * n + tid, slot = it / IPR, u = it % IPR;
    if (slot < pp.lo || slot >= pp.hi) continue;
    const int i = pp.i0 + slot;
    if (key)
      load_items<VEC, true, HB>(a.rot, x + i * sl, sh, heads, b * a.rot.tsb + (int64_t)i * a.rot.pairs, u, v[m]);
    else
      load_items<VEC, false, HB>(a.rot, x + i * sl, sh, heads, 0, u, v[m]);
  }
  if constexpr (!FP8) {
    const int64_t ph = key ? a.kph : a.vph;
    bf16* out = static_cast<bf16*>(key ? a.kp : a.vp) + pp.page * (key ? a.kps : a.vps) + h * ph;
#pragma unroll
    for (int m = 0; m < NI; ++m) {
      const int it = m * n + tid, slot = it / IPR, u = it % IPR;
      if (slot < pp.lo || slot >= pp.hi) continue;
      const ItemPlace at = key ? stored_place<VEC, true>(a.rot, u) : stored_place<VEC, false>(a.rot, u);
#pragma unroll
      for (int e = 0; e < HB; ++e) {
        if (e >= heads) continue;
        store8(out + e * ph + slot * D + at.c0, v[m][e]);
        store8(out + e * ph + slot * D + at.c1, v[m][e] + 8);
      }
    }
  } else {
    float top = 0.f;
#pragma unroll
    for (int m = 0; m < NI; ++m) {
      const int slot = (m * n + tid) / IPR;
      if (slot < pp.lo || slot >= pp.hi) continue;
#pragma unroll
      for (int e = 0; e < kItem; ++e) {
        const float y = fabsf(v[m][0][e]);
        top = fmaxf(top, y < kPosInf ? y : 0.f);
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    int8_t* ep = (key ? a.ke + pp.page * a.kes : a.ve + pp.page * a.ves) + h;
    const int e0 = *ep;
    __syncthreads();  // (and e0 is read before it is written)
    top = red[0];
    for (int i = 1; i < n / 64; ++i) top = fmaxf(top, red[i]);
    int e = code_exponent(top);
    if (pp.lo > 0) e = max(e, e0);
    if (tid == 0) *ep = (int8_t)e;
    uint8_t* out = static_cast<uint8_t*>(key ? a.kp : a.vp);
    out += pp.page * (key ? a.kps : a.vps) + h * (key ? a.kph : a.vph);
    if (pp.lo > 0 && e > e0) {
      for (int it = tid; it < IPR << a.pages.shift; it += n) {
        if (it >= pp.lo * IPR && it < pp.hi * IPR) continue;
        u32x4* c = reinterpret_cast<u32x4*>(out + it * kItem);
        u32x4 y = *c;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = moved_codes(y[i], e0 - e);
        *c = y;
      }
    }
    const float unit = ldexpf(1.f, -e);  // (a page's own exponent may be 127: 2^-127 is subnormal)
#pragma unroll
    for (int m = 0; m < NI; ++m) {
      const int it = m * n + tid, slot = it / IPR, u = it % IPR;
      if (slot < pp.lo || slot >= pp.hi) continue;
      const ItemPlace at = key ? stored_place<VEC, true>(a.rot, u) : stored_place<VEC, false>(a.rot, u);
      *reinterpret_cast<u32x2*>(out + slot * D + at.c0) = codes8(v[m][0], unit);
      *reinterpret_cast<u32x2*>(out + slot * D + at.c1) = codes8(v[m][0] + 8, unit);
    }
  }
}

// 16 codes -> 16 bf16 per thread and round: (page, head, slot, channel) in order.
__global__ __launch_bounds__(256) void page_values_kernel(PageValuesArgs a) {
  const int64_t per = (int64_t)a.H << a.shift, n = (int64_t)a.pages * per * a.D / 16;
  const int w = blockIdx.y;
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < n; u += (int64_t)gridDim.x * 256) {
    const int64_t row = u * 16 / a.D;
    const int64_t page = row / per;
    const int r = (int)(row - page * per), h = r >> a.shift, slot = r - (h << a.shift);
    const int c = (int)(u * 16 - row * a.D);
    const uint8_t* src = a.codes[w] + page * a.ps[w] + h * a.hs[w] + (int64_t)slot * a.D + c;
    const int e = a.exponent[w][page * a.es[w] + h];
    const u32x4 x = *reinterpret_cast<const u32x4*>(src);
    u32x4 y[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = ldexpf(__builtin_amdgcn_cvt_f32_fp8((int)(x[i] >> (8 * k) & 0xffu), 0), e);
      y[i / 2][2 * (i & 1)] = pack_bf16x2(f[0], f[1]);
      y[i / 2][2 * (i & 1) + 1] = pack_bf16x2(f[2], f[3]);
    }
    bf16* o = a.out[w] + u * 16;
    *reinterpret_cast<u32x4*>(o) = y[0];
    *reinterpret_cast<u32x4*>(o + 8) = y[1];
  }
}

bool whole_chunks(const AppendArgs& a) {
  auto ok = [](const void* p, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
  };
  bool r = ok(a.k, a.ksb, a.ksh, a.ksl) && ok(a.v, a.vsb, a.vsh, a.vsl);
  if (a.q) r = r && ok(a.q, a.qsb, a.qsh, a.qsl) && ok(a.q_out, a.osb, a.osh, a.osl);
  if (a.rot.cos)
    r = r && a.rot.start % 8 == 0 && a.rot.pairs % (a.rot.half ? 8 : 4) == 0 && a.rot.tsb % 4 == 0 &&
        (reinterpret_cast<uintptr_t>(a.rot.cos) | reinterpret_cast<uintptr_t>(a.rot.sin)) % 16 == 0;
  return r;
}

template <int D, bool FP8, bool VEC>
void launch_items(const AppendArgs& a, int ni, int threads, unsigned grid, int nkv, hipStream_t stream) {
  if (ni == 1)
    hipLaunchKernelGGL((append_kernel<D, FP8, VEC, 1>), dim3(grid), dim3(threads), 0, stream, a, nkv);
  else if (ni == 2)
    hipLaunchKernelGGL((append_kernel<D, FP8, VEC, 2>), dim3(grid), dim3(threads), 0, stream, a, nkv);
  else if (ni == 4)
    hipLaunchKernelGGL((append_kernel<D, FP8, VEC, 4>), dim3(grid), dim3(threads), 0, stream, a, nkv);
  else
    hipLaunchKernelGGL((append_kernel<D, FP8, VEC, 8>), dim3(grid), dim3(threads), 0, stream, a, nkv);
}

}  // namespace

// Threads of a workgroup, items of a thread, and workgroups of either part.
struct AppendShape {
  int threads, ni;
  int64_t nkv, nq;
};
static AppendShape append_shape(const AppendArgs& a, int head_dim) {
  const int page = 1 << a.pages.shift, ipr = head_dim / kItem, items = page * ipr;
  AppendShape s;
  s.threads = items < 256 ? (items + 63) / 64 * 64 : 256;
  s.ni = items > 256 ? items / 256 : 1;
  const int heads = a.ke ? 1 : (s.ni == 1 ? kPageHeads<false, 1> : (s.ni == 2 ? kPageHeads<false, 2> : 1));
  s.nkv = 2 * (int64_t)a.B * ((a.L - 1) / page + 2) * ((a.Hkv + heads - 1) / heads);
  const int together = a.ke ? kQueryHeads<true> : kQueryHeads<false>;
  const int64_t nh = (a.Hq + together - 1) / together;
  s.nq = a.q ? ((int64_t)a.B * a.L * nh * ipr + s.threads - 1) / s.threads : 0;
  return s;
}

bool append_fits(const AppendArgs& a, int head_dim) {
  const AppendShape s = append_shape(a, head_dim);
  return (s.nkv + s.nq) * s.threads < (int64_t)1 << 32 && s.nkv < (int64_t)1 << 31;
}

hipError_t launch_append(const AppendArgs& args, int head_dim, hipStream_t stream) {
  AppendArgs a = args;
  const AppendShape s = append_shape(a, head_dim);
  a.nblocks = (a.L - 1) / (1 << a.pages.shift) + 2;
  const int ni = s.ni, threads = s.threads;
  const int64_t nkv = s.nkv, nq = s.nq;
  const unsigned grid = (unsigned)(nkv + nq);
  const bool vec = whole_chunks(a), fp8 = a.ke != nullptr;
  LaunchTimer timer(kKidAppend, stream);
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (fp8 && vec)
      launch_items<D, true, true>(a, ni, threads, grid, (int)nkv, stream);
    else if (fp8)
      launch_items<D, true, false>(a, ni, threads, grid, (int)nkv, stream);
    else if (vec)
      launch_items<D, false, true>(a, ni, threads, grid, (int)nkv, stream);
    else
      launch_items<D, false, false>(a, ni, threads, grid, (int)nkv, stream);
  };
  if (head_dim == 128)
    go(std::integral_constant<int, 128>());
  else
    go(std::integral_constant<int, 64>());
  return hipGetLastError();
}

hipError_t launch_page_values(const PageValuesArgs& a, hipStream_t stream) {
  const int64_t n = ((int64_t)a.pages * a.H << a.shift) * a.D / 16;
  if (n == 0) return hipSuccess;
  const int64_t blocks = (n + 255) / 256;
  LaunchTimer timer(kKidPageValues, stream);
  hipLaunchKernelGGL(page_values_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 2), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace avattn
