// What the few-row forwards share (attn_few.hip, attn_paged.hip): a block's rows
// and windows, and the join of the waves' parts of a workgroup.
#pragma once

#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

namespace {

constexpr int kWaves = 4, kTile = 32;

__device__ __forceinline__ float part_weight(float m, float top) {
  return m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
}

// A row's last steps: 1 / sum and the lse (see row_state in attn_fwd_kernel.h).
__device__ __forceinline__ void finish_row(float m, float l, float& inv, float& lse) {
  const float nan = __builtin_nanf("");
  inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : nan);
  lse = l > 0.f ? fmaf(m, kLn2, logf(l)) : (l == 0.f ? kNegInf : nan);
}

// Where row r of a unit's block lives: query i of head h.
struct RowPlace {
  int i, h;
};
__device__ __forceinline__ RowPlace row_place(const FewArgs& a, int hk, int r) {
  const int group = a.Hq / a.Hkv;
  return {r / group, hk * group + r % group};
}

// Union of the windows of a block's rows (lane l: row l % 32) and what every
// row's window covers.
struct BlockWindows {
  int lo, hi;          // this lane's row
  int glo, ghi;        // union (glo == ghi: no key)
  int all_lo, all_hi;  // intersection over the block's rows
};
__device__ __forceinline__ BlockWindows block_windows(int row_lo, int row_hi, bool valid) {
  BlockWindows w{row_lo, row_hi, 0, 0, 0, 0};
  const bool any = valid && w.lo < w.hi;
  int lo = any ? w.lo : 0x7fffffff, hi = any ? w.hi : 0;
  int al = valid ? w.lo : 0, ah = valid ? w.hi : 0x7fffffff;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off));
    hi = max(hi, __shfl_xor(hi, off));
    al = max(al, __shfl_xor(al, off));
    ah = min(ah, __shfl_xor(ah, off));
  }
  w.glo = __builtin_amdgcn_readfirstlane(min(lo, hi));
  w.ghi = __builtin_amdgcn_readfirstlane(hi);
  w.all_lo = __builtin_amdgcn_readfirstlane(al);
  w.all_hi = __builtin_amdgcn_readfirstlane(ah);
  return w;
}

__device__ __forceinline__ BlockWindows block_windows(const FewArgs& a, int b, int i, bool valid) {
  int lo = 0, hi = a.Lk;
  if (a.wlo != nullptr && valid) {
    lo = min(max(a.wlo[b * a.wsb + i], 0), a.Lk);
    hi = min(max(a.whi[b * a.wsb + i], lo), a.Lk);
  }
  return block_windows(lo, hi, valid);
}

// The bias of this lane's row (its clamped window in w; all of the wave).
struct RowBias {
  BiasRef at;
  float slope, slope2;
  uint32_t distance;
  __device__ __forceinline__ void init(const FewArgs& a, const BlockWindows& w, int b, const RowPlace& rp) {
    at = {0, 0}, slope = slope2 = 0.f, distance = 0;
    if (!(a.score.mode & kScoreDistance)) return;
    slope = a.score.slopes != nullptr ? a.score.slopes[rp.h] : 0.f;
    slope2 = slope * kLog2e;
    int lo = w.lo, hi = w.hi, hull_lo, hull_hi;
    const int p = rp.i + a.score.query_offset(b);
    rows_hull(a.score.slopes != nullptr && a.mask != nullptr ? a.mask + b * a.msb : nullptr, a.Lk, slope, p, lo, hi,
              hull_lo, hull_hi);
    within_hull(hull_lo, hull_hi, lo, hi);
    measure(p, lo, hi);
  }
  // The row at position p, its keys [lo, hi); slope is set.
  __device__ __forceinline__ void measure(int p, int lo, int hi) {
    at = bias_ref(p, lo, hi, slope < 0.f);
    distance = bias_distance(p, at);
  }
};

// A row's logsumexp from that of its computed scores, to both arrays.
__device__ __forceinline__ void store_lse(const FewArgs& a, int b, const RowPlace& p, float lse, uint32_t distance) {
  const int64_t at = ((int64_t)b * a.Hq + p.h) * a.Lq + p.i;
  a.lse[at] = a.score.slopes != nullptr ? lse_of_scores(lse, a.score.slopes[p.h], distance) : lse;
  if (a.row_lse != nullptr) a.row_lse[at] = lse;
}

// Changes one raw score (uniform mode); kd: the row's pos minus the key.
__device__ __forceinline__ float changed_score(const FewArgs& a, float s, float kd, float ref, float slope2) {
  float z;
  if (a.score.mode & kScoreCap)
    z = fmaf(-2.f * a.score.cap2, cap_complement(s, a.score.cap_arg), a.score.cap2);
  else
    z = s * a.scale_log2;
  return fmaf(-slope2, fabsf(kd) - ref, z);
}

// What the waves of a workgroup leave of their rows, to be joined.
template <int D, int ROWS>
struct Join {
  static constexpr int kPitch = D + 4;
  float o[kWaves][ROWS * kPitch];
  float m[kWaves][ROWS], l[kWaves][ROWS];
  uint32_t distance[ROWS];  // bias_distance (wave 0 writes it)
};

// The waves' parts of the block's rows, in order: to the rows themselves, or to
// the workgroup's slot.  Every thread; the waves have written jn.
template <int D, class T, int ROWS>
__device__ __forceinline__ void join_waves(const FewArgs& a, const Join<D, ROWS>& jn, int unit, int split, int rows) {
  const int rb = unit % a.row_blocks, bhk = unit / a.row_blocks;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  constexpr int CPR = D / 8;  // threads per row, 8 channels each
  for (int u = threadIdx.x; u < rows * CPR; u += 64 * kWaves) {
    const int r = u / CPR, ch = 8 * (u % CPR);
    float top = kNegInf;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) top = fmaxf(top, jn.m[v][r]);
    float sum = 0.f, o[8] = {};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float wt = part_weight(jn.m[v][r], top);
      sum = fmaf(jn.l[v][r], wt, sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(jn.o[v][r * jn.kPitch + ch + e], wt, o[e]);
    }
    if (a.nsplit > 1) {
      float* part = a.part + ((int64_t)unit * a.nsplit + split) * few_slot_floats(a.block_rows, D);
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(part + r * D + ch + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
      if (ch == 0) {
        float* ml = part + a.block_rows * D + 3 * r;
        ml[0] = top, ml[1] = sum, ml[2] = __uint_as_float(jn.distance[r]);
      }
    } else {
      float inv, lse;
      finish_row(top, sum, inv, lse);
      const RowPlace p = row_place(a, hk, rb * ROWS + r);
      T* out = static_cast<T*>(a.o) + b * a.osb + p.h * a.osh + (int64_t)p.i * a.osl + ch;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= inv;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4*>(out) = u32x4{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                               pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])};
      } else {
        *reinterpret_cast<f32x4*>(out) = f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(out + 4) = f32x4{o[4], o[5], o[6], o[7]};
      }
      if (ch == 0) store_lse(a, b, p, lse, jn.distance[r]);
    }
  }
}

}  // namespace

}  // namespace avattn
