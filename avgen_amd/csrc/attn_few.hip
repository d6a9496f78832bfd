// Attention forward of few query rows per kv head against many keys (one token
// of every sequence, a handful of drafted ones), and of small calls, with or
// without changed scores: the general forward's 128- or 256-row workgroups
// would idle, and its operand copies read and write the whole cache first.
//
// HBM-bound: k and v are read once, in place, by as many workgroups as fill
// the chip.  The rows of one kv head, Lq queries of its group of heads, form
// blocks of up to 32; the keys that a block's windows reach are split over
// `nsplit` workgroups, and a workgroup's 32-key tiles over its 4 waves.  A wave
// stages its own tiles (direct global->LDS loads, one tile ahead, no barrier),
// keeps its own running maximum, sum and output, and the waves are joined
// through LDS at the end, the workgroups by few_combine_kernel.  The products
// are those of the general forward (S^T = K Q^T, O^T += V^T P^T on 32x32x16
// MFMAs, P in registers); with fewer than 32 rows the matrix pipe works on
// empty columns, for which it has time: a tile's 16 KB take longer to arrive
// than its MFMAs to run.  One token against 205 MB of bf16 cache (D 128, 16
// kv heads): 36 us, 5.7 TB/s, and 4 us to combine.
#include "attn_few_parts.h"

namespace avattn {

namespace {

template <int D>
__global__ __launch_bounds__(256) void attn_few_kernel(FewArgs a) {
  constexpr int KS = D / 16, DT = D / 32, TE = kTile * D;
  struct Stage {
    bf16 k[TE];  // K rows: TileLayout<D>
    bf16 v[TE];  // V rows: TileLayout<D>
  };
  __shared__ __attribute__((aligned(16))) union Smem {
    Stage st[kWaves][2];
    Join<D, kTile> join;
  } sm;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int prow = perm23(l32);
  const int unit = blockIdx.x / a.nsplit, split = blockIdx.x % a.nsplit;
  const int rb = unit % a.row_blocks, bhk = unit / a.row_blocks;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  const int rows = min(a.Lq * (a.Hq / a.Hkv) - rb * kTile, kTile);  // of this block
  const bool valid = l32 < rows;
  const RowPlace rp = row_place(a, hk, rb * kTile + (valid ? l32 : 0));
  const BlockWindows w = block_windows(a, b, rp.i, valid);

  // This lane's row of Q: channels 16*ks + 8*hh + [0, 8).
  bf16x8 qf[KS];
  {
    const bf16* qp = static_cast<const bf16*>(a.q) + b * a.qsb + rp.h * a.qsh + (int64_t)rp.i * a.qsl + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (valid) x = *reinterpret_cast<const u32x4*>(qp + 16 * ks);
      qf[ks] = bits_to_bf16x8(x);
    }
  }
  RowBias rbias;
  rbias.init(a, w, b, rp);
  const int qpos = rbias.at.pos;
  const float slope2 = rbias.slope2, ref = (float)rbias.at.ref;

  // Tiles of this wave: the block's tiles, a range per workgroup, every
  // fourth of it per wave.
  const int tile0 = w.glo / kTile, ntile = w.ghi > w.glo ? (w.ghi + kTile - 1) / kTile - tile0 : 0;
  const int t0 = tile0 + (int)((int64_t)ntile * split / a.nsplit) + wave;
  const int t1 = tile0 + (int)((int64_t)ntile * (split + 1) / a.nsplit);

  const bf16* kp = static_cast<const bf16*>(a.k) + b * a.ksb + hk * a.ksh;
  const bf16* vp = static_cast<const bf16*>(a.v) + b * a.vsb + hk * a.vsh;
  TileStager<kTile, D, 1> kst, vst;
  kst.init(a.ksl, 0, lane);
  vst.init(a.vsl, 0, lane);
  // Rows past the last key read as zeros (or again, for strides below D).
  auto rsrc = [&](const bf16* base, int64_t sl, int t) {
    const int last = min(a.Lk - 1 - t * kTile, kTile - 1);
    return make_rsrc(base + (int64_t)t * kTile * sl, (uint32_t)((last * sl + D) * 2));
  };
  auto stage = [&](int t, Stage& sg) {
    kst.stage(sg.k, rsrc(kp, a.ksl, t), 0u);
    vst.stage(sg.v, rsrc(vp, a.vsl, t), 0u);
  };
  // Whether key l32 of tile t is one that a row of the block may attend.
  auto key_live = [&](int t) {
    const int key = t * kTile + l32;
    bool ok = key >= w.glo && key < w.ghi;
    if (a.mask != nullptr && ok) ok = a.mask[b * a.msb + key] != 0;
    return (int)ok;
  };

  float m = kNegInf, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();

  retire_prologue_loads();
  int live = 0;
  if (t0 < t1) {
    live = key_live(t0);
    stage(t0, sm.st[wave][0]);
  }
  for (int t = t0, buf = 0; t < t1; t += kWaves, buf ^= 1) {
    Stage& sg = sm.st[wave][buf];
    // Everything in flight belongs to this tile: its rows and its key mask.
    wait_vmem_n<0>();
    const uint32_t keys = (uint32_t)__builtin_amdgcn_ballot_w64(opaque(live) != 0);
    if (t + kWaves < t1) {
      // The other stage's reads have returned before it is filled again.
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      live = key_live(t + kWaves);
      stage(t + kWaves, sm.st[wave][buf ^ 1]);
    }
    if (keys != 0xffffffffu) {
      // What a key outside the mask and every window holds must not reach the
      // rows through 0 * NaN.
#pragma unroll
      for (int i = 0; i < TE / 8 / 64; ++i) {
        const int c = i * 64 + lane, row = c / (D / 8);
        if (!(keys >> row & 1)) *reinterpret_cast<u32x4*>(sg.v + TileLayout<D>::off(row, 8 * (c % (D / 8)))) = u32x4{};
      }
    }
    // Register 8*k2 + e of lane l: key 16*k2 + 8*hh + e of the tile, row l32.
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma32(row_operand<D>(sg.k, prow, 16 * ks + 8 * hh), qf[ks], s);
    const float kd = (float)(qpos - (t * kTile + 8 * hh));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = changed_score(a, s[r], kd - (float)(16 * (r >> 3) + (r & 7)), ref, slope2);
    if (keys != 0xffffffffu || t * kTile < w.all_lo || t * kTile + kTile > w.all_hi) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 16 * (r >> 3) + 8 * hh + (r & 7), key = t * kTile + j;
        if (!(keys >> j & 1) || key < w.lo || key >= w.hi) s[r] = kNegInf;
      }
    }
    float mx = kNegInf;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = halves_max(mx);
    // The reference maximum moves only for a score 2^8 above it (as in the
    // general forward); both lanes of a row agree.
    if (mx > m + 8.f || (m == kNegInf && mx > m)) {
      const float alpha = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - mx);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] *= alpha;
      m = mx;
    }
    const float mc = m == kNegInf ? 0.f : m;
    bf16x8 pf[2];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      u32x4 u;
#pragma unroll
      for (int e2 = 0; e2 < 4; ++e2) {
        const float p0 = __builtin_amdgcn_exp2f(s[8 * k2 + 2 * e2] - mc);
        const float p1 = __builtin_amdgcn_exp2f(s[8 * k2 + 2 * e2 + 1] - mc);
        l += p0 + p1;
        u[e2] = pack_bf16x2(p0, p1);  // the PV operand, rounded as in the general forward
      }
      pf[k2] = bits_to_bf16x8(u);
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x4 lo = lds_read_tr16(sg.v + tr_read_off<D>(lane, dt, 0) + 16 * k2 * D);
        const bf16x4 hi = lds_read_tr16(sg.v + tr_read_off<D>(lane, dt, 1) + 16 * k2 * D);
        acc[dt] = mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[k2], acc[dt]);
      }
  }

  // Join the waves: each leaves its rows' maxima, sums and outputs.
  l = halves_sum(l);
  __syncthreads();  // every wave is done with its stages
  auto& jn = sm.join;
  if (hh == 0) {
    jn.m[wave][l32] = m, jn.l[wave][l32] = l;
    if (wave == 0) jn.distance[l32] = rbias.distance;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(&jn.o[wave][l32 * jn.kPitch + 32 * dt + 8 * g + 4 * hh]) =
          f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
  __syncthreads();
  join_waves<D, bf16>(a, jn, unit, split, rows);
}

// float32, RB rows at a time on the vector ALUs: 268 MB of cache in 41 us with
// one row per kv head, 6.5 TB/s (part of it from the last-level cache), 52 us
// with 4, and 4 us to combine; every 4 more rows read K and V again, about 38
// us.  (The fp32 matrix instructions, which this kernel does not use, would
// multiply 32 rows whatever their number: 4.3 GFLOP, 28 us beside these loads.)
// Scores: lane l owns key l % 32 of the wave's tile and half of the channels, K
// from LDS (staged as above, rows of 256 bytes), q by broadcast reads.  P V: a
// lane owns D / 64 channels, V's rows come straight from memory a tile ahead
// (whole rows per load), p_j by readlane.
template <int D, int RB>
__global__ __launch_bounds__(256) void attn_few_f32_kernel(FewArgs a) {
  constexpr int HD = D / 2, CL = D / 64, NS = D / 64;  // channels per lane in P V; 64-channel K sub-tiles
  using vrow = std::conditional_t<CL == 2, f32x2, float>;
  __shared__ __attribute__((aligned(16))) union Smem {
    bf16 k[kWaves][2][NS][kTile * 128];  // 64 floats per row: TileLayout<128>
    Join<D, RB> join;
  } sm;
  __shared__ __attribute__((aligned(16))) float sq[RB][D];
  __shared__ float sneg[RB][2];  // the rows' slopes < 0, negated, and BiasRef::ref

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int unit = blockIdx.x / a.nsplit, split = blockIdx.x % a.nsplit;
  const int rb = unit % a.row_blocks, bhk = unit / a.row_blocks;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  const int rows = min(a.Lq * (a.Hq / a.Hkv) - rb * RB, RB);
  const bool valid = l32 < rows;
  const RowPlace rp = row_place(a, hk, rb * RB + (valid ? l32 : 0));
  const BlockWindows w = block_windows(a, b, rp.i, valid);
  // Row r's values are lane r's.
  RowBias rbias;
  rbias.init(a, w, b, rp);
  const int qpos = rbias.at.pos;
  const float slope2 = fmaxf(rbias.slope2, 0.f);
  // A slope < 0: its bias is added in a step of its own (with a reference to
  // subtract in the other slopes' code 4 rows took 59 us in place of 55).
  if (wave == 0 && lane < RB) sneg[lane][0] = fmaxf(-rbias.slope2, 0.f), sneg[lane][1] = (float)rbias.at.ref;
  const bool farthest = __builtin_amdgcn_ballot_w64(rbias.slope2 < 0.f) != 0;
  for (int u = tid; u < RB * (D / 4); u += 256) {
    const int r = u / (D / 4), c = 4 * (u % (D / 4));
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const RowPlace p = row_place(a, hk, rb * RB + r);
      x = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + b * a.qsb + p.h * a.qsh +
                                          (int64_t)p.i * a.qsl + c);
    }
    *reinterpret_cast<f32x4*>(&sq[r][c]) = x;
  }
  __syncthreads();

  const int tile0 = w.glo / kTile, ntile = w.ghi > w.glo ? (w.ghi + kTile - 1) / kTile - tile0 : 0;
  const int t0 = tile0 + (int)((int64_t)ntile * split / a.nsplit) + wave;
  const int t1 = tile0 + (int)((int64_t)ntile * (split + 1) / a.nsplit);
  const float* kp = static_cast<const float*>(a.k) + b * a.ksb + hk * a.ksh;
  const float* vp = static_cast<const float*>(a.v) + b * a.vsb + hk * a.vsh + CL * lane;
  TileStager<kTile, 128, 1> kst;  // in 2-byte units
  kst.init(2 * a.ksl, 0, lane);
  vrow vn[kTile];
  auto stage = [&](int t, int buf) {
    const int last = min(a.Lk - 1 - t * kTile, kTile - 1);
    const float* base = kp + (int64_t)t * kTile * a.ksl;
#pragma unroll
    for (int h = 0; h < NS; ++h)
      kst.stage(sm.k[wave][buf][h], make_rsrc(base + 64 * h, (uint32_t)((last * a.ksl + 64) * 4)), 0u);
#pragma unroll
    for (int j = 0; j < kTile; ++j)  // rows past the end read the last one again: their p is 0
      vn[j] = *reinterpret_cast<const vrow*>(vp + (int64_t)(t * kTile + min(j, last)) * a.vsl);
  };
  auto key_live = [&](int t) {
    const int key = t * kTile + l32;
    bool ok = key >= w.glo && key < w.ghi;
    if (a.mask != nullptr && ok) ok = a.mask[b * a.msb + key] != 0;
    return (int)ok;
  };

  float m[RB], l[RB];
  float acc[RB][CL];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = kNegInf, l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < CL; ++e) acc[r][e] = 0.f;
  }
  retire_prologue_loads();
  int live = 0;
  if (t0 < t1) {
    live = key_live(t0);
    stage(t0, 0);
  }
  for (int t = t0, buf = 0; t < t1; t += kWaves, buf ^= 1) {
    wait_vmem_n<0>();  // this tile's K, V and key mask
    const uint32_t keys = (uint32_t)__builtin_amdgcn_ballot_w64(opaque(live) != 0);
    vrow v[kTile];
#pragma unroll
    for (int j = 0; j < kTile; ++j) v[j] = vn[j];
    if (t + kWaves < t1) {
      // The other stage's reads have returned before it is filled again.
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      live = key_live(t + kWaves);
      stage(t + kWaves, buf ^ 1);
    }
    if (keys != 0xffffffffu) {
      // (see attn_few_kernel)
#pragma unroll
      for (int j = 0; j < kTile; ++j)
        if (!(keys >> j & 1)) v[j] = vrow{};
    }
    float s[RB] = {};
    const bf16* kr = sm.k[wave][buf][NS == 2 ? hh : 0];
#pragma unroll
    for (int c = 0; c < HD / 4; ++c) {
      const int chunk = NS == 2 ? c : hh * HD / 4 + c;
      const f32x4 k4 = *reinterpret_cast<const f32x4*>(kr + TileLayout<128>::off(l32, 8 * chunk));
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const f32x4 q4 = *reinterpret_cast<const f32x4*>(&sq[r][hh * HD + 4 * c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r] = fmaf(k4[e], q4[e], s[r]);
      }
    }
    const int key = t * kTile + l32;
    const bool live_key = keys >> l32 & 1;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int lo = __builtin_amdgcn_readlane(w.lo, r), hi = __builtin_amdgcn_readlane(w.hi, r);
      const int pos = __builtin_amdgcn_readlane(qpos, r);
      const float sl = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(slope2), r));
      float f;
      const float d = fabsf((float)(pos - key));
      float z = changed_score_exact(a.score, halves_sum(s[r]), a.scale_log2, d, sl, f);
      if (farthest) {
        __asm__ volatile("; a negative slope");
        z = fmaf(sneg[r][0], d - sneg[r][1], z);
      }
      if (!live_key || key < lo || key >= hi) z = kNegInf;
      if (__builtin_amdgcn_ballot_w64(z > m[r] + 8.f) != 0) {  // rare after the first tiles
        float mx = z;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        const float alpha = m[r] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[r] - mx);
        l[r] *= alpha;
#pragma unroll
        for (int e = 0; e < CL; ++e) acc[r][e] *= alpha;
        m[r] = mx;
      }
      const float p = __builtin_amdgcn_exp2f(z - (m[r] == kNegInf ? 0.f : m[r]));
      l[r] += p;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j));
        if constexpr (CL == 2) {
          acc[r][0] = fmaf(pj, v[j][0], acc[r][0]);
          acc[r][1] = fmaf(pj, v[j][1], acc[r][1]);
        } else {
          acc[r][0] = fmaf(pj, v[j], acc[r][0]);
        }
      }
    }
  }

  __syncthreads();  // every wave is done with its stages
  auto& jn = sm.join;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    float sum = l[r];  // both halves hold the same keys' shares
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) jn.m[wave][r] = m[r], jn.l[wave][r] = sum;
    if (wave == 0 && lane == r) jn.distance[r] = rbias.distance;
#pragma unroll
    for (int e = 0; e < CL; ++e) jn.o[wave][r * jn.kPitch + CL * lane + e] = acc[r][e];
  }
  __syncthreads();
  join_waves<D, float>(a, jn, unit, split, rows);
}

// A row from its joined parts.
template <int D, bool F32>
__device__ __forceinline__ void write_joined(const FewArgs& a, int unit, int r, float top, float sum,
                                             uint32_t distance, const f32x4& o, int ch) {
  const int rb = unit % a.row_blocks, bhk = unit / a.row_blocks;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  float inv, lse;
  finish_row(top, sum, inv, lse);
  const RowPlace rp = row_place(a, hk, rb * a.block_rows + r);
  const int64_t at = b * a.osb + rp.h * a.osh + (int64_t)rp.i * a.osl + ch;
  if constexpr (F32)
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.o) + at) = f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  else
    *reinterpret_cast<u32x2*>(static_cast<bf16*>(a.o) + at) =
        u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  if (ch == 0) store_lse(a, b, rp, lse, distance);
}

// The parts of one row, in order: a workgroup of 256 threads takes one row;
// D / 4 threads of four channels each per part, the parts dealt out over the
// thread groups, joined through LDS in a fixed order.
template <int D, bool F32>
__global__ __launch_bounds__(256) void few_combine_kernel(FewArgs a) {
  constexpr int TP = D / 4, G = 256 / TP;
  __shared__ float so[G][D], sl[G], st[4];
  const int unit = blockIdx.x / a.block_rows, r = blockIdx.x % a.block_rows;
  // (With one block of rows block_rows is their number, else a full block's.)
  if (unit % a.row_blocks * a.block_rows + r >= a.Lq * (a.Hq / a.Hkv)) return;  // the whole workgroup
  const int64_t slot = few_slot_floats(a.block_rows, D);
  const float* part = a.part + (int64_t)unit * a.nsplit * slot;
  const float* ml = part + (int64_t)a.block_rows * D + 3 * r;
  float top = kNegInf;
  for (int p = threadIdx.x; p < a.nsplit; p += 256) top = fmaxf(top, ml[p * slot]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if ((threadIdx.x & 63) == 0) st[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]));
  const int g = threadIdx.x / TP, ch = 4 * (threadIdx.x % TP);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int p = g; p < a.nsplit; p += G) {
    const float wt = part_weight(ml[p * slot], top);
    const f32x4 x = *reinterpret_cast<const f32x4*>(part + p * slot + (int64_t)r * D + ch);
    sum = fmaf(ml[p * slot + 1], wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], wt, o[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) so[g][ch + e] = o[e];
  if (ch == 0) sl[g] = sum;
  __syncthreads();
  if (g > 0) return;
#pragma unroll
  for (int i = 1; i < G; ++i) {
    sum += sl[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += so[i][ch + e];
  }
  write_joined<D, F32>(a, unit, r, top, sum, __float_as_uint(ml[2]), o, ch);
}

// The same for up to kFewParts parts of many rows: D / 4 threads join a row
// by themselves, in order.
constexpr int kFewParts = 4;
template <int D, bool F32>
__global__ __launch_bounds__(256) void few_combine_rows_kernel(FewArgs a) {
  constexpr int TP = D / 4;
  const int64_t u = (int64_t)blockIdx.x * (256 / TP) + threadIdx.x / TP;
  const int ch = 4 * (threadIdx.x % TP);
  const int64_t unit = u / a.block_rows;
  const int r = (int)(u - unit * a.block_rows);
  if (unit >= (int64_t)a.B * a.Hkv * a.row_blocks ||
      (int)(unit % a.row_blocks) * a.block_rows + r >= a.Lq * (a.Hq / a.Hkv))
    return;
  const int64_t slot = few_slot_floats(a.block_rows, D);
  const float* part = a.part + unit * a.nsplit * slot;
  const float* ml = part + (int64_t)a.block_rows * D + 3 * r;
  f32x4 x[kFewParts];
  float m[kFewParts], l[kFewParts];
#pragma unroll
  for (int p = 0; p < kFewParts; ++p) {
    const int64_t at = min(p, a.nsplit - 1) * slot;  // (a part again, left out below)
    x[p] = *reinterpret_cast<const f32x4*>(part + at + (int64_t)r * D + ch);
    m[p] = ml[at];
    l[p] = ml[at + 1];
  }
  float top = m[0];
#pragma unroll
  for (int p = 1; p < kFewParts; ++p) top = fmaxf(top, m[p]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll
  for (int p = 0; p < kFewParts; ++p) {
    if (p >= a.nsplit) break;
    const float wt = part_weight(m[p], top);
    sum = fmaf(l[p], wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[p][e], wt, o[e]);
  }
  write_joined<D, F32>(a, (int)unit, r, top, sum, __float_as_uint(ml[2]), o, ch);
}

template <int D, bool F32>
void launch_combine(const FewArgs& a, unsigned units, hipStream_t stream) {
  const unsigned rows = units * (unsigned)a.block_rows;
  if (a.nsplit <= kFewParts)
    hipLaunchKernelGGL((few_combine_rows_kernel<D, F32>), dim3((rows + 1024 / D - 1) / (1024 / D)), dim3(256), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((few_combine_kernel<D, F32>), dim3(rows), dim3(256), 0, stream, a);
}

template <int D>
void launch_few_f32(const FewArgs& a, dim3 grid, hipStream_t stream) {
  const int rows = a.Lq * (a.Hq / a.Hkv);
  if (rows == 1)
    hipLaunchKernelGGL((attn_few_f32_kernel<D, 1>), grid, dim3(256), 0, stream, a);
  else if (rows == 2)
    hipLaunchKernelGGL((attn_few_f32_kernel<D, 2>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attn_few_f32_kernel<D, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

FewPlan few_plan(int B, int Hq, int Hkv, int Lq, int Lk, int D, bool f32) {
  FewPlan p{};
  const int64_t rows = (int64_t)Lq * (Hq / Hkv);
  if (Lk < 1) return p;
  // Rows of a block: up to a tile's 32; float32 up to 4 (those of 8 spill).
  const int most_rows = f32 ? 4 : kTile;
  p.block_rows = (int)(rows < most_rows ? rows : most_rows);
  const int64_t units = (int64_t)B * Hkv * ((rows + most_rows - 1) / most_rows);
  // Workgroups the chip holds at once: one per CU at D 128 (LDS), two at 64.
  const int64_t slots = D == 128 ? 256 : 512;
  // How many query rows are few.  Few queries: a block's time grows with the
  // rows of its kv head, the general forward's with the heads.  8 sequences of
  // 4,096 keys, 8 kv heads of D 128, capped scores, this path against the
  // general one (at one more query): bf16, 32 queries 51 / 122 us in groups of
  // two heads, 83 / 171 of 4, 213 / 533 of 16, and 64 queries of single heads
  // 51 / 93; float32, 16 queries 171 / 178 us of single heads, 523 / 648 in
  // groups of 4, 1,035 / 1,242 of 8.
  const bool few_queries = f32 ? Lq <= kFewQueriesF32 : Lq <= kFewQueries || rows <= kFewRows;
  // Small calls, whose blocks the chip holds at once (of long keys, a part of
  // it): the general forward's workgroups are fewer and longer, and its copies
  // a launch.  D 128: (1,4,128) 8 / 13 us, (1,4,1024) 18 / 31, (1,4,2048) 32 /
  // 41, (1,8 on 2 heads,2048) 512 blocks 60 / 72 (not taken), (2,8,1024) 512 36
  // / 34; (1,8 on 2 heads,128) x 8,192 keys 24 / 55, (1,32 on 8 heads,256) x
  // 4,096 256 blocks 56 / 52.  float32: (1,4,256) 256 blocks 16 / 32, (1,4,512)
  // 512 46 / 35, (1,8 on 2 heads,64) x 2,048 44 / 60, twice the heads 73 / 63.
  const bool few_blocks = f32 ? units <= (Lk <= 512 ? slots : slots / 2) : units <= (Lk <= 2048 ? slots : slots / 4);
  if (!few_queries && !few_blocks) return FewPlan{};
  p.row_blocks = (int)((rows + most_rows - 1) / most_rows);
  // Parts of a block's keys, each with a tile for every wave: rounds of
  // workgroups at the measured times of a wave's tile (with one and with two
  // workgroups on a CU) against the combination's launch and traffic.
  const int tiles = (Lk + kTile - 1) / kTile, most = (tiles + kWaves - 1) / kWaves;
  const float one = f32 ? (D == 128 ? 4.3f : 2.7f) : (D == 128 ? 1.55f : 1.4f);
  const float two = f32 ? (D == 128 ? 4.3f : 4.4f) : (D == 128 ? 1.55f : 1.75f);
  float best = 3e38f;
  for (int n = 1; n <= most && n <= 256; ++n) {
    const int64_t wgs = units * n;
    const int turns = (tiles + kWaves * n - 1) / (kWaves * n);
    const float cost = (float)((wgs + slots - 1) / slots) * (turns * (wgs <= 256 ? one : two) + 4.5f) +
                       (n > 1 ? 4.f + (float)wgs * p.block_rows * D * 1.1e-6f : 0.f);
    if (cost < best) {
      best = cost;
      p.nsplit = n;
    }
    if (wgs >= slots) break;
  }
  // Grids of 256 threads each, within 2^32: past that the general path, whose
  // grid is the smaller one.
  constexpr int64_t kMaxGrid = (1 << 24) - 1;
  if (units * p.nsplit > kMaxGrid || units * p.block_rows > kMaxGrid) return FewPlan{};
  p.bytes = p.nsplit > 1 ? (size_t)units * p.nsplit * few_slot_floats(p.block_rows, D) * sizeof(float) : 0;
  return p;
}

void launch_few_combine(const FewArgs& a, int D, hipStream_t stream) {
  LaunchTimer timer(kKidMerge, stream);
  const unsigned units = (unsigned)(a.B * a.Hkv * a.row_blocks);
  if (D == 128)
    launch_combine<128, false>(a, units, stream);
  else
    launch_combine<64, false>(a, units, stream);
}

hipError_t launch_few(const FewArgs& args, const FewPlan& p, int D, bool f32, hipStream_t stream) {
  FewArgs a = args;
  a.nsplit = p.nsplit;
  a.row_blocks = p.row_blocks;
  a.block_rows = p.block_rows;
  const unsigned units = (unsigned)(a.B * a.Hkv * p.row_blocks);
  {
    LaunchTimer timer(kKidFwdFew, stream);
    const dim3 grid(units * p.nsplit);
    if (f32 && D == 128)
      launch_few_f32<128>(a, grid, stream);
    else if (f32)
      launch_few_f32<64>(a, grid, stream);
    else if (D == 128)
      hipLaunchKernelGGL(attn_few_kernel<128>, grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL(attn_few_kernel<64>, grid, dim3(256), 0, stream, a);
  }
  if (p.nsplit > 1 && f32) {
    LaunchTimer timer(kKidMerge, stream);
    if (D == 128)
      launch_combine<128, true>(a, units, stream);
    else
      launch_combine<64, true>(a, units, stream);
  } else if (p.nsplit > 1) {
    launch_few_combine(a, D, stream);
  }
  return hipGetLastError();
}

}  // namespace avattn
