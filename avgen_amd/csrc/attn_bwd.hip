// Attention backward for gfx950, recomputing the probabilities from (q, k,
// lse) instead of storing them.  No atomics (bitwise reproducible):
//   1. preprocess: per query row, lse2 = lse * log2(e) and
//      ndelta = -rowsum(dout * out) (the `D` term of dS = P * (dP - D)), in
//      arrays padded to whole 64-row tiles (+inf / 0 past the end so padded
//      rows get P = 0); plus the padded operand copies (prep.hip):
//      head_dim-major k (row-major k, v for 3''), and row-major q where it is
//      rotated first;
//   2. dK/dV: one workgroup per 128 keys (32 per wave, kept in registers as
//      MFMA operands); loops over 64-row query tiles of every query head
//      that reads this KV head; with staged dS it also stores dS (bf16) to
//      the workspace;
//   3. dQ, either
//      3'. from the staged dS: dQ = scale * dS K, one product, one workgroup
//          per 256 query rows streaming the dS once (bwd_dq_ds_kernel), or
//      3''. recomputing S and dP: one workgroup per 256 query rows (32 per
//          wave), 32-key tiles (bwd_dq_kernel).
// Every MFMA operand read from LDS is one 16-byte chunk of a tile row or two
// 8-byte transposed reads (ds_read_b64_tr_b16) of a row-major tile: the
// products contracting over the sequence read their operands across the
// rows, and the rows feeding the first product are read in perm23 order so
// that their C layout lines up with those eight consecutive rows.
// With out/lse the merged result over all KV chunks, the outputs are one
// chunk's contributions, which is how the ring backward calls the op
// (torch/.../_context_parallel/_attention.py:567-575).
#include "attn_bwd_dkdv.h"

namespace avattn {

// dk/dv of the split key blocks: one thread per (block, role, key, 4
// channels) adds the parts' fp32 sums in part order, then scales, rounds to
// bf16 and rotates dk back as the dK/dV kernel's own epilogue does.
template <int D>
__global__ __launch_bounds__(256) void dkv_reduce_kernel(BwdArgs a) {
  constexpr int BK = 128, CQ = D / 4;
  const int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (u >= (int64_t)a.nsplit * 2 * BK * CQ) return;
  const int c = (int)(u % CQ);
  const int r = (int)((u / CQ) % BK);
  const int role = (int)((u / (CQ * BK)) % 2);
  const int s = (int)(u / (CQ * BK * 2));
  const int nkt = (a.Lk + BK - 1) / BK;
  const int bid = nkt * a.nkv - a.nsplit + s;
  int kt = bid % nkt, pair = bid / nkt;
  if (a.score.mode != 0 && a.wlo != nullptr && a.nsplit < nkt * a.nkv) longest_first(bid, nkt, a.nkv, kt, pair);
  const int bhk = a.kv0 + pair;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  const int key = kt * BK + r;
  if (key >= a.Lk) return;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  const bool attended = a.mask == nullptr || a.mask[b * a.msb + key] != 0;
  for (int p = 0; attended && p < a.nparts; ++p)
    t += *reinterpret_cast<const f32x4*>(a.split_part + ((((int64_t)s * a.nparts + p) * 2 + role) * BK + r) * D + 4 * c);
  const float sc = role == 0 ? 1.f : a.scale;
  u32x2 w;
  w[0] = pack_bf16x2(t[0] * sc, t[1] * sc);
  w[1] = pack_bf16x2(t[2] * sc, t[3] * sc);
  if (role == 1 && a.cos_k != nullptr) {
    const int64_t ti = b * a.rksb + (int64_t)key * (D / 2) + 2 * c;  // pairs 2c, 2c + 1
    const f32x2 c2 = *reinterpret_cast<const f32x2*>(a.cos_k + ti);
    const f32x2 s2 = *reinterpret_cast<const f32x2*>(a.sin_k + ti);
    w = rotate4(w, c2[0], s2[0], c2[1], s2[1], true);
  }
  bf16* op = role == 0 ? a.dv + b * a.dvsb + hk * a.dvsh + (int64_t)key * a.dvsl
                       : a.dk + b * a.dksb + hk * a.dksh + (int64_t)key * a.dksl;
  *reinterpret_cast<u32x2*>(op + 4 * c) = w;
}

// ---------------------------------------------------------------------------
// 3. dQ
// ---------------------------------------------------------------------------
// One workgroup = 256 query rows of one (batch, head): 8 waves x 32 rows
// (lane % 32 owns query column q0w + lane % 32), 1 workgroup per CU, so each
// K/V tile is staged once for 256 rows.  For each 32-key tile (lane l supplies
// key row perm23(l % 32) to the first two products):
//   S^T  = K Q^T    A = K rows (LDS)          B = Q^T (registers)
//   dP^T = V dO^T   A = V rows (LDS)          B = dO^T (registers)
//   dS^T = P^T * (dP^T + ndelta[q])           (fp32, key bias masks P^T)
//   dQ^T += K^T dS^T   A = K^T (LDS, head_dim-major)  B = dS^T (C layout reused)
// Ping-pong: waves 0-3 (group A) and 4-7 (group B) share the SIMDs pairwise.
// Group A runs S/dP(t), dS(t), dQ(t) in iteration t; group B is one tile
// behind and runs dS(t-1), dQ(t-1), S/dP(t), carrying S^T/dP^T across the
// barrier.  So while one wave of a SIMD computes dS (VALU), the other issues
// MFMAs, and the per-tile barrier no longer lines both up on the same phase.
// Tiles come from the padded copies through four LDS stages: tile t+2 is
// loaded during iteration t (spread between MFMAs) and tile t-1 stays
// resident for group B.
template <int D>
__global__ __launch_bounds__(512, 1) void bwd_dq_kernel(BwdArgs a) {
  constexpr int NW = 8, BM = 32 * NW, BN = 32;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int TE = BN * D;
  // One LDS object per stage (see bwd_dkdv_kernel).
  struct Stage {
    bf16 k[TE];      // K rows: TileLayout<D>
    bf16 v[TE];      // V rows: TileLayout<D>
    bf16 kt[TE];     // K^T: D rows of BN keys, TileLayout<BN>
    float bias[64];  // key bias (this tile and the next)
    int flags[64];   // "all attended" flag of this tile (and the next 63)
  };
  __shared__ __attribute__((aligned(16))) Stage st0, st1, st2, st3;
  auto stage_ref = [&](auto bufc) __attribute__((always_inline)) -> Stage& {
    constexpr int buf = decltype(bufc)::value;
    return buf == 0 ? st0 : (buf == 1 ? st1 : (buf == 2 ? st2 : st3));
  };

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int prow = perm23(l32);

  const int nqt = (a.Lq + BM - 1) / BM;
  const int total = nqt * a.B * a.Hq;
  const int bid = xcd_remap(blockIdx.x, total);
  const int qt = bid % nqt;
  const int bh = bid / nqt;
  const int b = bh / a.Hq, h = bh % a.Hq;
  const int hk = h / (a.Hq / a.Hkv);

  const int qrow = qt * BM + wave * 32 + l32;
  const bool qvalid = qrow < a.Lq;
  const int64_t srow = (int64_t)bh * a.Lqp + qrow;
  const float lse2 = qvalid ? a.lse2[srow] : kPosInf;
  const float ndelta = qvalid ? a.ndelta[srow] : 0.f;

  bf16x8 qf[KS], df[KS];
  {
    const bf16* qp = a.q + b * a.qsb + h * a.qsh + (int64_t)qrow * a.qsl + 8 * hh;
    const bf16* dp = a.dout + b * a.dosb + h * a.dosh + (int64_t)qrow * a.dosl + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
      if (qvalid) {
        x = *reinterpret_cast<const u32x4*>(qp + 16 * ks);
        y = *reinterpret_cast<const u32x4*>(dp + 16 * ks);
        if (a.cos_q) {
          const int64_t t = b * a.rqsb + (int64_t)qrow * (D / 2) + 8 * ks + 4 * hh;
          x = rotate8(x, *reinterpret_cast<const f32x4*>(a.cos_q + t), *reinterpret_cast<const f32x4*>(a.sin_q + t),
                      false);
        }
      }
      qf[ks] = bits_to_bf16x8(x);
      df[ks] = bits_to_bf16x8(y);
    }
  }

  const int64_t bhk = (int64_t)(b * a.Hkv + hk);
  const uint32_t slice = (uint32_t)a.Lkp * D * 2;
  const u32x4 rk = make_rsrc(a.kr + bhk * a.Lkp * D, slice);
  const u32x4 rv = make_rsrc(a.vr + bhk * a.Lkp * D, slice);
  const u32x4 rkt = make_rsrc(a.kt + bhk * D * a.Lkp, slice);
  // Biases and flags: both arrays are padded by 64 entries, so the 64 read
  // from a tile start stay inside them.
  const u32x4 rb = make_rsrc(a.kbias + (int64_t)b * a.Lkp, (uint32_t)(a.Lkp + 64) * 4);
  const u32x4 rf = make_rsrc(a.kfull + (int64_t)b * (a.Lkp / 32), (uint32_t)(a.Lkp / 32 + 64) * 4);

  using RowStager = TileStager<BN, D, NW>;  // 32 rows of D channels (row stride D)
  using ColStager = TileStager<D, BN, NW>;  // D rows of 32 keys (row stride Lkp)
  RowStager rst;
  ColStager ktst;
  rst.init(D, wave, lane);
  ktst.init(a.Lkp, wave, lane);
  // Vector-memory loads one stage issues per wave: K, V, K^T, bias, flags.
  constexpr int kStageLoads = 2 * RowStager::kPer + ColStager::kPer + 2;
  auto stage_op = [&](int t, auto bufc, int i) __attribute__((always_inline)) {
    Stage& sg = stage_ref(bufc);
    const uint32_t k0 = (uint32_t)t * BN;
    if (i < RowStager::kPer)
      rst.stage_one(sg.k, rk, k0 * D * 2, i);
    else if (i < 2 * RowStager::kPer)
      rst.stage_one(sg.v, rv, k0 * D * 2, i - RowStager::kPer);
    else if (i < 2 * RowStager::kPer + ColStager::kPer)
      ktst.stage_one(sg.kt, rkt, k0 * 2, i - 2 * RowStager::kPer);
    else if (i == kStageLoads - 2)
      dma4(rb, lds_addr(sg.bias), lane * 4, k0 * 4);
    else
      dma4(rf, lds_addr(sg.flags), lane * 4, (uint32_t)t * 4);
  };

  // Per-lane LDS byte offsets inside a tile.  Each iteration passes them
  // through opaque() once (Off), so every read of that iteration adds its
  // stage's base as an instruction immediate instead of the compiler keeping
  // one hoisted copy of every offset per stage in registers.
  struct Off {
    int k[KS];  // K/V row perm23(l32), chunk 16*ks + 8*hh
    int t[2];   // K^T row l32, key chunk 16*k2 + 8*hh (+32*dt rows)
  };
  Off off0;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) off0.k[ks] = 2 * TileLayout<D>::off(prow, 16 * ks + 8 * hh);
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) off0.t[k2] = 2 * TileLayout<BN>::off(l32, 16 * k2 + 8 * hh);
  auto fresh = [&]() __attribute__((always_inline)) {
    Off o;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) o.k[ks] = opaque(off0.k[ks]);
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) o.t[k2] = opaque(off0.t[k2]);
    return o;
  };
  auto lds16 = [](const void* base, int byte_off) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(base) + byte_off);
  };

  f32x16 dq[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) dq[i] = zero16();

  const float c = a.scale_log2;
  const int nkt = (a.Lk + BN - 1) / BN;

  // S^T and dP^T of one tile (2*KS MFMAs, the two chains alternating); dP^T
  // starts at ndelta (one value per query column, i.e. per lane), so the MFMAs
  // deliver dP^T + ndelta directly.  Operand reads run two k-steps (four
  // MFMAs) ahead; `slot(j)` runs extra work after MFMA j; sched_barrier(0)
  // pins the order.
  auto sdp = [&](const Stage& sg, const Off& o, f32x16& s, f32x16& dp, auto&& slot) __attribute__((always_inline)) {
    auto krow = [&](int ks) __attribute__((always_inline)) { return lds16(sg.k, o.k[ks]); };
    auto vrow = [&](int ks) __attribute__((always_inline)) { return lds16(sg.v, o.k[ks]); };
    bf16x8 ka[2], va[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      ka[j] = krow(j);
      va[j] = vrow(j);
    }
    s = zero16();
    dp = splat16(ndelta);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mfma32(ka[ks & 1], qf[ks], s);
      if (ks + 2 < KS) ka[ks & 1] = krow(ks + 2);
      slot(2 * ks);
      __builtin_amdgcn_sched_barrier(0);
      dp = mfma32(va[ks & 1], df[ks], dp);
      if (ks + 2 < KS) va[ks & 1] = vrow(ks + 2);
      slot(2 * ks + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // dS^T of one tile (its S^T, dP^T and stage) as the bf16 B operands of dQ;
  // registers 8*k2 + e hold key 16*k2 + 8*hh + e.
  auto dsm = [&](const Stage& sg, f32x16& s, const f32x16& dp, bf16x8* dsb, auto&& slot) __attribute__((always_inline)) {
    if (!__builtin_amdgcn_readfirstlane(sg.flags[0])) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 bb = *reinterpret_cast<const f32x4*>(sg.bias + 16 * (g >> 1) + 8 * hh + 4 * (g & 1));
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * g + r] += bb[r];
      }
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      u32x4 u;
#pragma unroll
      for (int e2 = 0; e2 < 4; ++e2) {
        const int r = 8 * k2 + 2 * e2;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse2));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -lse2));
        u[e2] = pack_bf16x2(p0 * dp[r], p1 * dp[r + 1]);
        slot(4 * k2 + e2);
      }
      dsb[k2] = bits_to_bf16x8(u);
    }
  };
  // dQ^T += K^T dS^T (2*DT MFMAs).  The first four K^T operands are read
  // before dsm runs (their latency hides behind it), the rest four MFMAs
  // ahead.
  auto kt_op = [&](const Stage& sg, const Off& o, int j) __attribute__((always_inline)) {
    return lds16(sg.kt + (j % DT) * 32 * BN, o.t[j / DT]);
  };
  auto kt_read = [&](const Stage& sg, const Off& o, bf16x8* kta) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) kta[j] = kt_op(sg, o, j);
  };
  auto dqm = [&](const Stage& sg, const Off& o, bf16x8* kta, const bf16x8* dsb, auto&& slot) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j) {
      dq[j % DT] = mfma32(kta[j & 3], dsb[j / DT], dq[j % DT]);
      if (j + 4 < 2 * DT) kta[j & 3] = kt_op(sg, o, j + 4);
      slot(j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Where a tile's loads are issued: between the dQ MFMAs when they fit there
  // (measured ~1% faster than between the S/dP MFMAs), else between the S/dP
  // MFMAs (0); 2 would spread them over the dS VALU steps (measured slower).
  constexpr int kLoadsAt = kStageLoads <= 2 * DT ? 1 : 0;
  static_assert(kStageLoads <= 2 * KS && kStageLoads <= 8, "tile loads must fit the slots");
  auto no_slot = [](int) __attribute__((always_inline)) {};
  auto loads_in = [&](int t, auto nextc) __attribute__((always_inline)) {  // tile t's loads, one after each of the first MFMAs
    return [&, t, nextc](int j) __attribute__((always_inline)) {
      if (j < kStageLoads) stage_op(t, nextc, j);
    };
  };
  // Top of iteration t: tile t landed (only tile t+1's loads may still be in
  // flight) for every wave; the stage tile t-2 used is free for tile t+2.
  auto top = [&]() __attribute__((always_inline)) {
    wait_vmem_n<kStageLoads>();
    barrier_lds();
  };

  retire_prologue_loads();
  {
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
#pragma unroll
    for (int i = 0; i < kStageLoads; ++i) stage_op(0, B0(), i);
#pragma unroll
    for (int i = 0; i < kStageLoads; ++i) stage_op(min(1, nkt - 1), B1(), i);
  }

  f32x16 s, dp;
  bf16x8 kta[4], dsb[2];
  if (wave < NW / 2) {
    // Group A: S/dP(t), dS(t), dQ(t).
    auto body = [&](int t, auto bufc) __attribute__((always_inline)) {
      constexpr int buf = decltype(bufc)::value;
      using Next2 = std::integral_constant<int, (buf + 2) % 4>;
      top();
      const Stage& sg = stage_ref(bufc);
      const Off o = fresh();
      auto ld = loads_in(min(t + 2, nkt - 1), Next2());
      __builtin_amdgcn_s_setprio(2);
      if constexpr (kLoadsAt == 0) sdp(sg, o, s, dp, ld); else sdp(sg, o, s, dp, no_slot);
      kt_read(sg, o, kta);
      __builtin_amdgcn_s_setprio(0);
      if constexpr (kLoadsAt == 2) dsm(sg, s, dp, dsb, ld); else dsm(sg, s, dp, dsb, no_slot);
      __builtin_amdgcn_s_setprio(2);
      if constexpr (kLoadsAt == 1) dqm(sg, o, kta, dsb, ld); else dqm(sg, o, kta, dsb, no_slot);
    };
    for (int t = 0; t < nkt; t += 4) {
      body(t, std::integral_constant<int, 0>());
      if (t + 1 < nkt) body(t + 1, std::integral_constant<int, 1>());
      if (t + 2 < nkt) body(t + 2, std::integral_constant<int, 2>());
      if (t + 3 < nkt) body(t + 3, std::integral_constant<int, 3>());
    }
  } else {
    // Group B: dS(t-1), dQ(t-1), S/dP(t); S^T/dP^T of tile t are carried to
    // the next iteration.
    auto body = [&](int t, auto bufc) __attribute__((always_inline)) {
      constexpr int buf = decltype(bufc)::value;
      using Prev = std::integral_constant<int, (buf + 3) % 4>;
      using Next2 = std::integral_constant<int, (buf + 2) % 4>;
      top();
      const Stage& sp = stage_ref(Prev());
      const Off o = fresh();
      auto ld = loads_in(min(t + 2, nkt - 1), Next2());
      kt_read(sp, o, kta);
      __builtin_amdgcn_s_setprio(0);
      if constexpr (kLoadsAt == 2) dsm(sp, s, dp, dsb, ld); else dsm(sp, s, dp, dsb, no_slot);
      __builtin_amdgcn_s_setprio(2);
      if constexpr (kLoadsAt == 1) dqm(sp, o, kta, dsb, ld); else dqm(sp, o, kta, dsb, no_slot);
      if constexpr (kLoadsAt == 0) sdp(stage_ref(bufc), o, s, dp, ld); else sdp(stage_ref(bufc), o, s, dp, no_slot);
    };
    {
      // Iteration 0: only S/dP(0).
      using B2 = std::integral_constant<int, 2>;
      top();
      const Off o = fresh();
      if constexpr (kLoadsAt == 0) {
        sdp(stage_ref(std::integral_constant<int, 0>()), o, s, dp, loads_in(min(2, nkt - 1), B2()));
      } else {
        sdp(stage_ref(std::integral_constant<int, 0>()), o, s, dp, no_slot);
#pragma unroll
        for (int i = 0; i < kStageLoads; ++i) stage_op(min(2, nkt - 1), B2(), i);
      }
    }
    for (int t = 1; t < nkt; t += 4) {
      body(t, std::integral_constant<int, 1>());
      if (t + 1 < nkt) body(t + 1, std::integral_constant<int, 2>());
      if (t + 2 < nkt) body(t + 2, std::integral_constant<int, 3>());
      if (t + 3 < nkt) body(t + 3, std::integral_constant<int, 0>());
    }
    // Tail: dS and dQ of the last tile (its stage is not refilled).
    const int bl = (nkt - 1) % 4;
    const Stage& sl = bl == 0 ? st0 : (bl == 1 ? st1 : (bl == 2 ? st2 : st3));
    const Off o = fresh();
    kt_read(sl, o, kta);
    __builtin_amdgcn_s_setprio(0);
    dsm(sl, s, dp, dsb, no_slot);
    dqm(sl, o, kta, dsb, no_slot);
  }
  __builtin_amdgcn_s_setprio(0);
  wait_vmem();  // the last (re-staged) tile loads

  if (qvalid && a.dq_acc) {
    // fp32 accumulation: dq_acc += this chunk's dq (each element owned by
    // exactly one lane, so a plain load-add-store).
    float* op = a.dq_acc + b * a.dqsb + h * a.dqsh + (int64_t)qrow * a.dqsl;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4* p = reinterpret_cast<f32x4*>(op + dt * 32 + 8 * g + 4 * hh);
        f32x4 w = *p;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] += dq[dt][4 * g + r] * a.scale;
        *p = w;
      }
  } else if (qvalid) {
    bf16* op = a.dq + b * a.dqsb + h * a.dqsh + (int64_t)qrow * a.dqsl;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 w;
        w[0] = pack_bf16x2(dq[dt][4 * g] * a.scale, dq[dt][4 * g + 1] * a.scale);
        w[1] = pack_bf16x2(dq[dt][4 * g + 2] * a.scale, dq[dt][4 * g + 3] * a.scale);
        *reinterpret_cast<u32x2*>(op + dt * 32 + 8 * g + 4 * hh) = w;
      }
  }
}

// ---------------------------------------------------------------------------
// 3'. dQ from staged dS
// ---------------------------------------------------------------------------
// dQ^T[d, q] = scale * sum_key K^T[d, key] dS^T[key, q], a plain product
// (the S and dP recomputation of bwd_dq_kernel is replaced by reading the dS
// the dK/dV kernel stored).  One workgroup = 256 query rows of one (batch,
// head) of the pass: wave w owns query group 8*qb + w (32 rows, lane % 32 one
// row) and all D channels (DT accumulators).  64-key stages through three LDS
// buffers: K^T (D rows of 64 keys, TileLayout<64>, shared) and each wave's
// own 4 KB of dS, the stage's keys of its unit copied as stored
// ([k2][64 keys][16 rows]); the B operand (8 consecutive keys of one row per
// lane) comes from two transposed reads per 16-key step.  The kernel streams
// dS from HBM once; K^T comes from L2 (the query groups of one head run on
// one XCD).
// WIN: only the stages that meet the union of the workgroup's rows' key
// windows are staged, and a wave multiplies only those that meet its own
// 32 rows' windows (the dK/dV kernel wrote the dS of exactly those: a
// group's window union lies inside its 64-row tile's).
// NW: waves (32 rows each) per workgroup; 4 for short grids of changed scores
// (launch_dq_ds_d).  By their LDS two of those fit a CU at D 64 (72 KB each), one
// at D 128 (96 KB).  The bits are the same.
template <int D, int BK, int NSTG, bool WIN, bool CT, int NW = 8>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 1 : 2) void bwd_dq_ds_kernel(BwdArgs a) {
  static_assert(!CT || WIN, "the compact dS layout (BwdArgs::ds_tab) is for windows");
  constexpr int DT = D / 32;
  static_assert(BK == 32 || BK == 64, "stage of 32 or 64 keys");
  struct Stage {
    bf16 kt[D * BK];             // K^T: D rows of BK keys, TileLayout<BK>
    bf16 ds[NW][2 * BK * 16];    // per wave: [k2][BK keys][16 rows]
  };
  __shared__ __attribute__((aligned(16))) Stage st[NSTG];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;

  const int group = a.Hq / a.Hkv;
  const int nqg = a.Lqp / 32;
  const int nqb = (nqg + NW - 1) / NW;
  const int total = nqb * a.nkv * group;
  const int bid = xcd_remap_pairs(blockIdx.x, total, nqb * group, a.mask != nullptr);
  int qb = bid % nqb;
  int bq_rel = bid / nqb;                   // (b, hq) within the pass
  if constexpr (WIN) {
    // Changed scores (causal and prefix masks): the row blocks with the most
    // keys first, from whichever end the windows are wider (batch row 0 stands
    // for all: any order is right).  (2,20,2304,128) with a prefix of 512: 76 ->
    // 64 us.
    if (a.score.mode != 0) {
      longest_first(blockIdx.x, nqb, a.nkv * group, qb, bq_rel);
      const int n = min(NW * 32, a.Lq);
      if (a.whi[a.Lq - 1] - a.wlo[a.Lq - n] >= a.whi[n - 1] - a.wlo[0]) qb = nqb - 1 - qb;
    }
  }
  const int bq = a.kv0 * group + bq_rel;    // b*Hq + hq
  const int b = bq / a.Hq, h = bq % a.Hq;
  const int hk = h / group;
  const int qg = qb * NW + wave;
  const int qgl = min(qg, nqg - 1);  // groups past the end re-read the last one and write nothing
  const int qrow = qg * 32 + l32;
  const bool qvalid = qrow < a.Lq;
  const int nkt = (a.Lk + 127) / 128;
  int s0 = 0, s1 = a.Lkp / BK;  // stages of the workgroup
  int w0 = s0, w1 = s1;         // stages this wave multiplies
  if constexpr (!WIN) {
    s0 = load_const_i32(a.khull, 2 * (b * a.Hkv + hk)) * (64 / BK);
    s1 = load_const_i32(a.khull, 2 * (b * a.Hkv + hk) + 1) * (64 / BK);
  }
  if constexpr (WIN) {
    // Monotone windows: a row range's key union is [lo(first), hi(last)).
    const int* lo = a.wlo + b * a.wsb;
    const int* hi = a.whi + b * a.wsb;
    auto range = [&](int r0, int r1, int& st0, int& st1) {  // rows [r0, r1)
      r1 = min(r1, a.Lq);
      st0 = st1 = 0;
      if (r1 > r0) {
        const int l = min(max(lo[r0], 0), a.Lk);
        const int lol = min(max(lo[r1 - 1], 0), a.Lk);
        const int h = min(max(hi[r1 - 1], lol), a.Lk);
        if (h > l) {
          st0 = l / BK;
          st1 = (h + BK - 1) / BK;
        }
      }
    };
    range(qb * NW * 32, qb * NW * 32 + NW * 32, s0, s1);
    range(qg * 32, qg * 32 + 32, w0, w1);
    s0 = __builtin_amdgcn_readfirstlane(s0);
    s1 = __builtin_amdgcn_readfirstlane(s1);
    w0 = __builtin_amdgcn_readfirstlane(w0);
    w1 = __builtin_amdgcn_readfirstlane(w1);
  }

  const u32x4 rkt = make_rsrc(a.kt + (int64_t)(b * a.Hkv + hk) * D * a.Lkp, (uint32_t)a.Lkp * D * 2);
  // This wave's dS units: dense, every 128-key block of its group in order;
  // compact (WIN with a table), the blocks [kb_lo, kb_lo + nblk) of its
  // tile.  A stage is loaded by every wave (the counted waits need the same
  // loads everywhere); a stage outside this wave's blocks re-loads one of
  // them, or the head's first unit when the tile has none, and is not
  // multiplied (w0 .. w1 lies inside the tile's blocks).
  u32x4 rds;
  int ds_kb_lo = 0, ds_nblk = nkt;
  if (CT) {
    const int64_t e = ((int64_t)b * a.ds_tsb + (qgl >> 1)) * 4;
    const int kb_lo = __builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e));
    const int nblk = __builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e + 1));
    const int gbase = __builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e + 2));
    const bool ok = nblk > 0 && gbase >= 0 && (int64_t)gbase + 2 * nblk <= a.ds_units;
    const int64_t unit = (int64_t)bq_rel * a.ds_units + (ok ? gbase + (qgl & 1) * nblk : 0);
    ds_kb_lo = ok ? kb_lo : 0;
    ds_nblk = ok ? nblk : 1;
    rds = make_rsrc(reinterpret_cast<const char*>(a.ds) + unit * 8192, (uint32_t)ds_nblk * 8192);
  } else {
    rds = make_rsrc(reinterpret_cast<const char*>(a.ds) + ((int64_t)bq_rel * nqg + qgl) * nkt * 8192,
                    (uint32_t)nkt * 8192);
  }
  using KtStager = TileStager<D, BK, NW>;
  KtStager ktst;
  ktst.init(a.Lkp, wave, lane);
  constexpr int kPerK2 = BK / 32;            // 1 KB loads per k2 half and stage
  constexpr int kDsOps = 2 * kPerK2;         // this wave's 32 rows x BK keys
  constexpr int kStageLoads = KtStager::kPer + kDsOps;
  // Stage s = keys [BK s, BK s + BK): in unit BK*s/128, the BK*32 bytes at
  // (BK*s % 128)*32 of each k2 half (k2 at 4096 bytes).
  auto stage_load = [&](int s, Stage& sg) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KtStager::kPer; ++i) ktst.stage_one(sg.kt, rkt, (uint32_t)s * BK * 2, i);
    // Unit of stage s among this wave's units (clamped into them), then the
    // stage's keys within it.
    const int ku = min(max(s * BK / 128 - ds_kb_lo, 0), ds_nblk - 1);
    const uint32_t soff = (uint32_t)ku * 8192 + DsUnit::stage_src<BK>(s % (128 / BK), 0, 0);
#pragma unroll
    for (int i = 0; i < kDsOps; ++i)
      dma16_nt(rds, lds_addr(&sg.ds[wave][512 * i]), DsUnit::stage_src<BK>(0, i, lane), soff);
  };
  // Transposed B-operand reads: in 16-lane group G (k2 = G % 2, hh = G / 2),
  // lane i reads rows 16*k2 + 4*(i%4) .. +3 of key 16*ks + 8*hh + i/4 (+4 for
  // the second read) and receives keys +0..3 (+4..7) of row 16*k2 + i.
  const int tr_off = DsUnit::tr_elem<BK>(lane, 0, 0);

  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = zero16();

  auto compute = [&](const Stage& sg) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      const bf16* src = sg.ds[wave] + tr_off + ks * 16 * 16;
      const bf16x4 lo = lds_read_tr16(src), hi = lds_read_tr16(src + 4 * 16);
      const bf16x8 bop = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        acc[dt] = mfma32(row_operand<BK>(sg.kt, 32 * dt + l32, 16 * ks + 8 * hh), bop, acc[dt]);
    }
  };

  retire_prologue_loads();
  if (s1 > s0) {  // same for every wave of the workgroup
#pragma unroll
    for (int p = 0; p < NSTG - 1; ++p) stage_load(min(s0 + p, s1 - 1), st[p]);
    // Iteration s: stage s is waited for (NSTG - 2 later stages may still be
    // in flight), then stage s + NSTG - 1 (clamped: the last stage is
    // re-loaded, same bytes) goes into the buffer stage s - 1 used.
    int cur = 0;
    for (int s = s0; s < s1; ++s) {
      wait_vmem_n<(NSTG - 2) * kStageLoads>();
      barrier_lds();
      const int nxt = cur == 0 ? NSTG - 1 : cur - 1;
      stage_load(min(s + NSTG - 1, s1 - 1), st[nxt]);
      if (!WIN || (s >= w0 && s < w1)) compute(st[cur]);
      cur = cur == NSTG - 1 ? 0 : cur + 1;
    }
  }
  wait_vmem();  // the last (re-staged) loads

  if (a.dq_acc) {
    if (!qvalid) return;
    float* op = a.dq_acc + b * a.dqsb + h * a.dqsh + (int64_t)qrow * a.dqsl;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4* p = reinterpret_cast<f32x4*>(op + dt * 32 + 8 * g + 4 * hh);
        f32x4 w = *p;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] += acc[dt][4 * g + r] * a.scale;
        *p = w;
      }
  } else if (a.dq) {
    // bf16 rows leave through LDS (no stage is read any more), whole rows per
    // store instruction (see the forward's epilogue).
    barrier_lds();
    bf16* ep = reinterpret_cast<bf16*>(st) + wave * 32 * D;
    static_assert(sizeof(st) >= NW * 32 * D * sizeof(bf16), "the output rows fit the stages");
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 w;
        w[0] = pack_bf16x2(acc[dt][4 * g] * a.scale, acc[dt][4 * g + 1] * a.scale);
        w[1] = pack_bf16x2(acc[dt][4 * g + 2] * a.scale, acc[dt][4 * g + 3] * a.scale);
        *reinterpret_cast<u32x2*>(ep + TileLayout<D>::off(l32, dt * 32 + 8 * g) + 4 * hh) = w;
      }
    constexpr int kCpr = D / 8, kRpi = 64 / kCpr;  // chunks per row, rows per store
    const int er = lane / kCpr, ec = 8 * (lane % kCpr);
    bf16* op = a.dq + b * a.dqsb + h * a.dqsh + ec;
#pragma unroll
    for (int i = 0; i < 32 / kRpi; ++i) {
      const int r = i * kRpi + er, row = qg * 32 + r;
      const u32x4 x = *reinterpret_cast<const u32x4*>(ep + TileLayout<D>::off(r, ec));
      if (row < a.Lq) *reinterpret_cast<u32x4*>(op + (int64_t)row * a.dqsl) = x;
    }
  }
}

// Zero-fill rows of a strided (B, H, L, D) bf16 tensor (gradients of an empty
// attention).
__global__ void zero_rows_kernel(bf16* x, int64_t sb, int64_t sh, int64_t sl, int B, int H, int L, int D) {
  const int64_t units = (int64_t)B * H * L * (D / 8);
  for (int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; u < units; u += (int64_t)gridDim.x * blockDim.x) {
    const int c = (int)(u % (D / 8));
    const int64_t row = u / (D / 8);
    const int i = (int)(row % L);
    const int h = (int)((row / L) % H);
    const int b = (int)(row / ((int64_t)L * H));
    *reinterpret_cast<u32x4*>(x + b * sb + h * sh + (int64_t)i * sl + 8 * c) = u32x4{0u, 0u, 0u, 0u};
  }
}

// Compute units of the current device (0 if the query fails: no split).
static int cu_count() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
  return n;
}

// Split of every key block of a short dK/dV grid (no windows) over 2..8 ranges
// of query tiles (at least 8 each), or {0, 0}: for grids of at most one round
// (beyond it the tail split shares out the last round).  Estimated from the
// time per 64-row tile and per workgroup and the parts' traffic at 4 TB/s; a
// partial round clocks higher (see fwd_split_plan).  A key mask changes
// nothing: how many blocks it leaves without an attended key is known on the
// device only, and a plan that counted on half of them made fully attended
// calls slower ((1,5,12000,128) x 6,656 keys, 260 blocks, 552 us unsplit,
// 623 split; (2,20,40000) x 1,024 with one row empty 1,511 against 1,612).
// Backward: (1,16,20000,128) x 256 keys 498 -> 198 us, (1,20,10000) x 128 keys
// 255 -> 104, (1,4,4096) self-attention 171 -> 150.
TailSplit dkv_split_plan(int64_t total, int tiles, int D) {
  constexpr int kCus = 256;
  TailSplit best{0, 0};
  if (total > kCus) return best;
  const float work_us = tiles * (D == 64 ? 1.1f : 1.9f), fixed_us = 8.f;
  auto cost = [&](int p) {
    const int n = (int)total * p, rem = n % kCus;
    const float rounds = n / kCus + (rem == 0 ? 0.f : 1.f - 0.38f * (1.f - (float)rem / kCus));
    return rounds * (work_us / p + fixed_us) + (p > 1 ? 5.f + n * (1024.f * D) * 0.5e-6f : 0.f);
  };
  float c = cost(1) - 4.f;
  for (int p = 2; p <= 8 && tiles / p >= 8; ++p) {
    if (cost(p) < c) {
      c = cost(p);
      best = TailSplit{(int)total, p};
    }
  }
  return best;
}

// The same with changed scores, where also grids with windows are split: a
// block's tiles are then known on the device only and differ, so rounds after
// the first are taken to level out.  The model was fitted to 1 to 8 parts of
// 204 backward passes (12 to 256 blocks of 6 to 260 tiles; no windows, causal,
// five documents; D 64 and 128): its choice is 1.1% slower than the best of
// them on average, 13% (no windows) and 20% at most; two rounds of parts, 8
// tiles or more each, with every window were 6.4% and 48%.  (1,16 / 4
// heads,4133,64), 132 blocks, with 1 / 2 / 3 / 4 / 5 / 6 / 8 parts: five
// documents 254 / 167 / 160 / 147 / 155 / 157 / 160 us, causal 416 / 263 / 283 /
// 223 / 259 / 235 / 241, no windows 455 / 483 / 383 / 418 / 381 / 400 / 401.
TailSplit dkv_scored_split_plan(int64_t total, int tiles, int D, bool windows) {
  constexpr int kCus = 256;
  TailSplit best{0, 0};
  if (total > kCus) return best;
  const float tile_us = D == 64 ? 1.1f : 1.55f, slot_us = D == 64 ? 0.03f : 0.048f;
  auto cost = [&](int p) {
    const int n = (int)total * p, rem = n % kCus;
    float rounds = n / kCus + (rem == 0 ? 0.f : 1.f - 0.2f * (1.f - (float)rem / kCus));
    if (windows) rounds = n > kCus ? (float)n / kCus + 0.25f : 1.f;
    return rounds * (tiles * tile_us / p + 3.f) + (p > 1 ? 4.f + n * slot_us : 0.f);
  };
  float c = cost(1);
  for (int p = 2; p <= 8 && p <= tiles; ++p) {
    if (cost(p) < c) {
      c = cost(p);
      best = TailSplit{(int)total, p};
    }
  }
  return best;
}

template <int D>
static void launch_dq_ds_d(const BwdArgs& a, hipStream_t stream) {
  const int group = a.Hq / a.Hkv;
  const int nqb = (a.Lqp / 32 + 7) / 8;  // 256 query rows per workgroup
  const dim3 grid(nqb * a.nkv * group);
  LaunchTimer timer(kKidBwdDqDs, stream);
  // 64-key stages, three buffers: measured faster than 32-key stages with
  // four or six buffers (4.75 vs 4.9-5.4 ms per c3 chunk).  The grid's
  // partial last round is not split as the dK/dV one is: this kernel is
  // bound by HBM, and the last round's workgroups share all of it (measured:
  // no gain at c3).
  // With changed scores, short grids in workgroups of 128 rows: twice as many
  // spread over CUs that would idle (and at D 64 two share a CU), but K is staged
  // twice as often.  Backward in 256 against 128 rows, D 128: causal (1,4,1024)
  // 16 workgroups of 256 rows 53.0 / 47.8 us, (1,16,2048) 128 115.8 / 105.4, (1,16
  // on 4 heads,4133) 272 299 / 286, (1,40,2304) 360 243.1 / 241.4 (with a prefix of
  // 512 dQ alone 64 / 67), (1,16 on 8 heads,8192) 512 856 / 881; no windows
  // (1,2,16384) 128 849 / 796, (1,20,2304) 180 212 / 216, (1,8,8192) 256 795 / 818.
  if (a.score.mode != 0 && !a.ds_tab && grid.x <= (a.wlo ? 300 : 160)) {
    const dim3 short_grid((a.Lqp / 32 + 3) / 4 * a.nkv * group);
    if (a.wlo)
      hipLaunchKernelGGL((bwd_dq_ds_kernel<D, 64, 3, true, false, 4>), short_grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((bwd_dq_ds_kernel<D, 64, 3, false, false, 4>), short_grid, dim3(256), 0, stream, a);
  } else if (a.wlo && a.ds_tab)
    hipLaunchKernelGGL((bwd_dq_ds_kernel<D, 64, 3, true, true>), grid, dim3(512), 0, stream, a);
  else if (a.wlo)
    hipLaunchKernelGGL((bwd_dq_ds_kernel<D, 64, 3, true, false>), grid, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((bwd_dq_ds_kernel<D, 64, 3, false, false>), grid, dim3(512), 0, stream, a);
}

// Whether the dK/dV kernel can read 64-row tiles of rows `row_stride` elements
// apart in place: rows that do not overlap (so that a row past the end starts
// past the tile's buffer range) and a tile span within 32-bit byte offsets.
static bool tiles_in_place(int64_t row_stride, int D) { return row_stride >= D && row_stride < (int64_t)1 << 23; }

template <int D>
static hipError_t launch_bwd_d(const BwdArgs& args, int kv_per_pass, hipStream_t stream) {
  BwdArgs a = args;
  const bool mask = a.mask != nullptr;
  // Sources of the dK/dV kernel's Q and dO tiles: the caller's tensors, or
  // padded copies where q is rotated first or the rows cannot be read in
  // place.  A copy is one read and one write of the tensor at HBM rate, which
  // the tile loads then repeat: without the two of them 75,600 queries x 512
  // keys (2 x 40 heads, D 128) went from 8.53 to 7.35 ms forward + backward,
  // a 13x15x27-token block from 1.218 to 1.192 ms; at 16k tokens the copies
  // are under 1% of the step.
  const int64_t ch = (int64_t)a.Lqp * D;  // a copy's head stride
  if (a.cos_q == nullptr && tiles_in_place(a.qsl, D)) {
    a.qt = a.q, a.qtb = a.qsb, a.qth = a.qsh, a.qtl = a.qsl;
  } else {
    a.qt = a.qr, a.qtb = a.Hq * ch, a.qth = ch, a.qtl = D;
  }
  if (tiles_in_place(a.dosl, D)) {
    a.dt = a.dout, a.dtb = a.dosb, a.dth = a.dosh, a.dtl = a.dosl;
  } else {
    a.dt = a.dor, a.dtb = a.Hq * ch, a.dth = ch, a.dtl = D;
  }
  const hipError_t e = launch_prep_bwd(a, D, stream);
  if (e != hipSuccess) return e;
  // dK/dV (and, with staged dS, dQ) per pass over (b, kv head) pairs.
  const int nkv_all = a.B * a.Hkv;
  const int step = a.ds ? kv_per_pass : nkv_all;
  const int nkt = (a.Lk + 127) / 128;
  const int cus = cu_count();
  for (int kv0 = 0; kv0 < nkv_all; kv0 += step) {
    BwdArgs p = a;
    p.kv0 = kv0;
    p.nkv = min(step, nkv_all - kv0);
    // One 128-key block per workgroup, one workgroup per CU: a grid of
    // total blocks runs in ceil(total / cus) rounds, the last one with
    // total % cus blocks and the other CUs idle.  Those blocks are split
    // over several workgroups each (ranges of query tiles) so that the last
    // round is fuller and shorter.
    const int total = nkt * p.nkv;
    TailSplit ts = p.split_part ? plan_tail_split(total, cus, kSplitSlots) : TailSplit{0, 0};
    if (p.split_all != nullptr) {
      // Every block split (the region holds the plan's parts).
      const int tiles = (a.Lqp / 64) * (a.Hq / a.Hkv);
      ts = p.score.mode != 0 ? dkv_scored_split_plan(total, tiles, D, p.wlo != nullptr)
                             : dkv_split_plan(total, tiles, D);
      p.split_part = p.split_all;
    }
    p.nsplit = ts.nsplit;
    p.nparts = ts.nparts;
    {
      const dim3 grid(total - p.nsplit + p.nsplit * p.nparts);
      LaunchTimer timer(kKidBwdDkdv, stream);  // 1 workgroup (8 waves) per CU: LDS-bound occupancy
      if (p.score.mode != 0) {
        launch_dkdv_scored(p, D, grid, stream);
      } else if (p.wlo && p.ds_tab) {  // windows, compact dS layout
        if (mask)
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, true, true, true, true>), grid, dim3(512), 0, stream, p);
        else
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, true, true>), grid, dim3(512), 0, stream, p);
      } else if (p.wlo) {  // windows (staged dS only)
        if (mask)
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, true, true, true, false>), grid, dim3(512), 0, stream, p);
        else
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, true, false>), grid, dim3(512), 0, stream, p);
      } else if (mask) {
        if (p.ds)
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, true, true, false, false>), grid, dim3(512), 0, stream, p);
        else
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, true, false, false, false>), grid, dim3(512), 0, stream, p);
      } else {
        if (p.ds)
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, false, false>), grid, dim3(512), 0, stream, p);
        else
          hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, false, false, false>), grid, dim3(512), 0, stream, p);
      }
    }
    if (p.nsplit > 0) {
      const int64_t threads = (int64_t)p.nsplit * 2 * 128 * (D / 4);
      LaunchTimer timer(kKidDkdvReduce, stream);
      hipLaunchKernelGGL(dkv_reduce_kernel<D>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p);
    }
    if (p.ds && !p.defer_dq) launch_dq_ds_d<D>(p, stream);
  }
  if (!a.ds) {
    constexpr int BM = 256;  // 8 waves x 32 query rows
    const int nqt = (a.Lq + BM - 1) / BM;
    const dim3 grid(nqt * a.B * a.Hq);
    LaunchTimer timer(kKidBwdDq, stream);
    hipLaunchKernelGGL(bwd_dq_kernel<D>, grid, dim3(512), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_bwd(const BwdArgs& a, int head_dim, int kv_per_pass, hipStream_t stream) {
  return head_dim == 128 ? launch_bwd_d<128>(a, kv_per_pass, stream) : launch_bwd_d<64>(a, kv_per_pass, stream);
}

hipError_t launch_bwd_dq_staged(const BwdArgs& a, int head_dim, hipStream_t stream) {
  if (head_dim == 128)
    launch_dq_ds_d<128>(a, stream);
  else
    launch_dq_ds_d<64>(a, stream);
  return hipGetLastError();
}

hipError_t launch_zero_rows(bf16* x, int64_t sb, int64_t sh, int64_t sl, int B, int H, int L, int D,
                            hipStream_t stream) {
  const int64_t units = (int64_t)B * H * L * (D / 8);
  if (units == 0) return hipSuccess;
  const int64_t blocks = (units + 255) / 256;
  hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream, x,
                     sb, sh, sl, B, H, L, D);
  return hipGetLastError();
}

}  // namespace avattn
