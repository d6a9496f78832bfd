// The dK/dV kernel of the attention backward (see attn_bwd.hip for the whole).
#pragma once

#include <type_traits>

#include "avattn_device.h"
#include "avattn_kernels.h"

namespace avattn {

// ---------------------------------------------------------------------------
// 2. dK / dV
// ---------------------------------------------------------------------------
// One workgroup = 128 keys and 8 waves in two roles; waves w and w+4 own the
// same 32 keys (lane % 32 owns key column kt*128 + 32*(w%4) + lane % 32) and
// run on the same SIMD.  For each 32-row half `sub` of a 64-row query tile
// (lane l supplies query row 32*sub + perm23(l % 32) to the first products):
//   P waves (w < 4):   S  = Q K^T      A = Q rows (LDS)   B = K^T (registers)
//                      P  = exp2(S*c - lse2[q])   -> bf16, handed to the partner
//                      dV^T += dO^T P  A = dO^T (LDS, transposed reads), B = P
//   dS waves (w >= 4): dP = dO V^T     A = dO rows (LDS)  B = V^T (registers)
//                      dS = P * (dP + ndelta[q])  (P from the partner)
//                      dK^T += Q^T dS  A = Q^T (LDS, transposed reads), B = dS
// C-layout register 8*k2 + e of lane l holds query 32*sub + 16*k2 + 8*(l/32)
// + e, so the A operands of the last products are two transposed reads of
// the row tiles (rows +0..3, +4..7), the row statistics 16-byte LDS reads,
// and P travels between the partners as each lane's own registers (one
// 16-byte LDS write and read per 16 rows).
//
// One barrier per tile (T: tile staged).  The dS waves run their dS phase one
// tile behind, so the P they need was written before the last barrier: in
// iteration t a P wave runs QK^T and the softmax of tile t, then dV; its
// partner runs dO V^T of tile t (low priority, MFMAs only), then dS and dK of
// tile t - 1 (high priority), so one wave's VALU work always has the other's
// MFMAs to hide behind.  Keys that are masked (or past the end) are
// not special-cased in the loop: each key's dK/dV column depends only on that
// key, and those columns are written as zeros (or not at all) at the end.
// With STAGE the dS waves also store their dS tiles (BwdArgs::ds).  With WIN
// (key windows non-decreasing in the row, BwdArgs::wlo/whi; staged dS only)
// the workgroup visits only the 64-row tiles whose rows' window union meets
// its keys, and the P waves set the scores outside a row's window to -inf
// in tiles not inside every window (so P and dS are 0 there).
//
// SCORE (kScoreCap, kScoreDistance or both; BwdArgs::score): the P waves change
// the scores as the forward does before exp2.  With the cap, the dS waves need
// P (1 - tanh^2) in place of P: the P waves hand over that product (rounded to
// bf16 like P) and keep P itself for dV, so the exchange stays one value per
// score and the dS waves do not change.  A score outside its row's window gets
// lse2 = +inf (P = 0 whatever the capped score is).
// Distances are measured as BiasRef says.  A tile's rows mostly have their pos
// among their keys in steps of one per row, or in steps of none (all of them
// behind their last key, or before their first); with a slope < 0 the bias is
// that of the distance from the far end of a row's keys, which moves by none or
// two per row where the wave's keys lie on one side of pos.  Such tiles share
// one form of the bias; in the others (`far`) each score's goes into its lse2
// before its softmax step.
template <int D, bool MASK, bool STAGE, bool WIN, bool CT, int SCORE = 0>
__global__ __launch_bounds__(512, 1) void bwd_dkdv_kernel(BwdArgs a) {
  static_assert(!SCORE || (STAGE && !MASK), "changed scores with staged dS only");
  static_assert(!WIN || STAGE, "windows with staged dS only");
  static_assert(!CT || WIN, "the compact dS layout (BwdArgs::ds_tab) is for windows");
  constexpr int BK = 128, BQ = 64, NW = 8;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int TE = BQ * D;
  // Query tiles are staged as Q rows and as dO rows plus the rows'
  // statistics, three slots of each (tile t in slot t % 3).  The first
  // products read the rows; the last two read the same tiles transposed
  // (ds_read_b64_tr_b16), so no head_dim-major copy is staged.  Tile t's Q
  // is read until the end of iteration t + 1 (dK^T), its dO and statistics
  // until the end of iteration t: during iteration t the Q rows of tile t + 1
  // and the rest of tile t + 2 are loaded, into the slots tiles t - 2 and
  // t - 1 used.
  struct RowStage {
    bf16 dout[TE];  // dO rows: TileLayout<D>
    float lse2[BQ];
    float ndl[BQ];  // ndelta: the dP accumulators start from it
    int wlo[WIN ? BQ : 4];  // key windows of the tile's rows (WIN)
    int whi[WIN ? BQ : 4];
  };
  struct Smem {
    bf16 q[3][TE];  // Q rows: TileLayout<D>
    RowStage rs[3];
    // P hand-over, one buffer per slot (tile t's P is written in iteration t
    // and read in iteration t + 1): 1 KB per (key group, sub, k2),
    // lane-major.
    u32x4 xp[3][4 * 2 * 2 * 64];
  };
  __shared__ __attribute__((aligned(16))) Smem sm;
  // Byte strides of the slots (the reads below add them to per-lane bases).
  constexpr uint32_t kQS = TE * 2, kRS = sizeof(RowStage), kXS = sizeof(sm.xp[0]);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int role = wave >> 2, kw = wave & 3;
  const int l32 = lane & 31, hh = lane >> 5;
  const int prow = perm23(l32);

  // SCORE variants look for a key mask at run time (MASK false): the mask is
  // read once, before the loop.
  const bool masked = SCORE ? a.mask != nullptr : MASK;
  const int nkt = (a.Lk + BK - 1) / BK;
  const int total = nkt * a.nkv;
  // Key blocks 0 .. nfull-1 take one workgroup each (query tiles all); the
  // last a.nsplit blocks (the grid's partial last round, or all of them)
  // take a.nparts workgroups each, one per range of query tiles, whose fp32
  // partial dK/dV dkv_reduce_kernel sums.
  const int nfull = total - a.nsplit;
  int bid, part = -1;
  if (nfull == 0) {
    // A pair's key blocks of one part next to each other: they stream the
    // same query tiles.
    const int per = nkt * a.nparts;
    const int u = xcd_remap_pairs(blockIdx.x, total * a.nparts, per, masked);
    bid = u / per * nkt + u % nkt;
    part = u % per / nkt;
  } else if ((int)blockIdx.x < nfull) {
    bid = xcd_remap_pairs(blockIdx.x, nfull, nkt, masked);
  } else {
    const int i = blockIdx.x - nfull;
    bid = nfull + i / a.nparts;
    part = i % a.nparts;
  }
  int kt = bid % nkt, pair = bid / nkt;
  if constexpr (SCORE && WIN) {
    // Causal and prefix masks give the first keys the most rows: those blocks
    // first (dkv_reduce_kernel finds the split ones in the same order).  With
    // every block split its parts stay together on their XCD instead: in this
    // order 132 blocks in 4 parts took 125 us in place of 106.
    if (nfull > 0) longest_first((int)blockIdx.x < nfull ? blockIdx.x : bid, nkt, a.nkv, kt, pair);
  }
  const int bhk = a.kv0 + pair;
  const int b = bhk / a.Hkv, hk = bhk % a.Hkv;
  const int group = a.Hq / a.Hkv;

  const int key = kt * BK + kw * 32 + l32;
  // Whether this lane's key is attended; read again for the epilogue rather
  // than held through the loop, which has no register to spare.
  auto key_valid = [&]() {
    bool ok = key < a.Lk;
    if (masked && ok) ok = a.mask[b * a.msb + key] != 0;
    return ok;
  };
  // SCORE: the key is one some row may attend; what others hold must not count.
  bool live = true;
  if constexpr (SCORE != 0) {
    int klo, khi;
    key_hull(nullptr, a.wlo, a.whi, a.wsb, b, a.Lq, a.Lk, klo, khi);
    live = key_valid() && key >= klo && key < khi;
  }

  // This wave's B operand: K (P waves, rotated when the backward carries the
  // key's rotation) or V (dS waves) of the lane's key, read once from the
  // caller's tensors; zeros past the end.
  bf16x8 kv[KS];
  {
    const bool in = SCORE ? live : key < a.Lk;
    const bf16* src = role == 0 ? a.k + b * a.ksb + hk * a.ksh + (int64_t)key * a.ksl + 8 * hh
                                : a.v + b * a.vsb + hk * a.vsh + (int64_t)key * a.vsl + 8 * hh;
    const bool rot = role == 0 && a.cos_k != nullptr;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (in) {
        x = *reinterpret_cast<const u32x4*>(src + 16 * ks);
        if (rot) {
          const int64_t t = b * a.rksb + (int64_t)key * (D / 2) + 8 * ks + 4 * hh;
          x = rotate8(x, *reinterpret_cast<const f32x4*>(a.cos_k + t), *reinterpret_cast<const f32x4*>(a.sin_k + t),
                      false);
        }
      }
      kv[ks] = bits_to_bf16x8(x);
    }
  }

  f32x16 acc[DT];  // dV^T (P waves) or dK^T (dS waves)
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = zero16();

  // Loop-invariant per-lane LDS element offsets.
  int ro[KS];  // row tiles: chunk (16*ks + 8*hh) of row perm23(l32)
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) ro[ks] = TileLayout<D>::off(prow, 16 * ks + 8 * hh);
  // Transposed reads of the same tiles (A operands of dV^T += dO^T P and
  // dK^T += Q^T dS): channel block dt, rows 16*(2*sub + k2) + 8*hh + 4*h ..
  // +3 for the read h = 0, 1 (tr_read_off).  Rows advance by 16 per
  // (sub, k2), which keeps the row swizzle, so the offsets are
  // loop-invariant.
  int tro[DT][2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int h = 0; h < 2; ++h) tro[dt][h] = tr_read_off<D>(lane, dt, h);
  // Per-lane LDS byte addresses in slot 0 (opaque: slot and row-block
  // offsets go into the reads' offset fields).  P waves read Q as rows and
  // dO transposed, dS waves dO as rows and Q transposed.
  uint32_t rb[KS], tb[DT][2];
  {
    const uint32_t q0 = lds_addr(&sm.q[0][0]), d0 = lds_addr(&sm.rs[0].dout[0]);
    const uint32_t rrow = role == 0 ? q0 : d0, rtr = role == 0 ? d0 : q0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) rb[ks] = opaque(rrow + 2 * ro[ks]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int h = 0; h < 2; ++h) tb[dt][h] = opaque(rtr + 2 * tro[dt][h]);
  }
  // Row statistics of the lane's rows 8*hh + ...: lse2 at sb, ndelta and
  // the windows at the offsets below.
  const uint32_t sb = opaque(lds_addr(&sm.rs[0].lse2[0]) + 32 * hh);
  // The lane's row's window (SCORE with a bias).
  const uint32_t wb = SCORE & kScoreDistance && WIN ? opaque(lds_addr(&sm.rs[0].wlo[0]) + 4 * lane) : 0u;
  constexpr uint32_t kNdlOff = BQ * 4, kWloOff = 2 * BQ * 4, kWhiOff = kWloOff + sizeof(sm.rs[0].wlo);
  static_assert(offsetof(RowStage, ndl) - offsetof(RowStage, lse2) == kNdlOff &&
                    offsetof(RowStage, wlo) - offsetof(RowStage, lse2) == kWloOff &&
                    offsetof(RowStage, whi) - offsetof(RowStage, lse2) == kWhiOff,
                "row statistics offsets");
  // This lane's 16 bytes of the P hand-over: + kXS*slot + 1024*(2*sub + k2).
  const uint32_t xb = opaque(lds_addr(&sm.xp[0][0]) + 16 * (kw * 4 * 64 + lane));

  const int nqt = a.Lqp / BQ;
  // Query tiles visited: tq0 .. tq0 + ntq - 1 of every query head of the
  // group (all of them without windows).  With monotone windows, tile T
  // meets this block's keys [k0, k1) iff lo(first row of T) < k1 and
  // hi(last row of T) > k0; both conditions hold on a prefix / suffix of the
  // tiles, so their counts give the range.
  int tq0 = 0, ntq = nqt;
  // WIN: tiles [w_ia, w_ib) hold only rows whose windows cover all 32 keys
  // of this wave (hi(first row) >= kk0 + 32 and lo(last row) <= kk0; each
  // condition holds on a suffix / prefix of the tiles); the others mask
  // scores per (row, key).
  int w_ia = 0, w_ib = 0;
  if constexpr (WIN) {
    __shared__ int cred[NW][2];
    const int k0 = kt * BK, k1 = min(k0 + BK, a.Lk);
    const int* lo = a.wlo + b * a.wsb;
    const int* hi = a.whi + b * a.wsb;
    const int nvt = (a.Lq + BQ - 1) / BQ;  // tiles holding valid rows
    int c_lo = 0, c_hi = 0;
    for (int T = tid; T < nvt; T += NW * 64) {
      const int f = T * BQ, l = min(f + BQ - 1, a.Lq - 1);
      const int lof = min(max(lo[f], 0), a.Lk);
      const int lol = min(max(lo[l], 0), a.Lk);
      const int hil = min(max(hi[l], lol), a.Lk);
      c_hi += lof < k1;
      c_lo += hil <= k0;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      c_lo += __shfl_xor(c_lo, off);
      c_hi += __shfl_xor(c_hi, off);
    }
    if (lane == 0) {
      cred[wave][0] = c_lo;
      cred[wave][1] = c_hi;
    }
    __syncthreads();
    int s_lo = 0, s_hi = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      s_lo += cred[w][0];
      s_hi += cred[w][1];
    }
    tq0 = __builtin_amdgcn_readfirstlane(s_lo);
    ntq = __builtin_amdgcn_readfirstlane(max(s_hi - s_lo, 0));
    const int kk0 = kt * BK + kw * 32;
    int c_a = 0, c_b = 0;
    for (int T = lane; T < nvt; T += 64) {
      const int f = T * BQ, l = min(f + BQ - 1, a.Lq - 1);
      c_a += hi[f] < kk0 + 32;
      c_b += lo[l] <= kk0;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      c_a += __shfl_xor(c_a, off);
      c_b += __shfl_xor(c_b, off);
    }
    w_ia = __builtin_amdgcn_readfirstlane(c_a);
    w_ib = __builtin_amdgcn_readfirstlane(c_b);
  }
  // A block outside the pair's hull of contributing tiles (every key masked):
  // dK and dV are zeros and dS is not read.
  if (masked && STAGE && !WIN) {
    if (2 * kt >= load_const_i32(a.khull, 2 * bhk + 1) || 2 * kt + 2 <= load_const_i32(a.khull, 2 * bhk)) {
      if (part >= 0) return;  // the reduction reads no part of a masked key
      ntq = 0;
    }
  }
  if (part >= 0) {  // this part's share of the tiles (possibly none)
    const int p0 = ntq * part / a.nparts, p1 = ntq * (part + 1) / a.nparts;
    tq0 += p0;
    ntq = p1 - p0;
  }
  const int niter = ntq * group;
  auto tile_head = [&](int it) { return it / ntq; };     // query head within the group
  auto tile_idx = [&](int it) { return tq0 + it % ntq; };  // 64-row tile of that head
  // The tiles this wave loads (dO for a P wave, Q for a dS wave), read where
  // BwdArgs::dt / qt point: the caller's tensor (rows past the end read as
  // zeros, see tile_rsrc) or a padded copy.
  const int64_t bq0 = (int64_t)(b * a.Hq + hk * group);
  const int64_t th = role == 0 ? a.dth : a.qth;
  const int tl = (int)(role == 0 ? a.dtl : a.qtl);
  const bf16* t00 = role == 0 ? a.dt + b * a.dtb : a.qt + b * a.qtb;
  t00 += (int64_t)hk * group * th;
  const u32x4 rl2 = make_rsrc(a.lse2 + bq0 * a.Lqp, (uint32_t)group * a.Lqp * 4);
  const u32x4 rnd = make_rsrc(a.ndelta + bq0 * a.Lqp, (uint32_t)group * a.Lqp * 4);
  // A tile is loaded in two parts, one load at a time between MFMAs (a burst
  // of them at the start of a phase would hold up the wave's instruction
  // stream): the dS waves load its Q rows (kQOps loads per wave) during their
  // dP phase of the iteration before, the P waves its dO rows and statistics
  // (kROps) during their dV phase of the iteration before that.
  TileStager<BQ, D, 4> rst;  // 64 rows of D channels (row stride tl) over 4 waves
  rst.init(tl, kw, lane);
  constexpr int kQOps = TileStager<BQ, D, 4>::kPer;
  constexpr int kROps = kQOps + 2 + (WIN ? 2 : 0);
  auto tile_rows = [&](int it) {  // first row of tile `it` in the group's statistics
    return (uint32_t)tile_head(it) * a.Lqp + (uint32_t)tile_idx(it) * BQ;
  };
  // Buffer over tile `it`'s rows of this wave's source: from its first row to
  // the end of its last valid one, so that loads of rows past the end (tl >=
  // D, so they start past the range) return zeros.
  auto tile_rsrc = [&](int it) {
    const int row0 = tile_idx(it) * BQ;
    const int last = min(a.Lq - 1 - row0, BQ - 1);
    return make_rsrc(t00 + tile_head(it) * th + (int64_t)row0 * tl, (uint32_t)(last * tl + D) * 2);
  };
  // Window arrays of this batch (WIN); rows past Lq read as 0 (empty).
  u32x4 rwl = {0u, 0u, 0u, 0u}, rwh = {0u, 0u, 0u, 0u};
  if constexpr (WIN) {
    rwl = make_rsrc(a.wlo + b * a.wsb, (uint32_t)a.Lq * 4);
    rwh = make_rsrc(a.whi + b * a.wsb, (uint32_t)a.Lq * 4);
  }
  // Q load i of a tile (its buffer rq) into Q slot `qd`.
  auto q_op = [&](const u32x4& rq, bf16* qd, int i) { rst.stage_one(qd, rq, 0u, i); };
  // Row load i of tile `it` (its dO buffer rdo) into row slot `rsg`.
  auto r_op = [&](int it, const u32x4& rdo, RowStage& rsg, int i) {
    if (i < kQOps)
      rst.stage_one(rsg.dout, rdo, 0u, i);
    else if (i == kQOps)
      dma4(rl2, lds_addr(rsg.lse2), lane * 4, tile_rows(it) * 4);  // every wave loads the stats: no branch
    else if (i == kQOps + 1)
      dma4(rnd, lds_addr(rsg.ndl), lane * 4, tile_rows(it) * 4);
    else if (i == kQOps + 2)
      dma4(rwl, lds_addr(rsg.wlo), lane * 4, (uint32_t)tile_idx(it) * BQ * 4);
    else
      dma4(rwh, lds_addr(rsg.whi), lane * 4, (uint32_t)tile_idx(it) * BQ * 4);
  };
  // Vector-memory operations complete in issue order (a load issued behind a
  // store only counts as done once the store has been written).  A P wave
  // issues rows(t + 1) in iteration t - 1 and rows(t + 2) in iteration t, so
  // at tile t + 1's T wait only the kROps loads of rows(t + 2) may still be
  // outstanding.  A dS wave issues Q(t + 1) in iteration t, followed only by
  // the dS stores of tile t - 1 (STAGE, t >= 1): kDsStores of them.
  constexpr int kDsStores = 4;
  // Slots of a phase that issue its `count` loads: every slot from 4 on (the
  // start of a phase is left to its operand and statistics reads); the rest
  // follow the phase's loop.
  constexpr int kLoad0 = 4;
  auto load_slot = [](int j, int nslots, int count) { return j >= kLoad0 && j - kLoad0 < count && j < nslots; };
  auto loads_in_loop = [](int nslots) { return nslots > kLoad0 ? nslots - kLoad0 : 0; };
  // Operand reads in flight ahead of the MFMAs (three measured faster than
  // four or six: fewer LDS requests queued at once).
  constexpr int kRA = 3;

  // dS staging (STAGE): per tile each dS wave stores its 32 keys x 64 rows
  // of dS as four 16-byte stores per lane (group g = 2*sub + k2: the lane's
  // key, its 8 consecutive rows), each instruction 1 KB contiguous in unit
  // `sub`, in the first slot of each group's dK^T MFMAs.
  // dS of masked / past-the-end keys is stored as 0.
  const uint32_t ds_keep = STAGE && (SCORE ? live : key_valid()) ? 0xffffffffu : 0u;
  const uint32_t ds_voff = DsUnit::store_offset(kw * 32 + l32, lane, 0, 0, 0);

  const float c = a.scale_log2;
  // Distance bias: lane g holds the slope of the group's query head g; the hull
  // of the attended keys (BiasRef).
  float slope_of = 0.f;
  int qoff = 0, hull_lo = 0, hull_hi = a.Lk;
  if constexpr (SCORE & kScoreDistance) {
    slope_of = a.score.slopes && lane < group ? a.score.slopes[hk * group + lane] * kLog2e : 0.f;
    qoff = __builtin_amdgcn_readfirstlane(a.score.query_offset(b));
    if (masked && a.score.slopes) {
      hull_lo = 64 * load_const_i32(a.khull, 2 * bhk);
      hull_hi = min(64 * load_const_i32(a.khull, 2 * bhk + 1), a.Lk);
    }
  }

  // The loop bodies below are explicitly software-pipelined: each "slot" is
  // one MFMA plus the LDS read it needs kRA slots later, at most one load of
  // the next tile, and a share of the VALU work; sched_barrier(0) pins the
  // slot order (the scheduler would otherwise sink each read next to its
  // MFMA and bunch the loads and the VALU work).
  // Iteration `it` of a P wave; uc = it % 3 (compile-time), the slot.
  auto body_p = [&](int it, auto uc) {
    constexpr int u = decltype(uc)::value;
    wait_vmem_n<kROps>();  // this tile's rows landed (for this wave)
    barrier_lds();             // T: ... for every wave; the slots loaded into below are free
    // The wave whose phase ends in VALU-dependent work gets issue priority:
    // P waves up to the end of the softmax (2, then 0 in dV), dS waves in
    // their dS phase (2; 1 in their dP phase, which measured 0.8% faster
    // than 0).
    __builtin_amdgcn_s_setprio(2);
    // Loads during dV: rows of tile it + 2 (the last tiles re-load into
    // slots nothing reads any more).
    const int itr = min(it + 2, niter - 1);
    RowStage& lrs = sm.rs[(u + 2) % 3];

    constexpr int NS = 2 * KS;  // QK^T MFMAs: (sub, ks)
    auto qop = [&](int j) { return lds_ld<bf16x8>(rb[j % KS] + u * kQS + (j / KS) * 64 * D); };
    bf16x8 qa[kRA];
#pragma unroll
    for (int j = 0; j < kRA; ++j) qa[j] = qop(j);
    // lse2 of this lane's 16 rows per sub (8 consecutive rows per k2), read
    // one f32x4 per slot from slot 1 on (the softmax needs them only later;
    // reading them up front delays the first MFMAs' operands).
    f32x4 l2[2][2][2];
    auto l2_read = [&](int q8) {
      l2[q8 >> 2][(q8 >> 1) & 1][q8 & 1] =
          lds_ld<f32x4>(sb + u * kRS + 4 * (32 * (q8 >> 2) + 16 * ((q8 >> 1) & 1) + 4 * (q8 & 1)));
    };
    // The bias as the fast path has it: near2 (|slope2|; 0: far) times the
    // distance of the lane's key from a point that moves by `step` per row (kd:
    // from that of row 0 of the lane's first eight in this tile).
    float kd = 0.f, slope2 = 0.f, step = 1.f, near2 = 0.f;
    bool far = false;
    int rlo = 0, rhi = 0;  // lane l: the window of row l of the tile
    if constexpr (SCORE & kScoreDistance && WIN)
      rlo = lds_ld<int>(wb + u * kRS), rhi = lds_ld<int>(wb + u * kRS + (kWhiOff - kWloOff));
    __builtin_amdgcn_sched_barrier(0);

    f32x16 s[2] = {zero16(), zero16()};
    bf16x8 pb[2][2];
    // Row l's keys: its window, clamped, within the hull.
    auto keys_of = [&](int lo, int hi, int& wl, int& wh) {
      wl = min(max(lo, hull_lo), a.Lk);
      wh = max(min(hi, hull_hi), wl);
    };
    auto place_bias = [&]() {
      if constexpr (SCORE & kScoreDistance) {
        slope2 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(slope_of), tile_head(it)));
        const int r0 = tile_idx(it) * BQ, p0 = r0 + qoff;  // row 0 and its position
        int wl = hull_lo, wh = hull_hi;
        bool plain = !(slope2 < 0.f);  // every row's position is among its keys
        if constexpr (WIN) {
          keys_of(rlo, rhi, wl, wh);
          const bool out = wl < wh && (uint32_t)(p0 + lane - wl) >= (uint32_t)(wh - wl);
          plain = plain && __builtin_amdgcn_ballot_w64(out) == 0;
        } else {
          plain = plain && p0 >= wl && p0 + min(BQ, a.Lq - r0) <= wh;
        }
        kd = (float)(p0 + 8 * hh - key);
        near2 = slope2;
        if (__builtin_expect(!plain, 0)) {
          const bool alive = wl < wh && (WIN || r0 + lane < a.Lq);
          const uint64_t rows = __builtin_amdgcn_ballot_w64(alive);
          const int f = rows != 0 ? __builtin_ctzll(rows) : 0;
          auto all = [&](bool x) { return (rows & ~__builtin_amdgcn_ballot_w64(x)) == 0; };
          const bool neg = slope2 < 0.f;
          const BiasRef br = bias_ref(p0 + lane, wl, wh, neg);
          int e = br.pos;
          if (neg) {
            // From the side of the row's pos on which its keys of this wave lie:
            // ref - |pos - j| = |pos -+ ref - j|.
            const int k0 = kt * BK + kw * 32;
            const bool left = all(min(wh - 1, k0 + 31) <= br.pos), right = all(max(wl, k0) >= br.pos);
            e += left ? -br.ref : br.ref;
            far = !left && !right;
          }
          const int e0 = __builtin_amdgcn_readlane(e, f), n = lane - f;
          int st = 1;
          if (!all(e - e0 == n)) {
            st = all(e == e0) ? 0 : 2;
            far = far || (st == 2 && !all(e - e0 == 2 * n));
          }
          step = (float)st;
          kd = (float)(e0 + st * (8 * hh - f) - key);
          near2 = far ? 0.f : fabsf(slope2);
        }
      }
    };
    u32x4 up[2][2];
    // WIN: a tile outside [w_ia, w_ib) masks the scores of a row half per
    // (row, key) before its softmax steps: one wave-uniform branch per half,
    // not taken on the (common) inside tiles.
    bool edge = false;
    if constexpr (WIN) {
      const int T = tile_idx(it);
      edge = T < w_ia || T >= w_ib;
    }
    auto mask_sub = [&](int sub) {
      if constexpr (WIN) {
        if (__builtin_expect(edge, 0)) {
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int h4 = 0; h4 < 2; ++h4) {
              // rows 32*sub + 16*k2 + 8*hh + 4*h4 + [0, 4) of the tile
              const uint32_t r0 = sb + u * kRS + 4 * (32 * sub + 16 * k2 + 4 * h4);
              const u32x4 lo = lds_ld<u32x4>(r0 + kWloOff), hi = lds_ld<u32x4>(r0 + kWhiOff);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (key < (int)lo[r] || key >= (int)hi[r]) {
                  if constexpr (SCORE != 0) {
                    s[sub][8 * k2 + 4 * h4 + r] = 0.f;
                    l2[sub][k2][h4][r] = kPosInf;
                  } else {
                    s[sub][8 * k2 + 4 * h4 + r] = kNegInf;
                  }
                }
            }
        }
      }
    };
    // Softmax step (sub, k2, e2): two probabilities, packed; the last step
    // of a (sub, k2) hands its 16 bytes to the partner wave.
    auto far_sub = [&](int sub) {
      if constexpr (SCORE & kScoreDistance) {
        if (__builtin_expect(far, 0)) {
          // Lane l has row l's bias; each lane fetches those of its rows.
          int wl = hull_lo, wh = hull_hi;
          if constexpr (WIN)
            keys_of(lds_ld<int>(wb + u * kRS), lds_ld<int>(wb + u * kRS + (kWhiOff - kWloOff)), wl, wh);
          const BiasRef br = bias_ref(tile_idx(it) * BQ + lane + qoff, wl, wh, slope2 < 0.f);
          const int pos = __float_as_int((float)(br.pos - kt * BK)), ref = __float_as_int((float)br.ref);
          const float kf = (float)(kw * 32 + l32);
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int from = 4 * (32 * sub + 16 * k2 + 8 * hh + e);
              const float d = fabsf(__int_as_float(__builtin_amdgcn_ds_bpermute(from, pos)) - kf) -
                              __int_as_float(__builtin_amdgcn_ds_bpermute(from, ref));
              l2[sub][k2][e >> 2][e & 3] = fmaf(slope2, d, l2[sub][k2][e >> 2][e & 3]);
            }
        }
      }
    };
    // P and, capped, P (1 - tanh^2) are rounded to bf16 here, as the operands
    // of dV's products and the factors of dS; everything before is fp32.  (The
    // fp32 matrix instructions run at an eighth of the rate.)
    u32x4 ux;  // SCORE: P (1 - tanh^2) of one (sub, k2)
    auto smx = [&](int sub, int k2, int e2) {
      const int e = 2 * e2;
      const f32x4& lv = l2[sub][k2][e >> 2];
      const float s0 = s[sub][8 * k2 + e], s1 = s[sub][8 * k2 + e + 1];
      if constexpr (SCORE != 0) {
        float p[2], f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float z = i ? s1 : s0;
          f[i] = 1.f;
          if constexpr (SCORE & kScoreCap) {
            // The statistics hold lse2 - cap2, and a quarter of 1 - tanh^2 =
            // 4 r (1 - r) goes out: the 4 is in a.scale.
            const float r = cap_complement(z, a.score.cap_arg);
            z = fmaf(-2.f * a.score.cap2, r, -lv[(e & 3) + i]);
            f[i] = fmaf(-r, r, r);
          } else {
            z = fmaf(z, c, -lv[(e & 3) + i]);
          }
          if constexpr (SCORE & kScoreDistance)
            z = fmaf(-near2, fabsf(fmaf(step, (float)(32 * sub + 16 * k2 + e + i), kd)), z);
          p[i] = __builtin_amdgcn_exp2f(z);
        }
        up[sub][k2][e2] = pack_bf16x2(p[0], p[1]);
        if constexpr (SCORE & kScoreCap) ux[e2] = pack_bf16x2(p[0] * f[0], p[1] * f[1]);
        if (e2 == 3) {
          lds_st<u32x4>(xb + u * kXS + 1024 * (2 * sub + k2), SCORE & kScoreCap ? ux : up[sub][k2]);
          pb[sub][k2] = bits_to_bf16x8(up[sub][k2]);
        }
        return;
      }
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s0, c, -lv[e & 3]));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s1, c, -lv[(e & 3) + 1]));
      up[sub][k2][e2] = pack_bf16x2(p0, p1);
      if (e2 == 3) {
        lds_st<u32x4>(xb + u * kXS + 1024 * (2 * sub + k2), up[sub][k2]);
        pb[sub][k2] = bits_to_bf16x8(up[sub][k2]);
      }
    };
    // Softmax steps of sub 0 (8 of them) go into the slots after S(sub 0) is
    // complete (two slots of MFMA latency after its last MFMA).
    constexpr int kLo = KS + 2 < NS ? KS + 2 : NS;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int sub = j / KS, ks = j % KS;
      s[sub] = mfma32(qa[j % kRA], kv[ks], s[sub]);
      if (j + kRA < NS) qa[j % kRA] = qop(j + kRA);
      if (j >= 1 && j <= 8) l2_read(j - 1);
      if (j == 2) place_bias();
      if (j >= kLo) {
        const int n = NS - kLo;
        if (j == kLo) far_sub(0), mask_sub(0);
        for (int st = (j - kLo) * 8 / n; st < (j - kLo + 1) * 8 / n; ++st) smx(0, st >> 2, st & 3);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q8 = NS - 1; q8 < 8; ++q8) l2_read(q8);  // what the loop had no slot for
    if (kLo >= NS) {
      far_sub(0);
      mask_sub(0);
#pragma unroll
      for (int st = 0; st < 8; ++st) smx(0, st >> 2, st & 3);
    }
    far_sub(1);
    mask_sub(1);
#pragma unroll
    for (int st = 0; st < 8; ++st) smx(1, st >> 2, st & 3);
    // P goes out with the next barrier (T of tile it + 1, where the partner
    // picks it up for its dS phase).
    __builtin_amdgcn_s_setprio(0);

    // dV^T += dO^T P over the (sub, k2, dt) steps, reads kRA steps ahead.
    constexpr int NJ = 4 * DT;
    auto dot_op = [&](int j) {
      const int sk = j / DT, dt = j % DT;  // sk = 2*sub + k2
      const uint32_t off = u * kRS + sk * 32 * D;
      const bf16x4 lo = lds_read_tr16_at(tb[dt][0] + off), hi = lds_read_tr16_at(tb[dt][1] + off);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bf16x8 opq[kRA];
#pragma unroll
    for (int j = 0; j < kRA; ++j) opq[j] = dot_op(j);
    const u32x4 lrd = tile_rsrc(itr);  // scalar work, here behind the first reads' latency
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const bf16x8 op = opq[j % kRA];
      if (j + kRA < NJ) opq[j % kRA] = dot_op(j + kRA);
      const int sk = j / DT, dt = j % DT;
      acc[dt] = mfma32(op, pb[sk >> 1][sk & 1], acc[dt]);
      if (load_slot(j, NJ, kROps)) r_op(itr, lrd, lrs, j - kLoad0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = loads_in_loop(NJ); i < kROps; ++i) r_op(itr, lrd, lrs, i);
  };

  // dS waves, dP phase of the tile in slot uc: dp = dO V^T + ndelta, and the
  // Q loads of tile itq into lq.
  auto dp_phase = [&](auto uc, f32x16(&dp)[2], int itq, bf16* lq) {
    constexpr int u = decltype(uc)::value;
    constexpr int NS = 2 * KS;  // dO V^T MFMAs: (sub, ks)
    auto dop = [&](int j) { return lds_ld<bf16x8>(rb[j % KS] + u * kRS + (j / KS) * 64 * D); };
    bf16x8 da[kRA];
#pragma unroll
    for (int j = 0; j < kRA; ++j) da[j] = dop(j);
    // dP starts at ndelta of its row (registers 8*k2 + e: row 32*sub + 16*k2
    // + 8*hh + e), so the MFMAs deliver dP + ndelta directly.  Sub 0's values
    // are read now, sub 1's in the first slots (its MFMAs start at slot KS).
    auto nd_read = [&](int sub, int q4) {
      const int k2 = q4 >> 1, hf = q4 & 1;
      const f32x4 n4 = lds_ld<f32x4>(sb + u * kRS + kNdlOff + 4 * (32 * sub + 16 * k2 + 4 * hf));
#pragma unroll
      for (int r = 0; r < 4; ++r) dp[sub][8 * k2 + 4 * hf + r] = n4[r];
    };
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) nd_read(0, q4);
    const u32x4 lrq = tile_rsrc(itq);  // scalar work, here behind the first reads' latency
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int sub = j / KS, ks = j % KS;
      dp[sub] = mfma32(da[j % kRA], kv[ks], dp[sub]);
      if (j + kRA < NS) da[j % kRA] = dop(j + kRA);
      if (j < 4) nd_read(1, j);  // KS >= 4: before sub 1's first MFMA
      if (load_slot(j, NS, kQOps)) q_op(lrq, lq, j - kLoad0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = loads_in_loop(NS); i < kQOps; ++i) q_op(lrq, lq, i);
  };

  // Where tile `it`'s dS goes (STAGE): a buffer over its two units (query
  // groups 2*tile_idx(it) and +1) and the byte distance between them.
  struct DsDest {
    u32x4 rds;
    uint32_t unit1;
  };
  // Compact layout (WIN with a table): the tile's table entry, read by a
  // scalar load.  Scalar loads return out of order with LDS reads, so while
  // one is outstanding every counted LDS wait would have to become a full
  // one: the entry of the tile whose dS phase comes next is loaded at the
  // end of an iteration (after its last LDS read) and used right after the
  // next barrier, whose wait has drained it.
  struct DsEntry {
    int kb_lo, nblk, gbase;
  };
  auto ds_entry = [&](int it) {
    const int64_t e = ((int64_t)b * a.ds_tsb + tile_idx(it)) * 4;
    return DsEntry{__builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e)),
                   __builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e + 1)),
                   __builtin_amdgcn_readfirstlane(load_const_i32(a.ds_tab, e + 2))};
  };
  auto ds_dest = [&](int it, const DsEntry& en) {
    DsDest d{{0u, 0u, 0u, 0u}, 0u};
    if constexpr (STAGE) {
      const int64_t bq = (int64_t)(bhk - a.kv0) * group + tile_head(it);
      if (CT) {
        // A block outside the entry's range (an inconsistent table) gets an
        // empty buffer, so its stores are dropped; the store offsets are then
        // wholly per-lane (range-checked), see ds_store.
        const bool ok = kt >= en.kb_lo && kt - en.kb_lo < en.nblk && en.gbase >= 0 &&
                        (int64_t)en.gbase + 2 * en.nblk <= a.ds_units;
        const int64_t unit = bq * a.ds_units + (ok ? en.gbase + (kt - en.kb_lo) : 0);
        d.rds = make_rsrc(reinterpret_cast<char*>(a.ds) + unit * 8192, ok ? (uint32_t)(en.nblk + 1) * 8192 : 0u);
        d.unit1 = (uint32_t)en.nblk * 8192;
      } else {
        const int64_t unit = (bq * (2 * nqt) + 2 * tile_idx(it)) * nkt + kt;
        d.rds = make_rsrc(reinterpret_cast<char*>(a.ds) + unit * 8192, (uint32_t)(nkt + 1) * 8192);
        d.unit1 = (uint32_t)nkt * 8192;
      }
    }
    return d;
  };

  // dS waves, dS phase of tile `it` (slot uc), one iteration after its dP
  // phase, so the partner's P has been handed over by the barrier in
  // between: dS = P * dp, dK^T += Q^T dS and, with STAGE, the dS stores
  // (kDsStores per lane) to `dd`.
  auto ds_phase = [&](int it, auto uc, const f32x16(&dp)[2], const DsDest& hoisted) {
    constexpr uint32_t u = decltype(uc)::value;
    // The compact layout's destination was computed at the top of the
    // iteration (see DsEntry); the dense one here, where its few scalar
    // operations schedule best.
    const DsDest dd = (CT) ? hoisted : ds_dest(it, DsEntry{0, 0, 0});
    const u32x4 rds = dd.rds;
    const uint32_t ds_unit1 = dd.unit1;

    // dS for group g = 2*sub + k2 (4 steps of two elements) interleaved with
    // the dK^T MFMAs of group g-1; every LDS read is issued up front or kRA
    // MFMAs ahead.
    u32x4 pv[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) pv[g] = lds_ld<u32x4>(xb + u * kXS + 1024 * g);
    constexpr int NJ = 4 * DT;
    auto qt_op = [&](int j) {
      const int g = j / DT, dt = j % DT;
      const uint32_t off = u * kQS + g * 32 * D;
      const bf16x4 lo = lds_read_tr16_at(tb[dt][0] + off), hi = lds_read_tr16_at(tb[dt][1] + off);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bf16x8 opq[kRA];
#pragma unroll
    for (int j = 0; j < kRA; ++j) opq[j] = qt_op(j);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 ud[4];
    auto dstep = [&](int g, int e2) {
      const int sub = g >> 1, k2 = g & 1, e = 2 * e2;
      const float p0 = __uint_as_float(pv[g][e2] << 16), p1 = __uint_as_float(pv[g][e2] & 0xffff0000u);
      ud[g][e2] = pack_bf16x2(p0 * dp[sub][8 * k2 + e], p1 * dp[sub][8 * k2 + e + 1]);
    };
    // Group g's dS: rows 16*k2 + 8*hh .. +7 of unit `sub`, at ((k2*128 +
    // key)*16 + 8*hh) bf16 into the unit.
    auto ds_store = [&](int g) {
      const int sub = g >> 1, k2 = g & 1;
      const u32x4 w = {ud[g][0] & ds_keep, ud[g][1] & ds_keep, ud[g][2] & ds_keep, ud[g][3] & ds_keep};
      const uint32_t unit_off = (sub ? ds_unit1 : 0u) + (uint32_t)k2 * 4096;  // = DsUnit::store_offset
      if (CT)
        store_b128_nt(rds, ds_voff + unit_off, 0u, w);  // the whole offset range-checked
      else
        store_b128_nt(rds, ds_voff, unit_off, w);
    };
#pragma unroll
    for (int e2 = 0; e2 < 4; ++e2) dstep(0, e2);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int g = j / DT, dt = j % DT;
      const bf16x8 op = opq[j % kRA];
      if (j + kRA < NJ) opq[j % kRA] = qt_op(j + kRA);
      acc[dt] = mfma32(op, bits_to_bf16x8(ud[g]), acc[dt]);
      if (g + 1 < 4) {
        // the next group's 4 steps, spread over this group's DT MFMAs
        for (int st = dt * 4 / DT; st < (dt + 1) * 4 / DT; ++st) dstep(g + 1, st);
      }
      if constexpr (STAGE) {
        if (dt == 0) ds_store(g);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  retire_prologue_loads();
  if (niter > 0 && role == 0) {  // niter is 0 when no window meets this block's keys
#pragma unroll
    for (int i = 0; i < kROps; ++i) r_op(0, tile_rsrc(0), sm.rs[0], i);
#pragma unroll
    for (int i = 0; i < kROps; ++i) r_op(min(1, niter - 1), tile_rsrc(min(1, niter - 1)), sm.rs[1], i);
  } else if (niter > 0) {
#pragma unroll
    for (int i = 0; i < kQOps; ++i) q_op(tile_rsrc(0), sm.q[0], i);
  }
  // Tile it lives in slot it % 3 (Q, rows and P hand-over); the loops are
  // unrolled by 3 so that every slot is a compile-time constant.  Every wave
  // passes one barrier per tile (T) and one after the last (F).
  if (niter > 0 && role == 0) {
    for (int it0 = 0;; it0 += 3) {
      const bool more = unrolled_while<3>([&](auto uc) {
        body_p(it0 + uc, uc);
        return it0 + uc + 1 < niter;
      });
      if (!more) break;
    }
    barrier_lds();  // F: the last tile's P handed over
  } else if (niter > 0) {
    // dP of tile it (slot it % 3), kept for the tile's dS phase in the next
    // iteration.
    f32x16 dpb[3][2];
    DsEntry ent{0, 0, 0};  // compact layout: tile it - 1's entry at the top of iteration it
    // Iterations 0 .. niter: iteration niter has only the last tile's dS
    // phase (its barrier pairs with the P waves' F).
    for (int it0 = 0;; it0 += 3) {
      const bool more = unrolled_while<3>([&](auto uc) {
        constexpr int u = decltype(uc)::value, up = (u + 2) % 3;  // slots of tiles it, it - 1
        const int it = it0 + u;
        // Q(it) landed: issued in iteration it - 1, followed there by the dS
        // stores of tile it - 2 if that iteration had a dS phase.
        if (STAGE && it >= 2)
          wait_vmem_n<kDsStores>();
        else
          wait_vmem_n<0>();
        barrier_lds();  // T: tile it staged, tile it - 1's P handed over
        DsDest dd{{0u, 0u, 0u, 0u}, 0u};
        if (CT && it > 0) dd = ds_dest(it - 1, ent);
        if (it < niter) {
          __builtin_amdgcn_s_setprio(1);
          // Loads: Q of tile it + 1 (the last tile re-loads into a slot
          // nothing reads any more).
          dp_phase(uc, dpb[u], min(it + 1, niter - 1), sm.q[(u + 1) % 3]);
        }
        if (it > 0) {
          __builtin_amdgcn_s_setprio(2);
          ds_phase(it - 1, std::integral_constant<int, up>(), dpb[up], dd);
        }
        if (CT && it < niter) ent = ds_entry(it);
        return it < niter;
      });
      if (!more) break;
    }
  }

  const bool kvalid = SCORE ? ds_keep != 0 : key_valid();
  if (part >= 0) {
    // Unscaled fp32 partial sums (masked keys and keys past the end as 0);
    // dkv_reduce_kernel scales, rounds and rotates their total.
    float* pp = a.split_part +
                ((((int64_t)(bid - nfull) * a.nparts + part) * 2 + role) * BK + kw * 32 + l32) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 w = {0.f, 0.f, 0.f, 0.f};
        if (kvalid) w = f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
        *reinterpret_cast<f32x4*>(pp + dt * 32 + 8 * g + 4 * hh) = w;
      }
  } else if (key < a.Lk) {
    const float sc = role == 0 ? 1.f : a.scale;
    bf16* op = role == 0 ? a.dv + b * a.dvsb + hk * a.dvsh + (int64_t)key * a.dvsl
                         : a.dk + b * a.dksb + hk * a.dksh + (int64_t)key * a.dksl;
    // dk of an unrotated key: the rotated key's gradient rounded to bf16,
    // then the transposed rotation (what the reference's autograd does
    // through src/avgen/models/rope.py:332-338).
    const bool rot = role == 1 && a.cos_k != nullptr;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 w = {0u, 0u};
        if (kvalid) {
          w[0] = pack_bf16x2(acc[dt][4 * g] * sc, acc[dt][4 * g + 1] * sc);
          w[1] = pack_bf16x2(acc[dt][4 * g + 2] * sc, acc[dt][4 * g + 3] * sc);
          if (rot) {
            // channels dt*32 + 8g + 4hh .. +3: pairs (that)/2 and +1
            const int64_t t = b * a.rksb + (int64_t)key * (D / 2) + 16 * dt + 4 * g + 2 * hh;
            const f32x2 c2 = *reinterpret_cast<const f32x2*>(a.cos_k + t);
            const f32x2 s2 = *reinterpret_cast<const f32x2*>(a.sin_k + t);
            w = rotate4(w, c2[0], s2[0], c2[1], s2[1], true);
          }
        }
        *reinterpret_cast<u32x2*>(op + dt * 32 + 8 * g + 4 * hh) = w;
      }
  }
}

}  // namespace avattn
