// Attention forward over a cache of pages (PageTable), bf16 or e4m3 with an
// exponent per page and head.
//
// Few query rows per kv head (a decode step, drafted tokens, a piece of a prompt;
// paged_plan): the few-row forward
// of attn_few.hip, whose waves stage their 32-key tiles from two runs of 16 slots
// each, since a page is a multiple of 16.  The entries of the block table and the
// exponents are read for 32 tiles at once, a lane each half tile, so that they add
// a latency per 32 tiles.  e4m3 codes stay codes in LDS (half the bytes, two workgroups
// on a CU) and become bf16 on the way into the MFMAs, c 2^e exactly: K as 16
// bytes of a key's row, V by transposed 8-bit reads.  HBM-bound: the pages are
// read once.
// More rows: the pages are copied once into the general forward's operands (K
// rows, V^T, in bf16), which costs 3 bytes per code next to 4 x rows x channels
// operations.
#include "attn_few_parts.h"

namespace avattn {

namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));

// Eight codes times `scale`, a power of two: exact in bf16.
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return bits_to_bf16x8(u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                              __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)});
}
__device__ __forceinline__ float exponent_scale(int e) {
  return __uint_as_float((uint32_t)(127 + max(e, -126)) << 23);
}

// Eight bytes of a transposed LDS read (ds_read_b64_tr_b8): in each group of 16
// lanes, lane i supplies the address of 8 consecutive bytes, the piece (i % 2) of
// row i / 2 of an 8 x 16 block, and lane j receives byte j of rows 0..7 (checked
// on the GPU).
__device__ __forceinline__ i32x2 lds_read_tr8(const bf16* p) {
  typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(const_cast<bf16*>(p)));
}

// A value that is the same in the whole wave, by a scalar load.
__device__ __forceinline__ int load_uniform(const int* p) {
  return *(const __attribute__((address_space(4))) int*)p;
}
// A sequence's tokens and how many of them are the call's; `uniform`: b is the
// whole wave's.
struct PagedSequence {
  int len, count;
  __device__ __forceinline__ PagedSequence(const PagedArgs& p, int b, bool uniform = false) {
    len = max(uniform ? load_uniform(p.lengths + b) : p.lengths[b], 0);
    count = p.few.Lq;
    if (p.counts) count = min(max(uniform ? load_uniform(p.counts + b) : p.counts[b], 0), count);
  }
};
// A query's position and keys.
struct PagedRow {
  int pos, lo, hi;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& p, const PagedSequence& s, int i) {
  const int pos = (int)((unsigned)(s.len - s.count) + (unsigned)i);
  PagedRow r{pos, 0, 0};                // (a row behind the last one: any position)
  if (i >= s.count || pos < 0) return r;
  r.hi = pos < p.few.Lk ? pos + 1 : p.few.Lk;
  r.lo = p.window > 0 ? min(max(pos - p.window + 1, 0), r.hi) : 0;
  return r;
}

// The hull of the keys of rows i0 .. i1 (a block's), whose windows never move
// back, and the keys that all of them see.
__device__ __forceinline__ void paged_hull(const PagedArgs& p, const PagedSequence& s, int i0, int i1,
                                           BlockWindows& w) {
  w.glo = w.ghi = w.all_lo = w.all_hi = 0;
  if (i0 >= s.count) return;
  const PagedRow first = paged_row(p, s, i0), last = paged_row(p, s, min(i1, s.count - 1));
  w.ghi = last.hi;
  w.glo = min(first.lo, last.hi);
  w.all_lo = last.lo;
  w.all_hi = i1 < s.count ? first.hi : 0;
}

template <int D, bool FP8>
__global__ __launch_bounds__(256, FP8 || D == 64 ? 2 : 1) void attn_paged_kernel(PagedArgs p) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int RL = FP8 ? D / 2 : D, TE = kTile * RL;  // rows and tiles, in 2-byte units
  const FewArgs& a = p.few;
  struct Stage {
    bf16 k[TE];  // rows: TileLayout<RL>
    bf16 v[TE];
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
  const PagedSequence seq(p, b, true);
  const int group = a.Hq / a.Hkv;
  const int rows = min(a.Lq * group - rb * kTile, kTile);  // of this block
  const bool valid = l32 < rows;
  const RowPlace rp = row_place(a, hk, rb * kTile + (valid ? l32 : 0));
  // This lane's row of Q: per 16-channel step channels 16*ks + 8*hh + [0, 8); with
  // codes, whose rows are read 16 bytes at a time, 32*(ks/2) + 16*hh + 8*(ks%2).
  bf16x8 qf[KS];
  {
    const bf16* qp = static_cast<const bf16*>(a.q) + b * a.qsb + rp.h * a.qsh + (int64_t)rp.i * a.qsl;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (valid)
        x = *reinterpret_cast<const u32x4*>(qp + (FP8 ? 32 * (ks / 2) + 16 * hh + 8 * (ks % 2) : 16 * ks + 8 * hh));
      qf[ks] = bits_to_bf16x8(x);
    }
  }
  RowBias rbias{{0, 0}, 0.f, 0.f, 0};
  if (a.score.slopes != nullptr) {
    rbias.slope = a.score.slopes[rp.h];
    rbias.slope2 = rbias.slope * kLog2e;
  }
  const PagedRow pr = paged_row(p, seq, rp.i);
  BlockWindows w{pr.lo, pr.hi, 0, 0, 0, 0};
  paged_hull(p, seq, rb * kTile / group, (rb * kTile + rows - 1) / group, w);

  // Tiles of this wave: the block's tiles, a range per workgroup, every
  // fourth of it per wave.
  const int tile0 = w.glo / kTile, ntile = w.ghi > w.glo ? (w.ghi + kTile - 1) / kTile - tile0 : 0;
  const int each = ntile / a.nsplit, more = ntile % a.nsplit;
  const int first = tile0 + each * split + min(split, more);
  const int t0 = first + wave, t1 = first + each + (split < more);

  TileStager<16, RL, 1> rows16;  // both tensors' slots are D apart
  rows16.init(RL, 0, lane);
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int kLoads = 4 * decltype(rows16)::kPer;  // of a stage
  const char* kp = static_cast<const char*>(p.kp) + hk * p.kph * ES;
  const char* vp = static_cast<const char*>(p.vp) + hk * p.vph * ES;
  // The pages of 32 of the wave's tiles at once, batch n: lane 2i + g has that of
  // slots 16*g .. + 15 of tile t0 + kWaves*(32n + i) (-1: none of them is looked
  // at, or the entry names no page) and its exponents.  A batch is loaded when its
  // first tile is staged, before the last batch's last tile is computed.
  int page = -1, ke = 0, ve = 0, old_ke = 0, old_ve = 0;
  auto load_batch = [&](int n) {
    const int key0 = (t0 + kWaves * (32 * n + (lane >> 1))) * kTile + 16 * (lane & 1);
    const bool in = key0 < w.ghi && key0 + 16 > w.glo;
    const int entry = p.pages.table[b * p.pages.tsb + (in ? key0 >> p.pages.shift : 0)];
    page = in && entry >= 0 && entry < p.pages.pages ? entry : -1;
  };
  auto load_exponents = [&] {
    if constexpr (FP8) {
      old_ke = ke, old_ve = ve;
      const int64_t at = page < 0 ? 0 : page;
      ke = p.ke[at * p.kes + hk], ve = p.ve[at * p.ves + hk];
    }
  };
  // Stages the wave's tile i (of this batch, at t); returns which of its keys have
  // a page.
  auto stage = [&](int i, int t, Stage& sg) {
    uint32_t has = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int pg = __builtin_amdgcn_readlane(page, 2 * (i % 32) + g);
      const int64_t at = pg < 0 ? 0 : pg;
      const int slot = (t * kTile + 16 * g) & ((1 << p.pages.shift) - 1);
      const uint32_t bytes = pg < 0 ? 0u : 16u * D * ES;  // no page: zeros
      has |= pg < 0 ? 0u : 0xffffu << (16 * g);
      rows16.stage(sg.k + 16 * g * RL, make_rsrc(kp + (at * p.kps + slot * D) * ES, bytes), 0u);
      rows16.stage(sg.v + 16 * g * RL, make_rsrc(vp + (at * p.vps + slot * D) * ES, bytes), 0u);
    }
    return has;
  };

  float m = kNegInf, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();

  // Two tiles of the wave are in flight: while one is computed the other, then
  // both.
  uint32_t has = 0, has_next = 0;
  load_batch(0);
  retire_prologue_loads();
  if (t0 < t1) has = stage(0, t0, sm.st[wave][0]);
  if (t0 + kWaves < t1) has_next = stage(1, t0 + kWaves, sm.st[wave][1]);
  load_exponents();  // (behind the tiles, which wait for the table's entries only)
  if (a.score.slopes != nullptr) rbias.measure(pr.pos, pr.lo, pr.hi);
  const int qpos = rbias.at.pos;
  const float slope2 = rbias.slope2, ref = (float)rbias.at.ref;
  for (int t = t0, i = 0; t < t1; t += kWaves, ++i) {
    Stage& sg = sm.st[wave][i & 1];
    // This tile's rows; the next one's may be on the way.
    if (t + kWaves < t1)
      wait_vmem_n<kLoads>();
    else
      wait_vmem_n<0>();
    uint32_t keys = has;
    float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;
    if constexpr (FP8) {
      const bool old = i % 32 == 31 && t + kWaves < t1;
      const int ek = old ? old_ke : ke, ev = old ? old_ve : ve, lane0 = 2 * (i % 32);
      ks0 = exponent_scale(__builtin_amdgcn_readlane(ek, lane0));
      ks1 = exponent_scale(__builtin_amdgcn_readlane(ek, lane0 + 1));
      vs0 = exponent_scale(__builtin_amdgcn_readlane(ev, lane0));
      vs1 = exponent_scale(__builtin_amdgcn_readlane(ev, lane0 + 1));
    }
    {
      const int from = w.glo - t * kTile, to = w.ghi - t * kTile;
      if (from > 0) keys &= 0xffffffffu << from;  // from < 32: the tile meets the window
      if (to < 32) keys &= ~(0xffffffffu << to);
    }
    if (keys != 0xffffffffu) {
      // What a slot without a token holds must not reach the rows through 0 * NaN.
#pragma unroll
      for (int i = 0; i < TE / 8 / 64; ++i) {
        const int c = i * 64 + lane, row = c / (RL / 8);
        if (!(keys >> row & 1))
          *reinterpret_cast<u32x4*>(sg.v + TileLayout<RL>::off(row, 8 * (c % (RL / 8)))) = u32x4{};
      }
    }
    // Register 8*k2 + e of lane l: key 16*k2 + 8*hh + e of the tile, row l32.
    f32x16 s = zero16();
    if constexpr (FP8) {
      const float ksc = l32 & 16 ? ks1 : ks0;
#pragma unroll
      for (int j = 0; j < KS / 2; ++j) {
        const u32x4 c = *reinterpret_cast<const u32x4*>(sg.k + TileLayout<RL>::off(prow, 16 * j + 8 * hh));
        s = mfma32(codes_to_bf16(c[0], c[1], ksc), qf[2 * j], s);
        s = mfma32(codes_to_bf16(c[2], c[3], ksc), qf[2 * j + 1], s);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = mfma32(row_operand<D>(sg.k, prow, 16 * ks + 8 * hh), qf[ks], s);
    }
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
    // The reference maximum moves only for a score 2^8 above it; both lanes of a
    // row agree.
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
        // The PV operand in bf16, as in the general forward: wider products run at
        // a fraction of the rate, and of the result's relative error of
        // 0.0020 the output's own rounding is 0.0017.  The sum takes the unrounded ones.
        u[e2] = pack_bf16x2(p0, p1);
      }
      pf[k2] = bits_to_bf16x8(u);
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if constexpr (FP8) {
          const int row = 8 * hh + ((lane & 15) >> 1), col = 16 * dt + 8 * ((lane >> 4) & 1) + 4 * (lane & 1);
          const i32x2 c = lds_read_tr8(sg.v + TileLayout<RL>::off(row, col) + 16 * k2 * RL);
          acc[dt] = mfma32(codes_to_bf16((uint32_t)c[0], (uint32_t)c[1], k2 ? vs1 : vs0), pf[k2], acc[dt]);
        } else {
          const bf16x4 lo = lds_read_tr16(sg.v + tr_read_off<D>(lane, dt, 0) + 16 * k2 * D);
          const bf16x4 hi = lds_read_tr16(sg.v + tr_read_off<D>(lane, dt, 1) + 16 * k2 * D);
          acc[dt] = mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[k2], acc[dt]);
        }
      }
    has = has_next;
    if (t + 2 * kWaves < t1) {
      if ((i + 2) % 32 == 0) load_batch((i + 2) / 32), load_exponents();
      // The stage's reads have returned before it is filled again.
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      has_next = stage(i + 2, t + 2 * kWaves, sg);
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

// The general forward's operands from pages, as prep_fwd_kernel makes them from k
// and v: workgroups [0, nk) a 64-key tile of K rows with its largest squared row
// norm, then a tile of V^T each, those of kv head 0 also the tile's key bias and
// flags, then the rows' windows and row 0's positions.  Keys outside the hull of a sequence's windows,
// or without a page, are zeros; tiles without a key in the hull are left alone,
// apart from their norm.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void prep_paged_kernel(FwdArgs a, PagedArgs p, int* wlo, int* whi, int* offsets,
                                                         int nk) {
  constexpr int S = 64, CPR = D / 8, LD = D + 2;
  __shared__ bf16 tile[S * LD];
  __shared__ float wmax[4];
  const int nt = a.Lkp / S, tid = threadIdx.x;
  if ((int)blockIdx.x >= 2 * nk) {
    const int64_t u = ((int64_t)blockIdx.x - 2 * nk) * 256 + tid;
    if (u >= (int64_t)a.B * a.Lq) return;
    const int b = (int)(u / a.Lq), i = (int)(u % a.Lq);
    const PagedSequence seq(p, b);
    PagedRow r = paged_row(p, seq, i);
    // Non-decreasing in the row: a row behind the last token ends where it ends.
    if (i >= seq.count && seq.count > 0) r.lo = r.hi = paged_row(p, seq, seq.count - 1).hi;
    wlo[u] = r.lo, whi[u] = r.hi;
    if (offsets != nullptr && i == 0) offsets[b] = r.pos;
    return;
  }
  const bool is_k = (int)blockIdx.x < nk;
  const int u = is_k ? blockIdx.x : blockIdx.x - nk;
  const int t = u % nt, bh = u / nt;
  const int b = bh / a.Hkv, h = bh % a.Hkv, s0 = S * t;
  const PagedSequence seq(p, b, true);
  int lo = 0, hi = 0;
  if (seq.count > 0) lo = paged_row(p, seq, 0).lo, hi = paged_row(p, seq, seq.count - 1).hi;
  if (s0 + S <= lo || s0 >= hi) {
    if (is_k && tid == 0) a.kmax2[(int64_t)bh * nt + t] = 0;
    if (!is_k && h == 0 && tid < 64) {
      a.kbias[(int64_t)b * a.Lkp + s0 + tid] = kNegInf;
      if (tid < 2) a.kfull[(int64_t)b * (a.Lkp / 32) + s0 / 32 + tid] = 0;
    }
    return;
  }
  const char* base = static_cast<const char*>(is_k ? p.kp : p.vp);
  const int64_t ps = is_k ? p.kps : p.vps, hs = is_k ? p.kph : p.vph, es = is_k ? p.kes : p.ves;
  const int8_t* ex = is_k ? p.ke : p.ve;
  auto page_of = [&](int key) { return key >= lo && key < hi ? p.pages.page(b, key >> p.pages.shift) : -1; };
  bf16* xr = a.kr + ((int64_t)bh * a.Lkp + s0) * D;
  float nmax = 0.f;
#pragma unroll
  for (int i = 0; i < S * CPR / 256; ++i) {
    const int c = tid + i * 256, row = c / CPR, ch = c % CPR, key = s0 + row;
    const int page = page_of(key);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (page >= 0) {
      const int64_t at = page * ps + h * hs + (key & ((1 << p.pages.shift) - 1)) * D + 8 * ch;
      if constexpr (FP8) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(base + at);
        v = bf16x8_to_bits(codes_to_bf16(x[0], x[1], exponent_scale(ex[page * es + h])));
      } else {
        v = *reinterpret_cast<const u32x4*>(base + 2 * at);
      }
    }
    if (is_k) {
      *reinterpret_cast<u32x4*>(xr + row * D + ch * 8) = v;
      float n = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) n = fmaf(bf16_lo(v[w]), bf16_lo(v[w]), fmaf(bf16_hi(v[w]), bf16_hi(v[w]), n));
#pragma unroll
      for (int off = 1; off < CPR; off <<= 1) n += __shfl_xor(n, off);
      nmax = fmaxf(nmax, n);
    } else {
      uint32_t* dst = reinterpret_cast<uint32_t*>(tile + row * LD + ch * 8);
#pragma unroll
      for (int w = 0; w < 4; ++w) dst[w] = v[w];
    }
  }
  if (is_k) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) nmax = fmaxf(nmax, __shfl_xor(nmax, off));
    if ((tid & 63) == 0) wmax[tid >> 6] = nmax;
    __syncthreads();
    if (tid == 0)
      a.kmax2[(int64_t)bh * nt + t] = __float_as_uint(fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3])));
    return;
  }
  if (h == 0 && tid < 64) {
    const uint64_t has = __builtin_amdgcn_ballot_w64(page_of(s0 + tid) >= 0);
    a.kbias[(int64_t)b * a.Lkp + s0 + tid] = has >> tid & 1 ? 0.f : kNegInf;
    if (tid < 2) a.kfull[(int64_t)b * (a.Lkp / 32) + s0 / 32 + tid] = (uint32_t)(has >> (32 * tid)) == 0xffffffffu;
  }
  __syncthreads();
  bf16* xt = a.vt + (int64_t)bh * D * a.Lkp + s0;
#pragma unroll
  for (int i = 0; i < D * (S / 8) / 256; ++i) {
    const int c = tid + i * 256, d = c / (S / 8), j = c % (S / 8);
    u32x4 v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint16_t x = __builtin_bit_cast(uint16_t, tile[(8 * j + 2 * w) * LD + d]);
      const uint16_t y = __builtin_bit_cast(uint16_t, tile[(8 * j + 2 * w + 1) * LD + d]);
      v[w] = (uint32_t)x | ((uint32_t)y << 16);
    }
    *reinterpret_cast<u32x4*>(xt + (int64_t)d * a.Lkp + 8 * j) = v;
  }
}

}  // namespace

// Few rows or many: the smaller of two estimates, both for sequences that fill
// their room (us, few-row against general):
//   e4m3, 32 heads over 8 of 128, 12,000 keys: 33 tokens 27, 64; 128 54, 68; 192 86, 70; 512 164, 105
//   the same twice: 96 tokens 89, 102; 192 140, 109; bf16: 64 tokens 88, 110; 96 128, 113
//   bf16, eight sequences of 4,000: 48 tokens 130, 136; 96 160, 141; of 1,000: 64 49, 39
//   e4m3, 64 heads over 8, 1,000 keys: 96 tokens 18, 31; 256 23, 33; 512 39, 34
//   e4m3, 16 heads over 2 of 64, 12,000 keys: 128 tokens 33, 41; 192 44, 43; 512 82, 49
// Of 576 such shapes (1 to 16 sequences, alike, of a quarter of their room on, or with
// windows; up to 512 tokens, both types) the slower way is taken at 17 by 5 to 25 %.  Near
// the crossing nine of ten estimates are within a quarter of what was measured.
// The few-row kernel computes no row that is not there (its blocks hold rows of all
// heads of a kv head) and needs no copy; the general one has twice its rate.
// Its split n of a block's keys is the fastest by the same estimate: whole rounds
// of workgroups, and no parts to join where the keys are few (128 blocks of 1,000
// keys 18 us, split in 4 19; 304 of 6,000 keys 88 whole, 72 in 3).
FewPlan paged_plan(int B, int Hq, int Hkv, int Lq, int64_t cap, int window, int D, bool fp8) {
  FewPlan p{};
  const int64_t rows = (int64_t)Lq * (Hq / Hkv);
  if (cap < 1) return p;
  const int64_t reach = window > 0 && (int64_t)window + Lq - 1 < cap ? (int64_t)window + Lq - 1 : cap;
  p.block_rows = (int)(rows < kTile ? rows : kTile);
  p.row_blocks = (int)((rows + kTile - 1) / kTile);
  const int64_t units = (int64_t)B * Hkv * p.row_blocks;
  constexpr int64_t kCus = 256, kMaxGrid = (1 << 24) - 1;
  if (units > kMaxGrid || units * p.block_rows > kMaxGrid) return FewPlan{};
  // Workgroups per CU, a wave's tile among them (and 0.7 of it with a CU to itself).
  const int per_cu = D == 128 && !fp8 ? 1 : 2;
  const float tile_us = D == 64 ? 1.6f : (fp8 ? 1.9f : 1.5f);
  const float slot_bytes = 4.f * few_slot_floats(p.block_rows, D);
  const int64_t slots = kCus * per_cu, tiles = reach / kTile + 1, most = (tiles + kWaves - 1) / kWaves;
  // A call's time with n parts, its sequences holding `filled` of their room on the
  // mean and the longest all of it.
  auto estimate = [&](int64_t n, float filled) {
    const int64_t grid = units * n, rem = grid % slots;
    const int64_t mine = ((tiles + n - 1) / n + kWaves - 1) / kWaves;
    float us;
    if (B == 1) {
      const float rounds = (float)(grid / slots) + (rem == 0 ? 0.f : (rem <= kCus && per_cu > 1 ? 0.7f : 1.f));
      us = rounds * (mine * tile_us + 4.f);
    } else {
      const float longest = mine * tile_us * (grid <= kCus && per_cu > 1 ? 0.7f : 1.f) + 5.f;
      const float mean = (float)grid / slots * (mine * tile_us * filled + 5.f) + 0.4f * longest;
      us = longest > mean ? longest : mean;
    }
    return 0.88f * (us + 6.f + (n > 1 ? 3.f + grid * slot_bytes * 2.f / 3.5e6f : 0.f));
  };
  // The workgroups of a batch's longest sequences end last, so more rounds of smaller
  // ones pay (16 sequences of 1,016 to 16,001 keys 126 us in one round, 106 in two; e4m3
  // 77, 66; alike ones 104, 107).
  const float filled = window > 0 ? 1.f : 0.75f;
  float best = 0.f;
  auto consider = [&](int64_t n) {
    if (n > most) n = most;
    if (n < 1 || units * n > kMaxGrid) return;
    const float us = estimate(n, filled);
    if (p.nsplit == 0 || us < best) best = us, p.nsplit = (int)n;
  };
  consider(1);
  for (int64_t r = 1; r <= 4; ++r) consider(r * slots / units);  // whole rounds
  if (per_cu > 1) consider(kCus / units);
  // Against three launches, the copy of the pages (from and to caches in part) and the
  // general forward, both for sequences that fill their room.  Two workgroups on a CU
  // fill each other's waits over a batch's many rounds; bf16 rows of 128 run into the
  // caches' rate, each block reading all pages, though of a batch's shorter sequences less,
  // while the general forward's time is that of the longest (four sequences of 3,000 to
  // 12,000 keys, 64 tokens: 158 in place, 188; all of 12,000: 228, 212).
  const float rate = per_cu == 1 ? (B == 1 ? 1.16f : 1.04f) : (B == 1 ? 1.f : (D == 64 ? 0.82f : 0.78f));
  const float copy = (float)(B * Hkv) * (float)reach * D * 2.f * (fp8 ? 3.f : 4.f) / 9e6f;
  const float forward = fwd_split_plan(B, Hq, Lq, (int)reach, D, false, false).us;
  const float general = 18.f + copy + 0.65f * (forward > 14.f ? forward : 14.f);
  if (rows > kFewRows && general < rate * estimate(p.nsplit, 1.f)) return FewPlan{};
  p.bytes = p.nsplit > 1 ? (size_t)units * p.nsplit * few_slot_floats(p.block_rows, D) * sizeof(float) : 0;
  return p;
}

hipError_t launch_paged_few(const PagedArgs& args, const FewPlan& plan, int D, hipStream_t stream) {
  PagedArgs p = args;
  FewArgs& a = p.few;
  a.nsplit = plan.nsplit;
  a.row_blocks = plan.row_blocks;
  a.block_rows = plan.block_rows;
  const dim3 grid((unsigned)(a.B * a.Hkv * plan.row_blocks * plan.nsplit));
  {
    LaunchTimer timer(kKidFwdPaged, stream);
    const bool fp8 = p.ke != nullptr;
    if (D == 128 && fp8)
      hipLaunchKernelGGL((attn_paged_kernel<128, true>), grid, dim3(256), 0, stream, p);
    else if (D == 128)
      hipLaunchKernelGGL((attn_paged_kernel<128, false>), grid, dim3(256), 0, stream, p);
    else if (fp8)
      hipLaunchKernelGGL((attn_paged_kernel<64, true>), grid, dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL((attn_paged_kernel<64, false>), grid, dim3(256), 0, stream, p);
  }
  if (plan.nsplit > 1) launch_few_combine(a, D, stream);
  return hipGetLastError();
}

hipError_t launch_prep_paged(const FwdArgs& a, int head_dim, hipStream_t stream) {
  const PagedArgs& p = *a.paged;
  const int64_t nk = (int64_t)a.B * a.Hkv * (a.Lkp / 64), nw = ((int64_t)a.B * a.Lq + 255) / 256;
  if (2 * nk + nw >= (int64_t)1 << 24) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(2 * nk + nw));
  int *wlo = const_cast<int*>(a.wlo), *whi = const_cast<int*>(a.whi);  // written here, read by the forward
  int* offsets = const_cast<int*>(a.score.offsets);
  LaunchTimer timer(kKidPrepPaged, stream);
  const bool fp8 = p.ke != nullptr;
  if (head_dim == 128 && fp8)
    hipLaunchKernelGGL((prep_paged_kernel<128, true>), grid, dim3(256), 0, stream, a, p, wlo, whi, offsets, (int)nk);
  else if (head_dim == 128)
    hipLaunchKernelGGL((prep_paged_kernel<128, false>), grid, dim3(256), 0, stream, a, p, wlo, whi, offsets, (int)nk);
  else if (fp8)
    hipLaunchKernelGGL((prep_paged_kernel<64, true>), grid, dim3(256), 0, stream, a, p, wlo, whi, offsets, (int)nk);
  else
    hipLaunchKernelGGL((prep_paged_kernel<64, false>), grid, dim3(256), 0, stream, a, p, wlo, whi, offsets, (int)nk);
  return hipGetLastError();
}

}  // namespace avattn
