// Attention forward over a cache of pages (PageTable), bf16 or e4m3 with an
// exponent per page and head.
//
// Few query rows per kv head (a decode step, drafted tokens): the few-row forward
// of attn_few.hip, whose waves stage their 32-key tiles from two runs of 16 slots
// each, since a page is a multiple of 16.  The entries of the block table are read
// two tiles ahead of their use and the exponents one, so neither adds a latency
// to the tile's.  e4m3 codes stay codes in LDS (half the bytes, two workgroups
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

// A query's position and keys.
struct PagedRow {
  int pos, lo, hi;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& p, int b, int i) {
  const int len = max(p.lengths[b], 0), count = p.counts ? min(max(p.counts[b], 0), p.few.Lq) : p.few.Lq;
  const int64_t pos = (int64_t)len - count + i;
  PagedRow r{(int)pos, 0, 0};  // (a row behind the last one: any position)
  if (i >= count || pos < 0) return r;
  const int64_t lo = p.window > 0 ? pos - p.window + 1 : 0;
  r.hi = (int)(pos + 1 < p.few.Lk ? pos + 1 : p.few.Lk);
  r.lo = (int)(lo < 0 ? 0 : (lo < r.hi ? lo : r.hi));
  return r;
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
  const int rows = min(a.Lq * (a.Hq / a.Hkv) - rb * kTile, kTile);  // of this block
  const bool valid = l32 < rows;
  const RowPlace rp = row_place(a, hk, rb * kTile + (valid ? l32 : 0));
  const PagedRow pr = paged_row(p, b, rp.i);
  const BlockWindows w = block_windows(pr.lo, pr.hi, valid);

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
    rbias.measure(pr.pos, pr.lo, pr.hi);
  }
  const int qpos = rbias.at.pos;
  const float slope2 = rbias.slope2, ref = (float)rbias.at.ref;

  // Tiles of this wave: the block's tiles, a range per workgroup, every
  // fourth of it per wave.
  const int tile0 = w.glo / kTile, ntile = w.ghi > w.glo ? (w.ghi + kTile - 1) / kTile - tile0 : 0;
  const int t0 = tile0 + (int)((int64_t)ntile * split / a.nsplit) + wave;
  const int t1 = tile0 + (int)((int64_t)ntile * (split + 1) / a.nsplit);

  TileStager<16, RL, 1> rows16;  // both tensors' slots are D apart
  rows16.init(RL, 0, lane);
  constexpr int ES = FP8 ? 1 : 2;
  const char* kp = static_cast<const char*>(p.kp) + hk * p.kph * ES;
  const char* vp = static_cast<const char*>(p.vp) + hk * p.vph * ES;
  // The table entry of slots t*32 + 16*(lane % 2) .. + 15 (-1: none of them is
  // looked at), as loaded: checked where it is used.
  auto load_entry = [&](int t) {
    const int key0 = t * kTile + 16 * (lane & 1);
    if (t >= t1 || key0 >= w.ghi || key0 + 16 <= w.glo) return -1;
    return p.pages.table[b * p.pages.tsb + (key0 >> p.pages.shift)];
  };
  int ke = 0, ve = 0;  // exponents of the staged tile, by lane % 2
  // Stages tile t from pages `entry`; returns which of its keys have a page.
  auto stage = [&](int t, int entry, Stage& sg) {
    if (entry < 0 || entry >= p.pages.pages) entry = -1;
    uint32_t has = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int page = __builtin_amdgcn_readlane(entry, g);
      const int64_t at = page < 0 ? 0 : page;
      const int slot = (t * kTile + 16 * g) & ((1 << p.pages.shift) - 1);
      const uint32_t bytes = page < 0 ? 0u : 16u * D * ES;  // no page: zeros
      has |= page < 0 ? 0u : 0xffffu << (16 * g);
      rows16.stage(sg.k + 16 * g * RL, make_rsrc(kp + (at * p.kps + slot * D) * ES, bytes), 0u);
      rows16.stage(sg.v + 16 * g * RL, make_rsrc(vp + (at * p.vps + slot * D) * ES, bytes), 0u);
    }
    if constexpr (FP8) {
      const int64_t at = entry < 0 ? 0 : entry;
      ke = p.ke[at * p.kes + hk];
      ve = p.ve[at * p.ves + hk];
    }
    return has;
  };

  float m = kNegInf, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();

  retire_prologue_loads();
  uint32_t has = 0;
  int entry = -1;
  if (t0 < t1) {
    entry = load_entry(t0);
    wait_vmem_n<0>();
    has = stage(t0, opaque(entry), sm.st[wave][0]);
    entry = load_entry(t0 + kWaves);
  }
  for (int t = t0, buf = 0; t < t1; t += kWaves, buf ^= 1) {
    Stage& sg = sm.st[wave][buf];
    // Everything in flight belongs to this tile (its rows, its exponents) or is
    // the next one's table entry.
    wait_vmem_n<0>();
    uint32_t keys = has;
    const int next = opaque(entry);
    float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;
    if constexpr (FP8) {
      const int ek = opaque(ke), ev = opaque(ve);
      ks0 = exponent_scale(__builtin_amdgcn_readlane(ek, 0)), ks1 = exponent_scale(__builtin_amdgcn_readlane(ek, 1));
      vs0 = exponent_scale(__builtin_amdgcn_readlane(ev, 0)), vs1 = exponent_scale(__builtin_amdgcn_readlane(ev, 1));
    }
    if (t + kWaves < t1) {
      // The other stage's reads have returned before it is filled again.
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      has = stage(t + kWaves, next, sm.st[wave][buf ^ 1]);
      entry = load_entry(t + 2 * kWaves);
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
        if (!(keys >> row & 1)) *reinterpret_cast<u32x4*>(sg.v + TileLayout<RL>::off(row, 8 * (c % (RL / 8)))) = u32x4{};
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
        u[e2] = pack_bf16x2(p0, p1);  // the PV operand, rounded as in the general forward
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
    PagedRow r = paged_row(p, b, i);
    const int count = p.counts ? min(max(p.counts[b], 0), a.Lq) : a.Lq;
    // Non-decreasing in the row: a row behind the last token ends where it ends.
    if (i >= count && count > 0) r.lo = r.hi = paged_row(p, b, count - 1).hi;
    wlo[u] = r.lo, whi[u] = r.hi;
    if (offsets != nullptr && i == 0) offsets[b] = r.pos;
    return;
  }
  const bool is_k = (int)blockIdx.x < nk;
  const int u = is_k ? blockIdx.x : blockIdx.x - nk;
  const int t = u % nt, bh = u / nt;
  const int b = bh / a.Hkv, h = bh % a.Hkv, s0 = S * t;
  const int count = p.counts ? min(max(p.counts[b], 0), a.Lq) : a.Lq;
  int lo = 0, hi = 0;
  if (count > 0) lo = paged_row(p, b, 0).lo, hi = paged_row(p, b, count - 1).hi;
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

FewPlan paged_plan(int B, int Hq, int Hkv, int Lq, int64_t cap, int window, int D, bool fp8) {
  FewPlan p{};
  const int64_t rows = (int64_t)Lq * (Hq / Hkv);
  if (cap < 1 || !(Lq <= kFewQueries || rows <= kFewRows)) return p;
  int64_t reach = window > 0 && (int64_t)window + Lq - 1 < cap ? (int64_t)window + Lq - 1 : cap;
  p.block_rows = (int)(rows < kTile ? rows : kTile);
  p.row_blocks = (int)((rows + kTile - 1) / kTile);
  const int64_t units = (int64_t)B * Hkv * p.row_blocks;
  const int64_t slots = D == 128 && !fp8 ? 256 : 512;
  const int64_t tiles = reach / kTile + 1, most = (tiles + kWaves - 1) / kWaves;
  int64_t n = units < slots ? slots / units : 1;
  if (n > most) n = most;
  p.nsplit = (int)n;
  constexpr int64_t kMaxGrid = (1 << 24) - 1;
  if (units * p.nsplit > kMaxGrid || units * p.block_rows > kMaxGrid) return FewPlan{};
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
