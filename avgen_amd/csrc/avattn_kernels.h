// Kernel argument blocks and launchers shared between the kernel files and
// the C-ABI layer.  All strides are in elements; head_dim is contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "avattn_device.h"

namespace avattn {

// Mark in the sign bit of a kmax2 entry (see FwdArgs).
constexpr uint32_t kTileSkip = 0x80000000u;

// Scores changed before the softmax: z = cap tanh(s / cap) (kScoreCap), then
// z - slopes[hq] * |position of the query - key| (kScoreDistance, see BiasRef),
// s = scale q.k; query i of batch b at position i + query_offset(b).  cap2 = cap
// * log2(e); cap_x = scale / cap; cap_arg = 2 log2(e) cap_x, so that
// exp2(cap_arg * q.k) is e^(2 s / cap).  slopes null: none (0).
constexpr int kScoreCap = 1, kScoreDistance = 2;
struct ScoreArgs {
  int mode;
  float cap2, cap_arg, cap_x;
  const float* slopes;
  const int* offsets;  // per batch (null: offset)
  int offset;
  __device__ __forceinline__ int query_offset(int b) const { return offsets ? offsets[b] : offset; }
};

// The bias of a row is measured from that of the key it favours most, since in
// fp32 slope * distance rounds the scores away long before the distances end (a
// query 2^20 behind its keys, slope 1/2: scores in steps of 1/16).  With the
// row's position p and its keys [lo, hi), pos is p moved into them, so that
// |p - j| = |p - pos| + |pos - j| for every key j; what is subtracted from a
// score is slope (|pos - j| - ref) >= 0, with ref 0 for a slope >= 0 (the nearest
// key has no bias) and pos's largest distance for one below (the farthest has
// none).  Integers until the difference is formed.  slope (|p - pos| + ref) is
// the constant that this leaves out: it moves the row's logsumexp, nothing else
// (bias_distance: the bracket).
// Keys: the row's window (every key without windows), with a key mask those of
// them between the first and the last 64-key tile with an attended key.
struct BiasRef {
  int pos, ref;
};
__device__ __forceinline__ BiasRef bias_ref(int p, int lo, int hi, bool farthest) {
  const int last = max(hi - 1, lo), pos = min(max(p, lo), last);
  return {pos, farthest ? max(pos - lo, last - pos) : 0};
}
__device__ __forceinline__ uint32_t bias_distance(int p, const BiasRef& r) {
  return (p < r.pos ? (uint32_t)r.pos - (uint32_t)p : (uint32_t)p - (uint32_t)r.pos) + (uint32_t)r.ref;
}
// The logsumexp of a row's scores from that of what the kernels compute, and
// back.
__device__ __forceinline__ float lse_of_scores(float lse, float slope, uint32_t distance) {
  return (float)((double)lse - (double)slope * (double)distance);
}
__device__ __forceinline__ float lse_from_scores(float lse, float slope, uint32_t distance) {
  return (float)((double)lse + (double)slope * (double)distance);
}

// The keys [lo, hi) from the first to the last 64-key tile with an attended key of
// a mask over n keys, as a wave of a group of `threads` sees it whose threads
// look at every threads-th key (none: lo large, hi 0).
__device__ __forceinline__ void attended_share(const uint8_t* mask, int n, int thread, int threads, int& lo, int& hi) {
  constexpr int U = 16;  // loads in flight
  lo = 0x7fffffff, hi = 0;
  for (int j0 = thread; j0 < n; j0 += U * threads) {
    uint8_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = j0 + u * threads < n ? mask[j0 + u * threads] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v[u] != 0) lo = min(lo, j0 + u * threads), hi = j0 + u * threads + 1;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
  lo = __builtin_amdgcn_readfirstlane(lo) & ~63;
  hi = min((__builtin_amdgcn_readfirstlane(hi) + 63) & ~63, n);
}
// A row's keys [lo, hi) without those outside that hull.
__device__ __forceinline__ void within_hull(int hull_lo, int hull_hi, int& lo, int& hi) {
  lo = max(lo, min(hull_lo, hull_hi));
  hi = max(min(hi, hull_hi), lo);
}
// The hull (0, n: not needed, it would change no row) for the rows of a wave, a
// row per lane at position p with keys [lo, hi): looked for where a slope is
// negative or a row's pos is masked.  The whole wave calls it.
__device__ __forceinline__ void rows_hull(const uint8_t* mask, int n, float slope, int p, int lo, int hi, int& hull_lo,
                                          int& hull_hi) {
  hull_lo = 0, hull_hi = n;
  if (mask == nullptr) return;
  const bool look = slope < 0.f || (lo < hi && mask[bias_ref(p, lo, hi, false).pos] == 0);
  if (__builtin_amdgcn_ballot_w64(look) == 0) return;
  attended_share(mask, n, threadIdx.x & 63, 64, hull_lo, hull_hi);
}

// 1 / (1 + exp2(arg s)) = (1 - tanh(s / cap)) / 2, in [0, 1].
__device__ __forceinline__ float cap_complement(float s, float arg) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * arg));
}

// The float32 kernels' changed score, in log2 units, from a raw one; d: the key's
// distance from the row's pos, less its ref (BiasRef); f = 1 - tanh^2 (1 without a cap).  tanh to a few
// units in the last place, small arguments too: below 0.35 its odd series to
// x^11 (the next term is below 2^-26), above it 1 - 2 r with r = 1 / (1 +
// e^2|x|), and then 1 - tanh^2 = 4 r (1 - r).
__device__ __forceinline__ float changed_score_exact(const ScoreArgs& a, float s, float scale_log2, float d,
                                                     float slope2, float& f) {
  float z = s * scale_log2;
  f = 1.f;
  if (a.mode & kScoreCap) {
    const float x = s * a.cap_x, x2 = x * x, ax = fabsf(x);
    const float series =
        x * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -8.8632355e-3f, 2.1869488e-2f), -5.3968254e-2f), 1.3333334e-1f),
                          -3.3333334e-1f),
                 1.f);
    const float r = cap_complement(ax, 2.f * kLog2e);
    const bool small = ax < 0.35f;
    const float t = small ? series : copysignf(fmaf(-2.f, r, 1.f), x);
    f = small ? fmaf(-t, t, 1.f) : 4.f * r * (1.f - r);
    z = a.cap2 * t;
  }
  return fmaf(-slope2, d, z);
}

// The keys [lo, hi) of batch b outside which no query row's window reaches:
// from `hull` (two ints per batch) where given, else the first row's lo and
// the last row's hi (windows non-decreasing in the row), clamped into
// 0 <= lo <= hi <= Lk; every key without windows.
__device__ __forceinline__ void key_hull(const int* hull, const int* wlo, const int* whi, int64_t wsb, int b, int Lq,
                                         int Lk, int& lo, int& hi) {
  lo = 0, hi = Lk;
  if (hull != nullptr) {
    lo = hull[2 * b], hi = hull[2 * b + 1];
  } else if (wlo != nullptr) {
    lo = wlo[b * wsb], hi = whi[b * wsb + Lq - 1];
  }
  lo = min(max(lo, 0), Lk);
  hi = min(max(hi, lo), Lk);
}

struct PagedArgs;

struct FwdArgs {
  const bf16* q;
  const bf16* k;
  const bf16* v;
  int64_t qsb, qsh, qsl;
  int64_t ksb, ksh, ksl;
  int64_t vsb, vsh, vsl;
  int B, Hq, Hkv, Lq, Lk;
  const uint8_t* mask;
  int64_t msb;
  const float* cos_q;
  const float* sin_q;
  int64_t rsb;
  float scale;       // softmax scale applied to q.k
  float scale_log2;  // scale * log2(e)
  bf16* o;
  int64_t osb, osh, osl;
  float* lse;
  // Padded copies (prep.hip), written by the launcher: k rows, element
  // (b, h, j, d) at ((b*Hkv + h)*Lkp + j)*D + d; v head_dim-major, element
  // (b, h, d, j) at ((b*Hkv + h)*D + d)*Lkp + j.
  bf16* kr;
  bf16* vt;
  float* kbias;  // (B, Lkp): 0 attended / -inf
  int* kfull;    // (B, Lkp/32): 1 if every key of the 32-key tile is attended
  int Lkp;
  // fp8 variant only (null otherwise): per-head scales and the e4m3
  // row-major k copy k8 = e4m3(k / k_scale[hk]), element (b, h, j, d) at byte
  // ((b*Hkv + h)*Lkp + j)*D + d.  q is quantized against the softmax
  // constant and k's scale (attn_fwd.hip); q_scale[h] only bounds |q| / 448.
  const float* q_scale;
  const float* k_scale;
  uint8_t* k8;
  // Largest squared row norm of k (bf16 path) or of k8 in e4m3 units (fp8)
  // per 64-key tile, (b, kv head, tile) at ((b*Hkv + h)*(Lkp/64) + tile),
  // float bits (written by the k copy): the largest over a head bounds every
  // score of a query row by |q_row| * sqrt(max).  The sign bit (kTileSkip,
  // bf16 path with a mask only) marks a tile that contributes nothing: no
  // key of it is attended and its k and v are finite.
  uint32_t* kmax2;
  // Key windows (null: every key): query row i of batch b attends to keys
  // [wlo[b*wsb + i], whi[b*wsb + i]) (and the key mask), shared by all heads.
  const int* wlo;
  const int* whi;
  int64_t wsb;
  // K rotation (null: k is used as given): the k copy rotates row j of batch
  // b with the tables (b, 0, j, pair) at b*rksb + j*(D/2) + pair, as q is
  // rotated on load with cos_q/sin_q.
  const float* cos_k;
  const float* sin_k;
  int64_t rksb;
  // Ring step (null o_acc: a plain forward writing o and lse): this chunk's
  // (bf16-rounded output, lse) is merged into the running fp32 accumulator
  // o_acc (B, Hq, Lq, D) contiguous and lse_acc (B, Hq, Lq) with the ring
  // merge (lse_merge_coeffs); acc_first: the accumulator holds nothing yet
  // and takes this chunk's result; acc_final: also write bf16(merged) to o.
  float* o_acc;
  float* lse_acc;
  bool acc_first;
  bool acc_final;
  // Split of the grid's partial last round (null part: none; nsplit and
  // nparts are set by launch_fwd from fwd_split_plan): the last nsplit row
  // blocks each go to nparts workgroups, one per range of key tiles, which
  // store their accumulators, max and sum in slot (block - first split
  // block) * nparts + part of fwd_slot_floats floats; a combining kernel
  // writes the rows.
  float* part;
  int nsplit, nparts;
  // Changed scores (mode 0: none).  With them a key that is masked or outside
  // the hull of its batch row's windows is copied as zeros in k and v, so that
  // what it holds never reaches a row; hull as in key_hull.
  // lse is that of the changed scores; row_lse (null: not wanted) that
  // of what the kernels compute (BiasRef), which the backward starts from.
  ScoreArgs score;
  int* hull;
  float* row_lse;
  // Keys and values in pages (null: k and v): the copies are made from them, and
  // wlo and whi (here also an output of the preparation) from the lengths.
  const PagedArgs* paged;
};

// Floats of one part of `rows` rows: the accumulators, then per 32 rows their
// maxima and sums.
constexpr int fwd_slot_floats(int rows, int D) { return rows * (D + 2); }
// The forward's split for a shape (nsplit 0: none), the bytes of its slots and the
// estimated time of the whole forward.
struct FwdSplit {
  int nsplit, nparts;
  size_t bytes;
  float us;
};
FwdSplit fwd_split_plan(int B, int Hq, int Lq, int Lk, int head_dim, bool fp8, bool windows);

struct BwdArgs {
  const bf16* dout;
  const bf16* q;
  const bf16* k;
  const bf16* v;
  const bf16* out;
  const float* lse;
  int64_t dosb, dosh, dosl;
  int64_t qsb, qsh, qsl;
  int64_t ksb, ksh, ksl;
  int64_t vsb, vsh, vsl;
  int64_t osb, osh, osl;
  int B, Hq, Hkv, Lq, Lk;
  const uint8_t* mask;
  int64_t msb;
  float scale;
  float scale_log2;
  bf16* dq;
  int64_t dqsb, dqsh, dqsl;
  bf16* dk;
  int64_t dksb, dksh, dksl;
  bf16* dv;
  int64_t dvsb, dvsh, dvsl;
  // Workspace (written by the launcher's first kernels).
  // Per query row (b, hq, i) at index (b*Hq + hq)*Lqp + i, i < Lqp:
  float* ndelta;  // -rowsum(dout * out); 0 for padded rows
  float* lse2;    // lse * log2(e); +inf for rows with lse == -inf and padded rows
  // Padded copies (prep.hip) with H/Lp = Hq/Lqp (q, dout) or Hkv/Lkp
  // (k, v): row copies (*r) hold element (b, h, j, d) at ((b*H + h)*Lp + j)*D
  // + d, head_dim-major copies (*t) at ((b*H + h)*D + d)*Lp + j.  qr and dor
  // are written only where qt and dt point to them, kr and vr without staged
  // dS.
  bf16* qr;
  bf16* dor;
  bf16* kr;
  bf16* vr;
  bf16* kt;
  // Where the dK/dV kernel reads its Q and dO tiles (set by launch_bwd): q and
  // dout themselves or the copies qr and dor; row i of (b, hq) at b*qtb +
  // hq*qth + i*qtl (dtb, dth, dtl for dO).
  const bf16* qt;
  int64_t qtb, qth, qtl;
  const bf16* dt;
  int64_t dtb, dth, dtl;
  float* kbias;  // (B, Lkp): 0 attended / -inf
  int* kfull;    // (B, Lkp/32): 1 if every key of the 32-key tile is attended
  int Lqp, Lkp;
  // Staged dS without windows: khull[2 p], khull[2 p + 1] bound the 64-key
  // tiles of pair p = b*Hkv + hk that can contribute; outside them no key is
  // attended and k is finite, so dS is exactly 0 there: the dK/dV kernel does
  // not form it, the dQ kernel does not read it.  (With windows, a mask and a
  // bias: the tiles with an attended key, for BiasRef alone.)  kskip: per (p,
  // tile), the marks it is made from (null without a mask).
  int* khull;
  int* kskip;
  // dq as an fp32 accumulator (dq_acc += this chunk's dq; dq is then null),
  // strides dqsb/dqsh/dqsl in floats.
  float* dq_acc;
  // lse2, ndelta and a rotated q copy are already in the workspace: skip them.
  bool reuse_q;
  // Pass over the flattened (b, kv head) pairs kv0 .. kv0 + nkv - 1 (b*Hkv +
  // hk); the whole problem unless dS is staged in several passes.
  int kv0, nkv;
  // Staged dS (null: the dQ kernel recomputes S and dP from q, k, v, dout).
  // The dK/dV kernel stores dS = P * (dP - delta) in bf16 for every query
  // head of its pass (masked keys and keys past the end as 0) and the dQ
  // kernel contracts it with K^T.  Unit (bq, qg, kt), bq = b*Hq + hq -
  // kv0*group, qg = 32-row query group (Lqp/32 of them), kt = 128-key block
  // (ceil(Lk/128) of them), is 8 KB at byte ((bq*(Lqp/32) + qg)*nkt + kt) *
  // 8192, ordered [k2 (2)][128 keys][16 rows]: row 16*k2 + r of key j at
  // bf16 (k2*128 + j)*16 + r, so a dS wave stores 8 consecutive rows of its
  // key as 16 bytes (1 KB per instruction) and the dQ kernel reads 8
  // consecutive keys of a row with two transposed LDS reads.
  bf16* ds;
  // With ds: leave dq to launch_bwd_dq_staged (a later call on the same
  // workspace, possibly on another stream).
  bool defer_dq;
  // Key windows as in FwdArgs (null: every key); non-decreasing in the row
  // (lo and hi), staged dS only.
  const int* wlo;
  const int* whi;
  int64_t wsb;
  // Compact dS layout for key windows (null: the dense unit layout above).
  // Per 64-row query tile T of batch b, four ints at ds_tab + (b*ds_tsb +
  // T)*4: the first 128-key block the tile's rows admit (kb_lo), the number
  // of blocks (nblk; the dK/dV kernel visits tile T from block kt iff kb_lo
  // <= kt < kb_lo + nblk), the unit index of the tile's first 32-row group
  // within its query head's units (gbase), unused.  Group 2T + h, block kt is
  // unit bq*ds_units + gbase + h*nblk + (kt - kb_lo); each query head of a
  // pass owns ds_units units (at least twice the sum of nblk over its tiles).
  const int* ds_tab;
  int64_t ds_tsb;
  int64_t ds_units;
  // RoPE fused into the backward (null: q and k are used as given): q and k
  // are the unrotated inputs; the query-side copies and the recomputing dQ
  // kernel rotate q with cos_q/sin_q (b*rqsb + i*(D/2) + pair), the k copies
  // and the dK/dV kernel's own key rows rotate k with cos_k/sin_k, and dk is
  // written as the transposed rotation of the rotated key's gradient
  // (rounded to bf16 first).  dq stays the rotated query's gradient (the
  // ring finishes it once over all chunks, avattn_ring_dq_finish).
  const float* cos_q;
  const float* sin_q;
  int64_t rqsb;
  const float* cos_k;
  const float* sin_k;
  int64_t rksb;
  // Split of the dK/dV grid's partial last round (null: no split; see
  // plan_tail_split): the last nsplit 128-key blocks of a pass each go to
  // nparts workgroups, one per range of query tiles, which store fp32
  // partial sums in slot (block - first split block) * nparts + part of
  // 256 x D floats (dv rows, then dk rows); a reduction kernel adds the
  // parts in order and writes dk and dv.
  float* split_part;
  int nsplit, nparts;
  // Slots for a split of every block (null: none; see dkv_(scored_)split_plan), in
  // place of split_part.
  float* split_all;
  // Changed scores as in FwdArgs (mode 0: none; staged dS only).  lse is its
  // row_lse, or with shifted_lse its lse.  With the cap lse2 holds that times
  // log2(e) - cap2, the staged dS a quarter of it, and scale 4 times the softmax
  // scale (scale_log2 stays).
  ScoreArgs score;
  bool shifted_lse;
};

// Partial-sum slots of the dK/dV tail split, 256 x D floats each; the
// region is there when the grid (one workgroup per 128-key block) has more
// workgroups than a 256-CU device runs at once.
constexpr int kSplitSlots = 512;
inline size_t split_part_bytes(int64_t dkv_blocks, int D) {
  return dkv_blocks > 256 ? (size_t)kSplitSlots * 256 * D * sizeof(float) : 0;
}

// Split of a grid's partial last round.  A grid of `total` equal workgroups,
// one per CU at a time on `cus` CUs, leaves r = total % cus of them alone in
// its last round; giving each of those r to p workgroups of 1/p the work
// makes that round ceil(r p / cus) / p as long.  Returns the p in 2..8 (r p
// within max_slots) that makes it shortest, the smaller on ties, or no split
// ({0, 0}) when none is shorter or the grid fits in one round.
struct TailSplit {
  int nsplit, nparts;
};
inline TailSplit plan_tail_split(int64_t total, int cus, int max_slots) {
  TailSplit t{0, 0};
  if (cus <= 0 || total <= cus) return t;
  const int r = (int)(total % cus);
  if (r == 0) return t;
  int best_num = 1, best_den = 1;  // round length best_num / best_den
  for (int p = 2; p <= 8 && r * p <= max_slots; ++p) {
    const int num = (r * p + cus - 1) / cus;
    if (num * best_den < best_num * p) {
      best_num = num;
      best_den = p;
      t = TailSplit{r, p};
    }
  }
  return t;
}

// Split of every block of a short dK/dV grid of `total` 128-key blocks, each
// over `tiles` 64-row query tiles (attn_bwd.hip); {0, 0}: none.
TailSplit dkv_split_plan(int64_t total, int tiles, int D);
// The same with changed scores, with or without windows.
TailSplit dkv_scored_split_plan(int64_t total, int tiles, int D, bool windows);

// Bytes of staged dS per (b, kv head) pair: dense, or the compact layout's
// units_per_head units per query head.
inline size_t ds_bytes_per_kv(int group, int Lq, int Lk, int64_t units_per_head = 0) {
  if (units_per_head > 0) return (size_t)group * (size_t)units_per_head * 8192;
  const size_t Lqp = (size_t)(Lq + 63) / 64 * 64;
  return (size_t)group * (Lqp / 32) * (size_t)((Lk + 127) / 128) * 8192;
}

// Kernel ids of the opt-in launch timer (avattn_timing_* in include/avattn.h).
enum KernelId : int {
  kKidFwd = 0,
  kKidBwdPre = 1,
  kKidBwdDkdv = 2,
  kKidBwdDq = 3,
  kKidMerge = 4,
  kKidRopeApply = 5,
  kKidRopeTables = 6,
  kKidTranspose = 7,
  kKidFwdFp8 = 8,
  kKidAbsmax = 9,
  kKidBwdDqDs = 10,
  kKidQkNorm = 11,
  kKidQkNormBwd = 12,
  kKidDqFinish = 13,
  kKidDkdvReduce = 14,
  kKidDiag = 15,
  kKidAddNorm = 16,
  kKidAddNormBwd = 17,
  kKidFwdFew = 18,
  kKidWindowHull = 19,
  kKidAppend = 20,
  kKidPageValues = 21,
  kKidFwdPaged = 22,
  kKidPrepPaged = 23,
  kKidGatedNorm = 24,
  kKidGatedNormBwd = 25,
};

// Records HIP events around one launch on `stream` while timing is enabled.
class LaunchTimer {
 public:
  LaunchTimer(int kernel_id, hipStream_t stream);
  ~LaunchTimer();
  LaunchTimer(const LaunchTimer&) = delete;
  LaunchTimer& operator=(const LaunchTimer&) = delete;

 private:
  int slot_;
  hipStream_t stream_;
};

// Sequence length of a padded copy (prep.hip): whole 64-row tiles.  In 64
// bits, so that the validation of a length near INT32_MAX sees the true
// padded length; validated problems fit in int.
inline int64_t transpose_padded_len(int64_t L) { return (L + 63) / 64 * 64; }

// The forward's preparation (FwdArgs::kr, vt, kbias, kfull, kmax2; with k8
// set everything but the K copy and kmax2).
hipError_t launch_prep_fwd(const FwdArgs& a, int head_dim, hipStream_t stream);
// The same from pages (a.paged; with bias a.score.offsets is written too).
hipError_t launch_prep_paged(const FwdArgs& a, int head_dim, hipStream_t stream);
// The backward's (BwdArgs::kt, kbias, kfull, khull, the row copies it needs
// and, unless a.reuse_q, lse2 and ndelta; a.qt and a.dt must be set).
hipError_t launch_prep_bwd(const BwdArgs& a, int head_dim, hipStream_t stream);

// dq (bf16, strided) = transposed rotation of bf16(dq_acc) (fp32, strided);
// a plain cast when cos_t is null.
hipError_t launch_dq_finish(const float* acc, int64_t asb, int64_t ash, int64_t asl, int B, int H, int L, int D,
                            const float* cos_t, const float* sin_t, int64_t tsb, bf16* dq, int64_t dsb, int64_t dsh,
                            int64_t dsl, hipStream_t stream);

// Per-head e4m3 scales of x (B, H, L, D) strided: scale[h] = max|x[:, h]| / 448
// (1 for an all-zero head).  `bits` (H words) holds the running maxima; it
// may alias `scale`.
hipError_t launch_absmax_scales(const bf16* x, int64_t sb, int64_t sh, int64_t sl, int B, int H, int L, int D,
                                float* scale, uint32_t* bits, hipStream_t stream);

// x (B, H, L, D) strided -> e4m3 row-major copy (B*H, Lp, D) bytes of
// x * (1 / scale[h]), zero padded to Lp = transpose_padded_len(L); with
// rowmax2 set, also the largest squared norm of the quantized rows of each
// 64-row tile, rowmax2[(b*H + h)*(Lp/64) + tile] (float bits).
hipError_t launch_quantize_rows(const bf16* x, int64_t sb, int64_t sh, int64_t sl, int B, int H, int L, int D,
                                const float* scale, uint8_t* out, uint32_t* rowmax2, hipStream_t stream);

// Forward; the fp8 q k^T variant when a.k8 is set (a.q_scale, a.k_scale too).
hipError_t launch_fwd(const FwdArgs& a, int head_dim, hipStream_t stream);
// The changed-score kernels (attn_scored_fwd.hip, attn_scored_bwd.hip) of
// launch_fwd (its grid, in the 128-row workgroups or not) and of launch_bwd's
// dK/dV step.
void launch_fwd_scored(const FwdArgs& a, int head_dim, bool small, dim3 grid, hipStream_t stream);
void launch_dkdv_scored(const BwdArgs& a, int head_dim, dim3 grid, hipStream_t stream);
// hull[2 b], hull[2 b + 1] of key_hull, over windows in any order.
hipError_t launch_window_hull(const int* wlo, const int* whi, int64_t wsb, int B, int Lq, int Lk, int* hull,
                              hipStream_t stream);
hipError_t launch_empty(bf16* o, int64_t osb, int64_t osh, int64_t osl, int B, int H, int L, int D, float* lse,
                        hipStream_t stream);
// Backward.  With a.ds set, the (b, kv head) pairs go in passes of
// kv_per_pass, each staging its dS in a.ds (ds_bytes_per_kv bytes per pair).
hipError_t launch_bwd(const BwdArgs& a, int head_dim, int kv_per_pass, hipStream_t stream);
// dQ from the dS and K^T copy a deferred launch_bwd left in the workspace
// (every (b, kv head) pair in one pass).
hipError_t launch_bwd_dq_staged(const BwdArgs& a, int head_dim, hipStream_t stream);
// Fused q/k RMSNorm + rotation (qk_norm.hip).  Rows (b, h, i) of x, dy,
// out and dx at b*sb + h*sh + i*sl (elements), head_dim contiguous.
struct QkNormArgs {
  const bf16* x;
  int64_t xsb, xsh, xsl;
  int B, H, L;
  const bf16* w;     // (head_dim) gain, or null for none
  float eps;
  const float* ct;   // rotation tables (b, 0, i, pair) at b*tsb + i*head_dim/2 + pair; null: no rotation
  const float* st;
  int64_t tsb;
  bf16* out;         // forward output
  int64_t osb, osh, osl;
  const bf16* dy;    // backward: gradient of the output
  int64_t dsb, dsh, dsl;
  bf16* dx;          // backward: gradient of x
  int64_t xgb, xgh, xgl;
  float* wpart;      // backward: per-block dW partials (qk_norm_bwd_workspace_bytes), null without a gain
};
size_t qk_norm_bwd_workspace_bytes(int head_dim);
hipError_t launch_qk_norm(const QkNormArgs& a, int head_dim, hipStream_t stream);
// Backward; with a.wpart also dw (head_dim floats) = the gain's gradient.
hipError_t launch_qk_norm_bwd(const QkNormArgs& a, int head_dim, float* dw, hipStream_t stream);
// dw[0 .. head_dim) = 0 (the gain gradient of an empty input).
hipError_t launch_qk_norm_dw_zero(float* dw, int head_dim, hipStream_t stream);

// Forward of few query rows (attn_few.hip): at most kFewQueries of them, or
// kFewRows over the group of a kv head; float32 kFewQueriesF32; and small calls
// (few_plan).
constexpr int kFewQueries = 32, kFewRows = 64, kFewQueriesF32 = 16;
struct FewArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t qsb, qsh, qsl;
  int64_t ksb, ksh, ksl;
  int64_t vsb, vsh, vsl;
  int64_t osb, osh, osl;
  int B, Hq, Hkv, Lq, Lk;
  const uint8_t* mask;
  int64_t msb;
  const int* wlo;
  const int* whi;
  int64_t wsb;
  float scale_log2;
  ScoreArgs score;
  float* lse;
  float* row_lse;  // as in FwdArgs
  // Set by launch_few from few_plan: workgroups per (batch, kv head, block of
  // rows), blocks per kv head, rows of a block; part: few_slot_floats per
  // workgroup (nsplit > 1), outputs by row, then (maximum, sum, bias_distance)
  // by row.
  int nsplit, row_blocks, block_rows;
  float* part;
};
constexpr int few_slot_floats(int rows, int D) { return rows * D + (3 * rows + 3) / 4 * 4; }
// nsplit 0: more rows than this path takes.
struct FewPlan {
  int nsplit, row_blocks, block_rows;
  size_t bytes;
};
FewPlan few_plan(int B, int Hq, int Hkv, int Lq, int Lk, int head_dim, bool f32);
hipError_t launch_few(const FewArgs& a, const FewPlan& plan, int head_dim, bool f32, hipStream_t stream);
// The second step of a split bf16 call: joins the parts of a.row_blocks blocks
// of a.block_rows rows of every (batch, kv head).
void launch_few_combine(const FewArgs& a, int head_dim, hipStream_t stream);

// A cache of pages (paged_append.hip, attn_paged.hip): slot s of head h of page
// p at p*kps + h*kph + s*head_dim (values: vps, vph), 1 << shift slots; bf16, or
// e4m3 codes with the exponent of (p, h) at p*kes + h (values: ves).  Token t of
// sequence b is in slot t % page of page table[b*tsb + t / page], t / page <
// blocks; an entry outside [0, pages) names no page.
constexpr int kMinPageShift = 4, kMaxPageShift = 8;
// Exponents written: code * 2^e is then a normal bf16 number, or zero.
constexpr int kMinCodeExponent = -110, kMaxCodeExponent = 119;
struct PageTable {
  const int* table;
  int64_t tsb;
  int blocks, pages, shift;
  // The page of a sequence's block, -1 for none.
  __device__ __forceinline__ int page(int b, int64_t block) const {
    if (block < 0 || block >= blocks) return -1;
    const int p = table[b * tsb + block];
    return p >= 0 && p < pages ? p : -1;
  }
};
// The rotation of rotate_kernel for rows of 16-channel items; cos null: none.
struct AppendRotation {
  const float* cos;
  const float* sin;
  int64_t tsb;
  int pairs, start;
  bool half;
};
struct AppendArgs {
  const bf16* k;
  const bf16* v;
  const bf16* q;  // null: none
  bf16* q_out;
  int64_t ksb, ksh, ksl, vsb, vsh, vsl, qsb, qsh, qsl, osb, osh, osl;
  int B, Hq, Hkv, L;
  AppendRotation rot;
  PageTable pages;
  const int* lengths;
  const int* counts;  // null: L
  void* kp;
  void* vp;
  int64_t kps, kph, vps, vph;
  int8_t* ke;  // null: bf16 pages
  int8_t* ve;
  int64_t kes, ves;
  int nblocks;  // blocks that L tokens may touch (set by launch_append)
};
bool append_fits(const AppendArgs& a, int head_dim);
hipError_t launch_append(const AppendArgs& a, int head_dim, hipStream_t stream);
// bf16 values of all pages, (page, head, slot, channel) contiguous, of keys [0]
// and values [1].
struct PageValuesArgs {
  const uint8_t* codes[2];
  const int8_t* exponent[2];
  int64_t ps[2], hs[2], es[2];
  bf16* out[2];
  int pages, H, D, shift;
};
hipError_t launch_page_values(const PageValuesArgs& a, hipStream_t stream);

// Attention over pages (attn_paged.hip).  few: q, o, lse, their strides and
// sizes, scale and scores (k, v, masks and windows unused); few.Lk is blocks <<
// shift.  Query i < counts[b] (null: Lq) is at position p = lengths[b] -
// counts[b] + i and sees keys (p - window, p] (window 0: from 0 on).
struct PagedArgs {
  FewArgs few;
  PageTable pages;
  const int* lengths;
  const int* counts;
  int window;
  const void* kp;
  const void* vp;
  int64_t kps, kph, vps, vph;
  const int8_t* ke;  // null: bf16 pages
  const int8_t* ve;
  int64_t kes, ves;
};
// nsplit > 0: the few-row kernel, `bytes` of parts; else the general forward on
// bf16 copies of the pages (its workspace, then the windows).
FewPlan paged_plan(int B, int Hq, int Hkv, int Lq, int64_t cap, int window, int head_dim, bool fp8);
hipError_t launch_paged_few(const PagedArgs& a, const FewPlan& plan, int head_dim, hipStream_t stream);
// The float32 kernels with changed scores (attn_f32.hip): what their C entry
// points check, with a status code.  The forward's workspace: split parts, then
// the hull; the backward's tensors are float behind BwdArgs' pointers.
size_t bwd_f32_split_bytes(int B, int Hq, int Hkv, int Lq, int Lk, int head_dim, bool windows);
size_t fwd_f32_split_bytes(int B, int Hq, int Lq, int Lk, int head_dim);
int fwd_scored_f32(const FewArgs& c, int head_dim, float scale, bool sorted_windows, void* workspace,
                   size_t workspace_bytes, hipStream_t stream);
int bwd_scored_f32(const BwdArgs& c, int head_dim, void* workspace, size_t workspace_bytes, hipStream_t stream);

// Tables of integer positions (seq_rope.hip): position of token (b, i) at
// b*psb + i, pair p's frequency freq[p]; cos and sin, times amplitude, to
// (b, i, pair) contiguous.
constexpr int kMaxTablePairs = 256;
struct PositionTableArgs {
  int64_t psb;
  int B, L, P;
  double amplitude;
  double freq[kMaxTablePairs];
  float* cos_out;
  float* sin_out;
};
hipError_t launch_position_tables(const PositionTableArgs& a, const void* pos, bool wide, hipStream_t stream);

// Rotation of part of the heads of one or two tensors (the second with H[1]
// 0: none) with the same tables, (b, i, pair) at b*tsb + i*P + pair.  Row i
// of head h of tensor w at b*xs[w][0] + h*xs[w][1] + i*xs[w][2] (output: os).
struct RotateArgs {
  const void* x[2];
  void* o[2];
  int64_t xs[2][3], os[2][3];
  int H[2];
  int B, L, D, P, start;
  int64_t first;  // the launch's first token (b * L + i), set by launch_rotate
  const float* ct;
  const float* st;
  int64_t tsb;
  bool inverse;
};
hipError_t launch_rotate(const RotateArgs& a, bool half, bool f32, hipStream_t stream);

// Residual addition + RMS norm (add_norm.hip).  Forward: rows of x and r, xs
// and rs apart; h and n (e4m3 codes with scale per row, or the rows' type)
// contiguous.  Backward: x holds the stored h, h receives dx, part the dW
// partials (add_norm_bwd_workspace_bytes).
struct AddNormArgs {
  const void* x;
  const void* r;
  const void* w;
  void* h;
  void* n;
  float* scale;
  const void* dn;
  const void* dh;  // null: none
  float* part;
  int64_t xs, rs, dns, dhs;
  int64_t rows, W;
  float eps;
  bool w32;  // the gain is fp32
};
size_t add_norm_bwd_workspace_bytes(int64_t rows, int64_t W);
hipError_t launch_add_norm(const AddNormArgs& a, bool f32, bool fp8, hipStream_t stream);
hipError_t launch_add_norm_bwd(const AddNormArgs& a, bool f32, void* dw, bool dw32, hipStream_t stream);

// The gated residual step with its norms (gated_norm.hip, which has the
// formulas).  Rows of x, r, dn and dh their strides apart; h, n, dx and dr
// contiguous.  w and p: (W), null for none; g, s, t: a row for each group of R
// rows, gs, ss and ts apart (0: shared), null for none.  stats: rx and rh of a
// row, written by the forward if not null, read by the backward.
// Backward: dh null for none, dr null where it is dx; ds, dt, dg (a contiguous
// row per group), dw and dp null where not wanted.
struct GatedNormArgs {
  const void* x;
  const void* r;
  int64_t xs, rs;
  const void* w;
  const void* p;
  const void* g;
  const void* s;
  const void* t;
  int64_t gs, ss, ts;
  bool w32, p32, m32;  // fp32 in place of the rows' type
  int64_t rows, W, R;
  float alpha, eps;
  void* h;
  void* n;
  float* stats;
  const void* dn;
  const void* dh;
  int64_t dns, dhs;
  void* dx;
  void* dr;
  void* dg;
  void* ds;
  void* dt;
  void* dw;
  void* dp;
  float* part;
  // Set by the launchers: a launch's first worker (backward: workgroup), those of a
  // group, and threads per row of the rows that share a wave.
  int64_t first, per_group;
  int tpr;
};
size_t gated_norm_bwd_workspace_bytes(int64_t rows, int64_t R, int64_t W, bool modulated);
hipError_t launch_gated_norm(const GatedNormArgs& a, bool f32, hipStream_t stream);
hipError_t launch_gated_norm_bwd(const GatedNormArgs& a, bool f32, hipStream_t stream);

hipError_t launch_zero_rows(bf16* x, int64_t sb, int64_t sh, int64_t sl, int B, int H, int L, int D,
                            hipStream_t stream);
hipError_t launch_lse_merge(float* out_acc, float* lse_acc, const void* out_blk, const float* lse_blk, int64_t rows,
                            int D, bool blk_bf16, hipStream_t stream);
hipError_t launch_rope_tables(const float* coords, int64_t csb, int64_t csr, int B, int L, int P,
                              const float* inv_freq, const int32_t* axis_of_pair, const int32_t* apply_mul,
                              const float* pos_mul, const int32_t* apply_div, const float* pos_div, float* cos_out,
                              float* sin_out, hipStream_t stream);
hipError_t launch_rope_apply(const bf16* x, int64_t xsb, int64_t xsh, int64_t xsl, int B, int H, int L, int D,
                             const float* cos_tab, const float* sin_tab, int64_t tsb, bool inverse, bf16* out,
                             int64_t osb, int64_t osh, int64_t osl, hipStream_t stream);

}  // namespace avattn
