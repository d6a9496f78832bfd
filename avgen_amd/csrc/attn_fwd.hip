// Attention forward: launches of the kernels in attn_fwd_kernel.h.
#include "attn_fwd_kernel.h"

namespace avattn {

// Writes zeros to out and -inf to lse: attention over an empty key set
// (src/avgen/models/attention.py:261-262 returns zeros_like(query)).
__global__ void attn_empty_kernel(bf16* o, int64_t osb, int64_t osh, int64_t osl, int B, int H, int L, int D,
                                  float* lse) {
  const int64_t units = (int64_t)B * H * L * (D / 8);
  for (int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; u < units; u += (int64_t)gridDim.x * blockDim.x) {
    const int c = (int)(u % (D / 8));
    const int64_t row = u / (D / 8);
    const int i = (int)(row % L);
    const int h = (int)((row / L) % H);
    const int b = (int)(row / ((int64_t)L * H));
    *reinterpret_cast<u32x4*>(o + b * osb + h * osh + (int64_t)i * osl + 8 * c) = u32x4{0u, 0u, 0u, 0u};
    if (c == 0) lse[row] = kNegInf;
  }
}

// Which workgroups a bf16 forward runs in.  Measured on one MI355X, 256-row
// against 128-row (SMALL) workgroups:
//   D 64, any shape: SMALL (three workgroups per CU): (2,20,16384) 2833 ->
//     2617 us, (2,16,7176) 505 -> 467, 20,000 x 256 keys 51 -> 41, varlen
//     (1,20,37800) 2645 -> 2380, window (1,20,21600) 1106 -> 963;
//   D 128, many tiles per workgroup and several rounds of workgroups: 256
//     rows ((2,20,16384) 4174 against 4630 us, (1,20,5265) 256 against 302,
//     (2,40,2304) 220 against 236);
//   D 128, few keys, where the prologue and output are a large part: SMALL
//     (75,600 x 128 keys 521 -> 470 us, 20,000 x 256 74.7 -> 66.2, x 512
//     within noise);
//   D 128, at most one workgroup of 128 rows per CU and up to 1,024 keys:
//     SMALL, which spreads over more CUs ((1,8,1024) x 700 keys 25.4 -> 22.6
//     us, (1,64,511) 33.0 -> 30.1, (1,200,128) 46.0 -> 41.7).  With more
//     workgroups, CUs hold two of them and gain nothing on one of 256 rows
//     ((1,24,2013) x 10,752 keys 271 us in 192 workgroups of 256 rows, 314 in
//     384 of 128; (1,17,2048) x 1,500 44 against 54); with more keys, the
//     two LDS stages hide less of the loads' latency than four do ((1,200,128)
//     x 2,000 keys 120 against 129, (1,100,256) x 5,000 178 against 198) and
//     splitting 256-row workgroups gains more ((1,12,2560) x 6,169 106 against
//     117 us).
constexpr int kSmallKeys = 512, kSmallRoundKeys = 1024, kCus = 256;
static bool use_small(int B, int Hq, int Lq, int Lk, int head_dim) {
  return head_dim == 64 || Lk <= kSmallKeys ||
         (Lk <= kSmallRoundKeys && (int64_t)((Lq + 127) / 128) * B * Hq <= kCus);
}

// Split of the last round's row blocks over ranges of key tiles: the number
// of parts (2..8, at least 8 tiles each) with the smallest estimated time, if
// it saves 4 us or more.  Times per tile and round and per workgroup as
// measured on an MI355X; (1,4,4096,128) 78.7 -> 61.1 us, D 64 56.7 -> 41.0,
// (1,16,4725,128) x 18,900 keys 844 -> 666, (1,8,18900,128) 1330 -> 1190.
// An only round of 256-row workgroups on more than half the CUs stays whole:
// it clocks higher than the estimate has it, and the splits it picks took
// (1,20,1792,128) x 10,752 keys from 221 to 234 us, (1,24,1537) 245 to 253
// (20,000 keys 0.94-1.02 of the whole).
FwdSplit fwd_split_plan(int B, int Hq, int Lq, int Lk, int D, bool fp8, bool windows) {
  FwdSplit best{0, 0, 0, 0.f};
  // The tiles of a row block are known on the device only.  (Over pages, where
  // the rows are a sequence's newest tokens, they are about all of them: 1,024 rows
  // of 64 heads x 12,001 keys 313 -> 267 us.)
  if (windows) return best;
  const bool small = !fp8 && use_small(B, Hq, Lq, Lk, D);
  const int bm = small ? 128 : 256;
  const int per_cu = small ? (D == 64 ? 3 : 2) : 1;
  const int slots = kCus * per_cu;
  const int ntile = (Lk + 63) / 64;
  const int64_t blocks = (int64_t)((Lq + bm - 1) / bm) * B * Hq;
  const int r = (int)(blocks % slots);
  const float tile_us = fp8 ? 1.25f : (D == 64 ? 1.55f : 1.7f), fixed_us = 8.f;
  // Rounds n workgroups take.  A partial round is shorter than a full one:
  // one workgroup on a CU by itself takes less than per_cu sharing it, and
  // the chip, power-limited when full, clocks higher with CUs idle (measured:
  // splitting 80 workgroups of 295 tiles left after two rounds saved 140 us
  // of 1330, where full-length rounds would have made it 335).
  auto rounds = [&](int n) {
    const int rem = n % slots;
    if (rem == 0) return (float)(n / slots);
    const int k = (rem + kCus - 1) / kCus;
    const float idle = 1.f - (float)rem / (k * kCus);
    return n / slots + (k + 0.2f * (per_cu - k)) / per_cu * (1.f - (small ? 0.25f : 0.38f) * idle);
  };
  // The parts cost their partial sums, written and read at 4 TB/s, and the
  // combining launch.
  const float slot_bytes = 4.f * fwd_slot_floats(bm, D);
  const float whole = ntile * tile_us + fixed_us;
  best.us = blocks / slots * whole + rounds(r) * whole;
  if (!small && r == blocks && r > kCus / 2) return best;
  float cost = rounds(r) * whole - 4.f;
  for (int p = 2; p <= 8 && ntile / p >= 8; ++p) {
    const float c = rounds(r * p) * (ntile * tile_us / p + fixed_us) + 5.f + r * p * slot_bytes * 0.5e-6f;
    if (c < cost) {
      cost = c;
      best = FwdSplit{r, p, (size_t)r * p * fwd_slot_floats(bm, D) * sizeof(float), blocks / slots * whole + c};
    }
  }
  return best;
}

template <int D, bool SMALL>
static void launch_variant(const FwdArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(SMALL ? 256 : 512);
  if (a.wlo != nullptr)
    hipLaunchKernelGGL((attn_fwd_kernel<D, false, false, true, SMALL>), grid, block, 0, stream, a);
  else if (a.cos_q != nullptr)
    hipLaunchKernelGGL((attn_fwd_kernel<D, true, false, false, SMALL>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fwd_kernel<D, false, false, false, SMALL>), grid, block, 0, stream, a);
}

template <int D>
static hipError_t launch_fwd_d(const FwdArgs& args, hipStream_t stream) {
  FwdArgs a = args;
  const bool fp8 = a.k8 != nullptr;
  hipError_t e = a.paged ? launch_prep_paged(a, D, stream) : launch_prep_fwd(a, D, stream);
  if (e == hipSuccess && fp8) {
    LaunchTimer timer(kKidTranspose, stream);
    e = launch_quantize_rows(a.k, a.ksb, a.ksh, a.ksl, a.B, a.Hkv, a.Lk, D, a.k_scale, a.k8, a.kmax2, stream);
  }
  if (e != hipSuccess) return e;
  const bool small = !fp8 && use_small(a.B, a.Hq, a.Lq, a.Lk, D);
  const int bm = small ? 128 : 256;
  const int64_t blocks = (int64_t)((a.Lq + bm - 1) / bm) * a.B * a.Hq;
  const FwdSplit sp = fwd_split_plan(a.B, a.Hq, a.Lq, a.Lk, D, fp8, a.wlo != nullptr && a.score.mode == 0 && !a.paged);
  if (a.part != nullptr) {
    a.nsplit = sp.nsplit;
    a.nparts = sp.nparts;
  }
  const dim3 grid((unsigned)(blocks - a.nsplit + (int64_t)a.nsplit * a.nparts));
  {
    LaunchTimer timer(fp8 ? kKidFwdFp8 : kKidFwd, stream);
    if (a.score.mode != 0)
      launch_fwd_scored(a, D, small, grid, stream);
    else if (fp8)
      hipLaunchKernelGGL((attn_fwd_kernel<D, false, true, false, false>), grid, dim3(512), 0, stream, a);
    else if (small)
      launch_variant<D, true>(a, grid, stream);
    else if constexpr (D != 64)  // never at D 64 (use_small)
      launch_variant<D, false>(a, grid, stream);
  }
  if (a.nsplit > 0) {
    const bool log2_units = fp8 || a.score.mode != 0;
    const float c = log2_units ? 1.f : a.scale_log2, unit = log2_units ? kLn2 : a.scale;
    LaunchTimer timer(kKidMerge, stream);
    if (small)
      hipLaunchKernelGGL((fwd_combine_kernel<D, 128>), dim3(a.nsplit), dim3(256), 0, stream, a, c, unit);
    else
      hipLaunchKernelGGL((fwd_combine_kernel<D, 256>), dim3(2 * a.nsplit), dim3(256), 0, stream, a, c, unit);
  }
  return hipGetLastError();
}

hipError_t launch_fwd(const FwdArgs& a, int head_dim, hipStream_t stream) {
  return head_dim == 128 ? launch_fwd_d<128>(a, stream) : launch_fwd_d<64>(a, stream);
}

hipError_t launch_empty(bf16* o, int64_t osb, int64_t osh, int64_t osl, int B, int H, int L, int D, float* lse,
                        hipStream_t stream) {
  const int64_t units = (int64_t)B * H * L * (D / 8);
  const int blocks = (int)((units + 255) / 256 < 65536 ? (units + 255) / 256 : 65536);
  hipLaunchKernelGGL(attn_empty_kernel, dim3(blocks > 0 ? blocks : 1), dim3(256), 0, stream, o, osb, osh, osl, B, H,
                     L, D, lse);
  return hipGetLastError();
}

}  // namespace avattn
