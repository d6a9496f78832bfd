// Attention whose scores are capped by a tanh and / or biased by distance: the
// SCORE variants of the forward kernels (attn_fwd_kernel.h; those of dK/dV are
// in attn_scored_bwd.hip), and the hull of key windows given in any order.
// With z the changed score,
//   z_ij = cap tanh(s_ij / cap) - slope_h |i + offset - j|,  P = softmax(z)
//   dS = P (dP - delta) (1 - tanh^2(s / cap)),  dQ = scale dS K, dK = scale dS^T Q
// (the factor without a cap: 1); the distance bias has no gradient.
#include "attn_fwd_kernel.h"

namespace avattn {

namespace {

template <int D, bool SMALL, int SCORE>
void fwd_variant(const FwdArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(SMALL ? 256 : 512);
  if (a.wlo != nullptr)
    hipLaunchKernelGGL((attn_fwd_kernel<D, false, false, true, SMALL, SCORE>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((attn_fwd_kernel<D, false, false, false, SMALL, SCORE>), grid, block, 0, stream, a);
}

template <int SCORE>
void fwd_scored(const FwdArgs& a, int head_dim, bool small, dim3 grid, hipStream_t stream) {
  if (head_dim == 64)  // always in 128-row workgroups
    fwd_variant<64, true, SCORE>(a, grid, stream);
  else if (small)
    fwd_variant<128, true, SCORE>(a, grid, stream);
  else
    fwd_variant<128, false, SCORE>(a, grid, stream);
}

// One workgroup per batch row.
__global__ __launch_bounds__(1024) void window_hull_kernel(const int* __restrict__ wlo, const int* __restrict__ whi,
                                                           int64_t wsb, int Lq, int Lk, int* __restrict__ hull) {
  __shared__ int red[2][16];
  const int b = blockIdx.x;
  int lo = Lk, hi = 0;
  for (int i = threadIdx.x; i < Lq; i += 1024) {
    const int l = min(max(wlo[b * wsb + i], 0), Lk);
    const int h = min(max(whi[b * wsb + i], l), Lk);
    if (l < h) lo = min(lo, l), hi = max(hi, h);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = lo, red[1][threadIdx.x >> 6] = hi;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) lo = min(lo, red[0][w]), hi = max(hi, red[1][w]);
    hull[2 * b] = min(lo, hi), hull[2 * b + 1] = hi;
  }
}

}  // namespace

void launch_fwd_scored(const FwdArgs& a, int head_dim, bool small, dim3 grid, hipStream_t stream) {
  if (a.score.mode == kScoreCap)
    fwd_scored<kScoreCap>(a, head_dim, small, grid, stream);
  else if (a.score.mode == kScoreDistance)
    fwd_scored<kScoreDistance>(a, head_dim, small, grid, stream);
  else
    fwd_scored<kScoreCap | kScoreDistance>(a, head_dim, small, grid, stream);
}

hipError_t launch_window_hull(const int* wlo, const int* whi, int64_t wsb, int B, int Lq, int Lk, int* hull,
                              hipStream_t stream) {
  LaunchTimer timer(kKidWindowHull, stream);
  hipLaunchKernelGGL(window_hull_kernel, dim3((unsigned)B), dim3(1024), 0, stream, wlo, whi, wsb, Lq, Lk, hull);
  return hipGetLastError();
}

}  // namespace avattn
