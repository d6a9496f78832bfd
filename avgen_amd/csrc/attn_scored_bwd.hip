// The dK/dV kernel (attn_bwd_dkdv.h) with scores that are capped by a tanh and /
// or biased by distance; the formulas are in attn_scored_fwd.hip.
#include "attn_bwd_dkdv.h"

namespace avattn {

namespace {

template <int D, int SCORE>
void dkdv_variant(const BwdArgs& a, dim3 grid, hipStream_t stream) {
  if (a.wlo && a.ds_tab)
    hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, true, true, SCORE>), grid, dim3(512), 0, stream, a);
  else if (a.wlo)
    hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, true, false, SCORE>), grid, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((bwd_dkdv_kernel<D, false, true, false, false, SCORE>), grid, dim3(512), 0, stream, a);
}

template <int SCORE>
void dkdv_scored(const BwdArgs& a, int head_dim, dim3 grid, hipStream_t stream) {
  if (head_dim == 64)
    dkdv_variant<64, SCORE>(a, grid, stream);
  else
    dkdv_variant<128, SCORE>(a, grid, stream);
}

}  // namespace

void launch_dkdv_scored(const BwdArgs& a, int head_dim, dim3 grid, hipStream_t stream) {
  if (a.score.mode == kScoreCap)
    dkdv_scored<kScoreCap>(a, head_dim, grid, stream);
  else if (a.score.mode == kScoreDistance)
    dkdv_scored<kScoreDistance>(a, head_dim, grid, stream);
  else
    dkdv_scored<kScoreCap | kScoreDistance>(a, head_dim, grid, stream);
}

}  // namespace avattn
