// Backward pass of the typed block norms: RMS norms, and the choice.
#include "rf_block_norm_typed_bwd.cuh"

namespace rf {
namespace bn {

TypedTeam typed_team(int64_t d) { return team_for(d, d <= kMaxTyped / 2 ? 1 : 2); }

bool try_typed_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st) {
  return p.kind == RF_LAYER_NORM ? try_typed_layer_bwd(p, A, bias, st) : typed_bwd<false>(p, A, bias, st);
}

}  // namespace bn
}  // namespace rf
