// Backward pass of the typed block norms: LayerNorms.
#include "rf_block_norm_typed_bwd.cuh"

namespace rf {
namespace bn {

bool try_typed_layer_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st) {
  return typed_bwd<true>(p, A, bias, st);
}

}  // namespace bn
}  // namespace rf
