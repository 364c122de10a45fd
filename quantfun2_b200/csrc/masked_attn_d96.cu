// Masked attention at head dim 96.
#include "masked_attn.cuh"

namespace qf2 {
namespace mattn {

cudaError_t launch_d96(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s) {
  return launch_dim<96>(m, a, grid, form, f16, score, s);
}

}  // namespace mattn
}  // namespace qf2
