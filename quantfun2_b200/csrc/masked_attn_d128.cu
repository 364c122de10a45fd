// Masked attention at head dim 128.
#include "masked_attn.cuh"

namespace qf2 {
namespace mattn {

cudaError_t launch_d128(const Maps& m, const Args& a, unsigned grid, int nt, bool f16, bool score, cudaStream_t s) {
  return nt == 2 ? launch_nt<128, 2>(m, a, grid, f16, score, s) : launch_nt<128, 1>(m, a, grid, f16, score, s);
}

}  // namespace mattn
}  // namespace qf2
