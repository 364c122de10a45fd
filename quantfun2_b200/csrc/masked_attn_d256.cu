// Masked attention at head dim 256: one query tile per CTA (its fp32 output fills half of
// tensor memory).
#include "masked_attn.cuh"

namespace qf2 {
namespace mattn {

cudaError_t launch_d256(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s) {
  (void)form;
  return launch_form<256, kDeep>(m, a, grid, f16, score, s);
}

}  // namespace mattn
}  // namespace qf2
