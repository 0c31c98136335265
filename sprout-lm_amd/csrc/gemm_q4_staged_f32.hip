// Products with 4-bit weights for more than a few tokens of float32.
#include "gemm_q4_staged.h"

namespace sprout {

namespace {

template <typename S> void launch_rows(hipStream_t s, const Q4Args& a, const Q4Plan& p, int steps) {
  if (p.token_tiles == 1) launch_staged<float, S, 2, 1>(s, a, steps);
  else launch_staged<float, S, 2, 2>(s, a, steps);
}

}  // namespace

void gemm_q4_staged_f32(hipStream_t s, const Q4Args& a, const Q4Plan& p, int steps, int scales_bf16) {
  if (scales_bf16) launch_rows<uint16_t>(s, a, p, steps);
  else launch_rows<float>(s, a, p, steps);
}

}  // namespace sprout
