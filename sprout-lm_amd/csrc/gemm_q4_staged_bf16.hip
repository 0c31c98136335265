// Products with 4-bit weights for more than a few tokens of bfloat16.
#include "gemm_q4_staged.h"

namespace sprout {

namespace {

template <typename S> void launch_rows(hipStream_t s, const Q4Args& a, const Q4Plan& p, int steps) {
  if (p.row_tiles == 4 && p.token_tiles == 3) launch_staged<uint16_t, S, 4, 3>(s, a, steps);
  else if (p.row_tiles == 4) launch_staged<uint16_t, S, 4, 4>(s, a, steps);
  else if (p.token_tiles == 2) launch_staged<uint16_t, S, 2, 2>(s, a, steps);
  else if (p.token_tiles == 3) launch_staged<uint16_t, S, 2, 3>(s, a, steps);
  else launch_staged<uint16_t, S, 2, 4>(s, a, steps);
}

}  // namespace

void gemm_q4_staged_bf16(hipStream_t s, const Q4Args& a, const Q4Plan& p, int steps, int scales_bf16) {
  if (scales_bf16) launch_rows<uint16_t>(s, a, p, steps);
  else launch_rows<float>(s, a, p, steps);
}

}  // namespace sprout
