// Products with 4-bit weights for more than a few tokens of float32.
#include "gemm_q4_staged.h"

namespace sprout {

namespace {

template <typename S> bool launch_tiles(hipStream_t s, const Q4Args& a, int token_tiles, int steps) {
  if (token_tiles == 1) return launch_staged<float, S, 1>(s, a, steps);
  if (token_tiles == 2) return launch_staged<float, S, 2>(s, a, steps);
  return launch_staged<float, S, 3>(s, a, steps);
}

}  // namespace

bool gemm_q4_staged_f32(hipStream_t s, const Q4Args& a, int token_tiles, int steps, int scales_bf16) {
  return scales_bf16 ? launch_tiles<uint16_t>(s, a, token_tiles, steps) : launch_tiles<float>(s, a, token_tiles, steps);
}

}  // namespace sprout
