// Products with 4-bit weights for more than a few tokens: x through LDS.  The kernel and its launch, instantiated for bfloat16 and float32
// x side by side.
//
// A block's four waves hold 32 rows of weights each and share the tokens, 16 TT of them, in stages of 128 along K: as matrix-core operands,
// 1 KB a step of 32 and tile of 16 tokens, which LDS gives without conflicts.  bfloat16 x travels straight into LDS while the stage before is
// multiplied; float32 x through registers, where it is split into its three parts once for all waves.  Weights and scales are asked for
// a stage ahead.  One barrier a stage.  (64 rows a wave unpack x's operands half as often, but leave room for two blocks a compute unit
// instead of three: 64 tokens by 55,296 x 5,120 in groups of 32 90.0 us, with 32 rows 85.0.)
#pragma once
#include "gemm_q4.h"

namespace sprout {

using namespace q4;

namespace {

// K is whole eights, rows of x start at whole 16 bytes.
template <typename X, typename S, int TT, int STEPS>
__global__ __launch_bounds__(256, 2) void gemm_q4_staged_kernel(Q4Args a) {
  constexpr int NT = kStagedRowTiles;
  constexpr bool kF32 = sizeof(X) == 4;
  constexpr int PARTS = kF32 ? 3 : 1, GROUPS = 4 / STEPS, PLANE = 4096 * TT, STAGE = PARTS * PLANE;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];      // two stages of [part][step][token tile][lane] pieces
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, lj = lane >> 4;
  const int tile0 = (blockIdx.x * 4 + wave) * NT, tiles = a.padded / 16, t0 = blockIdx.y * 16 * TT, split = blockIdx.z;
  const int k_from = int((long long)(a.blocks) * split / a.splits), k_to = int((long long)(a.blocks) * (split + 1) / a.splits);
  const floatx4 zero = floatx4{0.f, 0.f, 0.f, 0.f};
  floatx4 total[NT][TT], sum[NT][TT], off[TT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < TT; ++t) total[n][t] = sum[n][t] = zero;
#pragma unroll
  for (int t = 0; t < TT; ++t) off[t] = zero;
  const bf16x8 minus24 = as_bf16x8(make_uint4(0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u));
  // (addresses the same in all lanes and 32 bits a lane beside them: registers are what this has least of)
  const unsigned char* words[NT];
  const unsigned char* scales[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int tile = min(tile0 + n, tiles - 1);
    words[n] = reinterpret_cast<const unsigned char*>(a.words) + size_t(tile) * a.blocks * 1024;
    scales[n] = static_cast<const unsigned char*>(a.scales) + sizeof(S) * 16 * tile;
  }
  uint4 w[NT], w_next[NT];
  ScaleBits<S> scale[GROUPS][NT];
  auto load_words = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) w_next[n] = *reinterpret_cast<const uint4*>(words[n] + size_t(kb) * 1024 + uint32_t(16 * lane));
  };
  auto load_scales = [&](int kb, int g) __attribute__((always_inline)) {      // (behind the last group x is zero)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      load_scale(reinterpret_cast<const S*>(scales[n] + size_t(min(GROUPS * kb + g, a.groups - 1)) * a.padded * sizeof(S) + uint32_t(4 * lj * sizeof(S))), scale[g][n]);
  };
  // A wave brings its step of 32 of every token tile; a lane's piece is eight numbers of a token.
  const X* x = static_cast<const X*>(a.x) + size_t(t0) * a.K;
  const uint64_t x_at = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uint64_t>(x) >> 32)))) << 32 |
                        uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uint64_t>(x))));
  const int piece_k = 32 * wave + 8 * lj;
  uint32_t piece_at[TT];
#pragma unroll
  for (int u = 0; u < TT; ++u) piece_at[u] = uint32_t(min(t0 + 16 * u + lr, a.T - 1) - t0) * uint32_t(a.K) * uint32_t(sizeof(X));
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
  RawF32 raw[TT];
  auto request = [&](int kb, int buffer) __attribute__((always_inline)) {
    const int k = kb * kBlockK + piece_k;
    const uint32_t in_row = k < a.K ? uint32_t(k) * uint32_t(sizeof(X)) : 0;      // behind K: the row's first, cleared before use
#pragma unroll
    for (int u = 0; u < TT; ++u) {
      if constexpr (kF32) {
        const float* p = reinterpret_cast<const float*>(reinterpret_cast<const unsigned char*>(x) + (piece_at[u] + in_row));
        raw[u].a = *reinterpret_cast<const float4*>(p);
        raw[u].b = *reinterpret_cast<const float4*>(p + 4);
      } else {
        lanes_to_lds(x_at, piece_at[u] + in_row, lds_base + buffer * STAGE + 1024 * (wave * TT + u));
      }
    }
  };
  auto split_to_lds = [&](int kb, int buffer) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < TT; ++u) {
      if ((kb + 1) * kBlockK > a.K && kb * kBlockK + piece_k >= a.K) clear(raw[u]);
      bf16x8 p[3];
      x_operands(raw[u], p);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(lds + buffer * STAGE + i * PLANE + 1024 * (wave * TT + u) + 16 * lane) = p[i];
    }
  };
  // A stage's end: what was asked for the next one is there.  (The compiler does not count the loads into LDS; where it may expect others
  // still to be on their way it would wait for those too, as soon as they have been asked for.)
  auto all_arrived = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0)
    asm volatile("" : : : "memory");
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      arrived(w_next[n]);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) arrived(scale[g][n]);
    }
  };
  if (k_from < k_to) {
    request(k_from, 0);
    load_words(k_from);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) load_scales(k_from, g);
    if (kF32) split_to_lds(k_from, 0);
    all_arrived();
  }
  int buffer = 0;
  for (int kb = k_from; kb < k_to; ++kb, buffer ^= 1) {
    if (!kF32) {
      if ((kb + 1) * kBlockK > a.K) {      // what lies behind K is zero
#pragma unroll
        for (int u = 0; u < TT; ++u)
          if (kb * kBlockK + piece_k >= a.K) *reinterpret_cast<uint4*>(lds + buffer * STAGE + 1024 * (wave * TT + u) + 16 * lane) = make_uint4(0, 0, 0, 0);
      }
    }
    __syncthreads();
    const int kb_next = min(kb + 1, k_to - 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = w_next[n];
    if (kb + 1 < k_to) request(kb + 1, buffer ^ 1);
    load_words(kb_next);
    __builtin_amdgcn_sched_barrier(0);
    const unsigned char* stage = lds + buffer * STAGE + 16 * lane;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 b[TT][PARTS];
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) b[t][p] = *reinterpret_cast<const bf16x8*>(stage + p * PLANE + 1024 * (s * TT + t));
      if (!kF32) {
#pragma unroll
        for (int t = 0; t < TT; ++t) off[t] = mfma16(minus24, b[t][0], s % STEPS == 0 ? zero : off[t]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8 c = weights_operand(s == 0 ? w[n].x : s == 1 ? w[n].y : s == 2 ? w[n].z : w[n].w, X());
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          floatx4 v = s % STEPS != 0 ? sum[n][t] : !kF32 && STEPS == 1 ? off[t] : zero;
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) v = mfma16(c, b[t][p], v);
          sum[n][t] = v;
        }
      }
      if (s % STEPS == STEPS - 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 f = scale_values(scale[s / STEPS][n]);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            const floatx4 v = !kF32 && STEPS > 1 ? sum[n][t] + off[t] : sum[n][t];
            total[n][t][0] += f.x * v[0];
            total[n][t][1] += f.y * v[1];
            total[n][t][2] += f.z * v[2];
            total[n][t][3] += f.w * v[3];
          }
        }
        load_scales(kb_next, s / STEPS);
      }
    }
    if (kF32 && kb + 1 < k_to) split_to_lds(kb + 1, buffer ^ 1);
    all_arrived();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int token = t0 + 16 * t + lr;
      if (token < a.T) store_four<X>(a, split, token, 16 * (tile0 + n) + 4 * lj, kF32 ? total[n][t] * kWeightsUnit : total[n][t]);
    }
}

template <typename X, typename S, int TT, int STEPS> bool launch_staged_steps(hipStream_t s, const Q4Args& a) {
  constexpr int lds = 2 * 4096 * TT * (sizeof(X) == 4 ? 3 : 1);
  if (lds > 64 * 1024) {      // more than a launch may have unasked
    static bool asked[64] = {};
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e == hipSuccess && (device >= 64 || !asked[device])) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_q4_staged_kernel<X, S, TT, STEPS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e == hipSuccess && device < 64) asked[device] = true;
    }
    if (e != hipSuccess) {
      set_error("sp_gemm_q4: cannot raise the LDS limit: %s", hipGetErrorString(e));
      return false;
    }
  }
  const dim3 grid((a.padded / 16 + 4 * kStagedRowTiles - 1) / (4 * kStagedRowTiles), (a.T + 16 * TT - 1) / (16 * TT), a.splits);
  gemm_q4_staged_kernel<X, S, TT, STEPS><<<grid, 256, lds, s>>>(a);
  return true;
}
template <typename X, typename S, int TT> bool launch_staged(hipStream_t s, const Q4Args& a, int steps) {
  return steps == 1 ? launch_staged_steps<X, S, TT, 1>(s, a) : steps == 2 ? launch_staged_steps<X, S, TT, 2>(s, a) : launch_staged_steps<X, S, TT, 4>(s, a);
}

}  // namespace

}  // namespace sprout
