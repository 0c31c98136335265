// Products with 4-bit weights for a few tokens, their packing, and the entry points.
#include "gemm_q4.h"

namespace sprout {

using namespace q4;

namespace {

// X, S: x's type and the scales'; STEPS: steps of 32 in a group.
template <typename X, typename S, int NT, int STEPS, bool VEC>
__global__ __launch_bounds__(256) void gemm_q4_kernel(Q4Args a) {
  constexpr bool kF32 = sizeof(X) == 4;
  constexpr int PARTS = kF32 ? 3 : 1, GROUPS = 4 / STEPS;
  __shared__ floatx4 s_sums[3][NT][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, lj = lane >> 4;
  const int tile0 = blockIdx.x * NT, tiles = a.padded / 16, token = blockIdx.y * 16 + lr, split = blockIdx.z;
  const int k_from = int((long long)(a.blocks) * split / a.splits), k_to = int((long long)(a.blocks) * (split + 1) / a.splits);
  const floatx4 zero = floatx4{0.f, 0.f, 0.f, 0.f};
  floatx4 total[NT], sum[NT], off = zero;
#pragma unroll
  for (int n = 0; n < NT; ++n) total[n] = sum[n] = zero;
  const bf16x8 minus24 = as_bf16x8(make_uint4(0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u));
  const X* x_row = static_cast<const X*>(a.x) + size_t(min(token, a.T - 1)) * a.K;
  const uint32_t* words[NT];
  const S* scales[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int tile = min(tile0 + n, tiles - 1);
    words[n] = a.words + size_t(tile) * a.blocks * 256 + 4 * lane;
    scales[n] = static_cast<const S*>(a.scales) + 16 * tile + 4 * lj;
  }
  // Loads come back in the order in which they were asked for: whoever waits for x waits for weights asked for before it.  So everything
  // of a block of 128 along K is asked for a whole block before, each part where its predecessor has been used.
  uint4 w[NT], w_next[NT];
  typename RawOf<X>::type raw[4];
  ScaleBits<S> scale[GROUPS][NT];
  auto load_words = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) w_next[n] = ldg128(words[n] + size_t(kb) * 256);
  };
  auto load_x = [&](int kb, int s) __attribute__((always_inline)) { x_load<VEC>(x_row, 128 * kb + 32 * s + 8 * lj, a.K, raw[s]); };
  auto load_scales = [&](int kb, int g) __attribute__((always_inline)) {      // (behind the last group x is zero)
#pragma unroll
    for (int n = 0; n < NT; ++n) load_scale(scales[n] + size_t(min(GROUPS * kb + g, a.groups - 1)) * a.padded, scale[g][n]);
  };
  int kb = k_from + wave;
  if (kb < k_to) {
    load_words(kb);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      load_x(kb, s);
      if (s % STEPS == 0) load_scales(kb, s / STEPS);
    }
  }
  for (; kb < k_to; kb += 4) {
    const int kb_next = min(kb + 4, k_to - 1);      // (behind the wave's last: something that is there)
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = w_next[n];
    load_words(kb_next);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 b[PARTS];
      if (VEC && 128 * kb + 128 > a.K && 128 * kb + 32 * s + 8 * lj >= a.K) clear(raw[s]);
      x_operands(raw[s], b);
      if (!kF32) off = mfma16(minus24, b[0], s % STEPS == 0 ? zero : off);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8 c = weights_operand(s == 0 ? w[n].x : s == 1 ? w[n].y : s == 2 ? w[n].z : w[n].w, X());
        floatx4 v = s % STEPS != 0 ? sum[n] : !kF32 && STEPS == 1 ? off : zero;
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) v = mfma16(c, b[p], v);
        sum[n] = v;
      }
      load_x(kb_next, s);
      if (s % STEPS == STEPS - 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 f = scale_values(scale[s / STEPS][n]);
          const floatx4 v = !kF32 && STEPS > 1 ? sum[n] + off : sum[n];
          total[n][0] += f.x * v[0];
          total[n][1] += f.y * v[1];
          total[n][2] += f.z * v[2];
          total[n][3] += f.w * v[3];
        }
        load_scales(kb_next, s / STEPS);
      }
    }
  }
  if (kF32) {
#pragma unroll
    for (int n = 0; n < NT; ++n) total[n] *= kWeightsUnit;
  }
  if (wave > 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s_sums[wave - 1][n][lane] = total[n];
  }
  __syncthreads();
  if (wave > 0 || token >= a.T) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    store_four<X>(a, split, token, 16 * (tile0 + n) + 4 * lj, ((total[n] + s_sums[0][n][lane]) + s_sums[1][n][lane]) + s_sums[2][n][lane]);
}

template <typename X> __global__ __launch_bounds__(256) void gemm_q4_join_kernel(Q4Args a) {
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x, results = size_t(a.T) * a.N;
  if (i >= results) return;
  float y = 0.f;
  for (int s = 0; s < a.splits; ++s) y += a.parts[s * results + i];
  store_result<X>(a, int(i / a.N), int(i % a.N), y);
}

// Codes two a byte along K (the first in the low half) -> the words of sp_gemm_q4; scales [N, groups] -> [groups, N padded].
__global__ void q4_pack_kernel(const uint8_t* __restrict__ codes, uint32_t* __restrict__ words, int N, int K, int blocks, size_t total) {
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int u = i & 3, lane = (i >> 2) & 63;
  const size_t kb = (i >> 8) % blocks, tile = (i >> 8) / blocks;
  const size_t row = tile * 16 + (lane & 15);
  const int k = int(kb) * kBlockK + 32 * u + 8 * (lane >> 4), row_bytes = (K + 1) / 2;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t c = 8;      // behind the matrix's end: weights of zero
    if (row < size_t(N) && k + j < K) c = (codes[row * row_bytes + (k + j) / 2] >> (4 * ((k + j) & 1))) & 15u;
    w |= c << (4 * (j / 2) + 16 * (j & 1));
  }
  words[i] = w;
}
template <typename S>
__global__ void q4_scales_kernel(const S* __restrict__ scales, S* __restrict__ out, int N, int groups, int padded) {
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= size_t(groups) * padded) return;
  const int n = int(i % padded), g = int(i / padded);
  out[i] = n < N ? scales[size_t(n) * groups + g] : from_float<S>(0.f);
}

// A wave a group: scale = max |w| / 7 as stored, code = w / scale to the nearest whole number (ties to even), plus 8.
template <typename W, typename S>
__global__ __launch_bounds__(256) void q4_quantize_kernel(const W* __restrict__ w, uint8_t* __restrict__ codes, S* __restrict__ scales, int N, int K,
                                                          int group, int groups) {
  const size_t i = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= size_t(N) * groups) return;
  const size_t row = i / groups;
  const int g = int(i % groups), first = g * group, n = min(group, K - first), lane = threadIdx.x & 63;
  const W* src = w + row * K + first;
  const float v[2] = {2 * lane < n ? to_float(src[2 * lane]) : 0.f, 2 * lane + 1 < n ? to_float(src[2 * lane + 1]) : 0.f};
  const bool nan = __builtin_amdgcn_ballot_w64(v[0] != v[0] || v[1] != v[1]) != 0;
  const float most = nan ? NAN : wave_max(fmaxf(fabsf(v[0]), fabsf(v[1])));
  const S stored = from_float<S>(most / 7.0f);
  const float scale = to_float(stored);
  uint32_t c[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float q = rintf(v[j] / scale);
    c[j] = q == q ? uint32_t(int(fminf(fmaxf(q, -8.f), 7.f)) + 8) : 8u;      // (no scale, or one that is not finite: weights of zero times it)
  }
  if (2 * lane < n) codes[row * ((K + 1) / 2) + first / 2 + lane] = uint8_t(c[0] | (c[1] << 4));
  if (lane == 0) scales[i] = stored;
}

// Which kernel, how many tiles of 16 rows and tokens a wave or block takes, and over how many blocks K is split (bfloat16 unless float32 is
// named; us, groups of 64 where nothing else stands; sizes as rows x K).
//  - x through LDS costs barriers and pays where x is read often and the weights are many: 3,584 x 18,944, 40 tokens 27.3 against
//    33.0; float32 37,888 x 3,584, 16 tokens 30.8 against 36.9, one token 27.2 against 31.4.  It is left out up to 16 tokens of bfloat16
//    (16 of 37,888 x 3,584: 22.7, and 22.8 with it), up to four of float32 on fewer rows (four of 3,584 x 18,944: 23.4, 23.2 with it),
//    and where 16 Mi weights or fewer are spread over few blocks (33 tokens of 9,728 x 896: 7.9 against 10.8).
//  - Without it, more tiles a wave read x less often, fewer keep more blocks in flight: one token of 37,888 rows 17.6 with two tiles, 18.8
//    with four, 21.9 with one; 16 tokens 22.7 with four, 27.6 with two; 3,584 x 3,584 7.1 with one, 7.8 with two.  A long K of few rows
//    is better split over blocks of four tiles (16 tokens of 3,584 x 18,944: 18.8, two tiles 22.6; one tile, not split, 28.0); splitting a short
//    one gains less than a second launch costs the host (one token of 896 x 4,864: 7.1, in four parts 6.5, called one by one 8 and 11.8).
//  - With it, as many tokens share a block as registers and LDS allow, 64 of bfloat16 (64 of 55,296 x 5,120: 65.6 in groups of 128, by 32 each
//    71.1) and 48 of float32, whose parts take three times the room (40 of 3,584 x 18,944: 38.9, by 16 each 43.7).  K is split until each
//    compute unit has two blocks (five of float32: 40 tokens of 37,888 x 3,584 60.8 in four parts, 70.3 in two).
Q4Plan q4_plan(int x_dtype, int T, int N, int K) {
  Q4Plan p;
  const bool f32 = x_dtype == kF32, small = int64_t(N) * K <= 16 << 20;
  const int tiles = (N + 15) / 16, blocks = (K + kBlockK - 1) / kBlockK, tokens = (T + 15) / 16;
  p.staged = small ? T > 48 : f32 ? T > 4 || tiles >= 1024 : T > 16;
  p.splits = 1;
  if (p.staged) {
    const int most = f32 ? 3 : 4, rounds = (tokens + most - 1) / most;
    p.token_tiles = (tokens + rounds - 1) / rounds;
    p.row_tiles = kStagedRowTiles;
    const int64_t grid = int64_t(tiles + 4 * p.row_tiles - 1) / (4 * p.row_tiles) * ((tokens + p.token_tiles - 1) / p.token_tiles);
    while (grid * p.splits * 4 < (f32 ? 1280 : 448) * 3 && p.splits < 16 && blocks >= 2 * p.splits) p.splits *= 2;
  } else {
    const int64_t units = int64_t(tiles) * tokens;
    const bool long_k = units < 400 && blocks >= 64;
    p.token_tiles = 1;
    p.row_tiles = long_k ? 4 : T <= 4 ? (units >= 1024 ? 2 : 1) : units >= 600 ? 4 : units >= 400 ? 2 : 1;
    const int64_t grid = int64_t(tiles + p.row_tiles - 1) / p.row_tiles * tokens;
    while (long_k && grid * p.splits * 2 <= 512 && blocks >= 32 * p.splits) p.splits *= 2;
  }
  return p;
}

template <typename X, typename S, int NT, bool VEC> void launch_q4_steps(hipStream_t s, const Q4Args& a, int steps) {
  const dim3 grid((a.padded / 16 + NT - 1) / NT, (a.T + 15) / 16, a.splits);
  if (steps == 1) gemm_q4_kernel<X, S, NT, 1, VEC><<<grid, 256, 0, s>>>(a);
  else if (steps == 2) gemm_q4_kernel<X, S, NT, 2, VEC><<<grid, 256, 0, s>>>(a);
  else gemm_q4_kernel<X, S, NT, 4, VEC><<<grid, 256, 0, s>>>(a);
}
template <typename X, typename S> bool launch_q4_of(hipStream_t s, const Q4Args& a, const Q4Plan& p, int steps, bool vec) {
  bool launched = true;
  if (!vec) launch_q4_steps<X, S, 1, false>(s, a, steps);
  else if (p.staged) launched = sizeof(X) == 4 ? gemm_q4_staged_f32(s, a, p.token_tiles, steps, sizeof(S) == 2) : gemm_q4_staged_bf16(s, a, p.token_tiles, steps, sizeof(S) == 2);
  else if (p.row_tiles == 1) launch_q4_steps<X, S, 1, true>(s, a, steps);
  else if (p.row_tiles == 2) launch_q4_steps<X, S, 2, true>(s, a, steps);
  else launch_q4_steps<X, S, 4, true>(s, a, steps);
  if (launched && a.splits > 1) gemm_q4_join_kernel<X><<<unsigned((size_t(a.T) * a.N + 255) / 256), 256, 0, s>>>(a);
  return launched;
}

constexpr size_t kMostBlocks = (size_t(1) << 24) - 1;      // a launch has less than 2^32 threads

bool q4_sizes(int N, int K, int group) { return N > 0 && K > 0 && (group == 32 || group == 64 || group == 128); }

}  // namespace

}  // namespace sprout

using namespace sprout;

extern "C" int64_t sp_q4_words(int N, int K) { return N <= 0 || K <= 0 ? 0 : (int64_t(N) + 15) / 16 * ((int64_t(K) + 127) / 128) * 256; }

extern "C" int sp_q4_pack(void* stream, const void* codes, int scale_dtype, const void* scales, int N, int K, int group, void* words, void* packed_scales) {
  SP_REQUIRE(q4_sizes(N, K, group), "sp_q4_pack: N=%d K=%d group=%d (groups of 32, 64 or 128)", N, K, group);
  SP_REQUIRE(scale_dtype == kF32 || scale_dtype == kBF16, "sp_q4_pack: unsupported dtype %d of the scales", scale_dtype);
  SP_REQUIRE(codes && scales && words && packed_scales, "sp_q4_pack: null argument");
  const size_t total = size_t(sp_q4_words(N, K));
  const int groups = (K + group - 1) / group, padded = (N + 15) / 16 * 16, blocks = (K + kBlockK - 1) / kBlockK;
  SP_REQUIRE(total / 256 < kMostBlocks && size_t(groups) * padded / 256 < kMostBlocks, "sp_q4_pack: the matrix is too large");
  hipStream_t s = (hipStream_t)stream;
  q4_pack_kernel<<<(total + 255) / 256, 256, 0, s>>>(static_cast<const uint8_t*>(codes), static_cast<uint32_t*>(words), N, K, blocks, total);
  const unsigned grid = unsigned((size_t(groups) * padded + 255) / 256);
  if (scale_dtype == kF32) q4_scales_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(scales), static_cast<float*>(packed_scales), N, groups, padded);
  else q4_scales_kernel<bf16_t><<<grid, 256, 0, s>>>(static_cast<const bf16_t*>(scales), static_cast<bf16_t*>(packed_scales), N, groups, padded);
  return check_launch("sp_q4_pack");
}

extern "C" int sp_q4_quantize(void* stream, int w_dtype, const void* w, int N, int K, int group, void* codes, int scale_dtype, void* scales) {
  SP_REQUIRE(q4_sizes(N, K, group), "sp_q4_quantize: N=%d K=%d group=%d (groups of 32, 64 or 128)", N, K, group);
  SP_REQUIRE((w_dtype == kF32 || w_dtype == kBF16) && (scale_dtype == kF32 || scale_dtype == kBF16), "sp_q4_quantize: unsupported dtypes %d, %d", w_dtype, scale_dtype);
  SP_REQUIRE(w && codes && scales, "sp_q4_quantize: null argument");
  const int groups = (K + group - 1) / group;
  const size_t units = size_t(N) * groups;
  SP_REQUIRE(units / 4 < kMostBlocks, "sp_q4_quantize: the matrix is too large");
  const unsigned grid = unsigned((units + 3) / 4);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* c = static_cast<uint8_t*>(codes);
  if (w_dtype == kF32 && scale_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(w), c, static_cast<float*>(scales), N, K, group, groups);
  else if (w_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(w), c, static_cast<bf16_t*>(scales), N, K, group, groups);
  else if (scale_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16_t*>(w), c, static_cast<float*>(scales), N, K, group, groups);
  else q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16_t*>(w), c, static_cast<bf16_t*>(scales), N, K, group, groups);
  return check_launch("sp_q4_quantize");
}

extern "C" int64_t sp_gemm_q4_workspace_floats(int x_dtype, int T, int N, int K) {
  if (T <= 0 || N <= 0 || K <= 0) return 0;
  const int splits = q4_plan(x_dtype, T, N, K).splits;
  return splits > 1 ? int64_t(splits) * T * N : 0;
}

extern "C" int sp_gemm_q4(void* stream, int x_dtype, const void* x, const void* words, int scale_dtype, const void* scales, int bias_dtype,
                          const void* bias, int mode, int out_dtype, void* out, int T, int N, int K, int group, float* workspace,
                          int64_t workspace_floats) {
  SP_REQUIRE(q4_sizes(N, K, group) && T >= 0, "sp_gemm_q4: T=%d N=%d K=%d group=%d (groups of 32, 64 or 128)", T, N, K, group);
  SP_REQUIRE((x_dtype == kF32 || x_dtype == kBF16) && (scale_dtype == kF32 || scale_dtype == kBF16) && (bias_dtype == kF32 || bias_dtype == kBF16),
             "sp_gemm_q4: unsupported dtypes %d, %d, %d", x_dtype, scale_dtype, bias_dtype);
  SP_REQUIRE((mode == 0 && out_dtype == x_dtype) || (mode == 1 && out_dtype == kF32), "sp_gemm_q4: stores x's dtype or adds to float32, not mode %d to dtype %d", mode, out_dtype);
  if (T == 0) return 0;
  SP_REQUIRE(x && words && scales && out, "sp_gemm_q4: null argument");
  SP_REQUIRE(reinterpret_cast<uintptr_t>(words) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0, "sp_gemm_q4: packed weights must start at a multiple of 16 bytes");
  SP_REQUIRE(T <= 65535 * 16 && K <= 1 << 24, "sp_gemm_q4: %d tokens, K=%d", T, K);      // (64 rows of x within 32 bits)
  Q4Args a;
  a.x = x; a.words = static_cast<const uint32_t*>(words); a.scales = scales; a.bias = bias; a.out = out;
  a.T = T; a.N = N; a.K = K; a.blocks = (K + kBlockK - 1) / kBlockK; a.groups = (K + group - 1) / group; a.padded = (N + 15) / 16 * 16;
  a.bias_bf16 = bias_dtype == kBF16; a.accumulate = mode == 1;
  const Q4Plan p = q4_plan(x_dtype, T, N, K);
  const int64_t need = sp_gemm_q4_workspace_floats(x_dtype, T, N, K);
  SP_REQUIRE(need == 0 || (workspace && workspace_floats >= need), "sp_gemm_q4: workspace of %lld floats is smaller than the %lld needed",
             (long long)workspace_floats, (long long)need);
  a.splits = p.splits;
  a.parts = workspace;
  a.fours = N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 == 0;
  const bool vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  const int steps = group / 32;
  const bool launched = x_dtype == kF32 ? (scale_dtype == kF32 ? launch_q4_of<float, float>(s, a, p, steps, vec) : launch_q4_of<float, uint16_t>(s, a, p, steps, vec))
                                        : (scale_dtype == kF32 ? launch_q4_of<uint16_t, float>(s, a, p, steps, vec) : launch_q4_of<uint16_t, uint16_t>(s, a, p, steps, vec));
  return launched ? check_launch("sp_gemm_q4") : 1;
}
