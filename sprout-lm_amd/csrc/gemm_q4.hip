// Products with weights of 4 bits and a scale per group of K, for the few tokens of decode and verify steps.
//
//   out[t, n] = sum over groups g of scale[n, g] * sum over k in g of (code[n, k] - 8) x[t, k]   (+ bias[n])       code 0 .. 15
//
// The weights' bytes bound it: they are laid out once (sp_q4_pack) so that a wave's 16-byte loads are the matrix instruction's operands,
// a lane's four words being its eight codes of each of four steps of 32 along K, of 16 rows of weights.  A code becomes a bfloat16
// number without a conversion: put into bits 3 to 6 of the mantissa of 16.0 it reads 16 + code, exactly, two codes an instruction
// and its shift.  The 24 too much is taken off by the matrix cores: the sums of a group start from the product of x with rows of -24,
// which is the same for all rows of weights and costs one product beside those of a wave's 16 NT rows.  So the codes, which are
// whole numbers, meet x unrounded; the sums of a group are float32 and multiplied by the scale in float32.
// float32 x is taken as the sum of three bfloat16 numbers, which holds all its bits: three products each.
#include "mfma.h"
#include "sprout_hip.h"

namespace sprout {

// bfloat16 x and results are handled as their bits
template <> __device__ __forceinline__ uint16_t from_float<uint16_t>(float f) { return f32_to_bf16_bits(f); }

namespace {

constexpr int kBlockK = 128;      // k of one 16-byte load of a lane: four steps of 32

struct Q4Args {
  const void* x;
  const uint32_t* words;      // [rows / 16][K / 128][64 lanes][4]
  const void* scales;         // [groups][rows up to a multiple of 16]
  const void* bias;
  void* out;
  int T, N, K, blocks, groups, padded;      // blocks: of 128 along K; padded: N up to a multiple of 16
  int scales_bf16, bias_bf16, accumulate;
};

__device__ __forceinline__ bf16x8 codes_plus_16(uint32_t w) {
  constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u;
  return as_bf16x8(make_uint4(((w << 3) & kMask) | kSixteen, ((w >> 1) & kMask) | kSixteen, ((w >> 5) & kMask) | kSixteen, ((w >> 9) & kMask) | kSixteen));
}
__device__ __forceinline__ float4 four_scales(const void* scales, int bf16, size_t at) {
  if (bf16) {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(scales) + at);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  }
  return *reinterpret_cast<const float4*>(static_cast<const float*>(scales) + at);
}

// Eight numbers of token t from k on, as PARTS operands.  VEC: rows start at whole 16 bytes and K is whole eights.
template <bool VEC>
__device__ __forceinline__ void x_operand(const uint16_t* x, int t, int k, int K, bf16x8 (&p)[1]) {
  const uint16_t* src = x + size_t(t) * K + k;
  if (VEC) {
    p[0] = as_bf16x8(k < K ? ldg128(src) : make_uint4(0, 0, 0, 0));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (k + 2 * j < K ? uint32_t(src[2 * j]) : 0u) | (k + 2 * j + 1 < K ? uint32_t(src[2 * j + 1]) << 16 : 0u);
    p[0] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
  }
}
template <bool VEC>
__device__ __forceinline__ void x_operand(const float* x, int t, int k, int K, bf16x8 (&p)[3]) {
  const float* src = x + size_t(t) * K + k;
  float f[8];
  if (VEC) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (k < K) { a = *reinterpret_cast<const float4*>(src); b = *reinterpret_cast<const float4*>(src + 4); }
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = k + j < K ? src[j] : 0.f;
  }
  uint4 q[3];
  three_parts(f[0], f[1], q[0].x, q[1].x, q[2].x);
  three_parts(f[2], f[3], q[0].y, q[1].y, q[2].y);
  three_parts(f[4], f[5], q[0].z, q[1].z, q[2].z);
  three_parts(f[6], f[7], q[0].w, q[1].w, q[2].w);
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = as_bf16x8(q[i]);
}

// A block of four waves: NT tiles of 16 rows of weights by TT tiles of 16 tokens, the waves take turns along K and join in LDS.
// X: x's type; STEPS: steps of 32 in a group.
template <typename X, int NT, int TT, int STEPS, bool VEC>
__global__ __launch_bounds__(256) void gemm_q4_kernel(Q4Args a) {
  constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
  __shared__ floatx4 s_sums[3][NT * TT][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lr = lane & 15, lj = lane >> 4;
  const int tile0 = blockIdx.x * NT, tiles = a.padded / 16, t0 = blockIdx.y * 16 * TT;
  floatx4 total[NT][TT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < TT; ++t) total[n][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 minus24 = as_bf16x8(make_uint4(0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u));
  for (int kb = wave; kb < a.blocks; kb += 4) {
    uint4 w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = ldg128(a.words + (size_t(min(tile0 + n, tiles - 1)) * a.blocks + kb) * 256 + 4 * lane);
#pragma unroll
    for (int gs = 0; gs < 4 / STEPS; ++gs) {
      bf16x8 b[TT][STEPS][PARTS];
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
          x_operand<VEC>(static_cast<const X*>(a.x), min(t0 + 16 * t + lr, a.T - 1), kBlockK * kb + 32 * (gs * STEPS + s) + 8 * lj, a.K, b[t][s]);
      floatx4 off[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        off[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) off[t] = mfma16(minus24, b[t][s][p], off[t]);
      }
      const int group = min((4 * kb) / STEPS + gs, a.groups - 1);      // (behind the last group x is zero)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float4 scale = four_scales(a.scales, a.scales_bf16, size_t(group) * a.padded + 16 * min(tile0 + n, tiles - 1) + 4 * lj);
        const uint32_t words[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
        bf16x8 c[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) c[s] = codes_plus_16(words[gs * STEPS + s]);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          floatx4 sum = off[t];
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int p = PARTS - 1; p >= 0; --p) sum = mfma16(c[s], b[t][s][p], sum);
          total[n][t][0] += scale.x * sum[0];
          total[n][t][1] += scale.y * sum[1];
          total[n][t][2] += scale.z * sum[2];
          total[n][t][3] += scale.w * sum[3];
        }
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int t = 0; t < TT; ++t) s_sums[wave - 1][n * TT + t][lane] = total[n][t];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const floatx4 v = total[n][t] + s_sums[0][n * TT + t][lane] + s_sums[1][n * TT + t][lane] + s_sums[2][n * TT + t][lane];
      const int token = t0 + 16 * t + lr;
      if (token >= a.T) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * (tile0 + n) + 4 * lj + r;
        if (row >= a.N) continue;
        float y = v[r];
        if (a.bias) y += a.bias_bf16 ? to_float(static_cast<const bf16_t*>(a.bias)[row]) : static_cast<const float*>(a.bias)[row];
        const size_t at = size_t(token) * a.N + row;
        if (a.accumulate) static_cast<float*>(a.out)[at] += y;
        else static_cast<X*>(a.out)[at] = from_float<X>(y);
      }
    }
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

template <typename X, int NT, int TT, bool VEC> void launch_q4(hipStream_t s, const Q4Args& a, int steps) {
  const dim3 grid((a.padded / 16 + NT - 1) / NT, (a.T + 16 * TT - 1) / (16 * TT));
  if (steps == 1) gemm_q4_kernel<X, NT, TT, 1, VEC><<<grid, 256, 0, s>>>(a);
  else if (steps == 2) gemm_q4_kernel<X, NT, TT, 2, VEC><<<grid, 256, 0, s>>>(a);
  else gemm_q4_kernel<X, NT, TT, 4, VEC><<<grid, 256, 0, s>>>(a);
}
template <typename X> void launch_q4_of(hipStream_t s, const Q4Args& a, int steps, bool vec) {
  if (vec) launch_q4<X, 1, 1, true>(s, a, steps);
  else launch_q4<X, 1, 1, false>(s, a, steps);
}

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
  SP_REQUIRE(total / 256 < (size_t(1) << 31) && size_t(groups) * padded / 256 < (size_t(1) << 31) - 1, "sp_q4_pack: the matrix is too large");
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
  SP_REQUIRE(units / 4 < (size_t(1) << 31) - 1, "sp_q4_quantize: the matrix is too large");
  const unsigned grid = unsigned((units + 3) / 4);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* c = static_cast<uint8_t*>(codes);
  if (w_dtype == kF32 && scale_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(w), c, static_cast<float*>(scales), N, K, group, groups);
  else if (w_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(w), c, static_cast<bf16_t*>(scales), N, K, group, groups);
  else if (scale_dtype == kF32) q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16_t*>(w), c, static_cast<float*>(scales), N, K, group, groups);
  else q4_quantize_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16_t*>(w), c, static_cast<bf16_t*>(scales), N, K, group, groups);
  return check_launch("sp_q4_quantize");
}

extern "C" int sp_gemm_q4(void* stream, int x_dtype, const void* x, const void* words, int scale_dtype, const void* scales, int bias_dtype,
                          const void* bias, int mode, int out_dtype, void* out, int T, int N, int K, int group) {
  SP_REQUIRE(q4_sizes(N, K, group) && T >= 0, "sp_gemm_q4: T=%d N=%d K=%d group=%d (groups of 32, 64 or 128)", T, N, K, group);
  SP_REQUIRE((x_dtype == kF32 || x_dtype == kBF16) && (scale_dtype == kF32 || scale_dtype == kBF16) && (bias_dtype == kF32 || bias_dtype == kBF16),
             "sp_gemm_q4: unsupported dtypes %d, %d, %d", x_dtype, scale_dtype, bias_dtype);
  SP_REQUIRE((mode == 0 && out_dtype == x_dtype) || (mode == 1 && out_dtype == kF32), "sp_gemm_q4: stores x's dtype or adds to float32, not mode %d to dtype %d", mode, out_dtype);
  if (T == 0) return 0;
  SP_REQUIRE(x && words && scales && out, "sp_gemm_q4: null argument");
  SP_REQUIRE(reinterpret_cast<uintptr_t>(words) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0, "sp_gemm_q4: packed weights must start at a multiple of 16 bytes");
  SP_REQUIRE(T <= 65535 * 16, "sp_gemm_q4: %d tokens", T);
  Q4Args a;
  a.x = x; a.words = static_cast<const uint32_t*>(words); a.scales = scales; a.bias = bias; a.out = out;
  a.T = T; a.N = N; a.K = K; a.blocks = (K + kBlockK - 1) / kBlockK; a.groups = (K + group - 1) / group; a.padded = (N + 15) / 16 * 16;
  a.scales_bf16 = scale_dtype == kBF16; a.bias_bf16 = bias_dtype == kBF16; a.accumulate = mode == 1;
  const int per = x_dtype == kF32 ? 4 : 8;
  const bool vec = K % 8 == 0 && K % per == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (x_dtype == kF32) launch_q4_of<float>((hipStream_t)stream, a, group / 32, vec);
  else launch_q4_of<uint16_t>((hipStream_t)stream, a, group / 32, vec);
  return check_launch("sp_gemm_q4");
}
