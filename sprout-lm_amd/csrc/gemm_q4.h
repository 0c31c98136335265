// Products with weights of 4 bits and a scale per group of K, for the few tokens of decode and verify steps.
//
//   out[t, n] = sum over groups g of scale[n, g] * sum over k in g of (code[n, k] - 8) x[t, k]   (+ bias[n])       code 0 .. 15
//
// The weights' bytes bound it up to some 16 tokens: they are laid out once (sp_q4_pack) so that a wave's 16-byte loads are the matrix
// instruction's operands, a lane's four words being its eight codes of each of four steps of 32 along K, of 16 rows of weights.  A code
// becomes a bfloat16 number without a conversion: put into bits 3 to 6 of the mantissa of 16.0 it reads 16 + code, exactly, two codes an
// instruction and its shift.  The 24 too much is taken off by the matrix cores: x times rows of -24 is the same for all rows of
// weights and costs one product beside those of a wave's 16 NT rows.  So the codes, which are whole numbers, meet x unrounded; the sums of a
// group are float32 and multiplied by the scale in float32.
// float32 x is taken as the sum of three bfloat16 numbers, which holds all its bits: three products each.  There the codes become
// (code - 8) / 16 before the product (14 instructions for eight codes instead of 8): sums of numbers five times as large lost as much of the last places.
//
// Two kernels.  For a few tokens (gemm_q4.hip) a wave reads its operands of x itself.  A load of them touches 16 rows, which the caches
// serve at a quarter of their rate: with 64 tokens that took four times as long as everything else.  With more tokens (gemm_q4_staged.h) x comes
// through LDS, once for the four waves of a block.  Where rows of weights alone do not fill the chip several blocks (`splits`)
// share out K and a second launch joins them, in a fixed order.
//
// One token of bfloat16 by 37,888 x 3,584 in groups of 128: 15.8 us, 4.4 TB/s of weights and scales, near what a copy reaches.  64 tokens by
// 55,296 x 5,120 in groups of 32: 85.7 us, 423 TFLOP/s, bound by the vector unit, which works 37 us beside the matrix cores' 22: a group of 32 along K of
// 16 rows and 16 tokens costs one matrix instruction of 16 cycles, four float32 multiply-adds by the scale, 16 cycles, and of unpacking codes and
// scales 11 more (in groups of 128: 66 us); 432 blocks are two on 176 CUs and one on 80.  40 tokens of float32 by 3,584 x 18,944: 36.9 us, three products of bfloat16 each, 147 TFLOP/s of float32.
#pragma once
#include "mfma.h"
#include "sprout_hip.h"

namespace sprout {

// bfloat16 x and results are handled as their bits
template <> __device__ __forceinline__ uint16_t from_float<uint16_t>(float f) { return f32_to_bf16_bits(f); }

namespace q4 {

constexpr int kStagedRowTiles = 2;      // tiles of 16 rows of a wave where x comes through LDS
constexpr int kBlockK = 128;      // k of one 16-byte load of a lane: four steps of 32

struct Q4Args {
  const void* x;
  const uint32_t* words;      // [rows / 16][K / 128][64 lanes][4]
  const void* scales;         // [groups][rows up to a multiple of 16]
  const void* bias;
  void* out;
  float* parts;               // [splits][T][N], where there are several
  int T, N, K, blocks, groups, padded, splits;      // blocks: of 128 along K; padded: N up to a multiple of 16
  int bias_bf16, accumulate, fours;      // fours: N is whole fours and results start at whole 16 bytes
};

__device__ __forceinline__ uint4 codes_plus_16(uint32_t w) {
  constexpr uint32_t kMask = 0x00780078u;
  uint32_t sixteen = 0x41804180u;      // in a vector register: one of the two constants may be a scalar, then "and" and "or" are one instruction
  asm("" : "+v"(sixteen));
  return make_uint4(((w << 3) & kMask) | sixteen, ((w >> 1) & kMask) | sixteen, ((w >> 5) & kMask) | sixteen, ((w >> 9) & kMask) | sixteen);
}
__device__ __forceinline__ bf16x8 weights_operand(uint32_t w, uint16_t) { return as_bf16x8(codes_plus_16(w)); }
// For float32: (code - 8) / 16, exactly, by the conversion of four-bit numbers with a sign; two upper halves make a pair.
constexpr float kWeightsUnit = 16.f;
__device__ __forceinline__ uint32_t two_codes(uint32_t first, uint32_t second) {
  return __builtin_amdgcn_perm(__float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(int(second))), __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(int(first))), 0x07060302u);
}
__device__ __forceinline__ bf16x8 weights_operand(uint32_t w, float) {
  const uint32_t t = w ^ 0x88888888u, u = t >> 4;
  return as_bf16x8(make_uint4(two_codes(t, t >> 16), two_codes(u, u >> 16), two_codes((t >> 8) & 255u, t >> 24), two_codes((u >> 8) & 255u, u >> 24)));
}

// Scales of a lane's four rows as they lie in memory (S: bfloat16 bits or float32), and their values.
template <typename S> struct ScaleBits;
template <> struct ScaleBits<uint16_t> { uint2 v; };
template <> struct ScaleBits<float> { float4 v; };
__device__ __forceinline__ void load_scale(const uint16_t* p, ScaleBits<uint16_t>& b) { b.v = *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ void load_scale(const float* p, ScaleBits<float>& b) { b.v = *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 scale_values(const ScaleBits<uint16_t>& b) {
  return make_float4(__uint_as_float(b.v.x << 16), __uint_as_float(b.v.x & 0xffff0000u), __uint_as_float(b.v.y << 16), __uint_as_float(b.v.y & 0xffff0000u));
}
__device__ __forceinline__ float4 scale_values(const ScaleBits<float>& b) { return b.v; }

// Words asked for earlier have come here, and not been asked for later: a load whose only use lies in a loop's next turn is otherwise
// moved there, to where it is waited for.
__device__ __forceinline__ void arrived(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
__device__ __forceinline__ void arrived(ScaleBits<uint16_t>& b) { asm volatile("" : "+v"(b.v.x), "+v"(b.v.y)); }
__device__ __forceinline__ void arrived(ScaleBits<float>& b) { asm volatile("" : "+v"(b.v.x), "+v"(b.v.y), "+v"(b.v.z), "+v"(b.v.w)); }

// Eight numbers of a token from k on as they lie in memory, and as operands.  VEC: rows start at whole 16 bytes and K is whole eights; behind K
// the row's first eight are read (a load under a condition is waited for where the condition ends) and cleared before use.  Otherwise zeros lie behind K.
struct RawBf16 { uint4 v; };
struct RawF32 { float4 a, b; };
template <bool VEC> __device__ __forceinline__ void x_load(const uint16_t* row, int k, int K, RawBf16& r) {
  if (VEC) {
    r.v = ldg128(row + (k < K ? k : 0));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (k + 2 * j < K ? uint32_t(row[k + 2 * j]) : 0u) | (k + 2 * j + 1 < K ? uint32_t(row[k + 2 * j + 1]) << 16 : 0u);
    r.v = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <bool VEC> __device__ __forceinline__ void x_load(const float* row, int k, int K, RawF32& r) {
  if (VEC) {
    const float* p = row + (k < K ? k : 0);
    r.a = *reinterpret_cast<const float4*>(p);
    r.b = *reinterpret_cast<const float4*>(p + 4);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = k + j < K ? row[k + j] : 0.f;
    r.a = make_float4(f[0], f[1], f[2], f[3]);
    r.b = make_float4(f[4], f[5], f[6], f[7]);
  }
}
__device__ __forceinline__ void x_operands(const RawBf16& r, bf16x8 (&p)[1]) { p[0] = as_bf16x8(r.v); }
__device__ __forceinline__ void x_operands(const RawF32& r, bf16x8 (&p)[3]) {
  uint4 q[3];
  three_parts(r.a.x, r.a.y, q[0].x, q[1].x, q[2].x);
  three_parts(r.a.z, r.a.w, q[0].y, q[1].y, q[2].y);
  three_parts(r.b.x, r.b.y, q[0].z, q[1].z, q[2].z);
  three_parts(r.b.z, r.b.w, q[0].w, q[1].w, q[2].w);
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = as_bf16x8(q[i]);
}
__device__ __forceinline__ void clear(RawBf16& r) { r.v = make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ void clear(RawF32& r) { r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f); }
template <typename X> struct RawOf;
template <> struct RawOf<uint16_t> { typedef RawBf16 type; };
template <> struct RawOf<float> { typedef RawF32 type; };

// One result: bias, and what becomes of it.
template <typename X> __device__ __forceinline__ void store_result(const Q4Args& a, int token, int row, float y) {
  if (a.bias) y += a.bias_bf16 ? to_float(static_cast<const bf16_t*>(a.bias)[row]) : static_cast<const float*>(a.bias)[row];
  const size_t at = size_t(token) * a.N + row;
  if (a.accumulate) static_cast<float*>(a.out)[at] += y;
  else static_cast<X*>(a.out)[at] = from_float<X>(y);
}
// Four results of a token, from `row` on (a multiple of four).  Rows of whole fours are written by 16 or 8 bytes where nothing else is to be done.
template <typename X> __device__ __forceinline__ void store_four(const Q4Args& a, int split, int token, int row, floatx4 v) {
  const size_t at = size_t(token) * a.N + row;
  if (row + 3 < a.N && a.fours && (a.splits > 1 || (!a.bias && !a.accumulate))) {
    if (a.splits > 1) *reinterpret_cast<floatx4*>(a.parts + size_t(split) * a.T * a.N + at) = v;
    else if (sizeof(X) == 4) *reinterpret_cast<floatx4*>(static_cast<float*>(a.out) + at) = v;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (row + r >= a.N) continue;
    if (a.splits > 1) a.parts[size_t(split) * a.T * a.N + at + r] = v[r];
    else store_result<X>(a, token, row + r, v[r]);
  }
}

// The plan: which kernel, row_tiles (of 16 rows a wave), token_tiles (of 16 tokens a block).
struct Q4Plan { int row_tiles, token_tiles, splits, staged; };

}  // namespace q4

bool gemm_q4_staged_bf16(hipStream_t s, const q4::Q4Args& a, int token_tiles, int steps, int scales_bf16);
bool gemm_q4_staged_f32(hipStream_t s, const q4::Q4Args& a, int token_tiles, int steps, int scales_bf16);

}  // namespace sprout
