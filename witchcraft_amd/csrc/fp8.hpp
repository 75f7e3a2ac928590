// fp8.hpp -- e4m3 operands with a scale per block of 128, as the 8-bit kernels share them (gfx950).
//
// Codes are OCP e4m3 (1-4-3, bias 7, largest value 448, no infinities, 0x7f / 0xff NaN), row-major.
// Every 128 values along the summed axis share a scale (the last block of a row may be shorter).
// Activations: blocks of one row, scale 2^(byte - 127) in a byte, stored block-major, [K / 128][M16]
// with M16 = M rounded up to 16, so that the rows of a tile read one contiguous stretch per K block.
// Weights: blocks of 128 x 128, [N / 128][K / 128], a byte or a float.
//
// A power of two per activation block costs no accuracy that e4m3 has: rounding is relative to the
// value whatever the scale, and only the exponent range, 2^-9 to 448 below the block's maximum,
// loses at most a factor of two at its lower end.  The MFMAs take such a scale as an operand.
#pragma once
#include "common.hpp"

#include <algorithm>

namespace t5k {
enum Fp8Type : int { FP8_IO_F32 = 0, FP8_IO_F16 = 1, FP8_IO_BF16 = 2, FP8_IO_NONE = 3 };
enum Fp8Scale : int { FP8_E8M0 = 0, FP8_F32 = 1 };
constexpr int FP8_BLOCK = 128;
// Longest row: 64 weight rows, or 8 activation rows 8 apart, fit a buffer descriptor's 31-bit offsets.
constexpr int FP8_MAX_K = 1 << 21;
__host__ __device__ __forceinline__ size_t fp8_scale_rows(int M) { return ((size_t)M + 15) & ~(size_t)15; }

hipError_t launch_fp8_quantize(const void* x, int type, int M, int K, uint8_t* codes, uint8_t* scales, hipStream_t s);
hipError_t launch_fp8_quantize_weights(const void* w, int type, int N, int K, int scale_type, uint8_t* codes,
                                       void* scales, hipStream_t s);
struct Fp8NormArgs {
  const void* x;
  const void* delta;  // null: no addition
  void* sum;          // null: not stored; may be x or delta
  const float* gamma;
  float eps;
  int M, D, x_type, delta_type;
  uint8_t *codes, *scales;
};
hipError_t launch_fp8_rmsnorm(const Fp8NormArgs& a, hipStream_t s);

struct Fp8GemmArgs {
  const uint8_t *a, *a_scales;  // activations [M][K], [K / 128][M16]
  const uint8_t *w, *w1;        // weights [N][K]; w1: the gated product's second matrix
  const void *w_scales, *w1_scales;
  int M, N, K, scale_type;
  void* out;        // product: [M][N] of out_type; gated: codes [M][N]
  uint8_t* out_scales;
  int out_type;
};
hipError_t launch_fp8_matmul(const Fp8GemmArgs& g, hipStream_t s);
hipError_t launch_fp8_gated_gelu(const Fp8GemmArgs& g, hipStream_t s);
}  // namespace t5k

#ifdef __HIPCC__
typedef __bf16 b4 __attribute__((ext_vector_type(4)));

// 2^(byte - 127) as a float: byte 0 is the subnormal 2^-127, byte 255 NaN.
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : (b == 255 ? 0x7fc00000u : b << 23));
}

// The byte of the smallest power of two s >= 2^-126 with top <= 448 s = 1.75 * 2^8 s: the exponent of
// `top` less 8, one more when its mantissa is over 1.75 (the addition carries).  top finite, >= 0.
__device__ __forceinline__ uint32_t e8m0_of(float top) {
  const int b = (int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(b < 1 ? 1 : b);
}
// 1 / 2^(byte - 127), exact for the bytes of e8m0_of (1 .. 247).
__device__ __forceinline__ float e8m0_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// |v|, and 0 for infinities and NaN, which do not count towards a block's maximum.
__device__ __forceinline__ float finite_abs(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return __uint_as_float(u < 0x7f800000u ? u : 0u);
}

// Four values to e4m3 codes, nearest, ties to even.  |v| <= 448 (1 + 2^-23), or not finite: NaN code.
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (uint32_t)r;
}

// The same of v / s for a power of two s: one instruction divides and rounds two values.
typedef short s2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t e4m3_pack4_scaled(f4 v, float s) {
  s2v r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, v[0], v[1], s, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, v[2], v[3], s, true);
  return __builtin_bit_cast(uint32_t, r);
}

// v combined over the 16 lanes of a DPP row; every lane gets the same bits (each rotation step joins
// two halves that both lanes see).
template <int N>
__device__ __forceinline__ float dpp_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max_row16(float v) {
  v = fmaxf(v, dpp_ror<8>(v));
  v = fmaxf(v, dpp_ror<4>(v));
  v = fmaxf(v, dpp_ror<2>(v));
  return fmaxf(v, dpp_ror<1>(v));
}
__device__ __forceinline__ float sum_row16(float v) {
  v += dpp_ror<8>(v);
  v += dpp_ror<4>(v);
  v += dpp_ror<2>(v);
  return v + dpp_ror<1>(v);
}
#endif
