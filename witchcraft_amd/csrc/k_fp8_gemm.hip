// k_fp8_gemm.hip -- products of e4m3 activations and e4m3 weights with a scale per block of 128, and
// the gated product gelu(a w0^T) * (a w1^T) that writes the next product's codes and scales.
//
//   c[m][n] = sum over K blocks b of sa[b][m] sw[n / 128][b] sum_{k in b} a[m][k] w[n][k]
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 takes one K block of a 16 x 16 tile.  Its lanes hold 32 bytes
// of one row each; which K bytes a lane holds does not matter as long as both operands agree and all
// 128 have the same scale.  Weights are its first operand and activations its second, so that lane l
// ends with 4 consecutive columns 4 (l / 16) .. +3 of row l % 16.  The activations' scale byte goes in
// as the instruction's own scale operand, and so does the weights' byte; float weight scales multiply
// the block's sum in f32 on the vector unit.
//
// Precision.  The fp8 MFMAs add their products in groups of 8 to 16 values, each aligned to the
// group's largest product with 14 bits or so (measured: 2^14 + 2^0 in one group gives 2^14, 2^14 +
// 2^2 is kept; sums of groups and blocks are f32).  On normal data that is an error of 1.3e-5 of the
// result's norm: below the rounding of f16 (2^-11 of a value) and bf16 results and of codes (2^-4),
// but not what an f32 result promises.  f32 results are therefore computed exactly to f32 sums on
// v_mfma_f32_16x16x32_f16, at half the rate, from codes widened to f16 (every e4m3 value is one).
#include "fp8.hpp"

namespace {
using namespace t5k;

typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));

// e4m3 codes of a lane's 32 bytes, 8 at a time, as f16: exact.
__device__ __forceinline__ h8 widen8(int lo, int hi) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return h8{(_Float16)a[0], (_Float16)a[1], (_Float16)b[0], (_Float16)b[1],
            (_Float16)c[0], (_Float16)c[1], (_Float16)d[0], (_Float16)d[1]};
}

// acc += one K block of a 16 x 16 tile.  sa: the scale byte of the lane's row (l % 16); swb / swf: the
// weights' byte or float.
template <bool EXACT, int ST>
__device__ __forceinline__ void block_product(const i8v& w, const i8v& a, uint32_t sa, uint32_t swb, float swf, f4& acc) {
  const f4 zero = f4{0.f, 0.f, 0.f, 0.f};
  if constexpr (EXACT) {
    f4 t = zero;
#pragma unroll
    for (int i = 0; i < 4; i++)
      t = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(w[2 * i], w[2 * i + 1]), widen8(a[2 * i], a[2 * i + 1]), t, 0, 0, 0);
    const float f = e8m0_value(sa) * (ST == FP8_E8M0 ? e8m0_value(swb) : swf);
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(t[e], f, acc[e]);
  } else if constexpr (ST == FP8_E8M0) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, (int)swb, 0, (int)sa);
  } else {
    const f4 t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, zero, 0, 0, 0, 127, 0, (int)sa);
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(t[e], swf, acc[e]);
  }
}

// A lane's 32 bytes of K block kb of a row: 16-byte chunks g and g + 4 of its eight (g = lane / 16).
// Chunks at or past K are zero and not read.
__device__ __forceinline__ i8v load_row(const uint8_t* row, int kb, int g, int K) {
  const int k = kb * FP8_BLOCK + 16 * g;
  i4v lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (k < K) lo = *reinterpret_cast<const i4v*>(row + k);
  if (k + 64 < K) hi = *reinterpret_cast<const i4v*>(row + k + 64);
  return i8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Four consecutive columns n .. n + 3 of row m of the product.
__device__ __forceinline__ void store_out(const Fp8GemmArgs& p, int m, int n, f4 v) {
  if (m >= p.M || n >= p.N) return;
  const size_t at = (size_t)m * p.N + n;
  if ((p.N & 3) == 0) {  // whole quads, aligned
    if (p.out_type == FP8_IO_F32) *reinterpret_cast<f4*>((float*)p.out + at) = v;
    else if (p.out_type == FP8_IO_F16) *reinterpret_cast<h4*>((_Float16*)p.out + at) = __builtin_convertvector(v, h4);
    else *reinterpret_cast<b4*>((__bf16*)p.out + at) = __builtin_convertvector(v, b4);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (n + e < p.N) {
      if (p.out_type == FP8_IO_F32) ((float*)p.out)[at + e] = v[e];
      else if (p.out_type == FP8_IO_F16) ((_Float16*)p.out)[at + e] = (_Float16)v[e];
      else ((__bf16*)p.out)[at + e] = (__bf16)v[e];
    }
}

// ---- few rows: 16 MB rows x 16 NB columns per workgroup, its waves on the K blocks in turn ---
// Each operand goes from memory straight to the wave that multiplies it; the waves' partial sums
// meet in LDS and are added in wave order.
template <bool EXACT, int ST, int MB, int NB, int KS>
__global__ __launch_bounds__(64 * KS) void fp8_small_kernel(Fp8GemmArgs p, int tiles_n, int64_t tiles) {
  __shared__ f4 red[KS][MB * NB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int kbs = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
  const size_t m16 = fp8_scale_rows(p.M);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int m0 = (int)(tile / tiles_n) * 16 * MB, n0 = (int)(tile % tiles_n) * 16 * NB;
    const uint8_t *arow[MB], *wrow[NB], *sa[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
      const int m = min(m0 + 16 * i + r, p.M - 1);
      arow[i] = p.a + (size_t)m * p.K;
      sa[i] = p.a_scales + m;
    }
#pragma unroll
    for (int j = 0; j < NB; j++) wrow[j] = p.w + (size_t)min(n0 + 16 * j + r, p.N - 1) * p.K;
    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
      for (int j = 0; j < NB; j++) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < kbs; kb += KS) {
      i8v a[MB], w[NB];
      uint32_t as[MB], wb[NB];
      float wf[NB];
#pragma unroll
      for (int j = 0; j < NB; j++) {
        w[j] = load_row(wrow[j], kb, g, p.K);
        const size_t at = (size_t)(min(n0 + 16 * j, p.N - 1) / FP8_BLOCK) * kbs + kb;
        wb[j] = ST == FP8_E8M0 ? ((const uint8_t*)p.w_scales)[at] : 0;
        wf[j] = ST == FP8_F32 ? ((const float*)p.w_scales)[at] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < MB; i++) {
        a[i] = load_row(arow[i], kb, g, p.K);
        as[i] = sa[i][kb * m16];
      }
#pragma unroll
      for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) block_product<EXACT, ST>(w[j], a[i], as[i], wb[j], wf[j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
      for (int j = 0; j < NB; j++) red[wave][i * NB + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < MB * NB; t += KS) {
      f4 v = red[0][t][lane];
#pragma unroll
      for (int k = 1; k < KS; k++) v += red[k][t][lane];
      store_out(p, m0 + 16 * (t / NB) + r, n0 + 16 * (t % NB) + 4 * g, v);
    }
    __syncthreads();  // red is written again for the next tile
  }
}

// ---- gated, few rows: 16 MB rows x one block of 128 columns per workgroup --------------------
// Eight waves side by side, 16 gate and the same 16 up columns each, KS such groups on the K blocks in
// turn.  gelu(gate) * up stays in registers; the rows' maxima over the 128 columns meet in LDS.
template <int ST, int MB, int KS>
__global__ __launch_bounds__(512 * KS) void fp8_small_gated_kernel(Fp8GemmArgs p, int tiles_n, int64_t tiles) {
  __shared__ f4 red[KS > 1 ? KS - 1 : 1][8][2 * MB][64];
  __shared__ float tops[8][16 * MB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int col = wave & 7, ks = wave >> 3;
  const int kbs = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
  const size_t m16 = fp8_scale_rows(p.M);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int m0 = (int)(tile / tiles_n) * 16 * MB, blk = (int)(tile % tiles_n), n0 = blk * FP8_BLOCK + 16 * col;
    const bool live = n0 < p.N;  // N % 16 == 0: whole waves
    f4 acc[2][MB];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[0][i] = acc[1][i] = f4{0.f, 0.f, 0.f, 0.f};
    if (live) {
      const uint8_t* wrow[2] = {p.w + (size_t)(n0 + r) * p.K, p.w1 + (size_t)(n0 + r) * p.K};
      const void* ws[2] = {p.w_scales, p.w1_scales};
      const uint8_t *arow[MB], *sa[MB];
#pragma unroll
      for (int i = 0; i < MB; i++) {
        const int m = min(m0 + 16 * i + r, p.M - 1);
        arow[i] = p.a + (size_t)m * p.K;
        sa[i] = p.a_scales + m;
      }
      for (int kb = ks; kb < kbs; kb += KS) {
        i8v a[MB], w[2];
        uint32_t as[MB], wb[2];
        float wf[2];
        const size_t at = (size_t)blk * kbs + kb;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          w[j] = load_row(wrow[j], kb, g, p.K);
          wb[j] = ST == FP8_E8M0 ? ((const uint8_t*)ws[j])[at] : 0;
          wf[j] = ST == FP8_F32 ? ((const float*)ws[j])[at] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < MB; i++) {
          a[i] = load_row(arow[i], kb, g, p.K);
          as[i] = sa[i][kb * m16];
        }
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) block_product<false, ST>(w[j], a[i], as[i], wb[j], wf[j], acc[j][i]);
      }
    }
    if constexpr (KS > 1) {
      if (ks > 0)
#pragma unroll
        for (int i = 0; i < MB; i++) red[ks - 1][col][2 * i][lane] = acc[0][i], red[ks - 1][col][2 * i + 1][lane] = acc[1][i];
      __syncthreads();
      if (ks == 0)
#pragma unroll
        for (int k = 0; k < KS - 1; k++)
#pragma unroll
          for (int i = 0; i < MB; i++) acc[0][i] += red[k][col][2 * i][lane], acc[1][i] += red[k][col][2 * i + 1][lane];
    }
    f4 y[MB];
    if (ks == 0) {
#pragma unroll
      for (int i = 0; i < MB; i++) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          y[i][e] = gelu_tanh_dev(acc[0][i][e]) * acc[1][i][e];
          top = fmaxf(top, finite_abs(y[i][e]));
        }
        top = max_xor32(max_xor16(top));
        if (g == 0) tops[col][16 * i + r] = live ? top : 0.f;
      }
    }
    __syncthreads();
    if (ks == 0) {
#pragma unroll
      for (int i = 0; i < MB; i++) {
        float top = tops[0][16 * i + r];
#pragma unroll
        for (int c = 1; c < 8; c++) top = fmaxf(top, tops[c][16 * i + r]);
        const uint32_t byte = e8m0_of(top);
        const float inv = e8m0_inverse(byte);
        const int m = m0 + 16 * i + r;
        if (live && m < p.M)
          *reinterpret_cast<uint32_t*>((uint8_t*)p.out + (size_t)m * p.N + n0 + 4 * g) =
              e4m3_pack4(y[i][0] * inv, y[i][1] * inv, y[i][2] * inv, y[i][3] * inv);
        if (col == 0 && g == 0 && m < p.M) p.out_scales[blk * m16 + m] = (uint8_t)byte;
      }
    }
    __syncthreads();  // tops and red are written again for the next tile
  }
}

constexpr int64_t kMostGroups = 1 << 20;  // workgroups of a launch; the kernels walk what is left

template <bool EXACT, int ST, int MB, int NB, int KS>
hipError_t launch_small(const Fp8GemmArgs& p, hipStream_t s) {
  const int tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
  const int64_t tiles = (int64_t)((p.M + 16 * MB - 1) / (16 * MB)) * tiles_n;
  T5K_LAUNCH((fp8_small_kernel<EXACT, ST, MB, NB, KS>), dim3((unsigned)std::min(tiles, kMostGroups)), dim3(64 * KS), 0,
             s, p, tiles_n, tiles);
  return hipGetLastError();
}

template <int ST, int MB, int KS>
hipError_t launch_small_gated(const Fp8GemmArgs& p, hipStream_t s) {
  const int tiles_n = (p.N + FP8_BLOCK - 1) / FP8_BLOCK;
  const int64_t tiles = (int64_t)((p.M + 16 * MB - 1) / (16 * MB)) * tiles_n;
  T5K_LAUNCH((fp8_small_gated_kernel<ST, MB, KS>), dim3((unsigned)std::min(tiles, kMostGroups)), dim3(512 * KS), 0, s,
             p, tiles_n, tiles);
  return hipGetLastError();
}
}  // namespace

namespace t5k {
hipError_t launch_fp8_matmul(const Fp8GemmArgs& p, hipStream_t s) {
  if (p.M == 0 || p.N == 0) return hipSuccess;
  if (p.M < 0 || p.N < 0 || p.K <= 0 || p.K % 16) return hipErrorInvalidValue;
  const bool exact = p.out_type == FP8_IO_F32;
  if (p.scale_type == FP8_E8M0)
    return exact ? launch_small<true, FP8_E8M0, 2, 2, 4>(p, s) : launch_small<false, FP8_E8M0, 2, 2, 4>(p, s);
  if (p.scale_type == FP8_F32)
    return exact ? launch_small<true, FP8_F32, 2, 2, 4>(p, s) : launch_small<false, FP8_F32, 2, 2, 4>(p, s);
  return hipErrorInvalidValue;
}

hipError_t launch_fp8_gated_gelu(const Fp8GemmArgs& p, hipStream_t s) {
  if (p.M == 0 || p.N == 0) return hipSuccess;
  if (p.M < 0 || p.N < 0 || p.N % 16 || p.K <= 0 || p.K % 16) return hipErrorInvalidValue;
  if (p.scale_type == FP8_E8M0) return launch_small_gated<FP8_E8M0, 2, 1>(p, s);
  if (p.scale_type == FP8_F32) return launch_small_gated<FP8_F32, 2, 1>(p, s);
  return hipErrorInvalidValue;
}
}  // namespace t5k
