// k_fp8.hip -- 8-bit operands for the block-scaled products: the quantizers of activations and
// weights, and T5LayerNorm (src/quantized_t5.rs:163-172) with the residual's addition in front and
// codes behind.  No counterpart in the reference, whose products are f32, bf16 or Q4_K x Q8_K.
//
// Per block of up to 128 values: a = max |x| over the finite ones; the scale s is the smallest power
// of two with a <= 448 s (activations), or a / 448 in f32 (weights with float scales); codes are
// e4m3(x / s), for float scales e4m3(x fl(448 / a)).  Both are bound below by s = 2^-126, so that no
// inverse overflows and an all-zero block has codes 0.  Values that are not finite get the NaN code.
//
// All three kernels read each value once and write each code once: what bounds them is memory, and a launch
// where there is little of it.
#include "fp8.hpp"

namespace {
using namespace t5k;

// 4 values at p[i..i+3] of an io type, as floats (i a multiple of 4, p 16-byte aligned).
template <int T>
__device__ __forceinline__ f4 load4(const void* p, size_t i) {
  if constexpr (T == FP8_IO_F32) {
    return *reinterpret_cast<const f4*>((const float*)p + i);
  } else if constexpr (T == FP8_IO_F16) {
    return __builtin_convertvector(*reinterpret_cast<const h4*>((const _Float16*)p + i), f4);
  } else {
    return __builtin_convertvector(*reinterpret_cast<const b4*>((const __bf16*)p + i), f4);
  }
}
template <int T>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&v)[8]) {
  if constexpr (T == FP8_IO_F32) {
    const f4 a = load4<T>(p, i), b = load4<T>(p, i + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
      v[e] = T == FP8_IO_F16 ? f16_bits_to_f32(h) : __uint_as_float(h << 16);
    }
  }
}

// ---- activations: 16 threads per block of 128, 8 values each --------------------------------
// 8 values are one 16-byte load of a 16-bit type and one 8-byte store, and 16 threads are a row of the wave's
// lanes, whose maximum takes four lane moves and no LDS.  74,640 x 768 takes 42 us from f32 (6.9 TB/s, some of it
// from the last-level cache), 28.5 from f16; 30,000 x 8,192 from bf16 128 us (5.8 TB/s).  A large copy has 5.0.
template <int T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const void* x, int K, int kb, uint32_t blocks,
                                                           size_t m16, uint8_t* codes, uint8_t* scales) {
  const int t = threadIdx.x & 15;
  for (uint32_t b = blockIdx.x * 16 + (threadIdx.x >> 4); b < blocks; b += gridDim.x * 16) {
    const uint32_t row = b / (uint32_t)kb, blk = b - row * (uint32_t)kb;
    const int k = (int)blk * FP8_BLOCK + 8 * t;
    const size_t at = (size_t)row * K + k;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < K) load8<T>(x, at, v);
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) top = fmaxf(top, finite_abs(v[e]));
    top = max_row16(top);
    const uint32_t byte = e8m0_of(top);
    const float inv = e8m0_inverse(byte);
    if (k < K) {
      uint2 q;
      q.x = e4m3_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      q.y = e4m3_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
      *reinterpret_cast<uint2*>(codes + at) = q;
    }
    if (t == 0) scales[blk * m16 + row] = (uint8_t)byte;
  }
}

// ---- weights: one workgroup per 128 x 128 block, all of it in registers ----------------------
// A block's scale needs all of it, so it is held (64 values a thread) rather than read twice.  8,192 x 4,096 from
// f32: 31.3 us (5.4 TB/s), from the same matrix again 25.8, as the last-level cache holds part of its 134 MB; byte
// scales 26.3.
template <int T>
__global__ __launch_bounds__(256) void fp8_quantize_weights_kernel(const void* w, int N, int K, int kb,
                                                                   uint32_t blocks, int f32_scales, uint8_t* codes, void* scales) {
  __shared__ float part[4];
  const int t = threadIdx.x & 15, r = threadIdx.x >> 4;
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int n0 = (int)(b / (uint32_t)kb) * FP8_BLOCK, k = (int)(b % (uint32_t)kb) * FP8_BLOCK + 8 * t;
    float v[8][8];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = 0.f;
      const int n = n0 + 16 * i + r;
      if (n < N && k < K) load8<T>(w, (size_t)n * K + k, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) top = fmaxf(top, finite_abs(v[i][e]));
    top = max_xor32(max_xor16(max_row16(top)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    __syncthreads();  // part is written again by the next block
    float inv;
    if (f32_scales) {
      top = fmaxf(top, 448.f * 0x1p-126f);
      inv = 448.f / top;
      if (threadIdx.x == 0) ((float*)scales)[b] = top / 448.f;
    } else {
      const uint32_t byte = e8m0_of(top);
      inv = e8m0_inverse(byte);
      if (threadIdx.x == 0) ((uint8_t*)scales)[b] = (uint8_t)byte;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int n = n0 + 16 * i + r;
      if (n < N && k < K) {
        uint2 q;
        q.x = e4m3_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        q.y = e4m3_pack4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        *reinterpret_cast<uint2*>(codes + (size_t)n * K + k) = q;
      }
    }
  }
}

// ---- residual's addition, T5LayerNorm, codes -------------------------------------------------
// h = x + delta rounded to x's type, as the stream stores it; the norm is of the stored values, so a
// later reader of the stream sees what this norm saw.  Sums of squares in f32.
template <int T>
__device__ __forceinline__ f4 round_to(f4 v) {
  if constexpr (T == FP8_IO_F16) return __builtin_convertvector(__builtin_convertvector(v, h4), f4);
  if constexpr (T == FP8_IO_BF16) return __builtin_convertvector(__builtin_convertvector(v, b4), f4);
  return v;
}
template <int T>
__device__ __forceinline__ void store4(void* p, size_t i, f4 v) {
  if constexpr (T == FP8_IO_F32) *reinterpret_cast<f4*>((float*)p + i) = v;
  else if constexpr (T == FP8_IO_F16) *reinterpret_cast<h4*>((_Float16*)p + i) = __builtin_convertvector(v, h4);
  else *reinterpret_cast<b4*>((__bf16*)p + i) = __builtin_convertvector(v, b4);
}
template <int XT, int DT>
__device__ __forceinline__ f4 load_h(const Fp8NormArgs& a, size_t at) {
  f4 h = load4<XT>(a.x, at);
  if constexpr (DT != FP8_IO_NONE) h = round_to<XT>(h + load4<DT>(a.delta, at));
  return h;
}

// codes and scale of 4 normed values per lane, 32 lanes per block
__device__ __forceinline__ void norm_codes(const Fp8NormArgs& a, size_t row, int k, f4 h, float rs, bool ok, int lane,
                                           size_t m16) {
  f4 y = f4{0.f, 0.f, 0.f, 0.f};
  if (ok) {
    const f4 g = *reinterpret_cast<const f4*>(a.gamma + k);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = h[e] * rs * g[e];
  }
  float top = fmaxf(fmaxf(finite_abs(y[0]), finite_abs(y[1])), fmaxf(finite_abs(y[2]), finite_abs(y[3])));
  top = max_xor16(max_row16(top));
  const uint32_t byte = e8m0_of(top);
  const float inv = e8m0_inverse(byte);
  if (ok) {
    *reinterpret_cast<uint32_t*>(a.codes + row * a.D + k) =
        e4m3_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    if ((lane & 31) == 0) a.scales[(size_t)(k / FP8_BLOCK) * m16 + row] = (uint8_t)byte;
  }
}

// A row stays in registers between its sum of squares and its codes: one wave for up to 1,024 values (four rows
// a workgroup, no barrier), 4 or 16 waves past that, so that a lane holds at most 16 values and a lone row of
// 8,192 takes 3.7 us, half of it the launch.  74,640 x 768, f32 with an f16 delta: 114 us, 5.5 TB/s; 4,616 x 768:
// 7.7 us, 5.1 TB/s; 74,640 x 768 all in bf16 77 us, 5.2 TB/s.  Four waves a row: 20,000 x 2,048 in bf16 54 us, 5.3
// TB/s.  Sixteen: 5,000 x 8,192 in f32 with an f16 delta 87 us, 5.2 TB/s, in bf16 73 to 77 us, 3.7 to 3.9 TB/s (two
// rows of 16 waves fill a compute unit, and each waits twice for its slowest wave).
// W waves per row, C chunks of 256 W values in registers; C = 0: a row of any length, read twice
// (the second time from the stored sum, where there is one: it may have replaced x or delta).
template <int XT, int DT, int W, int C>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void fp8_rmsnorm_kernel(Fp8NormArgs a) {
  constexpr int ROWS = W == 1 ? 4 : 1, N = C ? C : 1;
  __shared__ float part[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = W == 1 ? 0 : wave;
  const size_t m16 = fp8_scale_rows(a.M);
  const int chunks = (a.D + 256 * W - 1) / (256 * W), k0 = 256 * w + 4 * lane;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + (W == 1 ? wave : 0); row < a.M; row += (int64_t)gridDim.x * ROWS) {
    const size_t base = (size_t)row * a.D;
    f4 h[N];
    float ss = 0.f;
    if constexpr (C > 0) {
#pragma unroll
      for (int c = 0; c < C; c++) {
        h[c] = f4{0.f, 0.f, 0.f, 0.f};
        const int k = k0 + 256 * W * c;
        if (k < a.D) h[c] = load_h<XT, DT>(a, base + k);
      }
#pragma unroll
      for (int c = 0; c < C; c++) {
        const int k = k0 + 256 * W * c;
        if (DT != FP8_IO_NONE && a.sum && k < a.D) store4<XT>(a.sum, base + k, h[c]);
#pragma unroll
        for (int e = 0; e < 4; e++) ss = __builtin_fmaf(h[c][e], h[c][e], ss);
      }
    } else {
      for (int c = 0; c < chunks; c++) {
        const int k = k0 + 256 * W * c;
        if (k >= a.D) break;
        const f4 v = load_h<XT, DT>(a, base + k);
        if (DT != FP8_IO_NONE && a.sum) store4<XT>(a.sum, base + k, v);
#pragma unroll
        for (int e = 0; e < 4; e++) ss = __builtin_fmaf(v[e], v[e], ss);
      }
    }
    ss = sum_xor32(sum_xor16(sum_row16(ss)));
    if constexpr (W > 1) {
      if (lane == 0) part[w] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < W; i++) ss += part[i];
      __syncthreads();  // part is written again for the next row
    }
    const float rs = rsqrtf(ss / (float)a.D + a.eps);
    if constexpr (C > 0) {
#pragma unroll
      for (int c = 0; c < C; c++) {
        const int k = k0 + 256 * W * c;
        if (256 * (W * c + w) < a.D) norm_codes(a, row, k, h[c], rs, k < a.D, lane, m16);
      }
    } else {
      for (int c = 0; c < chunks; c++) {
        const int k = k0 + 256 * W * c;
        if (256 * (W * c + w) >= a.D) break;
        f4 v = f4{0.f, 0.f, 0.f, 0.f};
        if (k < a.D) v = DT != FP8_IO_NONE && a.sum ? load4<XT>(a.sum, base + k) : load_h<XT, DT>(a, base + k);
        norm_codes(a, row, k, v, rs, k < a.D, lane, m16);
      }
    }
  }
}

template <int XT, int DT>
hipError_t launch_norm(const Fp8NormArgs& a, hipStream_t s) {
  const int64_t most = 1 << 20;  // workgroups; the kernels walk what is left
  if (a.D <= 1024) {
    const int grid = (int)std::min<int64_t>(((int64_t)a.M + 3) / 4, most);
    T5K_LAUNCH((fp8_rmsnorm_kernel<XT, DT, 1, 4>), dim3(grid), dim3(256), 0, s, a);
  } else {
    const int grid = (int)std::min<int64_t>(a.M, most);
    if (a.D <= 4096) T5K_LAUNCH((fp8_rmsnorm_kernel<XT, DT, 4, 4>), dim3(grid), dim3(256), 0, s, a);
    else if (a.D <= 16384) T5K_LAUNCH((fp8_rmsnorm_kernel<XT, DT, 16, 4>), dim3(grid), dim3(1024), 0, s, a);
    else T5K_LAUNCH((fp8_rmsnorm_kernel<XT, DT, 16, 0>), dim3(grid), dim3(1024), 0, s, a);
  }
  return hipGetLastError();
}
template <int XT>
hipError_t launch_norm_x(const Fp8NormArgs& a, hipStream_t s) {
  if (!a.delta) return launch_norm<XT, FP8_IO_NONE>(a, s);
  switch (a.delta_type) {
    case FP8_IO_F32: return launch_norm<XT, FP8_IO_F32>(a, s);
    case FP8_IO_F16: return launch_norm<XT, FP8_IO_F16>(a, s);
    case FP8_IO_BF16: return launch_norm<XT, FP8_IO_BF16>(a, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace

namespace t5k {
hipError_t launch_fp8_quantize(const void* x, int type, int M, int K, uint8_t* codes, uint8_t* scales,
                               hipStream_t s) {
  const int kb = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const uint64_t blocks = (uint64_t)M * kb;
  if (M <= 0 || K <= 0 || K % 16 || blocks >> 31) return M == 0 ? hipSuccess : hipErrorInvalidValue;
  const dim3 grid((unsigned)std::min<uint64_t>((blocks + 15) / 16, 1 << 20));
  const size_t m16 = fp8_scale_rows(M);
  switch (type) {
    case FP8_IO_F32:
      T5K_LAUNCH((fp8_quantize_kernel<FP8_IO_F32>), grid, dim3(256), 0, s, x, K, kb, (uint32_t)blocks, m16, codes, scales);
      break;
    case FP8_IO_F16:
      T5K_LAUNCH((fp8_quantize_kernel<FP8_IO_F16>), grid, dim3(256), 0, s, x, K, kb, (uint32_t)blocks, m16, codes, scales);
      break;
    case FP8_IO_BF16:
      T5K_LAUNCH((fp8_quantize_kernel<FP8_IO_BF16>), grid, dim3(256), 0, s, x, K, kb, (uint32_t)blocks, m16, codes, scales);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_fp8_quantize_weights(const void* w, int type, int N, int K, int scale_type, uint8_t* codes,
                                       void* scales, hipStream_t s) {
  const int kb = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const uint64_t blocks = (uint64_t)((N + (int64_t)FP8_BLOCK - 1) / FP8_BLOCK) * kb;
  if (N <= 0 || K <= 0 || K % 16 || blocks >> 31) return N == 0 ? hipSuccess : hipErrorInvalidValue;
  const dim3 grid((unsigned)std::min<uint64_t>(blocks, 1 << 20));
  const int f32s = scale_type == FP8_F32;
  switch (type) {
    case FP8_IO_F32:
      T5K_LAUNCH((fp8_quantize_weights_kernel<FP8_IO_F32>), grid, dim3(256), 0, s, w, N, K, kb, (uint32_t)blocks, f32s, codes, scales);
      break;
    case FP8_IO_F16:
      T5K_LAUNCH((fp8_quantize_weights_kernel<FP8_IO_F16>), grid, dim3(256), 0, s, w, N, K, kb, (uint32_t)blocks, f32s, codes, scales);
      break;
    case FP8_IO_BF16:
      T5K_LAUNCH((fp8_quantize_weights_kernel<FP8_IO_BF16>), grid, dim3(256), 0, s, w, N, K, kb, (uint32_t)blocks, f32s, codes, scales);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_fp8_rmsnorm(const Fp8NormArgs& a, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  if (a.M < 0 || a.D <= 0 || a.D % 16) return hipErrorInvalidValue;
  switch (a.x_type) {
    case FP8_IO_F32: return launch_norm_x<FP8_IO_F32>(a, s);
    case FP8_IO_F16: return launch_norm_x<FP8_IO_F16>(a, s);
    case FP8_IO_BF16: return launch_norm_x<FP8_IO_BF16>(a, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace t5k
