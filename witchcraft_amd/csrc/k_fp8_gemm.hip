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
// Precision.  The fp8 MFMAs align the products of eight consecutive K of a lane to the largest of them and
// keep 2^-13 of it (measured: 2^16 + 2^3 is exact, 2^16 + 2^2 in one group gives 2^16); sums of groups
// and blocks are f32.  A product of two codes has eight bits, so only those under 2^-6 of the largest lose any.
// Ahead of the results' rounding that is an error of 1.5e-5 of their norm on normal data, 2.4e-5 to 4.1e-5 on
// hidden states with outlying channels, where f32 sums have 3e-8 to 1e-7; of the gated product 2.2e-5 to 5.8e-5.
// Roundings to f16 (2.1e-4), bf16 (1.7e-3) and codes (2.7e-2) are larger as a whole, which is why those results
// take these instructions at twice the f16 ones' rate; of single f16 results 3 to 6% have a sum further off than
// their half step, the small ones.  It is not what an f32 result promises: those are computed exactly to f32
// sums on v_mfma_f32_16x16x32_f16, at half the rate, from codes widened to f16 (every e4m3 value is one).
#include "fp8.hpp"

#include <atomic>

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

struct Wide {
  h8 v[4];
};
__device__ __forceinline__ Wide widen(const i8v& x) {
  Wide r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.v[i] = widen8(x[2 * i], x[2 * i + 1]);
  return r;
}

// acc += one K block of a 16 x 16 tile.  sa: the scale byte of the lane's row (l % 16); swb / swf: the
// weights' byte or float.
template <int ST>
__device__ __forceinline__ void wide_product(const Wide& w, const Wide& a, uint32_t sa, uint32_t swb, float swf, f4& acc) {
  f4 t = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; i++) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], t, 0, 0, 0);
  const float f = e8m0_value(sa) * (ST == FP8_E8M0 ? e8m0_value(swb) : swf);
#pragma unroll
  for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(t[e], f, acc[e]);
}
template <bool EXACT, int ST>
__device__ __forceinline__ void block_product(const i8v& w, const i8v& a, uint32_t sa, uint32_t swb, float swf, f4& acc) {
  const f4 zero = f4{0.f, 0.f, 0.f, 0.f};
  if constexpr (EXACT) {
    wide_product<ST>(widen(w), widen(a), sa, swb, swf, acc);
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

// Four values as f16 or bf16.
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
template <int OUT>
__device__ __forceinline__ u2v half4(f4 v) {
  if constexpr (OUT == FP8_IO_F16) return __builtin_bit_cast(u2v, __builtin_convertvector(v, h4));
  else return __builtin_bit_cast(u2v, __builtin_convertvector(v, b4));
}

// Four consecutive columns n .. n + 3 of row m of the product.
template <int OUT>
__device__ __forceinline__ void store_out(const Fp8GemmArgs& p, int m, int n, f4 v) {
  if (m >= p.M || n >= p.N) return;
  const size_t at = (size_t)m * p.N + n;
  if ((p.N & 3) == 0) {  // whole quads, aligned
    if constexpr (OUT == FP8_IO_F32) *reinterpret_cast<f4*>((float*)p.out + at) = v;
    else *reinterpret_cast<u2v*>((uint16_t*)p.out + at) = half4<OUT>(v);
    return;
  }
  const u2v h = half4<OUT>(v);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (n + e < p.N) {
      if constexpr (OUT == FP8_IO_F32) ((float*)p.out)[at + e] = v[e];
      else ((uint16_t*)p.out)[at + e] = (uint16_t)(h[e / 2] >> (16 * (e % 2)));
    }
}

// ---- few rows: 16 MB rows x 16 NB columns per workgroup, its waves on the K blocks in turn ---
// Each operand goes from memory straight to the wave that multiplies it; the waves' partial sums
// meet in LDS and are added in wave order.  What bounds it is memory: 1 x 8,192 x 4,096 takes 6.5 us in bf16, its
// 33.6 MB of weights at 5.1 TB/s; 32 x 2,304 x 768 3.1, a launch (1.7) and two trips to memory.  A wave has one K
// block on its way at a time, so with a long K and several rows the trips add up: 65 x 2,048 x 4,096 in f32 10.7 us.
template <int OUT, int ST, int MB, int NB, int KS>
__global__ __launch_bounds__(64 * KS) void fp8_small_kernel(Fp8GemmArgs p, int tiles_n) {
  __shared__ f4 red[KS][MB * NB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int kbs = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
  const size_t m16 = fp8_scale_rows(p.M);
  const int m0 = (int)(blockIdx.x / tiles_n) * 16 * MB, n0 = (int)(blockIdx.x % tiles_n) * 16 * NB;
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
      for (int j = 0; j < NB; j++) block_product<OUT == FP8_IO_F32, ST>(w[j], a[i], as[i], wb[j], wf[j], acc[i][j]);
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
    store_out<OUT>(p, m0 + 16 * (t / NB) + r, n0 + 16 * (t % NB) + 4 * g, v);
  }
}

// ---- tiles: BM rows x BN weight rows per workgroup, K blocks through a double buffer in LDS --------
// WM x WN waves, each MT x NT tiles of 16 x 16.  Both operands go global -> LDS without registers, a
// K block (128 bytes of every row) per step; a row's eight 16-byte chunks are stored rotated (xor) by a
// function of the row, so that the 16 rows that a wave reads at once spread over all banks.
//  * A wave's activation rows are dealt out as row = MT (l % 16) + i for tile i, so that a lane's
//    scale bytes of one K block are MT consecutive ones: a dword holds four tiles' scales, and the
//    instruction picks its byte.
//  * A step's scales come the same way, the rows' as dwords, the weights' one per block of 128 columns.
//  * Step kb + 1's data has been requested one step ahead; the wait for it, and the barrier after which
//    step kb's buffer is refilled, come before the last row of MFMAs of step kb, whose operands are
//    in registers by then, so the first operands of step kb + 1 are read behind those MFMAs.
// Out-of-range rows and K chunks past K read as zero through the buffer descriptors' range.
// For 16-bit results of launches between one and one and a half strips of 128 x 256 per compute unit, whose
// last round these smaller tiles fill better.  4,616 x 2,048 x 768: 12 us, 1.2 PFLOP/s; what bounds it is the
// last round, and LDS (64 KiB read and 32 written for 16 products of a wave).

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// Raw buffer of `bytes` bytes at a wave-uniform base; reads past it give zero.  The lane's and the scalar offset
// count together (measured: a scalar offset at the end or past it leaves no lane in range).
__device__ __forceinline__ i4v buffer_at(const void* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  return i4v{__builtin_amdgcn_readfirstlane((int)(uint32_t)b), __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff),
             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// Global -> LDS copies as inline asm, so that the compiler adds no waits for them at LDS reads: the
// kernel's own vmcnt waits and barriers order them.  Lane l's bytes land at m0 + 16 l (4 l).
// A vector-memory read of a scalar register needs five wait states after the vector unit has written it, as
// buffer_at does and the restoring of a spilled descriptor; the compiler does not look for that in here.
// The write of m0 and s_nop 3 are five whatever stands in front.  Over s_nop 0 they cost 0 to 3%, in turn: gated
// 4,616 x 2,048 x 768 20.7 to 21.0 us, 24,288 x 113 x 3,936 in f32 57.9 to 59.4, 16,391 x 8,192 x 4,096 in bf16 nothing.
__device__ __forceinline__ void lds_copy16(i4v rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m0)
               : "memory", "m0");
}
__device__ __forceinline__ void lds_copy4(i4v rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m0)
               : "memory", "m0");
}
// One scale per lane, a byte or a dword of memory, a dword in LDS either way.
template <int ST>
__device__ __forceinline__ void lds_copy_scale(i4v rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
  if constexpr (ST == FP8_F32) lds_copy4(rsrc, voff, soff, m0);
  else
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_ubyte %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
                 "s"(m0)
                 : "memory", "m0");
}
// Copies in a run, each 1024 bytes of LDS behind the last, with one wait for all of their descriptors: eight of
// weights at their own scalar offsets, and a stage's rows with their scales behind them.  For workgroups with two
// waves that only copy, whose issue can be what a step takes: 65 x 2,048 x 4,096 in bf16 8.3 us, with a wait in
// front of each copy 10.1.  Four such waves are faster with single copies, between which the compiler forms
// the next one's offset: gated 135 x 2,032 x 2,976 11.2 us, in runs 11.5.
#define T5K_RUN_FIRST(rsrc, soff) "s_mov_b32 m0, %[at]\n\ts_nop 3\n\tbuffer_load_dwordx4 %[v], %[" rsrc "], %[" soff "] offen lds\n\t"
#define T5K_RUN_NEXT(rsrc, soff) "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %[v], %[" rsrc "], %[" soff "] offen lds\n\t"
__device__ __forceinline__ void lds_copy_weights(i4v r, uint32_t voff, const uint32_t (&s)[8], uint32_t m0) {
  asm volatile(T5K_RUN_FIRST("r", "s0") T5K_RUN_NEXT("r", "s1") T5K_RUN_NEXT("r", "s2") T5K_RUN_NEXT("r", "s3")
               T5K_RUN_NEXT("r", "s4") T5K_RUN_NEXT("r", "s5") T5K_RUN_NEXT("r", "s6") T5K_RUN_NEXT("r", "s7")
               ::[v] "v"(voff), [r] "s"(r), [s0] "s"(s[0]), [s1] "s"(s[1]), [s2] "s"(s[2]), [s3] "s"(s[3]), [s4] "s"(s[4]),
               [s5] "s"(s[5]), [s6] "s"(s[6]), [s7] "s"(s[7]), [at] "s"(m0)
               : "memory", "m0", "scc");
}
template <int N>
__device__ __forceinline__ void lds_copy_rows(const i4v (&r)[N], uint32_t voff, uint32_t soff, uint32_t m0, i4v scales, uint32_t scale_voff,
                                              uint32_t scale_soff, uint32_t scale_m0) {
  static_assert(N == 2 || N == 4, "a stage's rows");
#define T5K_RUN_SCALES "s_mov_b32 m0, %[sat]\n\ts_nop 0\n\tbuffer_load_dword %[sv], %[sr], %[ss] offen lds"
#define T5K_RUN_IN [v] "v"(voff), [s] "s"(soff), [at] "s"(m0), [sr] "s"(scales), [sv] "v"(scale_voff), [ss] "s"(scale_soff), [sat] "s"(scale_m0)
  if constexpr (N == 2)
    asm volatile(T5K_RUN_FIRST("a", "s") T5K_RUN_NEXT("b", "s") T5K_RUN_SCALES ::T5K_RUN_IN, [a] "s"(r[0]), [b] "s"(r[1])
                 : "memory", "m0", "scc");
  else
    asm volatile(T5K_RUN_FIRST("a", "s") T5K_RUN_NEXT("b", "s") T5K_RUN_NEXT("c", "s") T5K_RUN_NEXT("d", "s") T5K_RUN_SCALES
                 ::T5K_RUN_IN, [a] "s"(r[0]), [b] "s"(r[1]), [c] "s"(r[2]), [d] "s"(r[3])
                 : "memory", "m0", "scc");
#undef T5K_RUN_SCALES
#undef T5K_RUN_IN
}
#undef T5K_RUN_FIRST
#undef T5K_RUN_NEXT
constexpr uint32_t kOutside = 0x7fffffffu;  // past every descriptor's range

// c + one K block of a 16 x 16 tile; sa4: four rows' scale bytes, sel the one; swb: the weights' byte.
template <int SEL>
__device__ __forceinline__ f4 scaled_mfma_sel(const i8v& w, const i8v& a, f4 c, uint32_t sa4, uint32_t swb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 0, (int)swb, SEL, (int)sa4);
}
__device__ __forceinline__ f4 scaled_mfma(const i8v& w, const i8v& a, f4 c, uint32_t sa4, int sel, uint32_t swb) {
  switch (sel) {  // a constant once the loops are unrolled
    case 0: return scaled_mfma_sel<0>(w, a, c, sa4, swb);
    case 1: return scaled_mfma_sel<1>(w, a, c, sa4, swb);
    case 2: return scaled_mfma_sel<2>(w, a, c, sa4, swb);
    default: return scaled_mfma_sel<3>(w, a, c, sa4, swb);
  }
}

// The products of a wave's stripe of 16 rows with its NT weight operands, in four parts, so that a
// caller can put its copies and reads between them.  With byte scales on both sides the instruction adds
// into the accumulators.  Otherwise a block's sums are multiplied by their scale on the vector unit: a
// stripe behind, so that the wave never waits for the sums that it has just asked for.  `fold` adds the
// last stripe's at the end of a tile.
template <bool EXACT, int ST, int MT, int NT>
struct Products {
  static constexpr bool DIRECT = !EXACT && ST == FP8_E8M0;
  f4 acc[MT][NT];
  f4 sums[DIRECT ? 1 : 2][DIRECT ? 1 : NT];
  float factor[DIRECT ? 1 : 2][DIRECT ? 1 : NT];

  __device__ __forceinline__ void clear() {
    const f4 zero = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) acc[i][j] = zero;
    if constexpr (!DIRECT) {
#pragma unroll
      for (int j = 0; j < NT; j++) sums[(MT - 1) & 1][j] = zero, factor[(MT - 1) & 1][j] = 0.f;
    }
  }
  __device__ __forceinline__ void add(int i, int j) {  // stripe i's sums
    if constexpr (!DIRECT) {
#pragma unroll
      for (int e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(sums[i & 1][j][e], factor[i & 1][j], acc[i][j][e]);
    }
  }
  __device__ __forceinline__ void fold() {
#pragma unroll
    for (int j = 0; j < NT; j++) add(MT - 1, j);
  }
  // EXACT: the operands as f16, a quarter (32 of 128 K) at a time.  A part's products need quarter x; while
  // they run, the weights' next quarter is widened (first stripe) and the next stripe's rows.
  Wide ww[EXACT ? NT : 1], wa[EXACT ? 2 : 1];
  __device__ __forceinline__ void widen_quarter(Wide& to, const i8v& from, int x) { to.v[x] = widen8(from[2 * x], from[2 * x + 1]); }
  __device__ __forceinline__ void first_row(const i8v& a) {
    if constexpr (EXACT) wa[0] = widen(a);
  }
  __device__ __forceinline__ void begin_step(const i8v (&w)[NT]) {
    if constexpr (EXACT) {
#pragma unroll
      for (int j = 0; j < NT; j++) widen_quarter(ww[j], w[j], 0);
    }
  }
  // Part x of stripe i: w the weight operands, a and next this stripe's rows and the next one's, sw(j) the
  // bits of the weights' scales.
  template <typename Scale>
  __device__ __forceinline__ void part(int i, int x, const i8v (&w)[NT], const i8v& a, const i8v& next, uint32_t sa4, Scale sw) {
    const f4 zero = f4{0.f, 0.f, 0.f, 0.f};
    const int before = i ? i - 1 : MT - 1;
    if constexpr (DIRECT) {
      acc[i][x] = scaled_mfma(w[x], a, acc[i][x], sa4, i % 4, sw(x));
    } else if constexpr (!EXACT) {
      sums[i & 1][x] = scaled_mfma(w[x], a, zero, sa4, i % 4, 127);
      factor[i & 1][x] = __uint_as_float(sw(x));
      add(before, x);
    } else {
#pragma unroll
      for (int j = 0; j < NT; j++)
        sums[i & 1][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ww[j].v[x], wa[i & 1].v[x], x ? sums[i & 1][j] : zero, 0, 0, 0);
      if (x == 0) {
        const float f = e8m0_value((sa4 >> (8 * (i % 4))) & 255);
#pragma unroll
        for (int j = 0; j < NT; j++) factor[i & 1][j] = f * (ST == FP8_E8M0 ? e8m0_value(sw(j)) : __uint_as_float(sw(j)));
      }
#pragma unroll
      for (int j = x * NT / 4; j < (x + 1) * NT / 4; j++) add(before, j);
      if (i == 0 && x < 3) {
#pragma unroll
        for (int j = 0; j < NT; j++) widen_quarter(ww[j], w[j], x + 1);
      }
      if (x > 0) widen_quarter(wa[(i + 1) & 1], next, x - 1);
      if (x == 3) widen_quarter(wa[(i + 1) & 1], next, 3);
    }
  }
};

// Tile of the launch's index: bands of 8 row tiles, walked column by column, a contiguous stretch of
// them per XCD (workgroups are dealt to the 8 XCDs in turn), so that what runs at one time on an XCD
// is a patch of 8 row tiles by a few column tiles and its L2 serves both operands.
__device__ __forceinline__ void tile_place(uint32_t tiles, int tiles_m, int tiles_n, uint32_t i, int& tm, int& tn) {
  const uint32_t x = i % 8, rest = tiles % 8;
  const uint32_t t = x * (tiles / 8) + min(x, rest) + i / 8;
  const uint32_t wide = 8u * (uint32_t)tiles_n, band = t / wide, in = t - band * wide;
  const uint32_t h = min(8u, (uint32_t)tiles_m - band * 8);
  tm = (int)(band * 8 + in % h);
  tn = (int)(in / h);
}

// A wave's MT stripes of 16 rows and 16 NT columns: lane l has row MT (l % 16) + i of the wave's rows in
// stripe i, columns 16 j + 4 (l / 16).  A stripe is laid out in the wave's LDS (16 rows of 128 bytes at a
// time, 16-byte pieces rotated by the row) and stored in whole lines, past the caches: 64-byte pieces
// straight from registers took 151 us instead of 114 for 74,640 x 2,048 (x 768) in bf16, whole lines
// without the non-temporal hint 141.  Rows of C that do not keep 16-byte alignment go value by value.
template <int OUT, int MT, int NT>
__device__ __forceinline__ void store_stripes(const Fp8GemmArgs& p, uint8_t* stage, int lane, int m0, int n0,
                                              const f4 (&v)[MT][NT]) {
  constexpr int SZ = OUT == FP8_IO_F32 ? 4 : 2, TJ = 8 / SZ;  // TJ: columns / 16 of 128 bytes
  static_assert(NT % TJ == 0, "whole lines");
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int h = 0; h < NT / TJ; h++) {
#pragma unroll
      for (int j = 0; j < TJ; j++) {
        const int b = (16 * j + 4 * g) * SZ;  // byte within the row
        uint8_t* at = stage + r * 128 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15);
        if constexpr (SZ == 4) *reinterpret_cast<f4*>(at) = v[i][h * TJ + j];
        else *reinterpret_cast<u2v*>(at) = half4<OUT>(v[i][h * TJ + j]);
      }
      const int nh = n0 + h * TJ * 16;
      if (p.N % (16 / SZ) == 0) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
          const int row = 8 * q + (lane >> 3), c = lane & 7, m = m0 + row * MT + i, n = nh + c * (16 / SZ);
          if (m < p.M && n < p.N)
            __builtin_nontemporal_store(*reinterpret_cast<const i4v*>(stage + row * 128 + ((c ^ (row & 7)) << 4)),
                                        reinterpret_cast<i4v*>((uint8_t*)p.out + ((size_t)m * p.N + n) * SZ));
        }
      } else {
#pragma unroll 8
        for (int q = 0; q < 4 * TJ; q++) {
          const int row = (q * 64 + lane) / (TJ * 16), c = lane % (TJ * 16), b = c * SZ, m = m0 + row * MT + i, n = nh + c;
          const uint8_t* at = stage + row * 128 + (((b >> 4) ^ (row & 7)) << 4) + (b & 15);
          if (m < p.M && n < p.N) {
            if constexpr (SZ == 4) ((float*)p.out)[(size_t)m * p.N + n] = *reinterpret_cast<const float*>(at);
            else ((uint16_t*)p.out)[(size_t)m * p.N + n] = *reinterpret_cast<const uint16_t*>(at);
          }
        }
      }
    }
}

// The gated product's end: a wave has MT stripes of 16 rows, 32 gate columns and the same 32 up columns
// (n0 + 32 wave ..) of the 128 whose scale four waves share.  The rows' maxima meet in tops [16 MT][4],
// the codes in stage [MT][16][128], from where they are stored in whole lines.
template <int MT>
__device__ __forceinline__ void gated_stripes(const Fp8GemmArgs& p, uint32_t* tops, uint8_t* stage, int lane, int wave, int m0,
                                              int n0, int m16, f4 (&acc)[MT][4]) {
  const int r = lane & 15, g = lane >> 4;
  const int left = p.N - n0 - wave * 32;  // columns past N do not count (N % 16 == 0: whole 16s)
  // Largest magnitude of a lane's values of stripe i, NaN left out, as bits, which order alike.  The instruction
  // takes two more values at a time; fmaxf would first quiet each (they are products, so they are quiet).
  auto largest = [&](int i, bool finite) {
    float t[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const f4 y = acc[i][j];
      if (finite) {
        t[j] = fmaxf(fmaxf(finite_abs(y[0]), finite_abs(y[1])), fmaxf(finite_abs(y[2]), finite_abs(y[3])));
      } else {
        asm("v_max3_f32 %0, |%1|, |%2|, 0" : "=v"(t[j]) : "v"(y[0]), "v"(y[1]));
        asm("v_max3_f32 %0, |%1|, |%2|, %3" : "=v"(t[j]) : "v"(y[2]), "v"(y[3]), "v"(t[j]));
      }
    }
    return max(left > 0 ? __float_as_uint(t[0]) : 0u, left > 16 ? __float_as_uint(t[1]) : 0u);
  };
  uint32_t top[MT], all = 0;
#pragma unroll
  for (int i = 0; i < MT; i++) {
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[i][j][e] = gelu_tanh_dev(acc[i][j][e]) * acc[i][j + 2][e];
    top[i] = largest(i, false);
    all = max(all, top[i]);
  }
  if (all >= 0x7f800000u) {  // infinities do not count
#pragma unroll
    for (int i = 0; i < MT; i++) top[i] = largest(i, true);
  }
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const auto x = __builtin_amdgcn_permlane16_swap(top[i], top[i], false, false);
    const uint32_t half = max(x[0], x[1]);
    const auto y = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    top[i] = max(y[0], y[1]);
  }
  uint32_t* trow = tops + 4 * r;
  if (g == 0) {
#pragma unroll
    for (int i = 0; i < MT; i++) trow[64 * i + wave] = top[i];
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  uint8_t* to[2];
#pragma unroll
  for (int j = 0; j < 2; j++) to[j] = stage + r * 128 + 16 * ((2 * wave + j) ^ (r & 7)) + 4 * g;  // 16-byte piece 2 wave + j
  uint32_t bytes[(MT + 3) / 4] = {};
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const uint4 t4 = *reinterpret_cast<const uint4*>(trow + 64 * i);
    const uint32_t byte = e8m0_of(__uint_as_float(max(max(t4.x, t4.y), max(t4.z, t4.w))));
    bytes[i / 4] |= byte << (8 * (i % 4));
#pragma unroll
    for (int j = 0; j < 2; j++)
      *reinterpret_cast<uint32_t*>(to[j] + 2048 * i) = e4m3_pack4_scaled(acc[i][j], __uint_as_float(byte << 23));
  }
  if (wave == 0 && g == 0) {
    const int m = m0 + r * MT;
    uint8_t* scales = p.out_scales + (size_t)(n0 / FP8_BLOCK) * m16 + m;
    if (MT % 4 == 0 && m + MT <= p.M) {
#pragma unroll
      for (int c = 0; c < MT / 4; c++) reinterpret_cast<uint32_t*>(scales)[c] = bytes[c];
    } else {
#pragma unroll
      for (int i = 0; i < MT; i++)
        if (m + i < p.M) scales[i] = (uint8_t)(bytes[i / 4] >> (8 * (i % 4)));
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  const int c = lane & 7, rr = 8 * (wave & 1) + (lane >> 3), n = n0 + 16 * c;
  const uint8_t* from = stage + (wave / 2) * 2048 + rr * 128 + 16 * (c ^ (rr & 7));
#pragma unroll
  for (int q = 0; q < MT / 2; q++) {
    const int m = m0 + rr * MT + 2 * q + wave / 2;
    if (m < p.M && n < p.N)  // whole pieces
      __builtin_nontemporal_store(*reinterpret_cast<const i4v*>(from + 4096 * q),
                                  reinterpret_cast<i4v*>((uint8_t*)p.out + (size_t)m * p.N + n));
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // stage is copied into again
}

template <int OUT, int ST, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tile_kernel(Fp8GemmArgs p, int tiles_m, int tiles_n) {
  constexpr int WSZ = ST == FP8_F32 ? 4 : 1;  // bytes of a weight scale
  constexpr int NW = WM * WN, MT = BM / 16 / WM, NT = BN / 16 / WN, STAGE = (BM + BN) * 128;
  constexpr int H = MT / 2;                                      // stripes of a half step
  constexpr int CA = BM / 16 / NW, CW = BN / 8 / NW;             // copies per wave: of each half of the rows, of weights
  constexpr int C1 = CA + 2 + CW;                                // with the scales': of cursor 1 together
  constexpr int SC = 512, SCALES = 2 * STAGE, REST = SCALES + 2 * SC;  // SC: a step's scales, rows' and weights'
  constexpr int LDS = REST + NW * 2048;
  static_assert(BM % (16 * NW) == 0 && BN % (8 * NW) == 0 && MT % 4 == 0 && BM <= 256, "whole copies, whole scale dwords");
  static_assert(BN <= FP8_BLOCK && FP8_BLOCK % BN == 0, "one weight scale per tile and K block");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4, wm = wave / WN, wn = wave % WN;
  const int kbs = (p.K + FP8_BLOCK - 1) / FP8_BLOCK, m16 = (int)fp8_scale_rows(p.M);
  const uint32_t tiles = (uint32_t)tiles_m * (uint32_t)tiles_n;

  // ---- copies.  One brings K block kb of 8 rows: lane l chunk (l % 8) ^ (l / 8) of its row l / 8, to place
  // l % 8.  In LDS the activation rows are ordered by stripe, [MT][WM][16]; consecutive rows there lie MT
  // apart in memory.  A copy whose rows are all past the matrix brings the tile's first ones, which
  // nothing uses.  The scalar offset stays below one row, and so within every descriptor.
  struct Cursor {
    uint32_t tile;
    int kb, limit;  // limit: K, or 0 past the last tile (zeros)
  };
  Cursor c1 = {blockIdx.x, 0, p.K}, c2 = c1;  // of weights and the first stripes, of the last stripes
  i4v rw[CW], ra[2][CA], rsa, rsw;
  auto row_buffer = [&](const uint8_t* base, int first, int row, int end, int rows) {
    if (first + row >= end) row = 0;
    return buffer_at(base + (size_t)(first + row) * p.K, (uint32_t)min(rows, end - first - row) * (uint32_t)p.K);
  };
  auto aim_rows = [&](int half, int m0) {
#pragma unroll
    for (int j = 0; j < CA; j++) {
      const int q = 8 * ((half * NW + wave) * CA + j);  // LDS row: stripe q / (16 WM)
      ra[half][j] = row_buffer(p.a, m0, (q / 16 % WM) * 16 * MT + (q & 8) * MT + q / (16 * WM), p.M, 7 * MT + 1);
    }
  };
  auto aim1 = [&]() {
    int tm, tn;
    tile_place(tiles, tiles_m, tiles_n, c1.tile, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
#pragma unroll
    for (int j = 0; j < CW; j++) {
      rw[j] = row_buffer(p.w, n0, 8 * (wave * CW + j), p.N, 8);
    }
    aim_rows(0, m0);
    // the rows' scale bytes of a K block: BM of them (whole dwords: m16 and m0 are multiples of 16)
    rsa = buffer_at(p.a_scales + m0, (uint32_t)((size_t)kbs * m16 - m0));
    rsw = buffer_at((const uint8_t*)p.w_scales + (size_t)(n0 / FP8_BLOCK) * kbs * WSZ, (uint32_t)(kbs * WSZ));
  };
  auto aim2 = [&]() {
    int tm, tn;
    tile_place(tiles, tiles_m, tiles_n, c2.tile, tm, tn);
    aim_rows(1, tm * BM);
  };
  auto advance = [&](Cursor& c, auto aim) {
    if (++c.kb < kbs) return;
    c.kb = 0;
    c.tile += gridDim.x;
    if (c.tile < tiles) aim();
    else c.limit = 0;
  };
  const uint32_t fx = 16u * ((lane & 7) ^ (lane >> 3)), vw = (lane >> 3) * (uint32_t)p.K + fx;
  const uint32_t va = (lane >> 3) * (uint32_t)(MT * p.K) + fx, vsc = lane < BM / 4 ? 4u * lane : kOutside;
  const uint32_t vws = lane == 0 ? 0 : kOutside;
  const uint32_t lds0 = lds_offset(lds);
  // copy j of what cursor 1 brings: the first half of the rows, the scales, the weights
  auto copy1 = [&](int j, uint32_t slot) {
    const bool in = c1.kb * 128 + (int)fx < c1.limit;
    if (j < CA) lds_copy16(ra[0][j], in ? va : kOutside, c1.kb * 128, lds0 + slot * STAGE + (wave * CA + j) * 1024);
    else if (j == CA) lds_copy4(rsa, vsc, c1.kb * (uint32_t)m16, lds0 + SCALES + SC * slot);  // the same by every wave
    else if (j == CA + 1) lds_copy_scale<ST>(rsw, vws, c1.kb * WSZ, lds0 + SCALES + SC * slot + 256);
    else lds_copy16(rw[j - CA - 2], in ? vw : kOutside, c1.kb * 128, lds0 + slot * STAGE + BM * 128 + (wave * CW + j - CA - 2) * 1024);
  };
  auto copy2 = [&](int j, uint32_t slot) {
    const bool in = c2.kb * 128 + (int)fx < c2.limit;
    lds_copy16(ra[1][j], in ? va : kOutside, c2.kb * 128, lds0 + slot * STAGE + ((NW + wave) * CA + j) * 1024);
  };
  // All copies but the newest CA + C1 (one step's) have landed, and this wave's reads are complete.
  auto arrive = [&]() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(CA + C1) : "memory"); };

  Products<false, ST, MT, NT> prod;
  i8v a[2], w[NT];
  uint32_t sa[MT / 4], sw;  // scales: of the rows' stripes, of the weights
  // lane's chunks g and g + 4 of its row: places (g ^ f) and (g ^ f) ^ 4
  const int arow = wm * 16 * MT + r * MT, wrow = wn * 16 * NT + r;
  const uint32_t place = 16 * (g ^ (r & 7));
  uint32_t alo = (wm * 16 + r) * 128 + place, ahi = (wm * 16 + r) * 128 + (place ^ 64);  // in the current step's buffer
  uint32_t wlo = (BM + wrow) * 128 + place, whi = (BM + wrow) * 128 + (place ^ 64), sat = SCALES + arow, swat = SCALES + 256;
  auto read = [&](uint32_t lo, uint32_t hi, i8v& v) {
    const i4v x = *reinterpret_cast<const i4v*>(lds + lo), y = *reinterpret_cast<const i4v*>(lds + hi);
    v = i8v{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  auto read_w = [&](int j) { read(wlo + 2048 * j, whi + 2048 * j, w[j]); };
  auto read_scales = [&]() {
#pragma unroll
    for (int c = 0; c < MT / 4; c++) sa[c] = *reinterpret_cast<const uint32_t*>(lds + sat + 4 * c);
    sw = *reinterpret_cast<const uint32_t*>(lds + swat);
  };

  int tm, tn;
  tile_place(tiles, tiles_m, tiles_n, blockIdx.x, tm, tn);
  aim1();
  aim2();
#pragma unroll
  for (int j = 0; j < C1; j++) copy1(j, 0);
#pragma unroll
  for (int j = 0; j < CA; j++) copy2(j, 0);
  advance(c1, aim1);
#pragma unroll
  for (int j = 0; j < C1; j++) copy1(j, 1);
  arrive();
  read_scales();
#pragma unroll
  for (int j = 0; j < NT; j++) read_w(j);
  read(alo, ahi, a[0]);
  uint32_t slot = 0;

  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int m0 = tm * BM, n0 = tn * BN;
    if (tile + gridDim.x < tiles) tile_place(tiles, tiles_m, tiles_n, tile + gridDim.x, tm, tn);
    prod.clear();
    int kb = 0;
    do {
      advance(c1, aim1);
      advance(c2, aim2);
      const uint32_t s = sw;
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const uint32_t sc = sa[i / 4];
        if (i < MT - 1) {
          // the second half's rows of this step have landed; the first half's, and the weights, are in registers
          if (i == H - 1) arrive();
          read(alo + (i + 1) * WM * 2048, ahi + (i + 1) * WM * 2048, a[(i + 1) & 1]);
        } else {
          // the next step's first half and weights have landed; this step's operands are all in registers
          arrive();
          const uint32_t step = slot ? -STAGE : STAGE;
          alo += step, ahi += step, wlo += step, whi += step, sat += slot ? -SC : SC, swat += slot ? -SC : SC;
          read_scales();
          read(alo, ahi, a[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < NT; x++) {
          prod.part(i, x, w, a[i & 1], a[(i + 1) & 1], sc, [&](int) { return s; });
          __builtin_amdgcn_sched_barrier(0);
          if (i == MT - 1) read_w(x);  // each weight operand is replaced as soon as it has been used
          // this step's share of copies, behind the products: the next step's last stripes into its buffer,
          // then, once this step's first half is read, the step after it into this one's
          if (i < H - 1) {
            constexpr int PARTS = (H - 1) * NT;
            const int at = i * NT + x;
#pragma unroll
            for (int c = at * CA / PARTS; c < (at + 1) * CA / PARTS; c++) copy2(c, slot ^ 1);
          } else if (i < MT - 1) {
            constexpr int PARTS = (MT - H) * NT;
            const int at = (i - H + 1) * NT + x;
#pragma unroll
            for (int c = at * C1 / PARTS; c < (at + 1) * C1 / PARTS; c++) copy1(c, slot);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      slot ^= 1;
      kb++;
    } while (kb < kbs);
    prod.fold();
    store_stripes<OUT>(p, lds + REST + wave * 2048, lane, m0 + wm * 16 * MT, n0 + wn * NT * 16, prod.acc);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies past the end have landed
}

// ---- strips: 16 MT rows x 64 NW weight rows per workgroup, two workgroups per compute unit ----------
// Wave w has all rows and 64 weight rows of its own (gated: 32 gate rows and the 32 up rows of the same
// columns).  Rows' codes are double-buffered in LDS; the weights have one buffer, a wave's own share:
// their operands are in registers from a step's start, when the next step's are requested.  The two
// workgroups run apart, so that one's results are formed and stored behind the other's products.  The large
// sizes: 16,391 x 8,192 x 4,096 in bf16 takes 424 to 456 us, 2.4 to 2.6 PFLOP/s, at the clock that power leaves (a
// library product of 8,192 cubed reaches 2.6), with float scales 476 to 510, for the multiply-add per result and K
// block; 74,640 x 2,048 x 768 115 to 122 us, float scales 126 to 135; gated 226 to 247 us, 1.9 to 2.1 PFLOP/s, the
// rest its gelu and codes on the vector unit, which adds to the matrix unit's time, float scales 261 to 284.  f32
// results from 9,232 x 768 x 2,048 33 us, 0.87 PFLOP/s: widening and scaling take the vector unit as long as the
// products take theirs.
// RING, for launches that leave each compute unit one workgroup, with one tile each: as many waves again do
// nothing but copy, through a ring of that many K blocks, weights and rows.  A copy holds its wave up for some 36
// clocks, and a compute unit receives 64 bytes per clock: in waves that also multiply, copies and products of one
// workgroup add up (0.52 us a K block of the gated product's 64 x 256), with copying waves a step takes 0.33, near
// the larger of the two.  Where two workgroups share a compute unit one's copies run behind the other's products, and the
// copying waves' registers would be missed.
template <int OUT, int ST, bool GATED, int MT, int NW, int RING>
__global__ __launch_bounds__(64 * NW * (RING ? 2 : 1), 2) void fp8_strip_kernel(Fp8GemmArgs p, int tiles_m, int tiles_n) {
  constexpr bool EXACT = OUT == FP8_IO_F32 && !GATED;
  constexpr int NT = 4, BM = 16 * MT, NM = GATED ? 2 : 1;                     // NM: matrices
  constexpr int STAGES = RING ? RING : 2, STAGE = BM * 128 + (RING ? NW * 8192 : 0);
  constexpr int COLS = (GATED ? 32 : 64) * NW, CA = BM / 8 / NW;              // CA: copies of rows per wave and K block
  constexpr int WEIGHTS = RING ? BM * 128 : 2 * STAGE;  // RING: within a stage
  constexpr int SCALES = STAGES * STAGE + (RING ? 0 : NW * 8192), REST = SCALES + STAGES * 256, OPS = 9 + CA;
  constexpr int LDS = REST + (GATED ? NW * BM * 4 : NW * 2048);
  static_assert(BM % (8 * NW) == 0 && (MT % 4 == 0 || MT == 2) && (!GATED || NW == 4), "whole copies; all columns of a scale");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) % NW), copies = RING ? __builtin_amdgcn_readfirstlane((tid >> 6) / NW) : 0;
  const int r = lane & 15, g = lane >> 4;
  const int kbs = (p.K + FP8_BLOCK - 1) / FP8_BLOCK, m16 = (int)fp8_scale_rows(p.M);
  const uint32_t tiles = (uint32_t)tiles_m * (uint32_t)tiles_n;

  // ---- copies of the next step: K block ckb of tile ctile.  One brings 8 rows, lane l chunk (l % 8) ^ (l / 8)
  // of its row l / 8 to place l % 8.  In LDS the activations are ordered by stripe, [MT][16]; consecutive
  // ones lie MT apart in memory.  Descriptors end with the matrix; one whose rows are all past it has
  // the tile's first rows, which nothing uses.  No scalar offset passes its descriptor's end (a copy of
  // weight rows past the matrix is held there): the range check may subtract it from the size.
  uint32_t ctile = blockIdx.x;
  int ckb = 0, climit = p.K;  // climit 0: past the last tile, zeros
  int tm, tn;                 // place of tile ctile
  i4v ra[CA], rsa, rw[NM];
  uint32_t ws[NM], wsn[NM];   // weight scales: lane k's are of K block k of a stretch of 64
  auto weight_scales = [&](int n0, int kb, uint32_t (&to)[NM]) {
    const size_t at = (size_t)(min(n0 + wave * (COLS / NW), p.N - 1) / FP8_BLOCK) * kbs + min(kb + lane, kbs - 1);
#pragma unroll
    for (int j = 0; j < NM; j++) {
      const void* s = j ? p.w1_scales : p.w_scales;
      to[j] = ST == FP8_E8M0 ? ((const uint8_t*)s)[at] : __float_as_uint(((const float*)s)[at]);
    }
  };
  auto aim = [&]() {
    tile_place(tiles, tiles_m, tiles_n, ctile, tm, tn);
    const int m0 = tm * BM, n = tn * COLS + wave * (COLS / NW);
#pragma unroll
    for (int j = 0; j < CA; j++) {
      const int q = wave * CA + j;
      int row = (q & 1) * 8 * MT + q / 2;
      if (m0 + row >= p.M) row = 0;
      ra[j] = buffer_at(p.a + (size_t)(m0 + row) * p.K, (uint32_t)min(7 * MT + 1, p.M - m0 - row) * (uint32_t)p.K);
    }
    rsa = buffer_at(p.a_scales + m0, (uint32_t)((size_t)kbs * m16 - m0));
#pragma unroll
    for (int j = 0; j < NM; j++)
      rw[j] = buffer_at((j ? p.w1 : p.w) + (size_t)min(n, p.N - 1) * p.K, (uint32_t)max(1, min(COLS / NW, p.N - n)) * (uint32_t)p.K);
  };
  const uint32_t fx = 16u * ((lane & 7) ^ (lane >> 3)), va = (lane >> 3) * (uint32_t)(MT * p.K) + fx;
  const uint32_t vsa = lane < BM / 4 ? 4u * lane : kOutside, vw = (lane >> 3) * (uint32_t)p.K + fx;
  const uint32_t lds0 = lds_offset(lds);
  uint32_t cva, cvw;  // this step's lane offsets; chunks past K lie outside
  auto copy = [&](int j, uint32_t slot) {
    if (j < 8)
      lds_copy16(rw[GATED ? j / 4 : 0], cvw,
                 min(ckb * 128u + (uint32_t)((GATED ? j % 4 : j) * 8) * (uint32_t)p.K, (uint32_t)rw[GATED ? j / 4 : 0][2]),
                 lds0 + (RING ? slot * STAGE : 0) + WEIGHTS + wave * 8192 + j * 1024);
    else if (j < 8 + CA) lds_copy16(ra[j - 8], cva, ckb * 128, lds0 + slot * STAGE + (wave * CA + j - 8) * 1024);
    else lds_copy4(rsa, vsa, ckb * (uint32_t)m16, lds0 + SCALES + 256 * slot);  // the same by every wave
  };
  // RING: all copies of a step, by a copying wave
  auto copy_stage = [&](uint32_t slot) {
    if constexpr (NW == 2) {
      uint32_t at[8];
#pragma unroll
      for (int j = 0; j < 8; j++) at[j] = min(ckb * 128u + (uint32_t)(j * 8) * (uint32_t)p.K, (uint32_t)rw[0][2]);
      lds_copy_weights(rw[0], cvw, at, lds0 + slot * STAGE + WEIGHTS + wave * 8192);
      lds_copy_rows<CA>(ra, cva, ckb * 128, lds0 + slot * STAGE + wave * CA * 1024, rsa, vsa, ckb * (uint32_t)m16,
                        lds0 + SCALES + 256 * slot);
    } else {
#pragma unroll
      for (int j = 0; j < OPS; j++) copy(j, slot);
    }
  };
  auto lane_offsets = [&]() {
    const bool in = ckb * 128 + (int)fx < climit;
    cva = in ? va : kOutside;
    cvw = in ? vw : kOutside;
  };

  Products<EXACT, ST, MT, NT> prod;
  i8v a[2], w[NT];
  uint32_t sa[(MT + 3) / 4];
  // lane's chunks g and g + 4 of its row
  const uint32_t place = 16 * (g ^ (r & 7));
  uint32_t alo = r * 128 + place, ahi = r * 128 + (place ^ 64), sat = SCALES + r * MT;  // in the current step's buffer
  auto read = [&](uint32_t lo, uint32_t hi, i8v& v) {
    const i4v x = *reinterpret_cast<const i4v*>(lds + lo), y = *reinterpret_cast<const i4v*>(lds + hi);
    v = i8v{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  uint32_t wat = WEIGHTS + wave * 8192 + r * 128;
  auto read_w = [&](int j) { read(wat + place + 2048 * j, wat + (place ^ 64) + 2048 * j, w[j]); };
  auto read_scales = [&]() {
    if constexpr (MT == 2) sa[0] = *reinterpret_cast<const uint16_t*>(lds + sat);
#pragma unroll
    for (int c = 0; c < MT / 4; c++) sa[c] = *reinterpret_cast<const uint32_t*>(lds + sat + 4 * c);
  };

  auto next_block = [&]() {
    if (++ckb == kbs) {
      ckb = 0;
      ctile += gridDim.x;
      if (ctile < tiles) aim();
      else climit = 0;
    }
    lane_offsets();
  };
  // the next step's copies have landed, those of the steps after it (RING) may be on their way; reads are complete
  constexpr int IN_FLIGHT = (STAGES - 2) * OPS, WAIT = (IN_FLIGHT & 15) | (IN_FLIGHT >> 4 << 14) | 0x70;

  if (copies) {
    aim();
    lane_offsets();
#pragma unroll
    for (int n = 0; n < STAGES - 1; n++) {
      if (n) next_block();
      copy_stage(n);
    }
    __builtin_amdgcn_s_waitcnt(WAIT);
    asm volatile("s_barrier" ::: "memory");
    uint32_t fill = STAGES - 1;
    for (int kb = 0; kb < kbs; kb++) {  // the last STAGES - 1 fill stages that nothing reads or uses for its end
      next_block();
      copy_stage(fill);
      fill = fill == STAGES - 1 ? 0 : fill + 1;
      __builtin_amdgcn_s_waitcnt(WAIT);
      asm volatile("s_barrier" ::: "memory");
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    return;  // barriers of the tile's end do not count waves that have ended
  }

  if (RING) tile_place(tiles, tiles_m, tiles_n, ctile, tm, tn);
  else aim();
  weight_scales(tn * COLS, 0, ws);
  int ptm = tm, ptn = tn;  // place of the tile that the products are at
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), so that the compiler knows its own loads to be complete
  if constexpr (!RING) {
    lane_offsets();
#pragma unroll
    for (int j = 0; j < OPS; j++) copy(j, 0);
    __builtin_amdgcn_s_waitcnt(WAIT);
  }
  asm volatile("s_barrier" ::: "memory");
  read_scales();
#pragma unroll
  for (int j = 0; j < NT; j++) read_w(j);
  read(alo, ahi, a[0]);
  prod.first_row(a[0]);
  uint32_t slot = 0, last = 0;

  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int m0 = ptm * BM, n0 = ptn * COLS;
    if (tile + gridDim.x < tiles) tile_place(tiles, tiles_m, tiles_n, tile + gridDim.x, ptm, ptn);
    weight_scales(ptn * COLS, 0, wsn);  // of the next tile
    prod.clear();
    int kb = 0;
    do {
      if (kb && (kb & 63) == 0) {
        weight_scales(n0, kb, ws);
        __builtin_amdgcn_s_waitcnt(0x0f70);
      }
      if (!RING) next_block();
      const uint32_t fill = slot == 0 ? STAGES - 1 : slot - 1, after = slot == STAGES - 1 ? 0 : slot + 1;
      uint32_t swb[NM];
#pragma unroll
      for (int j = 0; j < NM; j++) swb[j] = __builtin_amdgcn_readlane(ws[j], kb & 63);
      prod.begin_step(w);
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const uint32_t sc = sa[i / 4];
        if (i < MT - 1) {
          read(alo + (i + 1) * 2048, ahi + (i + 1) * 2048, a[(i + 1) & 1]);
        } else {
          // the next step's copies have landed; every wave has its rows in LDS, and this step's in registers
          __builtin_amdgcn_s_waitcnt(RING ? 0xc07f : WAIT);
          asm volatile("s_barrier" ::: "memory");
          const uint32_t step = after == 0 ? (uint32_t)-((STAGES - 1) * STAGE) : (uint32_t)STAGE;
          alo += step, ahi += step, sat += after == 0 ? -(STAGES - 1) * 256 : 256;
          if (RING) wat += step;
          read_scales();
          read(alo, ahi, a[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; x++) {
          prod.part(i, x, w, a[i & 1], a[(i + 1) & 1], sc, [&](int j) { return swb[GATED ? j / 2 : 0]; });
          __builtin_amdgcn_sched_barrier(0);
          if (i == MT - 1) read_w(x);  // each weight operand is replaced as soon as it has been used
          // Behind the products: the next step's weights, whose buffer has been read, and rows.
          constexpr int PARTS = (MT > 2 ? MT - 2 : 1) * 4;
          const int at = i * 4 + x;
          if (!RING && at == 0) __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): w is in registers
          if (!RING && at < PARTS) {
#pragma unroll
            for (int c = at * OPS / PARTS; c < (at + 1) * OPS / PARTS; c++) copy(c, fill);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      last = slot;
      slot = after;
      kb++;
    } while (kb < kbs);
#pragma unroll
    for (int j = 0; j < NM; j++) ws[j] = wsn[j];
    prod.fold();

    if constexpr (!GATED) {
      store_stripes<OUT>(p, lds + REST + wave * 2048, lane, m0, n0 + wave * 64, prod.acc);
    } else {
      // staged in the rows' buffer that the next step's copies go to
      gated_stripes<MT>(p, reinterpret_cast<uint32_t*>(lds + REST), lds + last * STAGE, lane, wave, m0, n0, m16, prod.acc);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies past the end have landed
}

template <int OUT, int ST, int MB, int NB, int KS>
hipError_t launch_small(const Fp8GemmArgs& p, hipStream_t s) {
  const int tiles_n = (p.N + 16 * NB - 1) / (16 * NB);
  const int64_t tiles = (int64_t)((p.M + 16 * MB - 1) / (16 * MB)) * tiles_n;  // few: see launch_product
  T5K_LAUNCH((fp8_small_kernel<OUT, ST, MB, NB, KS>), dim3((unsigned)tiles), dim3(64 * KS), 0, s, p, tiles_n);
  return hipGetLastError();
}

template <int OUT, int ST, int BM, int BN, int WM, int WN>
hipError_t launch_tile(const Fp8GemmArgs& p, int cus, hipStream_t s) {
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const int64_t tiles = (int64_t)tiles_m * tiles_n;
  if (tiles >> 30) return hipErrorInvalidValue;
  T5K_LAUNCH((fp8_tile_kernel<OUT, ST, BM, BN, WM, WN>), dim3((unsigned)std::min<int64_t>(tiles, cus * (8 / (WM * WN)))),
             dim3(64 * WM * WN), 0, s, p, tiles_m, tiles_n);
  return hipGetLastError();
}

template <int OUT, int ST, bool GATED, int MT, int NW, int RING>
hipError_t launch_strip(const Fp8GemmArgs& p, int cus, hipStream_t s) {
  constexpr int COLS = (GATED ? 32 : 64) * NW;
  const int tiles_m = (p.M + 16 * MT - 1) / (16 * MT), tiles_n = (p.N + COLS - 1) / COLS;
  const int64_t tiles = (int64_t)tiles_m * tiles_n;
  if (tiles >> 30) return hipErrorInvalidValue;
  const int64_t groups = RING ? tiles : std::min<int64_t>(tiles, cus * (8 / NW));
  T5K_LAUNCH((fp8_strip_kernel<OUT, ST, GATED, MT, NW, RING>), dim3((unsigned)groups), dim3(64 * NW * (RING ? 2 : 1)), 0, s, p,
             tiles_m, tiles_n);
  return hipGetLastError();
}

// Compute units of the current device, asked for once per device.
int compute_units() {
  static std::atomic<int> known[64];
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if ((cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// The smallest tiles that leave each compute unit at most a workgroup, of the kernel that is fastest at that.  us
// of small kernels of 1 x 1 / 1 x 2 / 2 x 2 / 4 x 2 tiles of 16, then strips through the ring of 32 x 128 / 64 x 128 /
// 64 x 256; in bf16
//   1 x 8,192 x 4,096  7.2 / 6.8 / 9.4 / 9.7, 9.9 / 11.7 / 14.1     33 x 2,048 x 4,096  8.4 / 7.9 / 10.5 / 11.3, 8.4 / 11.7 / 13.5
//   65 x 2,304 x 768   4.6 / 4.6 / 4.2 / 5.1, 3.8 / 4.8 / 5.4       256 x 768 x 2,048   8.0 / 8.0 / 6.6 / 8.4, 5.6 / 7.5 / 8.6
//   256 x 8,192 x 4,096  - / - / 62 / 48, 16.5 / 13.8 / 16.6        1,000 x 2,304 x 768  - / - / 16 / 15, 7.1 / 6.9 / 6.0
// and for f32 results, whose widening makes strips slower (32 x 256 in place of 64 x 128)
//   65 x 2,048 x 4,096  12.2 / 12.6 / 10.5 / 14.5, 20.5 / 21.8 / -  500 x 768 x 2,048   - / 11.1 / 10.5 / 8.9, 11.9 / 12.7 / 17.9
//   500 x 2,304 x 768  - / - / 10.6 / 12.9, 9.4 / 7.6 / 9.7         1,000 x 2,304 x 768  - / - / 17 / 21, 11.8 / 12.2 / 10.0
template <int OUT, int ST>
hipError_t launch_product(const Fp8GemmArgs& p, hipStream_t s) {
  const int cus = compute_units();
  auto groups = [&](int rows, int cols) { return (((int64_t)p.M + rows - 1) / rows) * (((int64_t)p.N + cols - 1) / cols); };
  if (groups(16, 16) <= cus) return launch_small<OUT, ST, 1, 1, 8>(p, s);
  if (groups(16, 32) <= cus) return launch_small<OUT, ST, 1, 2, 8>(p, s);
  if constexpr (OUT == FP8_IO_F32) {
    // two workgroups per compute unit: 14.8 against 20 for 1 x 16,384 x 4,096, 18 against 21 for 32 x 16,384 x 4,096
    if (p.M <= 16 && groups(16, 32) <= 2 * cus) return launch_small<OUT, ST, 1, 2, 8>(p, s);
    if (groups(32, 32) <= cus) return launch_small<OUT, ST, 2, 2, 4>(p, s);
    if (groups(64, 32) <= cus) return launch_small<OUT, ST, 4, 2, 8>(p, s);
    if (groups(32, 32) <= 2 * cus) return launch_small<OUT, ST, 2, 2, 4>(p, s);
    if (groups(32, 128) <= cus) return launch_strip<OUT, ST, false, 2, 2, 3>(p, cus, s);
    if (groups(32, 256) <= cus) return launch_strip<OUT, ST, false, 2, 4, 3>(p, cus, s);
    if (groups(64, 256) <= cus) return launch_strip<OUT, ST, false, 4, 4, 3>(p, cus, s);
    return launch_strip<OUT, ST, false, 4, 4, 0>(p, cus, s);  // 9,232 x 768 x 2,048: 32.6, through the ring 35
  } else {
    if (groups(32, 128) <= cus) return launch_strip<OUT, ST, false, 2, 2, 3>(p, cus, s);
    if (groups(64, 128) <= cus) return launch_strip<OUT, ST, false, 4, 2, 3>(p, cus, s);
    if (groups(64, 256) <= cus) return launch_strip<OUT, ST, false, 4, 4, 3>(p, cus, s);
    if (groups(128, 256) <= cus) return launch_strip<OUT, ST, false, 8, 4, 3>(p, cus, s);
    // us of 128 x 256 strips, two workgroups on a compute unit / through the ring / tiles of 128 x 128: 12.2 / 14.9 / 12.2
    // for 4,616 x 2,048 x 768 (296 strips), 48.7 / 48.2 / 47.5 for 1,500 x 8,192 x 4,096 (384); 13.3 / 15.1 / 15.8 for
    // 6,500 x 2,304 x 768 (459), 115 / 146 / 135 for 74,640 x 2,048 x 768, 427 / 441 / 497 for 16,391 x 8,192 x 4,096.
    // Over 34 sizes of 257 to 384 strips the tiles take 0.95 of the strips' time with byte scales, 0.97 with float ones.
    if (2 * groups(128, 256) > 3 * cus) return launch_strip<OUT, ST, false, 8, 4, 0>(p, cus, s);
    return launch_tile<OUT, ST, 128, 128, 2, 2>(p, cus, s);
  }
}

// A scale needs all of its 128 columns in one workgroup.  Up to one strip per compute unit, as few rows each as that
// allows, through the ring: us of 32 / 64 / 128 rows / 128 without the ring, 5.2 / 6.2 / 8.9 / 9.4 for 32 x 2,048 x 768,
// 16 / 17 / 24 / 35 for 32 x 8,192 x 4,096, 30 / 19 / 27 / - for 200 x 8,192 x 4,096, 30 / 19 / 16 / 21 for 4,616 x 768 x
// 2,048 (222 of 128).  Beyond that two workgroups on a compute unit: 21 against 24 for 4,616 x 2,048 x 768, 230
// against 300 for 74,640 x 2,048 x 768.  Few rows leave most compute units without work, and a strip's time is that of
// its weights through one of them, at 64 bytes per clock; operands straight to registers take 9.0 for 32 x 2,048 x 768.
template <int ST>
hipError_t launch_gated(const Fp8GemmArgs& p, hipStream_t s) {
  const int cus = compute_units();
  auto strips = [&](int rows) { return (((int64_t)p.M + rows - 1) / rows) * ((p.N + FP8_BLOCK - 1) / FP8_BLOCK); };
  if (strips(32) <= cus) return launch_strip<FP8_IO_NONE, ST, true, 2, 4, 3>(p, cus, s);
  if (strips(64) <= cus) return launch_strip<FP8_IO_NONE, ST, true, 4, 4, 3>(p, cus, s);
  if (strips(128) <= cus) return launch_strip<FP8_IO_NONE, ST, true, 8, 4, 3>(p, cus, s);
  return launch_strip<FP8_IO_NONE, ST, true, 8, 4, 0>(p, cus, s);
}
}  // namespace

namespace t5k {
hipError_t launch_fp8_matmul(const Fp8GemmArgs& p, hipStream_t s) {
  if (p.M == 0 || p.N == 0) return hipSuccess;
  if (p.M < 0 || p.N < 0 || p.K <= 0 || p.K % 16 || p.K > FP8_MAX_K) return hipErrorInvalidValue;
  switch (2 * p.out_type + p.scale_type) {
    case 2 * FP8_IO_F32 + FP8_E8M0: return launch_product<FP8_IO_F32, FP8_E8M0>(p, s);
    case 2 * FP8_IO_F32 + FP8_F32: return launch_product<FP8_IO_F32, FP8_F32>(p, s);
    case 2 * FP8_IO_F16 + FP8_E8M0: return launch_product<FP8_IO_F16, FP8_E8M0>(p, s);
    case 2 * FP8_IO_F16 + FP8_F32: return launch_product<FP8_IO_F16, FP8_F32>(p, s);
    case 2 * FP8_IO_BF16 + FP8_E8M0: return launch_product<FP8_IO_BF16, FP8_E8M0>(p, s);
    case 2 * FP8_IO_BF16 + FP8_F32: return launch_product<FP8_IO_BF16, FP8_F32>(p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_fp8_gated_gelu(const Fp8GemmArgs& p, hipStream_t s) {
  if (p.M == 0 || p.N == 0) return hipSuccess;
  if (p.M < 0 || p.N < 0 || p.N % 16 || p.K <= 0 || p.K % 16 || p.K > FP8_MAX_K) return hipErrorInvalidValue;
  if (p.scale_type == FP8_E8M0) return launch_gated<FP8_E8M0>(p, s);
  if (p.scale_type == FP8_F32) return launch_gated<FP8_F32>(p, s);
  return hipErrorInvalidValue;
}
}  // namespace t5k
