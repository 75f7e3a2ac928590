// k_rotary.hip -- queries and keys on their way from the projection to attention: a norm of each head and
// the rotation by positions, in one pass.  No counterpart in the reference, whose attention has a bias by
// distance instead.
//
//   z = x / sqrt(mean over the head of x^2 + eps) * gamma          (only x where there is no gamma)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)               for each pair of the first `rot` values
//
// in f32, rounded once.  Pairs are (i, i + rot / 2) or (2i, 2i + 1); t = position * frequency, each pair
// with its own frequency and its own one of the position's axes.
//
// Angles.  A frequency is held as a 61-bit fraction of a turn, so position * frequency modulo a turn is an
// integer product that wraps: no position loses bits to its size.  32 bits of the product's fraction, less
// their nearest quarter turn, give an angle within pi / 4, and the Taylor series of sine and cosine up to
// x^9 and x^8 are within 3e-8 there.
#include "rotary.hpp"

#include <algorithm>

#include "fp8.hpp"  // FP8_IO types

namespace {
using namespace t5k;

// V values of an io type, as they lie in memory and as floats.
template <int T, int V>
struct Chunk;
template <>
struct Chunk<FP8_IO_F32, 4> {
  f4 raw;
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = raw[e];
  }
  __device__ __forceinline__ void set(const float* v) { raw = f4{v[0], v[1], v[2], v[3]}; }
};
template <int T, int V>
struct Chunk {
  typedef uint32_t words __attribute__((ext_vector_type(V / 2)));
  words raw;
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int e = 0; e < V; e++) {
      const uint32_t w = raw[e / 2];
      if constexpr (T == FP8_IO_F16) v[e] = f16_bits_to_f32(e & 1 ? w >> 16 : w & 0xffffu);
      else v[e] = __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const f4 x = f4{v[e], v[e + 1], v[e + 2], v[e + 3]};
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      u2 w;
      if constexpr (T == FP8_IO_F16) w = __builtin_bit_cast(u2, __builtin_convertvector(x, h4));
      else w = __builtin_bit_cast(u2, __builtin_convertvector(x, b4));
      raw[e / 2] = w[0], raw[e / 2 + 1] = w[1];
    }
  }
};

// Sine and cosine of a fraction of a turn in 32 bits.
__device__ __forceinline__ void sincos_turn(uint32_t f, float& s, float& c) {
  const uint32_t quarter = (f + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(f - (quarter << 30)) * (float)(6.283185307179586 / 4294967296.0);
  const float y = x * x;
  const float sx = __builtin_fmaf(x * y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), x);
  const float cx = __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.f / 40320.f, -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const bool odd = quarter & 1;
  const float a = odd ? cx : sx, b = odd ? sx : cx;
  s = quarter & 2 ? -a : a;
  c = (quarter + 1) & 2 ? -b : b;
}

// v summed over aligned groups of L lanes; all of them get the sum.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int L>
__device__ __forceinline__ float sum_group(float v) {
  v = dpp_add<0xb1>(v);                         // lane ^ 1
  v = dpp_add<0x4e>(v);                         // lane ^ 2
  if constexpr (L >= 8) v = dpp_add<0x141>(v);  // mirrored within 8: the other four
  if constexpr (L >= 16) v = dpp_add<0x140>(v);  // mirrored within 16: the other eight
  if constexpr (L >= 32) v = sum_xor16(v);
  if constexpr (L >= 64) v = sum_xor32(v);
  return v;
}

struct Shape {
  int tokens, heads;  // a workgroup's
  int step_tokens, step_heads;  // of 256 / L heads, in whole rows of `heads`
};

// A lane holds two chunks of V values of a head, those whose values make pairs: c and c + rot / 2 / V for
// halves, neighbouring ones otherwise and behind the rotated part; L lanes (a power of two) hold the head.
// A workgroup walks the heads of some tokens, and computes each token's sines and cosines once, into LDS.
// What bounds it is memory; a value takes about 10 vector instructions, a third of the memory's time.
template <int T, int V, int L, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, Shape w) {
  extern __shared__ f4 lds[];
  float* turns = (float*)lds;  // [tokens][2][pairs]: cosines, sines
  const int pairs = a.rot / 2, unit = threadIdx.x & (L - 1), slot = threadIdx.x / L;
  const int n = a.D / V, m = pairs / V;  // chunks of a head, chunks of a half of its rotated part
  const bool turned = unit < m, first_ok = 2 * unit < n;
  const int c0 = HALVES && turned ? unit : 2 * unit, c1 = HALVES && turned ? unit + m : 2 * unit + 1;
  const bool second_ok = c1 < n && first_ok;
  const int h_first = blockIdx.y * w.heads, h_last = min(h_first + w.heads, a.q_heads + a.k_heads);
  const size_t size = T == FP8_IO_F32 ? 4 : 2;
  float gq[2 * V], gk[2 * V];
#pragma unroll
  for (int e = 0; e < 2 * V; e++) {
    const bool ok = e < V ? first_ok : second_ok;
    const int at = (e < V ? c0 * V + e : c1 * V + e - V);
    gq[e] = ok && a.q_gamma ? a.q_gamma[at] : 1.f;
    gk[e] = ok && a.k_gamma ? a.k_gamma[at] : 1.f;
  }
  for (int64_t t0 = (int64_t)blockIdx.x * w.tokens; t0 < a.T; t0 += (int64_t)gridDim.x * w.tokens) {
    const int tokens = (int)min((int64_t)w.tokens, a.T - t0);
    for (int i = threadIdx.x; i < tokens * pairs; i += 256) {
      const int t = i / pairs, p = i - t * pairs;
      const uint64_t entry = a.table[p];
      const int axis = (int)(entry & (ROTARY_MAX_AXES - 1));
      const int32_t at = axis < a.axes ? a.pos[(size_t)axis * a.T + t0 + t] : 0;
      const uint64_t turn = (uint64_t)(int64_t)at * (entry & ~(uint64_t)(ROTARY_MAX_AXES - 1));
      float s, c;
      sincos_turn((uint32_t)(turn >> 32), s, c);
      turns[2 * t * pairs + p] = c;
      turns[(2 * t + 1) * pairs + p] = s;
    }
    __syncthreads();
    int t = slot / w.heads, h = h_first + slot - t * w.heads;
    while (t < tokens) {
      if (h < h_last) {
        const bool is_q = h < a.q_heads;
        const int hh = is_q ? h : h - a.q_heads;
        const char* from = (const char*)(is_q ? a.q : a.k) + ((size_t)(t0 + t) * (is_q ? a.ldq : a.ldk) + (size_t)hh * a.D) * size;
        char* to = (char*)(is_q ? a.q_out : a.k_out) + ((size_t)(t0 + t) * (is_q ? a.ldq_out : a.ldk_out) + (size_t)hh * a.D) * size;
        Chunk<T, V> x0{}, x1{};
        if (first_ok) x0 = *(const Chunk<T, V>*)(from + c0 * V * size);
        if (second_ok) x1 = *(const Chunk<T, V>*)(from + c1 * V * size);
        float v[2 * V];
        x0.get(v), x1.get(v + V);
        if (is_q ? a.q_gamma != nullptr : a.k_gamma != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 2 * V; e++) ss = __builtin_fmaf(v[e], v[e], ss);
          const float rs = rsqrtf(sum_group<L>(ss) / (float)a.D + a.eps);
#pragma unroll
          for (int e = 0; e < 2 * V; e++) v[e] *= rs * (is_q ? gq[e] : gk[e]);
        }
        if (turned) {
          float cs[V], sn[V];
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            *(f4*)(cs + e) = *(const f4*)(turns + 2 * t * pairs + unit * V + e);
            *(f4*)(sn + e) = *(const f4*)(turns + (2 * t + 1) * pairs + unit * V + e);
          }
#pragma unroll
          for (int e = 0; e < V; e++) {
            float& x = v[HALVES ? e : 2 * e];
            float& y = v[HALVES ? e + V : 2 * e + 1];
            const float c = cs[e], s = sn[e], r = x * c - y * s;
            y = y * c + x * s;
            x = r;
          }
        }
        x0.set(v), x1.set(v + V);
        if (first_ok) *(Chunk<T, V>*)(to + c0 * V * size) = x0;
        if (second_ok) *(Chunk<T, V>*)(to + c1 * V * size) = x1;
      }
      t += w.step_tokens, h += w.step_heads;
      if (h - h_first >= w.heads) h -= w.heads, t++;
    }
    __syncthreads();  // the next tokens' sines take this one's place
  }
}

template <int T, int V, int L>
hipError_t launch(const RotaryArgs& a, int pairing, hipStream_t s) {
  const int heads = a.q_heads + a.k_heads, pairs = a.rot / 2, step = 256 / L;
  // Heads per workgroup: four rounds of its lanes, one where that leaves workgroups for every compute unit.
  const int64_t all = (int64_t)a.T * heads;
  const int want = all < (int64_t)1024 * step ? step : 4 * step;
  Shape w{};
  w.heads = std::min(heads, want);
  w.tokens = std::max(1, want / heads);
  if (pairs > 0) w.tokens = std::min(w.tokens, std::max(1, 4096 / (2 * pairs)));  // 16 KiB of sines
  w.tokens = (int)std::min<int64_t>(w.tokens, a.T);
  w.step_tokens = step / w.heads;
  w.step_heads = step % w.heads;
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)a.T + w.tokens - 1) / w.tokens, 1 << 20), (heads + w.heads - 1) / w.heads);
  const size_t lds = (size_t)w.tokens * 2 * pairs * 4;
  if (pairing == ROTARY_HALVES) T5K_LAUNCH((rotary_kernel<T, V, L, true>), grid, dim3(256), lds, s, a, w);
  else T5K_LAUNCH((rotary_kernel<T, V, L, false>), grid, dim3(256), lds, s, a, w);
  return hipGetLastError();
}
template <int T, int V>
hipError_t launch_lanes(const RotaryArgs& a, int pairing, hipStream_t s) {
  const int units = (a.D / V + 1) / 2;
  if (units <= 4) return launch<T, V, 4>(a, pairing, s);
  if (units <= 8) return launch<T, V, 8>(a, pairing, s);
  if (units <= 16) return launch<T, V, 16>(a, pairing, s);
  if (units <= 32) return launch<T, V, 32>(a, pairing, s);
  if (units <= 64) return launch<T, V, 64>(a, pairing, s);
  return hipErrorInvalidValue;
}
}  // namespace

namespace t5k {
hipError_t launch_rotary(const RotaryArgs& a, int pairing, hipStream_t s) {
  if (a.T == 0 || a.q_heads + a.k_heads == 0) return hipSuccess;
  if (a.T < 0 || a.D <= 0 || a.D % 8 || a.D > ROTARY_MAX_DIM || a.rot < 0 || a.rot > a.D || a.rot % 8) return hipErrorInvalidValue;
  // 16-bit values go eight to a load where a half of the rotated part is whole loads, four otherwise
  const bool wide = a.rot % 16 == 0;
  switch (a.type) {
    case FP8_IO_F32: return launch_lanes<FP8_IO_F32, 4>(a, pairing, s);
    case FP8_IO_F16: return wide ? launch_lanes<FP8_IO_F16, 8>(a, pairing, s) : launch_lanes<FP8_IO_F16, 4>(a, pairing, s);
    case FP8_IO_BF16: return wide ? launch_lanes<FP8_IO_BF16, 8>(a, pairing, s) : launch_lanes<FP8_IO_BF16, 4>(a, pairing, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace t5k
