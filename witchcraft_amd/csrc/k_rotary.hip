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

// Queries or keys alone: rows of `heads` heads, and how workgroups share them.
struct Part {
  const char* from;
  char* to;
  int64_t ld, ld_to;  // bytes from row to row
  const float* gamma;
  int heads;
  int tokens, group;        // rows and heads of a workgroup's share, 256 heads at most in all
  unsigned per_group;       // 2^16 / group, rounded up: i * per_group >> 16 is i / group for i < 256
  unsigned groups, blocks;  // groups of heads, workgroups for this part
};

// Of both parts.
struct Shared {
  float inverse;       // 1 / D
  unsigned per_pairs;  // 2^20 / pairs, rounded up: i * per_pairs >> 20 is i / pairs for i < 2,048
};

// x1 of the lower four lanes of each eight and x0 of the upper four change places.
template <int WORDS>
__device__ __forceinline__ void swap_quads(uint32_t* x0, uint32_t* x1) {
#pragma unroll
  for (int i = 0; i < WORDS; i++) {
    const int a = (int)x0[i], b = (int)x1[i];
    x1[i] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x104, 0xf, 0x5, false);  // lane + 4 to the lower four
    x0[i] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x114, 0xf, 0xa, false);  // lane - 4 to the upper four
  }
}

// Workgroups [0, q.blocks) take the queries, the others the keys.  A lane holds two chunks of V values of a head,
// c and c + rot / 2 / V, which are pairs in the one form and contain them in the other, and neighbouring chunks
// behind the rotated part; L lanes (a power of two) hold the head.  A workgroup walks the heads of some rows, the next
// head's values on their way while one is turned, and computes each row's sines and cosines once, into LDS.
// What bounds it is memory, and for few rows a launch and two trips to it: 16,391 x (32 + 8) heads of 128 in bf16, three
// axes, norms: 71 us, 4.7 TB/s; one row of it 3.8 us.  Stores go past the caches: 20.9 instead of 27.1 us for 10,007 x
// (16 + 16) heads of 80 whose input the last-level cache does not hold.
// EIGHT: heads of eight chunks, all turned, would be loaded and stored in halves of 64 bytes (74,640 x (12 + 12) heads of
// 64 in f16 with norms: 106 us, 4.3 TB/s); there eight lanes load a head's chunks into x0 and the next head's into x1,
// and the quads of lanes swap (93 us, 4.9 TB/s).
template <int T, int V, int L, bool HALVES, bool EIGHT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, Shared u, Part q, Part k) {
  extern __shared__ f4 lds[];
  float* turns = (float*)lds;  // [tokens][2][pairs]: cosines, sines
  typedef Chunk<T, V> C;
  constexpr int SIZE = T == FP8_IO_F32 ? 4 : 2, PIECE = V * SIZE, STEP = 256 / L, WORDS = PIECE / 4;
  const bool is_q = blockIdx.x < q.blocks;
  const Part& w = is_q ? q : k;
  const unsigned block = is_q ? blockIdx.x : blockIdx.x - q.blocks, stride = w.blocks / w.groups;
  const int pairs = a.rot / 2, unit = threadIdx.x & (L - 1), slot = threadIdx.x / L;
  const int n = a.D / V, m = pairs / V;  // chunks of a head, chunks of a half of its rotated part
  const bool turned = unit < m, first_ok = EIGHT || 2 * unit < n;
  const int c0 = turned ? unit : 2 * unit, c1 = turned ? unit + m : 2 * unit + 1;
  const bool second_ok = EIGHT || (c1 < n && first_ok);
  const int h0 = (int)(block % w.groups) * w.group, group = min(w.group, w.heads - h0);
  const int head = a.D * SIZE;
  // what a lane loads and stores: chunk l0 of item i + d0 and chunk l1 of item i + d1
  const int l0 = (EIGHT ? (int)(threadIdx.x & 7) : c0) * PIECE, l1 = (EIGHT ? (int)(threadIdx.x & 7) : c1) * PIECE;
  const int d0 = EIGHT ? -(slot & 1) : 0, d1 = EIGHT ? 1 - (slot & 1) : 0;
  for (int64_t t0 = (int64_t)(block / w.groups) * w.tokens; t0 < a.T; t0 += (int64_t)stride * w.tokens) {
    const int tokens = (int)min((int64_t)w.tokens, a.T - t0), items = tokens * w.group;
    const char* from = w.from + t0 * w.ld + (int64_t)h0 * head;
    char* to = w.to + t0 * w.ld_to + (int64_t)h0 * head;
    const auto place = [&](int i, int64_t ld, int64_t& at) {  // of item i; whether there is one
      const int t = (int)((unsigned)i * w.per_group >> 16), h = i - t * w.group;
      at = t * ld + h * head;
      return i < items && h < group;
    };
    const auto load = [&](int i, C& x0, C& x1) {
      int64_t at;
      const bool ok = place(i + d0, w.ld, at);
      if (ok && first_ok) x0 = *(const C*)(from + at + l0);
      const bool ok1 = EIGHT ? place(i + d1, w.ld, at) : ok;
      if (ok1 && second_ok) x1 = *(const C*)(from + at + l1);
    };
    C x0{}, x1{};
    load(slot, x0, x1);
    float g[2 * V];
    if (w.gamma) {
#pragma unroll
      for (int e = 0; e < 2 * V; e++) g[e] = (e < V ? first_ok : second_ok) ? w.gamma[(e < V ? c0 : c1 - 1) * V + e] : 0.f;
    }
    for (int i = threadIdx.x; i < tokens * pairs; i += 256) {
      const int r = (int)((unsigned)i * u.per_pairs >> 20), p = i - r * pairs;
      const uint64_t entry = a.table[p];
      const int axis = (int)(entry & (ROTARY_MAX_AXES - 1));
      int32_t pos;
      if (a.axes == 1) {  // on its way together with the table's entry
        pos = a.pos[t0 + r];
        if (axis) pos = 0;
      } else {
        pos = axis < a.axes ? a.pos[(size_t)axis * a.T + t0 + r] : 0;
      }
      const uint64_t turn = (uint64_t)(int64_t)pos * (entry & ~(uint64_t)(ROTARY_MAX_AXES - 1));
      float s, c;
      sincos_turn((uint32_t)(turn >> 32), s, c);
      turns[2 * r * pairs + p] = c;
      turns[(2 * r + 1) * pairs + p] = s;
    }
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += STEP) {
      C y0{}, y1{};
      load(i0 + STEP + slot, y0, y1);
      if constexpr (EIGHT) swap_quads<WORDS>((uint32_t*)&x0.raw, (uint32_t*)&x1.raw);
      float v[2 * V];
      x0.get(v), x1.get(v + V);
      if (w.gamma) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 2 * V; e++) ss = __builtin_fmaf(v[e], v[e], ss);
        const float rs = rsqrtf(__builtin_fmaf(sum_group<L>(ss), u.inverse, a.eps));
#pragma unroll
        for (int e = 0; e < 2 * V; e++) v[e] *= rs * g[e];
      }
      if (turned) {
        // halves: pair e is (c0's, c1's) value e; neighbours: two values of c0, then of c1
        const int t = min((int)((unsigned)(i0 + slot) * w.per_group >> 16), tokens - 1);
        const float* cs = turns + 2 * t * pairs;
        constexpr int W = HALVES ? 4 : V / 2;
        typedef float fw __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int i = 0; i < V; i += W) {
          const int p = HALVES ? c0 * V + i : (i == 0 ? c0 : c1) * W;
          const fw cw = *(const fw*)(cs + p), sw = *(const fw*)(cs + pairs + p);
#pragma unroll
          for (int e = i; e < i + W; e++) {
            float& x = v[HALVES ? e : 2 * e];
            float& y = v[HALVES ? e + V : 2 * e + 1];
            const float c = cw[e - i], s = sw[e - i], r = x * c - y * s;
            y = y * c + x * s;
            x = r;
          }
        }
      }
      x0.set(v), x1.set(v + V);
      if constexpr (EIGHT) swap_quads<WORDS>((uint32_t*)&x0.raw, (uint32_t*)&x1.raw);
      int64_t at;
      const bool ok = place(i0 + slot + d0, w.ld_to, at);
      if (ok && first_ok) __builtin_nontemporal_store(x0.raw, &((C*)(to + at + l0))->raw);
      const bool ok1 = EIGHT ? place(i0 + slot + d1, w.ld_to, at) : ok;
      if (ok1 && second_ok) __builtin_nontemporal_store(x1.raw, &((C*)(to + at + l1))->raw);
      x0 = y0, x1 = y1;
    }
    __syncthreads();  // the next rows' sines take this one's place
  }
}

// How the workgroups share `heads` heads of T rows, `step` heads at a time.
Part share(const RotaryArgs& a, const void* from, int64_t ld, void* to, int64_t ld_to, const float* gamma, int heads, int step) {
  const int size = a.type == FP8_IO_F32 ? 4 : 2, pairs = a.rot / 2;
  Part w{};
  w.from = (const char*)from, w.to = (char*)to;
  w.ld = ld * size, w.ld_to = ld_to * size;
  w.gamma = gamma;
  w.heads = heads;
  w.group = w.groups = 1;
  if (heads == 0) return w;
  // Up to four rounds of a workgroup's lanes while that leaves 400 workgroups a part.  4,616 x (12 + 12) heads of 64 in
  // f16: 7.8 us at two rounds, 8.7 at one; 10,007 x (16 + 16) heads of 80 in bf16 21.7 at four, 20.9 at two.
  const int want = step * (int)std::min<int64_t>(4, std::max<int64_t>(1, (int64_t)a.T * heads / (400 * step)));
  w.group = std::min(heads, want);
  w.tokens = std::max(1, want / w.group);
  if (pairs > 0) w.tokens = std::min(w.tokens, std::max(1, 4096 / (2 * pairs)));  // 16 KiB of sines
  w.tokens = std::min(w.tokens, a.T);
  w.per_group = (65536 + w.group - 1) / w.group;
  w.groups = (unsigned)((heads + w.group - 1) / w.group);
  const unsigned most = std::max(1u, (1u << 20) / w.groups);  // workgroups for a group; they walk what is left
  w.blocks = w.groups * std::min((unsigned)(((int64_t)a.T + w.tokens - 1) / w.tokens), most);
  return w;
}

template <int T, int V, int L>
hipError_t launch(const RotaryArgs& a, int pairing, hipStream_t s) {
  const Part q = share(a, a.q, a.ldq, a.q_out, a.ldq_out, a.q_gamma, a.q_heads, 256 / L);
  const Part k = share(a, a.k, a.ldk, a.k_out, a.ldk_out, a.k_gamma, a.k_heads, 256 / L);
  const Shared u{1.f / (float)a.D, a.rot ? (unsigned)((1 << 20) + a.rot / 2 - 1) / (unsigned)(a.rot / 2) : 0u};
  const dim3 grid(q.blocks + k.blocks);
  const size_t lds = (size_t)std::max(q.tokens, k.tokens) * a.rot * 4;
  if constexpr (L == 4 && (T == FP8_IO_F32 || V == 8)) {  // of 16-bit values, four to a load never are a whole such head
    if (a.D == 8 * V && a.rot == a.D) {
      if (pairing == ROTARY_HALVES) T5K_LAUNCH((rotary_kernel<T, V, L, true, true>), grid, dim3(256), lds, s, a, u, q, k);
      else T5K_LAUNCH((rotary_kernel<T, V, L, false, true>), grid, dim3(256), lds, s, a, u, q, k);
      return hipGetLastError();
    }
  }
  if (pairing == ROTARY_HALVES) T5K_LAUNCH((rotary_kernel<T, V, L, true, false>), grid, dim3(256), lds, s, a, u, q, k);
  else T5K_LAUNCH((rotary_kernel<T, V, L, false, false>), grid, dim3(256), lds, s, a, u, q, k);
  return hipGetLastError();
}
template <int T, int V>
hipError_t launch_lanes(const RotaryArgs& a, int pairing, hipStream_t s) {
  const int units = (a.D / V + 1) / 2;
  if (units <= 4) return launch<T, V, 4>(a, pairing, s);
  if (units <= 8) return launch<T, V, 8>(a, pairing, s);
  if (units <= 16) return launch<T, V, 16>(a, pairing, s);
  if (units <= 32) return launch<T, V, 32>(a, pairing, s);
  if constexpr (ROTARY_MAX_DIM > 64 * V) {
    if (units <= 64) return launch<T, V, 64>(a, pairing, s);
  }
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
