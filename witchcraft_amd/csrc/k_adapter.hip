// k_adapter.hip -- low-rank adapters of many requests at once beside a shared projection.  No counterpart in
// the reference, whose encoder has one set of weights.
//
//   h[t][j] = sum_k x[t][k] A_g[j][k]                      g = ids[t], j over S slices of R ranks
//   out[t][n] = y[t][n] + scale_g sum_r h[t][s(n) R + r] B_g[n][r]
//
// Two launches: h goes through a workspace.  A tile of rows may hold several adapters' rows; a workgroup takes the
// tile's adapters one after the other, each against all of the tile's rows (16 at a time, where one of them is its
// own), and keeps the results of the rows that are the adapter's.  Products run on the f16 / bf16 matrix
// instructions with the weights as the first operand and rows as the second, so that a lane's results belong to
// one row and the choice is one per lane; rows of other adapters cannot reach them.
#include "adapter.hpp"

#include <algorithm>

#include "fp8.hpp"

namespace {
using namespace t5k;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int ROWS = 16;        // of a matrix instruction
constexpr int STEP = 128;       // K values of a step
constexpr int WAVES = 4;
constexpr int TILE_COLS = 64;   // columns of a wave in the second product

template <bool BF>
__device__ __forceinline__ f4 mfma(const u4& a, const u4& b, f4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Eight e4m3 codes as f16 or bf16: exact.
template <bool BF>
__device__ __forceinline__ u4 widen8(uint32_t lo, uint32_t hi) {
  u4 r;
  if constexpr (BF) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.f, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, true));
  }
  return r;
}

// The adapters of a tile of NT x 16 rows, in the order of their first rows.  Lane l holds the ids of rows l % 16 of
// each sixteen, -1 where a row has none.  Every wave of a workgroup walks the same ones.
template <int NT>
struct Adapters {
  int id[NT];
  bool pending[NT];
  int current;
  bool use[NT];  // whether a row of this sixteen is the current one's (the same in all lanes)
  __device__ __forceinline__ Adapters(const AdapterArgs& p, int64_t row0) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const int64_t row = row0 + ROWS * i + (threadIdx.x & 15);
      const int v = row < p.T ? p.ids[row] : -1;
      id[i] = (unsigned)v < (unsigned)p.G ? v : -1;
      pending[i] = id[i] >= 0;
    }
  }
  __device__ __forceinline__ bool next() {
    current = -1;
#pragma unroll
    for (int i = NT - 1; i >= 0; i--) {
      const uint64_t m = __ballot(pending[i]);
      if (m) current = __builtin_amdgcn_readlane(id[i], __builtin_ctzll(m));
    }
    if (current < 0) return false;
#pragma unroll
    for (int i = 0; i < NT; i++) {
      use[i] = __ballot(id[i] == current) != 0;
      pending[i] = pending[i] && id[i] != current;
    }
    return true;
  }
};

// The adapter's rank, rounded up to whole eights: what its weights are read up to.
__device__ __forceinline__ int rank_of(const AdapterArgs& p, int g) {
  if (!p.ranks) return p.R;
  const int r = __builtin_amdgcn_readfirstlane(p.ranks[g]);
  return r <= 0 ? 0 : (r >= p.R ? p.R : (r + 7) & ~7);
}

// ---- h = x A^T: 16 NT rows x 16 RT ranks per workgroup, its waves on steps of 128 K in turn ----
// Lane (r = lane % 16, g = lane / 16) holds row r's K values 16 g .. + 15 and 64 + 16 g .. + 15 of a step, so that
// four lanes read whole lines of 16-bit values and half ones of codes.  The waves' sums meet in LDS and are added in
// wave order.  Workgroups split K further where there are few rows; their sums are parts of h.
template <bool CODES, bool BF, int NT, int RT>
__global__ __launch_bounds__(64 * WAVES) void adapter_down_kernel(AdapterArgs p, int splits, int groups) {
  __shared__ f4 red[WAVES][NT * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int SR = p.S * p.R, steps = (p.K + STEP - 1) / STEP;
  const int split = (int)blockIdx.y / groups, group = (int)blockIdx.y % groups;
  const size_t m16 = fp8_scale_rows(p.T);
  const int64_t tiles = ((int64_t)p.T + ROWS * NT - 1) / (ROWS * NT);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row0 = tile * ROWS * NT;
    Adapters<NT> ad(p, row0);
    for (unsigned seen = 0; ad.next(); seen++) {
      if (seen % gridDim.z != blockIdx.z) continue;
      const int rank = rank_of(p, ad.current);
      const uint16_t* arow[RT];
      bool live[RT];
#pragma unroll
      for (int q = 0; q < RT; q++) {
        const int j = ROWS * (group * RT + q) + r;
        const bool ok = j < SR && j % p.R < rank;
        live[q] = __ballot(ok) != 0;
        arow[q] = (const uint16_t*)p.a + ((size_t)ad.current * SR + (ok ? j : 0)) * p.K;
      }
      f4 acc[NT][RT];
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int q = 0; q < RT; q++) acc[i][q] = f4{0.f, 0.f, 0.f, 0.f};
      for (int kb = split * WAVES + wave; kb < steps; kb += splits * WAVES) {
        const int k0 = kb * STEP + 16 * g;
        const bool ok0 = k0 < p.K, ok1 = k0 + 64 < p.K;
        const u4 zero = u4{0, 0, 0, 0};
        u4 w[RT][4];
#pragma unroll
        for (int q = 0; q < RT; q++)
          if (live[q]) {
            w[q][0] = ok0 ? *(const u4*)(arow[q] + k0) : zero;
            w[q][1] = ok0 ? *(const u4*)(arow[q] + k0 + 8) : zero;
            w[q][2] = ok1 ? *(const u4*)(arow[q] + k0 + 64) : zero;
            w[q][3] = ok1 ? *(const u4*)(arow[q] + k0 + 72) : zero;
          }
#pragma unroll
        for (int i = 0; i < NT; i++)
          if (ad.use[i]) {
            const int64_t row = min(row0 + ROWS * i + r, (int64_t)p.T - 1);
            u4 v[4];
            float scale = 1.f;
            if constexpr (CODES) {
              const uint8_t* at = (const uint8_t*)p.x + row * p.ldx;
              const u4 c0 = ok0 ? *(const u4*)(at + k0) : zero, c1 = ok1 ? *(const u4*)(at + k0 + 64) : zero;
              scale = e8m0_value(p.x_scales[kb * m16 + row]);
              v[0] = widen8<BF>(c0[0], c0[1]), v[1] = widen8<BF>(c0[2], c0[3]);
              v[2] = widen8<BF>(c1[0], c1[1]), v[3] = widen8<BF>(c1[2], c1[3]);
            } else {
              const uint16_t* at = (const uint16_t*)p.x + row * p.ldx;
              v[0] = ok0 ? *(const u4*)(at + k0) : zero;
              v[1] = ok0 ? *(const u4*)(at + k0 + 8) : zero;
              v[2] = ok1 ? *(const u4*)(at + k0 + 64) : zero;
              v[3] = ok1 ? *(const u4*)(at + k0 + 72) : zero;
            }
#pragma unroll
            for (int q = 0; q < RT; q++)
              if (live[q]) {
                f4 t = CODES ? f4{0.f, 0.f, 0.f, 0.f} : acc[i][q];
#pragma unroll
                for (int e = 0; e < 4; e++) t = mfma<BF>(w[q][e], v[e], t);
                if constexpr (CODES) {
#pragma unroll
                  for (int e = 0; e < 4; e++) acc[i][q][e] = __builtin_fmaf(t[e], scale, acc[i][q][e]);
                } else {
                  acc[i][q] = t;
                }
              }
          }
      }
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int q = 0; q < RT; q++) red[wave][i * RT + q][lane] = acc[i][q];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const int64_t row = row0 + ROWS * i + r;
        if (ad.id[i] != ad.current) continue;
#pragma unroll
        for (int q = 0; q < RT; q++) {
          const int t = i * RT + q, j = ROWS * (group * RT + q) + 4 * g;
          if (t % WAVES != wave || j >= SR || j % p.R >= rank) continue;
          f4 v = red[0][t][lane];
#pragma unroll
          for (int k = 1; k < WAVES; k++) v += red[k][t][lane];
          *(f4*)(p.h + ((size_t)split * p.T + row) * SR + j) = v;
        }
      }
      __syncthreads();
    }
  }
}

// ---- out = y + scale h B^T: 16 NT rows x 256 columns of one slice per workgroup, 64 columns a wave -------
// h is f32 and stays so: its values go to the matrix instructions as sums of 16-bit parts, all of which multiply the
// same weights, as if K were `PARTS` times the rank.  bf16: three parts hold all 24 bits (results in f32), two the
// upper 16 (an error of 2^-17 of h, where the results' own rounding is 2^-9 or 2^-12).  f16: two parts hold 22 bits of
// a row scaled by a power of two to below 2^15, as f16 has neither the range nor, below 2^-14, the bits.
template <bool BF, int PARTS>
__device__ __forceinline__ void split_parts(float v, uint16_t (&part)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; i++) {
    float got;
    if constexpr (BF) {
      // cut, not rounded, up to the last part: the largest values round to infinity
      const uint32_t u = __float_as_uint(v);
      if (i < PARTS - 1 || PARTS == 3) part[i] = (uint16_t)(u >> 16), got = __uint_as_float(u & 0xffff0000u);
      else part[i] = __builtin_bit_cast(uint16_t, (__bf16)v), got = v;
    } else {
      const _Float16 f = i < PARTS - 1 ? (_Float16)__builtin_amdgcn_cvt_pkrtz(v, 0.f)[0] : (_Float16)v;
      part[i] = __builtin_bit_cast(uint16_t, f);
      got = (float)f;
    }
    // infinities and NaN are their first part
    v = (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? 0.f : v - got;
  }
}

template <int YT>
struct Out {  // 16 values of a row: f32 four at a time, 16-bit types eight
  static constexpr int PIECES = YT == FP8_IO_F32 ? 4 : 2, COUNT = 16 / PIECES;
  u4 raw[PIECES];
};
// The column, of a wave's 64, of value e of lane group g in matrix tile j: such that a lane holds whole pieces.
template <int YT>
__device__ __forceinline__ int column(int j, int g, int e) {
  return YT == FP8_IO_F32 ? 16 * j + 4 * g + e : 32 * (j / 2) + 8 * g + 4 * (j % 2) + e;
}
template <int YT>
__device__ __forceinline__ void add_to(u4& raw, const f4* v, float f) {  // raw += v f, rounded once
  if constexpr (YT == FP8_IO_F32) {
    f4 x = __builtin_bit_cast(f4, raw);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(v[0][e], f, x[e]);
    raw = __builtin_bit_cast(u4, x);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t w = raw[e];
      float lo, hi;
      if constexpr (YT == FP8_IO_F16) lo = f16_bits_to_f32(w & 0xffffu), hi = f16_bits_to_f32(w >> 16);
      else lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
      lo = __builtin_fmaf(v[e / 2][2 * (e % 2)], f, lo);
      hi = __builtin_fmaf(v[e / 2][2 * (e % 2) + 1], f, hi);
      typedef _Float16 hh __attribute__((ext_vector_type(2)));
      typedef __bf16 bb __attribute__((ext_vector_type(2)));
      typedef float ff __attribute__((ext_vector_type(2)));
      if constexpr (YT == FP8_IO_F16) raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((ff{lo, hi}), hh));
      else raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((ff{lo, hi}), bb));
    }
  }
}

template <int YT, bool BF, int NT, int PARTS>
__global__ __launch_bounds__(64 * WAVES) void adapter_up_kernel(AdapterArgs p, int splits) {
  extern __shared__ u4 lds[];
  constexpr int COUNT = Out<YT>::COUNT, PIECES = Out<YT>::PIECES, SIZE = YT == FP8_IO_F32 ? 4 : 2;
  constexpr int LANES = 64 * WAVES / (ROWS * NT), CHUNKS = (ADAPTER_MAX_RANK / 4 + LANES - 1) / LANES;  // of a row of h
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int SR = p.S * p.R, pitch = PARTS * p.R + 8;  // of a row of parts: its 16-byte reads spread over the banks
  uint16_t* parts = (uint16_t*)lds;                   // [16 NT][pitch]
  float* unscale = (float*)(parts + ROWS * NT * pitch);
  // this workgroup's columns
  int s = 0, n0 = 0, c = (int)blockIdx.x;
  while (true) {
    const int t = (p.cols[s] + WAVES * TILE_COLS - 1) / (WAVES * TILE_COLS);
    if (c < t) break;
    c -= t, n0 += p.cols[s], s++;
  }
  const int end = n0 + p.cols[s];
  n0 += c * WAVES * TILE_COLS + wave * TILE_COLS;
  const bool busy = n0 < end;
  const int64_t tiles = ((int64_t)p.T + ROWS * NT - 1) / (ROWS * NT);
  const bool in_place = p.y == p.out;
  for (int64_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
    const int64_t row0 = tile * ROWS * NT;
    Out<YT> y[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const int64_t row = row0 + ROWS * i + r;
#pragma unroll
      for (int q = 0; q < PIECES; q++) {
        const int n = n0 + column<YT>(q * (4 / PIECES), g, 0);
        if (row < p.T && n < end) y[i].raw[q] = *(const u4*)((const char*)p.y + (row * p.ldy + n) * SIZE);
      }
    }
    Adapters<NT> ad(p, row0);
    if (!in_place && blockIdx.z == 0) {  // rows without an adapter
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const int64_t row = row0 + ROWS * i + r;
        if (row >= p.T || ad.id[i] >= 0) continue;
#pragma unroll
        for (int q = 0; q < PIECES; q++) {
          const int n = n0 + column<YT>(q * (4 / PIECES), g, 0);
          if (n < end) *(u4*)((char*)p.out + (row * p.ldo + n) * SIZE) = y[i].raw[q];
        }
      }
    }
    for (unsigned seen = 0; ad.next(); seen++) {
      if (seen % gridDim.z != blockIdx.z) continue;
      const int rank = rank_of(p, ad.current), depth = PARTS * rank;
      {
        // h of the tile's rows, all of them, for they are there: rows of other adapters and behind the last give
        // results that nothing keeps
        const int t = threadIdx.x / LANES, q = threadIdx.x % LANES;
        const int64_t row = min(row0 + t, (int64_t)p.T - 1);
        const float scale = p.scales ? p.scales[ad.current] : 1.f;
        f4 v[CHUNKS];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) {
          const int at = 4 * (q + LANES * k);
          v[k] = f4{0.f, 0.f, 0.f, 0.f};
          if (at < rank) {
            const float* from = p.h + (size_t)row * SR + s * p.R + at;
            v[k] = *(const f4*)from;
            for (int i = 1; i < splits; i++) v[k] += *(const f4*)(from + (size_t)i * p.T * SR);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              v[k][e] *= scale;
              top = fmaxf(top, finite_abs(v[k][e]));
            }
          }
        }
        float up = 1.f;
        if constexpr (!BF) {
          // max over the row's lanes
          if constexpr (LANES == 4) {
            top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0xb1, 0xf, 0xf, false)));
            top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0x4e, 0xf, 0xf, false)));
          } else if constexpr (LANES == 8) {
            top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0xb1, 0xf, 0xf, false)));
            top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0x4e, 0xf, 0xf, false)));
            top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0x141, 0xf, 0xf, false)));
          } else {
            top = max_row16(top);
          }
          // the power of two that brings top to 2^14 .. 2^15, of 2^-112 .. 2^112
          const int e = (int)(__float_as_uint(top) >> 23) - 127;
          const int shift = top > 0.f ? min(max(14 - e, -112), 112) : 0;
          up = __uint_as_float((uint32_t)(127 + shift) << 23);
          if (q == 0) unscale[t] = __uint_as_float((uint32_t)(127 - shift) << 23);
        }
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) {
          const int at = 4 * (q + LANES * k);
          if (at < rank) {
            uint16_t w[4][PARTS];
#pragma unroll
            for (int e = 0; e < 4; e++) split_parts<BF, PARTS>(v[k][e] * up, w[e]);
#pragma unroll
            for (int i = 0; i < PARTS; i++) {
              typedef uint32_t u2 __attribute__((ext_vector_type(2)));
              *(u2*)(parts + t * pitch + i * rank + at) =
                  u2{(uint32_t)w[0][i] | (uint32_t)w[1][i] << 16, (uint32_t)w[2][i] | (uint32_t)w[3][i] << 16};
            }
          }
        }
      }
      __syncthreads();
      if (busy) {
        const uint16_t* brow[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int n = min(n0 + column<YT>(j, r / 4, r % 4), end - 1);
          brow[j] = (const uint16_t*)p.b + ((size_t)ad.current * p.N + n) * p.R;
        }
        f4 acc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < depth; k0 += 32) {
          const int k = k0 + 8 * g;
          const bool ok = k < depth;
          const int wk = ok ? k % rank : 0;  // the parts' weights are the same ones
          const u4 zero = u4{0, 0, 0, 0};
          u4 w[4];
#pragma unroll
          for (int j = 0; j < 4; j++) w[j] = ok ? *(const u4*)(brow[j] + wk) : zero;
#pragma unroll
          for (int i = 0; i < NT; i++)
            if (ad.use[i]) {
              const u4 v = ok ? *(const u4*)(parts + (ROWS * i + r) * pitch + k) : zero;
#pragma unroll
              for (int j = 0; j < 4; j++) acc[i][j] = mfma<BF>(w[j], v, acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; i++) {
          const int64_t row = row0 + ROWS * i + r;
          if (ad.id[i] != ad.current) continue;  // -1 behind the last row
          const float f = BF ? 1.f : unscale[ROWS * i + r];
#pragma unroll
          for (int q = 0; q < PIECES; q++) {
            const int n = n0 + column<YT>(q * (4 / PIECES), g, 0);
            if (n >= end) continue;
            add_to<YT>(y[i].raw[q], &acc[i][q * (4 / PIECES)], f);
            *(u4*)((char*)p.out + (row * p.ldo + n) * SIZE) = y[i].raw[q];
          }
        }
      }
      __syncthreads();
    }
  }
}

// 16-row tiles of a workgroup's rows in the two products, and workgroups that share a tile's adapters.
struct Plan {
  int down_tiles, up_tiles, share;
};
Plan plan_of(const AdapterArgs& a, int up_blocks) {
  Plan q{1, 1, 1};
  const int64_t rows = ((int64_t)a.T + ROWS - 1) / ROWS;
  if (rows >= 4 * 1024) q.down_tiles = 4;
  if (rows * up_blocks >= 4 * 512) q.up_tiles = 4;
  if (a.T <= 256) q.share = std::min(16, a.T);
  return q;
}

template <bool CODES, bool BF, int NT>
hipError_t launch_down(const AdapterArgs& a, int share, hipStream_t s) {
  const int SR = a.S * a.R, tiles = (SR + ROWS - 1) / ROWS, splits = adapter_splits(a.T, a.K, SR);
  const int rt = tiles == 1 ? 1 : (tiles == 2 ? 2 : (tiles == 3 ? 3 : 4)), groups = (tiles + rt - 1) / rt;
  const int64_t rows = ((int64_t)a.T + ROWS * NT - 1) / (ROWS * NT);
  const dim3 grid((unsigned)std::min<int64_t>(rows, 1 << 20), (unsigned)(splits * groups), (unsigned)share);
  switch (rt) {
    case 1: T5K_LAUNCH((adapter_down_kernel<CODES, BF, NT, 1>), grid, dim3(64 * WAVES), 0, s, a, splits, groups); break;
    case 2: T5K_LAUNCH((adapter_down_kernel<CODES, BF, NT, 2>), grid, dim3(64 * WAVES), 0, s, a, splits, groups); break;
    case 3: T5K_LAUNCH((adapter_down_kernel<CODES, BF, NT, 3>), grid, dim3(64 * WAVES), 0, s, a, splits, groups); break;
    default: T5K_LAUNCH((adapter_down_kernel<CODES, BF, NT, 4>), grid, dim3(64 * WAVES), 0, s, a, splits, groups); break;
  }
  return hipGetLastError();
}

template <int YT, bool BF, int NT>
hipError_t launch_up(const AdapterArgs& a, int blocks, int share, hipStream_t s) {
  constexpr int PARTS = BF && YT == FP8_IO_F32 ? 3 : 2;
  const int64_t rows = ((int64_t)a.T + ROWS * NT - 1) / (ROWS * NT);
  const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(rows, 65535), (unsigned)share);
  const size_t lds = (size_t)ROWS * NT * ((PARTS * a.R + 8) * 2 + 4);
  T5K_LAUNCH((adapter_up_kernel<YT, BF, NT, PARTS>), grid, dim3(64 * WAVES), lds, s, a, adapter_splits(a.T, a.K, a.S * a.R));
  return hipGetLastError();
}
template <bool BF, int NT>
hipError_t launch_up_type(const AdapterArgs& a, int blocks, int share, hipStream_t s) {
  switch (a.y_type) {
    case FP8_IO_F32: return launch_up<FP8_IO_F32, BF, NT>(a, blocks, share, s);
    case FP8_IO_F16: return launch_up<FP8_IO_F16, BF, NT>(a, blocks, share, s);
    case FP8_IO_BF16: return launch_up<FP8_IO_BF16, BF, NT>(a, blocks, share, s);
  }
  return hipErrorInvalidValue;
}
template <bool BF>
hipError_t launch(const AdapterArgs& a, hipStream_t s) {
  int blocks = 0;
  for (int i = 0; i < a.S; i++) blocks += (a.cols[i] + WAVES * TILE_COLS - 1) / (WAVES * TILE_COLS);
  const Plan q = plan_of(a, blocks);
  hipError_t e;
  if (a.x_type == ADAPTER_E4M3) e = q.down_tiles == 4 ? launch_down<true, BF, 4>(a, q.share, s) : launch_down<true, BF, 1>(a, q.share, s);
  else e = q.down_tiles == 4 ? launch_down<false, BF, 4>(a, q.share, s) : launch_down<false, BF, 1>(a, q.share, s);
  if (e != hipSuccess) return e;
  return q.up_tiles == 4 ? launch_up_type<BF, 4>(a, blocks, q.share, s) : launch_up_type<BF, 1>(a, blocks, q.share, s);
}
}  // namespace

namespace t5k {
int adapter_splits(int T, int K, int SR) {
  const int64_t tiles = ((int64_t)T + ROWS - 1) / ROWS;
  const int most = ((K + STEP - 1) / STEP + WAVES - 1) / WAVES;  // a step for each wave
  return (int)std::max<int64_t>(1, std::min<int64_t>({most, 16, 256 / std::max<int64_t>(1, tiles)}));
}

hipError_t launch_adapter(const AdapterArgs& a, hipStream_t s) {
  if (a.T == 0 || a.N == 0) return hipSuccess;
  if (a.T < 0 || a.K <= 0 || a.K % 16 || a.R <= 0 || a.R % 8 || a.R > ADAPTER_MAX_RANK || a.S < 1 || a.S > ADAPTER_MAX_SLICES)
    return hipErrorInvalidValue;
  if (a.w_type == FP8_IO_BF16) return launch<true>(a, s);
  if (a.w_type == FP8_IO_F16) return launch<false>(a, s);
  return hipErrorInvalidValue;
}
}  // namespace t5k
