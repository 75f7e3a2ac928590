// k_adapter.hip -- low-rank adapters of many requests at once beside a shared projection.  No counterpart in
// the reference, whose encoder has one set of weights.
//
//   h[t][j] = sum_k x[t][k] A_g[j][k]                      g = ids[t], j over S slices of R ranks
//   out[t][n] = y[t][n] + scale_g sum_r h[t][s(n) R + r] B_g[n][r]
//
// Two launches: scale_g h goes through a workspace.  A tile of rows may hold several adapters' rows; they are taken
// one adapter after the other, each against all of the tile's rows (16 at a time, where one of them is its own), and
// the results of the rows that are the adapter's are kept.  Products run on the f16 / bf16 matrix instructions with
// the weights as the first operand and rows as the second, so that a lane's results belong to one row and the choice
// is one per lane; rows of other adapters cannot reach them.
//
// h is f32 and stays so: it is stored as a sum of bf16 parts, all of which multiply the same weights in the second
// product, as if there were so many times the ranks.  Three parts hold all 24 bits (results in f32), two the upper 16
// (within 2^-17 of h, where the results' own rounding is 2^-9 or 2^-12).  bf16 has f32's range, which f16 has not; f16
// weights go in as two bf16 parts, which hold their 11 bits.
#include "adapter.hpp"

#include <algorithm>

#include "fp8.hpp"

namespace {
using namespace t5k;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int ROWS = 16;        // of a matrix instruction
constexpr int STEP = 64;        // K values of a step
constexpr int DOWN_WAVES = 8;   // waves of a workgroup of the first product, at most
constexpr int COLS = 64;        // columns of a wave in the second product
constexpr int UP_WAVES = 4;     // its waves, on columns beside each other

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

// The adapters of a tile of NT x 16 rows.  Lane l holds the ids of rows l % 16 of each sixteen, -1 where a row has none.
// Every wave of a workgroup walks the same ones: all of them, in the order of their first rows, or with `only` (one
// sixteen) the one of row `only`, where that is its first.
template <int NT>
struct Adapters {
  int64_t row0;
  int id[NT];
  bool pending[NT];
  int current;
  int64_t row;  // the current one's first
  __device__ __forceinline__ Adapters(const AdapterArgs& p, int64_t first) : row0(first) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const int64_t row = row0 + ROWS * i + (threadIdx.x & 15);
      const int v = row < p.T ? p.ids[row] : -1;
      id[i] = (unsigned)v < (unsigned)p.G ? v : -1;
      pending[i] = id[i] >= 0;
    }
  }
  __device__ __forceinline__ void only(int row) {
    const int first = __builtin_amdgcn_readlane(id[0], row);
    const uint64_t m = __ballot(id[0] == first);
    pending[0] = id[0] == first && first >= 0 && __builtin_ctzll(m) == row;
  }
  __device__ __forceinline__ bool next() {
    current = -1;
#pragma unroll
    for (int i = NT - 1; i >= 0; i--) {
      const uint64_t m = __ballot(pending[i]);
      if (m) {
        current = __builtin_amdgcn_readlane(id[i], __builtin_ctzll(m));
        row = row0 + ROWS * i + __builtin_ctzll(m);
      }
    }
    if (current < 0) return false;
#pragma unroll
    for (int i = 0; i < NT; i++) pending[i] = pending[i] && id[i] != current;
    return true;
  }
  // Which row a lane reads for its row of sixteen i: its own where that is the current adapter's, and otherwise, as
  // nothing keeps the result, one that is read anyway.
  __device__ __forceinline__ int64_t source(int i) const {
    return id[i] == current ? row0 + ROWS * i + (threadIdx.x & 15) : row;
  }
};

// The adapter's rank, rounded up to whole eights: what its weights are read up to.
__device__ __forceinline__ int rank_of(const AdapterArgs& p, int g) {
  if (!p.ranks) return p.R;
  const int r = __builtin_amdgcn_readfirstlane(p.ranks[g]);
  return r <= 0 ? 0 : (r >= p.R ? p.R : (r + 7) & ~7);
}

// The next bf16 part of v, which keeps the rest: cut, not rounded, up to the last of two, for the largest values round
// to infinity.  Infinities and NaN are their first part.
__device__ __forceinline__ uint32_t next_part(float& v, bool last_of_two) {
  const uint32_t u = __float_as_uint(v);
  const uint32_t part = last_of_two ? (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v) : u >> 16;
  v = (u & 0x7f800000u) != 0x7f800000u ? v - __uint_as_float(u & 0xffff0000u) : 0.f;
  return part;
}

// ---- h = scale x A^T: 16 NT rows x 16 RT ranks per workgroup, its waves on 64 K values in turn ----
// Lane (r = lane % 16, g = lane / 16) holds row r's K values 16 g .. + 15 of a step, so that four lanes read a whole
// line of 16-bit values or half of one of codes; the next step's are on their way while one is multiplied.  The waves'
// sums meet in LDS and are added in wave order.  With JOIN, for few rows, workgroups split K further, and leave their
// sums in f32 for the second product to add.
template <bool CODES, bool BF, int NT, int RT>
struct DownStep {
  u4 w[RT][2], x[NT][CODES ? 1 : 2];
  uint32_t scale[NT];
  bool ok;
};
constexpr int down_occupancy(int NT, int RT) { return NT * RT <= 2 ? 4 : (NT * RT <= 8 ? 3 : 2); }  // waves a SIMD

template <bool CODES, bool BF, int NT, int RT, bool JOIN>
__global__ __launch_bounds__(64 * DOWN_WAVES, down_occupancy(NT, RT)) void adapter_down_kernel(AdapterArgs p, int splits, int parts) {
  extern __shared__ f4 red[];  // [waves][NT * RT][64], where there is more than one
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int SR = p.S * p.R, steps = (p.K + STEP - 1) / STEP, waves = (int)(blockDim.x >> 6);
  const int split = JOIN ? (int)blockIdx.y % splits : 0, group = JOIN ? (int)blockIdx.y / splits : (int)blockIdx.y;
  const int first = split * waves + wave, stride = splits * waves;
  const size_t m16 = fp8_scale_rows(p.T);
  const int64_t tiles = ((int64_t)p.T + ROWS * NT - 1) / (ROWS * NT);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row0 = tile * ROWS * NT;
    Adapters<NT> ad(p, row0);
    if (JOIN) ad.only((int)blockIdx.z);
    while (ad.next()) {
      int64_t at[NT];  // the lane's rows of x
#pragma unroll
      for (int i = 0; i < NT; i++) at[i] = ad.source(i);
      const float scale = p.scales ? p.scales[ad.current] : 1.f;
      // ranks past the adapter's own give results that nothing keeps
      const int rank = rank_of(p, ad.current);
      const uint16_t* arow[RT];
#pragma unroll
      for (int q = 0; q < RT; q++) {
        const int j = ROWS * (group * RT + q) + r;
        arow[q] = (const uint16_t*)p.a + ((size_t)ad.current * SR + min(j, SR - 1)) * p.K;
      }
      f4 acc[NT][RT];
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int q = 0; q < RT; q++) acc[i][q] = f4{0.f, 0.f, 0.f, 0.f};
      typedef DownStep<CODES, BF, NT, RT> Step;
      // loads are unconditional, past the rows' end from their start: a branch around each would cost registers, and
      // the addresses of results are left to be computed behind the loop for the same reason
      const auto load = [&](Step& v, int n) {
        const int k0 = n * STEP + 16 * g, k = k0 < p.K ? k0 : 0;
        const int block = min(n, steps - 1) / (FP8_BLOCK / STEP);  // of the scales: the same for all lanes
#pragma unroll
        for (int i = 0; i < NT; i++) {
          if constexpr (CODES) {
            v.x[i][0] = *(const u4*)((const uint8_t*)p.x + at[i] * p.ldx + k);
            v.scale[i] = p.x_scales[(size_t)block * m16 + at[i]];
          } else {
            const uint16_t* from = (const uint16_t*)p.x + at[i] * p.ldx + k;
            v.x[i][0] = *(const u4*)from;
            v.x[i][1] = *(const u4*)(from + 8);
          }
        }
#pragma unroll
        for (int q = 0; q < RT; q++) {
          v.w[q][0] = *(const u4*)(arow[q] + k);
          v.w[q][1] = *(const u4*)(arow[q] + k + 8);
        }
        v.ok = k0 < p.K;
      };
      const auto multiply = [&](const Step& v) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
          const u4 zero = u4{0, 0, 0, 0};
          u4 x0 = v.ok ? v.x[i][0] : zero, x1 = CODES ? zero : (v.ok ? v.x[i][CODES ? 0 : 1] : zero);
          if constexpr (CODES) x1 = widen8<BF>(x0[2], x0[3]), x0 = widen8<BF>(x0[0], x0[1]);
#pragma unroll
          for (int q = 0; q < RT; q++) {
            f4 t = mfma<BF>(v.w[q][0], x0, CODES ? f4{0.f, 0.f, 0.f, 0.f} : acc[i][q]);
            t = mfma<BF>(v.w[q][1], x1, t);
            if constexpr (CODES) {
              const float f = e8m0_value(v.scale[i]);
#pragma unroll
              for (int e = 0; e < 4; e++) acc[i][q][e] = __builtin_fmaf(t[e], f, acc[i][q][e]);
            } else {
              acc[i][q] = t;
            }
          }
        }
      };
      Step u;
      load(u, first);
#pragma unroll 2
      for (int n = first; n < steps; n += stride) {
        Step v;
        load(v, n + stride);
        multiply(u);
        u = v;
      }
      if (waves > 1) {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int q = 0; q < RT; q++) red[(wave * NT * RT + i * RT + q) * 64 + lane] = acc[i][q];
        __syncthreads();
      }
      int gg = g;
      asm volatile("" : "+v"(gg));
#pragma unroll
      for (int i = 0; i < NT; i++) {
        if (ad.id[i] != ad.current) continue;  // -1 behind the last row
#pragma unroll
        for (int q = 0; q < RT; q++) {
          const int t = i * RT + q, j = ROWS * (group * RT + q) + 4 * gg;
          if (t % waves != wave || j >= SR || j % p.R >= rank) continue;
          f4 v = acc[i][q];
          if (waves > 1) {
            v = red[t * 64 + lane];
            for (int k = 1; k < waves; k++) v += red[(k * NT * RT + t) * 64 + lane];
          }
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] *= scale;
          const int64_t row = row0 + ROWS * i + r;
          if constexpr (JOIN) {
            *(f4*)((float*)p.h + ((size_t)split * p.T + row) * SR + j) = v;
          } else {
            float rest[4] = {v[0], v[1], v[2], v[3]};
            const int slice = j / p.R;
            uint16_t* to = (uint16_t*)p.h + ((size_t)row * p.S + slice) * parts * p.R + (j - slice * p.R);
            for (int k = 0; k < parts; k++) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; e++) w[e] = next_part(rest[e], k == 1 && parts == 2);
              typedef uint32_t u2 __attribute__((ext_vector_type(2)));
              *(u2*)(to + k * p.R) = u2{w[0] | w[1] << 16, w[2] | w[3] << 16};
            }
          }
        }
      }
      if (waves > 1) __syncthreads();
    }
  }
}

// ---- out = y + h B^T: 16 NT rows x 256 columns of one slice per workgroup, 64 columns a wave -------
// A wave's columns of a row are two pieces of 64 bytes in 16-bit types and four in f32.  Matrix tile j has columns such
// that a lane's results are 16 bytes of each piece; the lanes of rows 0 .. 7 and 8 .. 15 of a sixteen then swap pieces,
// so that eight lanes load and store whole lines.
template <int YT>
__device__ __forceinline__ int column(int j, int g, int e) {  // of value e of lane group g in tile j
  return YT == FP8_IO_F32 ? 16 * j + 4 * g + e : 32 * (j / 2) + 8 * g + 4 * (j % 2) + e;
}
// x1 of the lower eight lanes of each sixteen and x0 of the upper eight change places.
__device__ __forceinline__ void swap_eights(u4& x0, u4& x1) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int a = (int)x0[i], b = (int)x1[i];
    x1[i] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false);
    x0[i] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);
  }
}
template <int YT>
__device__ __forceinline__ void add_to(u4& raw, const f4* v) {  // raw += v, rounded once
  if constexpr (YT == FP8_IO_F32) {
    raw = __builtin_bit_cast(u4, __builtin_bit_cast(f4, raw) + v[0]);
  } else {
    typedef _Float16 hh __attribute__((ext_vector_type(2)));
    typedef __bf16 bb __attribute__((ext_vector_type(2)));
    typedef float ff __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t w = raw[e];
      ff x;
      if constexpr (YT == FP8_IO_F16) x = ff{f16_bits_to_f32(w & 0xffffu), f16_bits_to_f32(w >> 16)};
      else x = ff{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
      x[0] += v[e / 2][2 * (e % 2)];
      x[1] += v[e / 2][2 * (e % 2) + 1];
      if constexpr (YT == FP8_IO_F16) raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, hh));
      else raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bb));
    }
  }
}
// Eight f16 weights as two bf16 parts each.
__device__ __forceinline__ void split8(const u4& w, u4& hi, u4& lo) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float a = f16_bits_to_f32(w[e] & 0xffffu), b = f16_bits_to_f32(w[e] >> 16);
    const uint32_t ah = __float_as_uint(a) & 0xffff0000u, bh = __float_as_uint(b) & 0xffff0000u;
    hi[e] = ah >> 16 | bh;
    lo[e] = __float_as_uint(a - __uint_as_float(ah)) >> 16 | (__float_as_uint(b - __uint_as_float(bh)) & 0xffff0000u);
  }
}

// Eight ranks of a row's part, from parts of K that the first product left in f32.
template <int PARTS>
__device__ __forceinline__ void join8(const float* from, int splits, size_t stride, u4 (&part)[PARTS]) {
  f4 a = *(const f4*)from, b = *(const f4*)(from + 4);
#pragma unroll 4
  for (int k = 1; k < splits; k++) a += *(const f4*)(from + k * stride), b += *(const f4*)(from + k * stride + 4);
#pragma unroll
  for (int k = 0; k < PARTS; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float lo = e < 2 ? a[2 * e] : b[2 * e - 4], hi = e < 2 ? a[2 * e + 1] : b[2 * e - 3];
      const bool last = k == 1 && PARTS == 2;
      part[k][e] = next_part(lo, last);
      part[k][e] |= next_part(hi, last) << 16;
      if (e < 2) a[2 * e] = lo, a[2 * e + 1] = hi;
      else b[2 * e - 4] = lo, b[2 * e - 3] = hi;
    }
}

template <int YT, bool BF, int NT, bool JOIN>
__global__ __launch_bounds__(64 * UP_WAVES, (NT == 1) == (YT == FP8_IO_F32) ? 3 : (NT == 1 ? 4 : 2)) void adapter_up_kernel(AdapterArgs p, int splits) {
  constexpr int PARTS = YT == FP8_IO_F32 ? 3 : 2, SIZE = YT == FP8_IO_F32 ? 4 : 2, PAIRS = YT == FP8_IO_F32 ? 2 : 1;
  constexpr int PIECE = 64 / SIZE, COUNT = 16 / SIZE;  // values of a piece, and of a lane in it
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  // this wave's columns
  int s = 0, n0 = 0, c = (int)blockIdx.x;
  while (true) {
    const int t = (p.cols[s] + UP_WAVES * COLS - 1) / (UP_WAVES * COLS);
    if (c < t) break;
    c -= t, n0 += p.cols[s], s++;
  }
  const int end = n0 + p.cols[s];
  n0 += (c * UP_WAVES + wave) * COLS;
  if (n0 >= end) return;
  const int64_t tiles = ((int64_t)p.T + ROWS * NT - 1) / (ROWS * NT);
  const bool in_place = p.y == p.out, upper = r >= 8;
  const int nm = n0 + (upper ? PIECE : 0) + COUNT * g;  // the first column that the lane loads and stores, pairs 32 apart
  for (int64_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
    const int64_t row0 = tile * ROWS * NT;
    Adapters<NT> ad(p, row0);
    u4 y[NT][PAIRS][2];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int m = 0; m < PAIRS; m++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int64_t row = row0 + ROWS * i + (r & 7) + 8 * k;
          const int n = nm + 32 * m < end ? nm + 32 * m : n0;
          y[i][m][k] = *(const u4*)((const char*)p.y + (min(row, (int64_t)p.T - 1) * p.ldy + n) * SIZE);
        }
    // stores the rows of adapter `which`, -1: those of none
    const auto store = [&](int i, int which) {
      int column = nm;  // opaque, so that no address is held from before
      asm volatile("" : "+v"(column));
      const int other = __builtin_amdgcn_update_dpp(0, ad.id[i], 0x128, 0xf, 0xf, false);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int64_t row = row0 + ROWS * i + (r & 7) + 8 * k;
        if (((k == 1) == upper ? ad.id[i] : other) != which || row >= p.T) continue;
#pragma unroll
        for (int m = 0; m < PAIRS; m++)
          if (column + 32 * m < end) *(u4*)((char*)p.out + (row * p.ldo + column + 32 * m) * SIZE) = y[i][m][k];
      }
    };
    if (!in_place && (!JOIN || blockIdx.z == 0)) {
#pragma unroll
      for (int i = 0; i < NT; i++) store(i, -1);
    }
    if (JOIN) ad.only((int)blockIdx.z);
    while (ad.next()) {
      const int rank = rank_of(p, ad.current);
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
#pragma unroll 1
      for (int r0 = 0; r0 < p.R; r0 += 32) {
        // this lane's eight ranks, loaded where they are the matrix's and counted where they are the adapter's: the
        // loads do not wait for its rank
        const int at = r0 + 8 * g < p.R ? r0 + 8 * g : 0;
        const u4 zero = u4{0, 0, 0, 0};
        u4 w[4], lo[4], v[NT][PARTS];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = *(const u4*)(brow[j] + at);
#pragma unroll
        for (int i = 0; i < NT; i++) {
          const size_t row = ad.source(i);
          if constexpr (JOIN) {
            join8<PARTS>((const float*)p.h + row * p.S * p.R + s * p.R + at, splits, (size_t)p.T * p.S * p.R, v[i]);
          } else {
            const uint16_t* from = (const uint16_t*)p.h + (row * p.S + s) * PARTS * p.R + at;
#pragma unroll
            for (int k = 0; k < PARTS; k++) v[i][k] = *(const u4*)(from + k * p.R);
          }
        }
        if (r0 >= rank) break;
        const bool ok = r0 + 8 * g < rank;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          w[j] = ok ? w[j] : zero;
          if constexpr (!BF) {
            const u4 x = w[j];
            split8(x, w[j], lo[j]);
          }
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int k = 0; k < PARTS; k++) {
            const u4 x = ok ? v[i][k] : zero;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              acc[i][j] = mfma<true>(w[j], x, acc[i][j]);
              if constexpr (!BF) acc[i][j] = mfma<true>(lo[j], x, acc[i][j]);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < NT; i++) {
        const int other = __builtin_amdgcn_update_dpp(0, ad.id[i], 0x128, 0xf, 0xf, false);
#pragma unroll
        for (int m = 0; m < PAIRS; m++) {
          u4 a = y[i][m][0], b = y[i][m][1];
          swap_eights(a, b);
          add_to<YT>(a, &acc[i][YT == FP8_IO_F32 ? 2 * m : 0]);
          add_to<YT>(b, &acc[i][YT == FP8_IO_F32 ? 2 * m + 1 : 2]);
          swap_eights(a, b);
          // another adapter's rows keep theirs
          if ((upper ? other : ad.id[i]) == ad.current) y[i][m][0] = a;
          if ((upper ? ad.id[i] : other) == ad.current) y[i][m][1] = b;
        }
        store(i, ad.current);
      }
    }
  }
}

// How a call is cut up.
struct Plan {
  bool join;       // few rows: one of a sixteen's adapters to a workgroup, K split over workgroups
  int splits;      // parts of K of different workgroups
  int waves;       // of a workgroup, on parts of K
  int down, up;    // sixteens of rows of a workgroup
  int ranks;       // sixteens of ranks of a workgroup
};
Plan plan_of(int T, int K, int SR, int up_blocks) {
  Plan q{};
  const int steps = (K + STEP - 1) / STEP, tiles = (SR + ROWS - 1) / ROWS;
  const int64_t sixteens = ((int64_t)T + ROWS - 1) / ROWS;
  q.join = T <= 256;
  if (q.join) {
    q.waves = std::min(8, steps);
    q.splits = std::min((steps + q.waves - 1) / q.waves, 8);
    q.down = q.up = q.ranks = 1;
    return q;
  }
  q.splits = 1;
  q.ranks = std::min(tiles, 4);
  const int groups = (tiles + q.ranks - 1) / q.ranks;
  q.down = sixteens >= 4 * 1024 ? 4 : 2;
  q.waves = 1;
  while (q.waves < DOWN_WAVES && 2 * q.waves <= steps && sixteens / q.down * groups * q.waves < 4096) q.waves *= 2;
  q.up = sixteens * up_blocks >= 2 * 1024 ? 2 : 1;
  return q;
}

template <bool CODES, bool BF, int NT, int RT, bool JOIN>
hipError_t launch_down(const AdapterArgs& a, const Plan& q, hipStream_t s) {
  const int tiles = (a.S * a.R + ROWS - 1) / ROWS, groups = (tiles + RT - 1) / RT;
  const int64_t rows = ((int64_t)a.T + ROWS * NT - 1) / (ROWS * NT);
  const dim3 grid((unsigned)std::min<int64_t>(rows, 1 << 20), (unsigned)(groups * q.splits), JOIN ? std::min(ROWS, a.T) : 1);
  const size_t lds = q.waves > 1 ? (size_t)q.waves * NT * RT * 64 * sizeof(f4) : 0;
  T5K_LAUNCH((adapter_down_kernel<CODES, BF, NT, RT, JOIN>), grid, dim3(64 * q.waves), lds, s, a, q.splits, a.y_type == FP8_IO_F32 ? 3 : 2);
  return hipGetLastError();
}
template <bool CODES, bool BF, int NT>
hipError_t launch_down_ranks(const AdapterArgs& a, const Plan& q, hipStream_t s) {
  switch (q.ranks) {
    case 1: return launch_down<CODES, BF, NT, 1, false>(a, q, s);
    case 2: return launch_down<CODES, BF, NT, 2, false>(a, q, s);
    case 3: return launch_down<CODES, BF, NT, 3, false>(a, q, s);
  }
  return launch_down<CODES, BF, NT, 4, false>(a, q, s);
}
template <bool CODES, bool BF>
hipError_t launch_down_plan(const AdapterArgs& a, const Plan& q, hipStream_t s) {
  if (q.join) return launch_down<CODES, BF, 1, 1, true>(a, q, s);
  return q.down == 4 ? launch_down_ranks<CODES, BF, 4>(a, q, s) : launch_down_ranks<CODES, BF, 2>(a, q, s);
}

template <int YT, bool BF>
hipError_t launch_up(const AdapterArgs& a, const Plan& q, int blocks, hipStream_t s) {
  const int64_t sixteens = ((int64_t)a.T + ROWS - 1) / ROWS;
  const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>((sixteens + q.up - 1) / q.up, 65535), q.join ? std::min(ROWS, a.T) : 1);
  if (q.join) T5K_LAUNCH((adapter_up_kernel<YT, BF, 1, true>), grid, dim3(64 * UP_WAVES), 0, s, a, q.splits);
  else if (q.up == 2) T5K_LAUNCH((adapter_up_kernel<YT, BF, 2, false>), grid, dim3(64 * UP_WAVES), 0, s, a, 1);
  else T5K_LAUNCH((adapter_up_kernel<YT, BF, 1, false>), grid, dim3(64 * UP_WAVES), 0, s, a, 1);
  return hipGetLastError();
}
template <bool BF>
hipError_t launch(const AdapterArgs& a, hipStream_t s) {
  int blocks = 0;
  for (int i = 0; i < a.S; i++) blocks += (a.cols[i] + UP_WAVES * COLS - 1) / (UP_WAVES * COLS);
  const Plan q = plan_of(a.T, a.K, a.S * a.R, blocks);
  const hipError_t e = a.x_type == ADAPTER_E4M3 ? launch_down_plan<true, BF>(a, q, s) : launch_down_plan<false, BF>(a, q, s);
  if (e != hipSuccess) return e;
  switch (a.y_type) {
    case FP8_IO_F32: return launch_up<FP8_IO_F32, BF>(a, q, blocks, s);
    case FP8_IO_F16: return launch_up<FP8_IO_F16, BF>(a, q, blocks, s);
    case FP8_IO_BF16: return launch_up<FP8_IO_BF16, BF>(a, q, blocks, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace

namespace t5k {
size_t adapter_work_bytes(int T, int K, int SR) {
  const Plan q = plan_of(T, K, SR, 1);
  return (size_t)T * SR * (q.join ? 4 * (size_t)q.splits : 6);
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
