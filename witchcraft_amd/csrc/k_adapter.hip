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
// (within 2^-16 of h, where the results' own rounding is 2^-8 or 2^-11).  The third would show where y cancels the
// adapter's share, and in one of 50 f16 results elsewhere by a step; it costs 1 to 4% with up to 32 ranks (74,640 rows of
// codes 186 and 193 us) and 8 to 16% with more (16,391 x 4,096 -> 8,192, rank 64, bf16: 167 and 193), so 16-bit results go
// without.  bf16 has f32's range, which f16 has not; f16 weights go in as two bf16 parts, which hold their 11 bits; where
// the second is zero, an infinite h makes NaN of it.
#include "adapter.hpp"

#include <algorithm>

#include "fp8.hpp"
#include "lds_copy.hpp"

namespace {
using namespace t5k;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int ROWS = 16;        // of a matrix instruction
constexpr int FEW_STEP = 64;    // K values of a step of the first product for few rows
constexpr int FEW_WAVES = 8;    // its waves, at most
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
      const int v = p.ids[min(row, (int64_t)p.T - 1)];
      id[i] = row < p.T && (unsigned)v < (unsigned)p.G ? v : -1;
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

// The adapter's rank as it is given: inner products past it are zeros.  And (the same in all lanes) rounded up to whole
// eights: what the second product takes of them and of B.
__device__ __forceinline__ int given_rank(const AdapterArgs& p, int g) { return p.ranks ? p.ranks[g] : p.R; }
__device__ __forceinline__ int whole_rank(const AdapterArgs& p, int given) {
  const int r = __builtin_amdgcn_readfirstlane(given);
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

// Where the parts of h lie, in the second product's operand order: for each sixteen of rows, slice, part and eight of
// ranks 16 rows of 16 bytes, so that its lanes read consecutive ones.  Behind the last row up to a sixteen.
__device__ __forceinline__ size_t h_index(int64_t row, int slice, int part, int rank, int S, int parts, int R) {
  return ((((size_t)(row / ROWS) * S + slice) * parts + part) * (R / 8) + rank / 8) * (ROWS * 8) + (row % ROWS) * 8 + rank % 8;
}

// ---- h = scale x A^T, few rows: 16 rows x 16 ranks per workgroup, its waves on 64 K values in turn ----
// Lane (r = lane % 16, g = lane / 16) holds row r's K values 16 g .. + 15 of a step, the next step's are on their way
// while one is multiplied.  The waves' sums meet in LDS and are added in wave order.  Workgroups split K further, and
// leave their sums in f32 for the second product to add; each takes one adapter of the sixteen rows.  Bound by the launch
// and two trips to memory, ids and then rows: one row of 4,096 against 16 ranks 4.1 us, 64 rows of 64 adapters (8.4 MB) 5.2.
template <bool CODES>
struct FewStep {
  u4 w[2], x[CODES ? 1 : 2];
  uint32_t scale;
  bool ok;
};
template <bool CODES, bool BF>
__global__ __launch_bounds__(64 * FEW_WAVES) void adapter_down_few_kernel(AdapterArgs p, int splits) {
  __shared__ f4 red[FEW_WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int SR = p.S * p.R, steps = (p.K + FEW_STEP - 1) / FEW_STEP, waves = (int)(blockDim.x >> 6);
  const int split = (int)blockIdx.y % splits, group = (int)blockIdx.y / splits;
  const size_t m16 = fp8_scale_rows(p.T);
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  Adapters<1> ad(p, row0);
  ad.only((int)blockIdx.z);
  if (!ad.next()) return;
  const float scale = p.scales ? p.scales[ad.current] : 1.f;
  const int j0 = ROWS * group, given = given_rank(p, ad.current);
  const int64_t at = ad.source(0);
  const uint16_t* arow = (const uint16_t*)p.a + ((size_t)ad.current * SR + min(j0 + r, SR - 1)) * p.K;
  // loads are unconditional, past the rows' end from their start
  const auto load = [&](FewStep<CODES>& v, int n) {
    const int k0 = n * FEW_STEP + 16 * g, k = k0 < p.K ? k0 : 0;
    const int block = min(n, steps - 1) / (FP8_BLOCK / FEW_STEP);  // of the scales: the same for all lanes
    if constexpr (CODES) {
      v.x[0] = *(const u4*)((const uint8_t*)p.x + at * p.ldx + k);
      v.scale = p.x_scales[(size_t)block * m16 + at];
    } else {
      const uint16_t* from = (const uint16_t*)p.x + at * p.ldx + k;
      v.x[0] = *(const u4*)from;
      v.x[1] = *(const u4*)(from + 8);
    }
    v.w[0] = *(const u4*)(arow + k);
    v.w[1] = *(const u4*)(arow + k + 8);
    v.ok = k0 < p.K;
  };
  f4 acc = f4{0.f, 0.f, 0.f, 0.f};
  FewStep<CODES> u;
  load(u, split * waves + wave);
#pragma unroll 2
  for (int n = split * waves + wave; n < steps; n += splits * waves) {
    FewStep<CODES> v;
    load(v, n + splits * waves);
    const u4 zero = u4{0, 0, 0, 0};
    const u4 x = u.ok ? u.x[0] : zero;
    if constexpr (CODES) {
      f4 t = mfma<BF>(u.w[0], widen8<BF>(x[0], x[1]), f4{0.f, 0.f, 0.f, 0.f});
      t = mfma<BF>(u.w[1], widen8<BF>(x[2], x[3]), t);
      const float f = e8m0_value(u.scale);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(t[e], f, acc[e]);
    } else {
      acc = mfma<BF>(u.w[0], x, acc);
      acc = mfma<BF>(u.w[1], u.ok ? u.x[CODES ? 0 : 1] : zero, acc);
    }
    u = v;
  }
  red[wave][lane] = acc;
  __syncthreads();
  const int j = j0 + 4 * g;
  if (wave != 0 || ad.id[0] != ad.current || j >= SR) return;
  for (int k = 1; k < waves; k++) acc += red[k][lane];
  // values past the adapter's rank may come from anything
#pragma unroll
  for (int e = 0; e < 4; e++) acc[e] = j % p.R + e < given ? acc[e] * scale : 0.f;
  *(f4*)((float*)p.h + ((size_t)split * p.T + row0 + r) * SR + j) = acc;
}

// ---- h = scale x A^T, many rows: 16 RG rows x 16 RT ranks per workgroup ------------------------------
// Steps of 128 bytes of x's rows (64 values, or 128 codes) go through a ring of STAGES in LDS: copies in whole rows,
// eight of 128 bytes to an instruction, straight from memory.  A row's eight 16-byte chunks are stored rotated (xor) by
// its number, so that eight rows' same chunk, which a read takes at a time, lie in different banks.  Four waves: RG
// sixteens of rows, the ranks in 4 / RG parts.  A wait and a barrier per step: step n has been requested STAGES - 1 ahead.
// Chunks past K, and steps past the last, are copied from outside the descriptors' range, as zeros.  Bound by the way
// through LDS and the wait for a step where rows are few (4,616 of 768: 8.7 us), by memory where they are many
// (16,391 of 4,096 against 64 ranks: 51 us, 2.6 TB/s; 74,640 of 768 codes: 39).
template <bool CODES, int RT, int RG>
struct Ring {
  static constexpr int ROW_COPIES = RG / 2, HALVES = CODES ? 2 : 1;  // of a wave; pieces of 128 bytes of A's rows
  static constexpr int ROW_BYTES = RG * ROWS * 128, A_BYTES = HALVES * RT * ROWS * 128, A_COPIES = A_BYTES / 1024;  // of four waves
  // behind them the scales of codes, one copy a wave, or room for the copies of waves that have none of A's
  static constexpr int REST = CODES ? 4 * 256 : (A_COPIES % 4 ? 1024 : 0);
  static constexpr int STAGE = ROW_BYTES + A_BYTES + REST;
  // three where they leave room for two workgroups on a compute unit and more: 4,096 rows of 64 ranks 66 us, with two
  // stages 86; larger ones take 145 us with three, 122 with two (three slices' codes)
  static constexpr int STAGES = STAGE <= 16384 ? 3 : 2;
  static constexpr int COPIES = ROW_COPIES + (A_COPIES + 3) / 4 + (CODES ? 1 : 0);  // of a wave, the same for all
};
template <bool CODES, bool BF, int RT, int RG>
__global__ __launch_bounds__(256, 2) void adapter_down_kernel(AdapterArgs p, int parts) {
  typedef Ring<CODES, RT, RG> Lds;
  __shared__ __attribute__((aligned(1024))) char lds[Lds::STAGES * Lds::STAGE];
  constexpr int SIZE = CODES ? 1 : 2, K_STEP = 128 / SIZE, STAGES = Lds::STAGES, RQ = RT * RG / 4;  // RQ: sixteens of ranks of a wave
  static_assert(RG == 4 || (RG == 2 && RT % 2 == 0), "whole sixteens of ranks for each wave");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int rw = wave % RG, q0 = wave / RG * RQ;
  const int SR = p.S * p.R, steps = (p.K + K_STEP - 1) / K_STEP, group = (int)blockIdx.y;
  const size_t m16 = fp8_scale_rows(p.T);
  const int64_t tiles = ((int64_t)p.T + RG * ROWS - 1) / (RG * ROWS);
  const uint32_t lds0 = lds_offset(lds);
  const int cr = lane >> 3, cc = (lane & 7) ^ cr;  // the row of eight and the chunk that the lane copies
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row0 = tile * RG * ROWS;
    const int rows = (int)min((int64_t)RG * ROWS, p.T - row0);
    Adapters<RG> ad(p, row0);
    for (unsigned seen = 0; ad.next(); seen++) {
      if (seen % gridDim.z != blockIdx.z) continue;
      const float scale = p.scales ? p.scales[ad.current] : 1.f;
      const int given = given_rank(p, ad.current);
      const int id0 = ad.id[0], id1 = ad.id[1], id2 = ad.id[RG - 2], id3 = ad.id[RG - 1];
      const auto id_of = [&](int i) { return i == 0 ? id0 : (i == 1 ? id1 : (i == 2 ? id2 : id3)); };  // of the i-th sixteen
      const int id = id_of(rw);
      const int64_t row = row0 + ROWS * rw + r;
      // This wave's copies: eights of rows of x (in the place of those whose result nothing keeps, one that is
      // copied anyway), and pieces 4 i + wave of A: eight ranks, codes: of one half of a step.  A wave without one copies zeros
      // behind the last.
      const i4v x_at = buffer_at((const char*)p.x + row0 * p.ldx * SIZE, (uint32_t)((rows - 1) * p.ldx + p.K) * SIZE);
      const int j0 = ROWS * RT * group, ranks = min(ROWS * RT, SR - j0);
      const i4v a_at = buffer_at((const uint16_t*)p.a + ((size_t)ad.current * SR + j0) * p.K, (uint32_t)ranks * p.K * 2);
      const i4v s_at = buffer_at(CODES ? (const void*)p.x_scales : p.x, CODES ? (uint32_t)(steps * m16) : 0u);
      uint32_t x_off[Lds::ROW_COPIES], a_off[(Lds::A_COPIES + 3) / 4];
#pragma unroll
      for (int i = 0; i < Lds::ROW_COPIES; i++) {
        const int eight = Lds::ROW_COPIES * wave + i, at = 8 * eight + cr;
        const int other = __builtin_amdgcn_ds_bpermute(4 * (at % ROWS), id_of(eight / 2));
        const int from = other == ad.current ? at : (int)(ad.row - row0);
        x_off[i] = (uint32_t)(from * p.ldx * SIZE) + 16 * cc;
      }
#pragma unroll
      for (int i = 0; i < (Lds::A_COPIES + 3) / 4; i++) {
        const int c = 4 * i + wave, half = c / (2 * RT), j = c % (2 * RT) * 8 + cr;
        a_off[i] = c < Lds::A_COPIES && j < ranks ? (uint32_t)(j * p.K + 64 * half + 8 * cc) * 2 : kOutside;
      }
      const uint32_t s_off = lane < 4 ? (uint32_t)(row0 + ROWS * wave + 4 * lane) : kOutside;
      // Workgroups begin at different steps: with all at the same one the 32 compute units of an XCD, whose workgroups are
      // every eighth, want the same few lines of A at a time (16,391 rows of 4,096: 169 us for both products, 165 so).
      const int shift = (int)((tile / 8) % steps);
      const auto copy = [&](int at) {
        const int n = at + shift - (at + shift >= steps ? steps : 0);
        const uint32_t stage = lds0 + (uint32_t)(at % STAGES) * Lds::STAGE;
        const int left = at < steps ? p.K - n * K_STEP : 0;  // values of this step
        const uint32_t soff = (uint32_t)n * 128;
#pragma unroll
        for (int i = 0; i < Lds::ROW_COPIES; i++)
          lds_copy16(x_at, cc * (16 / SIZE) < left ? x_off[i] : kOutside, soff, stage + (Lds::ROW_COPIES * wave + i) * 1024);
#pragma unroll
        for (int i = 0; i < (Lds::A_COPIES + 3) / 4; i++) {
          const int c = 4 * i + wave, half = c / (2 * RT);
          lds_copy16(a_at, 64 * half + 8 * cc < left ? a_off[i] : kOutside, soff * Lds::HALVES,
                     stage + Lds::ROW_BYTES + min(c, (int)Lds::A_COPIES) * 1024);
        }
        if constexpr (CODES) lds_copy4(s_at, left > 0 ? s_off : kOutside, (uint32_t)(n * m16), stage + Lds::ROW_BYTES + Lds::A_BYTES + wave * 256);
      };
      f4 acc[RQ];
#pragma unroll
      for (int q = 0; q < RQ; q++) acc[q] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < STAGES - 1; i++) copy(i);
#pragma unroll 1
      for (int n = 0; n < steps; n++) {
        // this step's stage is whole, and the last one's has been read by all
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * Lds::COPIES) : "memory");
        copy(n + STAGES - 1);
        const char* stage = lds + n % STAGES * Lds::STAGE;
        const char* xs = stage + (ROWS * rw + r) * 128;
        const char* as = stage + Lds::ROW_BYTES + (ROWS * q0 + r) * 128;
        u4 x[CODES ? 4 : 2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const u4 c = *(const u4*)(xs + (((g + 4 * e) ^ r) & 7) * 16);
          if constexpr (CODES) x[2 * e] = widen8<BF>(c[0], c[1]), x[2 * e + 1] = widen8<BF>(c[2], c[3]);
          else x[e] = c;
        }
        const float f = CODES ? e8m0_value((uint8_t)stage[Lds::ROW_BYTES + Lds::A_BYTES + rw * 256 + r]) : 1.f;
#pragma unroll
        for (int q = 0; q < RQ; q++) {
          f4 t = CODES ? f4{0.f, 0.f, 0.f, 0.f} : acc[q];
#pragma unroll
          for (int e = 0; e < (CODES ? 4 : 2); e++) {
            // the chunk with the same K values, of which codes have two in one of x's
            const int c = CODES ? 2 * g + e % 2 : g + 4 * e, half = CODES ? e / 2 : 0;
            t = mfma<BF>(*(const u4*)(as + (half * RT + q) * ROWS * 128 + ((c ^ r) & 7) * 16), x[e], t);
          }
          if constexpr (CODES) {
#pragma unroll
            for (int e = 0; e < 4; e++) acc[q][e] = __builtin_fmaf(t[e], f, acc[q][e]);
          } else {
            acc[q] = t;
          }
        }
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the ring is free
      int gg = g;
      asm volatile("" : "+v"(gg));           // the addresses of results are left to be computed here
      if (id == ad.current) {  // -1 behind the last row
#pragma unroll
        for (int q = 0; q < RQ; q++) {
          const int j = j0 + ROWS * (q0 + q) + 4 * gg;
          if (j >= SR) continue;
          const f4 v = acc[q];
          const int slice = j / p.R, at_rank = j - slice * p.R;
          float rest[4];  // values past the adapter's rank may come from anything
#pragma unroll
          for (int e = 0; e < 4; e++) rest[e] = at_rank + e < given ? v[e] * scale : 0.f;
          uint16_t* to = (uint16_t*)p.h + h_index(row, slice, 0, at_rank, p.S, parts, p.R);
          for (int k = 0; k < parts; k++) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = next_part(rest[e], k == 1 && parts == 2);
            *(u2*)(to + k * p.R * ROWS) = u2{w[0] | w[1] << 16, w[2] | w[3] << 16};
          }
        }
      }
    }
  }
}

// ---- out = y + h B^T: 16 rows x 64 columns of one slice per wave and turn, four waves side by side --------
// A wave loads and stores y in whole rows, eight of 128 bytes or four of 256 to an instruction, lane after lane: with
// lanes in the matrix units' order, sixteen rows in turn, the address unit takes four times as long.  The products
// therefore change lanes, through LDS: rows of f32, 16 bytes apart in their banks.
// raw (16 bytes of y) += v (as many values as it has), rounded once.
template <int YT>
__device__ __forceinline__ u4 add_to(const u4& raw, const f4& v0, const f4& v1) {
  if constexpr (YT == FP8_IO_F32) {
    return __builtin_bit_cast(u4, __builtin_bit_cast(f4, raw) + v0);
  } else {
    typedef _Float16 hh __attribute__((ext_vector_type(2)));
    typedef __bf16 bb __attribute__((ext_vector_type(2)));
    typedef float ff __attribute__((ext_vector_type(2)));
    u4 out;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t w = raw[e];
      ff x;
      if constexpr (YT == FP8_IO_F16) x = ff{f16_bits_to_f32(w & 0xffffu), f16_bits_to_f32(w >> 16)};
      else x = ff{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
      x[0] += e < 2 ? v0[2 * e] : v1[2 * e - 4];
      x[1] += e < 2 ? v0[2 * e + 1] : v1[2 * e - 3];
      if constexpr (YT == FP8_IO_F16) out[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, hh));
      else out[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bb));
    }
    return out;
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

// Three forms: SHORT, ranks up to 16, where the matrix unit's 32 hold a row's parts one after the other; otherwise STEPS
// times 32 ranks for each part; JOIN, few rows, one sixteen and one of its adapters.  Except there, a wave walks sixteens
// of rows, the next one on its way while one is taken (two gain nothing), and loads weights where the adapter changes.
// Bound by the reads and writes of y: 74,640 rows of 2,304 columns
// 152 us (4.5 TB/s), 16,391 of 8,192 118 us (4.5 TB/s); 4,616 of 2,304 15 us (2.8 TB/s), of which sixteens with two
// adapters and the wait for weights behind them are 4.  JOIN: one row of 4,096 columns 4.6 us, 64 of 64 adapters 7.0.
enum UpForm : int { SHORT = 0, JOIN = -1 };  // else STEPS
// 64 columns are a whole line of y; f32 results from f16 weights of more than 64 ranks have registers for 32
constexpr int up_columns(int YT, bool BF, int FORM) { return FORM == 4 && !BF && YT == FP8_IO_F32 ? 32 : 64; }  // of a wave
constexpr int up_occupancy(int YT, bool BF, int FORM) {  // waves a SIMD
  if (YT == FP8_IO_F32) return FORM <= 0 || (FORM == 1 && BF) || up_columns(YT, BF, FORM) == 32 ? 3 : 2;
  return FORM == JOIN || (FORM == SHORT && BF) ? 4 : (FORM <= 1 || BF ? 3 : 2);
}
template <int YT, bool BF, int FORM>
__global__ __launch_bounds__(64 * UP_WAVES, up_occupancy(YT, BF, FORM)) void adapter_up_kernel(AdapterArgs p, int splits, int run) {
  constexpr int PARTS = YT == FP8_IO_F32 ? 3 : 2, SIZE = YT == FP8_IO_F32 ? 4 : 2;
  constexpr int COLS = up_columns(YT, BF, FORM), NJ = COLS / 16, PITCH = COLS + 4;
  constexpr int COUNT = 16 / SIZE, LANES = COLS / COUNT, STRIDE = 64 / LANES, PIECES = ROWS / STRIDE;
  constexpr int STEPS = FORM > 0 ? FORM : 1;
  constexpr int TURNS = YT == FP8_IO_F32 ? 2 : 1;  // SHORT: of four eights of ranks
  constexpr int EARLY = FORM == SHORT ? TURNS : (FORM == 1 || FORM == 2 ? FORM * PARTS : 0);  // pieces of h that come with y
  constexpr bool APART = !BF && FORM >= 0;  // f16 weights are kept as their parts
  __shared__ f4 stage_all[UP_WAVES][ROWS * PITCH / 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  float* stage = (float*)stage_all[wave];
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
  const int64_t tiles = ((int64_t)p.T + ROWS - 1) / ROWS;
  const bool in_place = p.y == p.out;
  // what the lane loads and stores: 16 bytes at column lc of rows lr, lr + STRIDE, ..; past the columns' end the first
  // ones are loaded.  Rows of a sixteen lie within 2^30 bytes.
  const int lr = lane / LANES, lc = COUNT * (lane % LANES);
  const bool inside = n0 + lc < end;
  const uint32_t column = (inside ? lc : 0) * SIZE, pitch_y = (uint32_t)p.ldy * SIZE, pitch_out = (uint32_t)p.ldo * SIZE;
  const u4 zero = u4{0, 0, 0, 0};
  const int eights = p.R / 8;  // SHORT: 1 or 2
  const int short_at = eights == 1 ? 0 : 8 * (g & 1);
  struct Tile {
    u4 y[PIECES], v[EARLY ? EARLY : 1];
  };
  const auto last_of = [&](int64_t tile) { return (int)min((int64_t)ROWS - 1, (int64_t)p.T - 1 - tile * ROWS); };  // its last row
  // loads are unconditional, behind the last row from it
  const auto load = [&](Tile& x, int64_t tile) {
    const int last = last_of(tile);
    const char* y = (const char*)p.y + (tile * ROWS * p.ldy + n0) * SIZE;
#pragma unroll
    for (int k = 0; k < PIECES; k++) x.y[k] = *(const u4*)(y + ((uint32_t)min(lr + STRIDE * k, last) * pitch_y + column));
    if constexpr (EARLY > 0) {
      const char* h = (const char*)p.h + 2 * h_index(tile * ROWS, s, 0, 0, p.S, PARTS, p.R);
#pragma unroll
      for (int k = 0; k < EARLY; k++) {
        // SHORT: piece 4 k + g of all; otherwise ranks 32 (k / PARTS) + 8 g of part k % PARTS
        const int rank0 = FORM == SHORT ? 8 * (4 * k + g) : 32 * (k / PARTS) + 8 * g;
        const int at = FORM == SHORT ? (rank0 < PARTS * p.R ? rank0 : 0) : (rank0 < p.R ? rank0 : 0) + k % PARTS * p.R;
        x.v[k] = *(const u4*)(h + (uint32_t)(at * ROWS + r * 8) * 2);
      }
    }
  };
  const auto id_of = [&](int64_t tile) {  // of row r, -1 without an adapter
    const int last = last_of(tile), v = p.ids[tile * ROWS + min(r, last)];
    return r <= last && (unsigned)v < (unsigned)p.G ? v : -1;
  };
  const auto store = [&](int64_t tile, int k, const u4& v) {
    char* out = (char*)p.out + (tile * ROWS * p.ldo + n0) * SIZE;
    if (lr + STRIDE * k <= last_of(tile) && inside) *(u4*)(out + ((uint32_t)(lr + STRIDE * k) * pitch_out + column)) = v;
  };
  const auto row_id = [&](int id, int k) { return __builtin_amdgcn_ds_bpermute(4 * (lr + STRIDE * k), id); };  // of a stored row
  const auto store_none = [&](const Tile& x, int64_t tile, int id) {
#pragma unroll
    for (int k = 0; k < PIECES; k++)
      if (row_id(id, k) == -1) store(tile, k, x.y[k]);
  };
  const auto weights = [&](u4 (&v)[NJ], int current, int at) {  // of ranks at .. + 7
    int first = n0 + r;
    asm volatile("" : "+v"(first));  // no address is held from before
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int n = min(first + 16 * j, end - 1);
      v[j] = *(const u4*)((const uint16_t*)p.b + ((size_t)current * p.N + n) * p.R + (at < p.R ? at : 0));
    }
  };
  const auto apart = [&](const u4 (&f)[NJ], u4 (&hi)[NJ], u4 (&low)[NJ]) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      if constexpr (BF) hi[j] = f[j];
      else split8(f[j], hi[j], low[j]);
    }
  };
  const auto multiply = [&](f4 (&acc)[NJ], const u4 (&hi)[NJ], const u4 (&low)[NJ], const u4& v) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      acc[j] = mfma<true>(hi[j], v, acc[j]);
      if constexpr (!BF) acc[j] = mfma<true>(low[j], v, acc[j]);
    }
  };
  // y and the products, in the order of memory, and the rows of adapter `current`
  const auto finish = [&](const f4 (&acc)[NJ], const Tile& x, int64_t tile, int id, int current) {
#pragma unroll
    for (int j = 0; j < NJ; j++) *(f4*)(stage + r * PITCH + 16 * j + 4 * g) = acc[j];
    // the wave's own region: its lanes' writes come before its reads, and these before the next writes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
      const float* from = stage + (lr + STRIDE * k) * PITCH + lc;
      const f4 v0 = *(const f4*)from, v1 = *(const f4*)(from + (COUNT > 4 ? 4 : 0));
      if (row_id(id, k) == current) store(tile, k, add_to<YT>(x.y[k], v0, v1));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // Values behind the last part or the adapter's rank count as zeros, like the weights' there: an infinity times zero
  // would be NaN.
  if constexpr (FORM == JOIN) {
    const int64_t tile = blockIdx.y;
    Tile x;
    load(x, tile);
    Adapters<1> ad(p, tile * ROWS);
    if (!in_place && blockIdx.z == 0) store_none(x, tile, ad.id[0]);
    ad.only((int)blockIdx.z);
    if (!ad.next()) return;
    const int rank = whole_rank(p, given_rank(p, ad.current));
    const int64_t row = ad.source(0);
    f4 acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int t = 0; 32 * t < p.R; t++) {
      const int at = 32 * t + 8 * g;
      u4 w[NJ], v[PARTS], hi[NJ], low[NJ];
      weights(w, ad.current, at);
      join8<PARTS>((const float*)p.h + (size_t)row * p.S * p.R + s * p.R + (at < p.R ? at : 0), splits, (size_t)p.T * p.S * p.R, v);
#pragma unroll
      for (int j = 0; j < NJ; j++) w[j] = at < rank ? w[j] : zero;
      apart(w, hi, low);
#pragma unroll
      for (int k = 0; k < PARTS; k++) multiply(acc, hi, low, at < rank ? v[k] : zero);
    }
    finish(acc, x, tile, ad.id[0], ad.current);
  } else {
    for (int64_t first = (int64_t)blockIdx.y * run; first < tiles; first += (int64_t)gridDim.y * run) {
      const int64_t stop = min(first + run, tiles);
      // the first adapter that rows of `id` wait for, -1: none
      const auto waiting = [&](int id) {
        const uint64_t m = __ballot(id >= 0);
        return m ? __builtin_amdgcn_readlane(id, __builtin_ctzll(m)) : -1;
      };
      Tile x, x1;
      int64_t tile = first;
      int id = id_of(tile), left = id, next_id = id_of(min(tile + 1, stop - 1));  // left: of rows not yet taken
      load(x, tile);
      bool fresh = true;  // rows without an adapter are yet to come
      while (tile < stop) {
        const int current = waiting(left);
        int rank = 0;
        u4 w[STEPS][NJ], lo[APART ? STEPS : 1][NJ];
        if (current >= 0) {
#pragma unroll
          for (int t = 0; t < STEPS; t++) weights(w[t], current, FORM == SHORT ? short_at : 32 * t + 8 * g);
          rank = whole_rank(p, given_rank(p, current));
#pragma unroll
          for (int t = 0; t < STEPS; t++)
#pragma unroll
            for (int j = 0; j < NJ; j++) {
              w[t][j] = (FORM == SHORT ? short_at : 32 * t + 8 * g) < rank ? w[t][j] : zero;
              if constexpr (APART) {
                const u4 f = w[t][j];
                split8(f, w[t][j], lo[t][j]);
              }
            }
        }
        // Takes the sixteen in `now` for the current adapter, the next one on its way to `later`.  False: another
        // adapter's turn, in the same sixteen (`same`) or in the next.
        bool same = false;
        const auto take = [&](const Tile& now, Tile& later) {
          const int later_id = id_of(min(tile + 2, stop - 1));
          load(later, min(tile + 1, stop - 1));
          if (!in_place && fresh) store_none(now, tile, id);
          if (current >= 0) {
            f4 acc[NJ];
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
            if constexpr (FORM == SHORT) {
#pragma unroll
              for (int t = 0; t < TURNS; t++)
                multiply(acc, w[0], lo[0], 4 * t + g < PARTS * eights && short_at < rank ? now.v[t] : zero);
            } else {
#pragma unroll
              for (int t = 0; t < STEPS; t++) {
                const int at = 32 * t + 8 * g;
                u4 v[PARTS];
                const char* from = (const char*)p.h + 2 * h_index(tile * ROWS, s, 0, 0, p.S, PARTS, p.R);
#pragma unroll
                for (int k = 0; k < PARTS; k++)
                  v[k] = EARLY ? now.v[EARLY ? PARTS * t + k : 0]
                               : *(const u4*)(from + (uint32_t)(((at < p.R ? at : 0) + k * p.R) * ROWS + r * 8) * 2);
#pragma unroll
                for (int k = 0; k < PARTS; k++) {
                  const u4 u = at < rank ? v[k] : zero;
                  multiply(acc, w[t], lo[APART ? t : 0], u);
                }
              }
            }
            finish(acc, now, tile, id, current);
            left = left == current ? -1 : left;
          }
          if (current >= 0 && waiting(left) >= 0) {
            fresh = false;
            same = true;
            return false;
          }
          tile++;
          id = left = next_id;
          next_id = later_id;
          fresh = true;
          return tile < stop && waiting(left) == current;
        };
        // the sixteens' registers take turns: moved from one to the next, they would have to have arrived
        while (true) {
          if (!take(x, x1)) {
            if (!same) x = x1;
            break;
          }
          if (!take(x1, x)) {
            if (same) x = x1;
            break;
          }
        }
      }
    }
  }
}

// How a call is cut up.
struct Plan {
  bool few;     // rows: one of a sixteen's adapters to a workgroup, K split over workgroups
  int splits;   // their parts of K
  int waves;    // few rows: of a workgroup, on parts of K
  int sixteens; // many rows: of a workgroup
  int ranks;    // sixteens of ranks of a workgroup
};
// The few rows' form reads A once for each sixteen of rows and adapter, and its second product splits h for each 64
// columns, so it is taken for fewer rows where ranks are many.  Rank 16, K -> columns, 16 requests, this form and the
// other: 512 rows of 768 codes -> 3 x 768 14.1 and 14.1 us, 4,096 -> 4,096 21.3 and 25.5 (64 adapters mixed 46 and 77); 700
// rows 17.5 and 15.3, 24.1 and 25.2.  Rank 64, two requests: 256 rows of 4,096 -> 8,192 28.9 and 28.7, of 2,048 -> 768 13.8
// and 20.0; 512 rows 49.3 and 30.4, 19.3 and 20.8.  It goes by rows and ranks alone, though the other form walks all of K in
// one workgroup: where K is 8,192, 700 rows of rank 16 -> 4,096 would take 26 us in this form and take 38, and 256 rows of
// rank 64 -> 8,192 take 32 and would take 44.
int few_rows(int R) { return std::min(512, 24576 / R); }
Plan plan_of(int T, int K, int S, int R) {
  Plan q{};
  const int SR = S * R, tiles = (SR + ROWS - 1) / ROWS;
  q.few = T <= few_rows(R);
  q.splits = 1;
  if (q.few) {
    const int steps = (K + FEW_STEP - 1) / FEW_STEP;
    q.waves = std::min(FEW_WAVES, steps);
    q.splits = std::min((steps + q.waves - 1) / q.waves, 8);
    q.ranks = 1;
    return q;
  }
  // Up to 64 ranks to a workgroup.  With 128 bf16 adapters of rank 128 take 1% less (16,391 rows), codes 70% more.
  const int groups = (tiles + 3) / 4;
  q.ranks = (tiles + groups - 1) / groups;
  const int64_t blocks = ((int64_t)T + 4 * ROWS - 1) / (4 * ROWS) * groups;
  // Halves of tiles while those are fewer than compute units, which read A twice as often but LDS less: 4,616 rows of
  // 2,048 against 64 ranks 29.0 us (both products), in whole tiles 31.1; past that it is the same or less (18,464 rows: 63.9 and 61.7).
  q.sixteens = q.ranks > 1 && blocks <= 256 ? 2 : 4;
  if (q.sixteens == 2) q.ranks = (q.ranks + 1) & ~1;
  return q;
}

template <bool CODES, bool BF, int RT, int RG>
hipError_t launch_down(const AdapterArgs& a, hipStream_t s) {
  const int tiles = (a.S * a.R + ROWS - 1) / ROWS, groups = (tiles + RT - 1) / RT;
  const int64_t rows = ((int64_t)a.T + RG * ROWS - 1) / (RG * ROWS);
  // A tile with the rows of several short requests takes as many turns; up to 16 workgroups share them while the grid
  // stays within 2,048: 1,000 rows of 64 adapters, mixed, take 83 us so and 193 with 4, 4,616 rows of 32 requests 23.5 and
  // 32 with one to a tile.  Past that the ones without a turn cost more: 9,232 rows 37.2 us, with twice as many 40.5.
  const int64_t share = std::max<int64_t>(1, std::min<int64_t>(ROWS, 2048 / (rows * groups)));
  const dim3 grid((unsigned)std::min<int64_t>(rows, 1 << 20), (unsigned)groups, (unsigned)share);
  T5K_LAUNCH((adapter_down_kernel<CODES, BF, RT, RG>), grid, dim3(256), 0, s, a, a.y_type == FP8_IO_F32 ? 3 : 2);
  return hipGetLastError();
}
template <bool CODES, bool BF>
hipError_t launch_down_plan(const AdapterArgs& a, const Plan& q, hipStream_t s) {
  if (q.few) {
    const int groups = (a.S * a.R + ROWS - 1) / ROWS;
    const dim3 grid((unsigned)((a.T + ROWS - 1) / ROWS), (unsigned)(groups * q.splits), (unsigned)std::min(ROWS, a.T));
    T5K_LAUNCH((adapter_down_few_kernel<CODES, BF>), grid, dim3(64 * q.waves), 0, s, a, q.splits);
    return hipGetLastError();
  }
  if (q.sixteens == 2) return q.ranks == 2 ? launch_down<CODES, BF, 2, 2>(a, s) : launch_down<CODES, BF, 4, 2>(a, s);
  switch (q.ranks) {
    case 1: return launch_down<CODES, BF, 1, 4>(a, s);
    case 2: return launch_down<CODES, BF, 2, 4>(a, s);
    case 3: return launch_down<CODES, BF, 3, 4>(a, s);
  }
  return launch_down<CODES, BF, 4, 4>(a, s);
}

// Workgroups side by side.
int up_blocks(const AdapterArgs& a, int columns) {
  int blocks = 0;
  for (int i = 0; i < a.S; i++) blocks += (a.cols[i] + UP_WAVES * columns - 1) / (UP_WAVES * columns);
  return blocks;
}
template <int YT, bool BF, int FORM>
hipError_t launch_up_form(const AdapterArgs& a, hipStream_t s) {
  const int blocks = up_blocks(a, up_columns(YT, BF, FORM));
  const int64_t sixteens = ((int64_t)a.T + ROWS - 1) / ROWS;
  // sixteens of rows of a workgroup, so that all workgroups have a place at once: 16,391 rows of 8,192 columns 165 us, with
  // one each 297
  const int64_t places = 256 * up_occupancy(YT, BF, FORM);
  const int run = (int)std::max<int64_t>(1, std::min<int64_t>(64, (sixteens * blocks + places - 1) / places));
  const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>((sixteens + run - 1) / run, 65535));
  T5K_LAUNCH((adapter_up_kernel<YT, BF, FORM>), grid, dim3(64 * UP_WAVES), 0, s, a, 1, run);
  return hipGetLastError();
}
template <int YT, bool BF>
hipError_t launch_up(const AdapterArgs& a, const Plan& q, hipStream_t s) {
  if (q.few) {
    const dim3 grid((unsigned)up_blocks(a, up_columns(YT, BF, JOIN)), (unsigned)((a.T + ROWS - 1) / ROWS), (unsigned)std::min(ROWS, a.T));
    T5K_LAUNCH((adapter_up_kernel<YT, BF, JOIN>), grid, dim3(64 * UP_WAVES), 0, s, a, q.splits, 1);
    return hipGetLastError();
  }
  if (a.R <= 16) return launch_up_form<YT, BF, SHORT>(a, s);
  if (a.R <= 32) return launch_up_form<YT, BF, 1>(a, s);
  if (a.R <= 64) return launch_up_form<YT, BF, 2>(a, s);
  return launch_up_form<YT, BF, 4>(a, s);
}
template <bool BF>
hipError_t launch(const AdapterArgs& a, hipStream_t s) {
  const Plan q = plan_of(a.T, a.K, a.S, a.R);
  const hipError_t e = a.x_type == ADAPTER_E4M3 ? launch_down_plan<true, BF>(a, q, s) : launch_down_plan<false, BF>(a, q, s);
  if (e != hipSuccess) return e;
  switch (a.y_type) {
    case FP8_IO_F32: return launch_up<FP8_IO_F32, BF>(a, q, s);
    case FP8_IO_F16: return launch_up<FP8_IO_F16, BF>(a, q, s);
    case FP8_IO_BF16: return launch_up<FP8_IO_BF16, BF>(a, q, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace

namespace t5k {
size_t adapter_work_bytes(int T, int K, int S, int R) {
  // no less than for fewer rows
  const int few = std::min(T, few_rows(R));
  const size_t sums = (size_t)plan_of(few, K, S, R).splits * few * S * R * 4;
  if (few == T) return sums;
  return std::max(sums, ((size_t)T + ROWS - 1) / ROWS * ROWS * S * R * 6);  // three parts of 16 bits, whole sixteens of rows
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
