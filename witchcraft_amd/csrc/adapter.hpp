// adapter.hpp -- low-rank adapters of many requests beside a shared projection (k_adapter.hip).
#pragma once
#include "common.hpp"

namespace t5k {
constexpr int ADAPTER_MAX_RANK = 128;
constexpr int ADAPTER_MAX_SLICES = 4;
constexpr int ADAPTER_E4M3 = 3;  // x_type: codes with scales; the others are the FP8_IO types

struct AdapterArgs {
  const void* x;            // [T] rows of K values, ldx values apart
  const uint8_t* x_scales;  // codes only: [K / 128][T rounded up to 16]
  int64_t ldx;
  int x_type, T, K;
  const int32_t* ids;  // [T]
  int G;
  const void *a, *b;  // [G][S R][K], [G][N][R] of w_type
  int w_type;
  const int32_t* ranks;  // [G], null: all R
  const float* scales;   // [G], null: all 1
  int R, S;
  int cols[ADAPTER_MAX_SLICES];  // columns of each slice
  int N;                         // their sum
  const void* y;
  void* out;
  int64_t ldy, ldo;  // values
  int y_type;
  void* h;  // bf16 parts in operand order, or for few rows f32 [splits][T][S R]: the kernels' own
};
size_t adapter_work_bytes(int T, int K, int S, int R);
hipError_t launch_adapter(const AdapterArgs& a, hipStream_t s);
}  // namespace t5k
