// rotary.hpp -- norms of queries' and keys' heads and the rotation by positions (k_rotary.hip).
#pragma once
#include "common.hpp"

namespace t5k {
// A table entry: the turns a pair makes per step of its position, as a 61-bit fraction of a turn in the
// upper bits, and the position's axis in the lower three.
constexpr int ROTARY_AXIS_BITS = 3;
constexpr int ROTARY_MAX_AXES = 1 << ROTARY_AXIS_BITS;
constexpr int ROTARY_MAX_DIM = 512;
enum RotaryPairing : int { ROTARY_HALVES = 0, ROTARY_NEIGHBOURS = 1 };

struct RotaryArgs {
  const void *q, *k;  // rows of q_heads, k_heads heads of D values; row strides in values
  int64_t ldq, ldk;
  void *q_out, *k_out;
  int64_t ldq_out, ldk_out;
  int q_heads, k_heads;
  int type;  // of all four
  int T, D;
  const float *q_gamma, *k_gamma;  // null: no norm
  float eps;
  const uint64_t* table;  // [rot / 2]
  int rot;
  const int32_t* pos;  // [axes][T]
  int axes;
};
hipError_t launch_rotary(const RotaryArgs& a, int pairing, hipStream_t s);
}  // namespace t5k
