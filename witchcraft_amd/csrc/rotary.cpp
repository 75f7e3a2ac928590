// rotary.cpp -- the C ABI entry points of the head norms and the rotation: the table of frequencies,
// argument checks, and the host-buffer form around the launch of k_rotary.hip.
#include <math.h>

#include "abi.hpp"
#include "fp8.hpp"
#include "rotary.hpp"

namespace {

using t5h_detail::fail;
using t5h_detail::HostCall;
using t5h_detail::known_type;
using t5h_detail::overlap;
using t5h_detail::Rows;
using t5h_detail::type_bytes;

static_assert(T5H_ROTARY_HALVES == t5k::ROTARY_HALVES && T5H_ROTARY_NEIGHBOURS == t5k::ROTARY_NEIGHBOURS,
              "the kernels take the ABI's pairings");

constexpr int32_t kMostRows = 1 << 30, kMostHeads = 65535;
constexpr int64_t kMostStride = (int64_t)1 << 30;  // 2^30 rows of it stay within 63 bits

int bad(const std::string& what) { return fail(T5H_ERR_INVALID, "rotary: " + what); }

int check_shape(int32_t q_heads, int32_t k_heads, int32_t type, int32_t T, int32_t D, float eps, int32_t rot,
                int32_t pairing, int32_t axes) {
  if (T < 0 || T > kMostRows) return bad("rows must lie in 0 .. 2^30");
  if (q_heads < 0 || q_heads > kMostHeads || k_heads < 0 || k_heads > kMostHeads) return bad("heads must lie in 0 .. 65535");
  if (D < 8 || D % 8 || D > t5k::ROTARY_MAX_DIM) return bad("head size must be a multiple of 8 in 8 .. 512");
  if (rot < 0 || rot % 8 || rot > D) return bad("rotated values must be a multiple of 8 in 0 .. head size");
  if (!known_type(type)) return bad("unknown type");
  if (pairing != T5H_ROTARY_HALVES && pairing != T5H_ROTARY_NEIGHBOURS) return bad("unknown pairing");
  if (axes < 1 || axes > t5k::ROTARY_MAX_AXES) return bad("axes must lie in 1 .. 8");
  if (!(eps >= 0.f) || isinf(eps)) return bad("eps must be finite and not negative");
  return T5H_OK;
}

int check_rows(const Rows& r, int64_t ld, int64_t heads_width) {
  if (!r.at) return bad(std::string("NULL ") + r.name);
  if (r.at % 16 || r.stride % 16) return bad(std::string(r.name) + "'s rows must start on 16 bytes");
  if (ld < heads_width || ld > kMostStride) return bad(std::string(r.name) + "'s rows must be as long as its heads, up to 2^30 apart");
  return T5H_OK;
}
}  // namespace

extern "C" {

int t5h_rotary_table(const double* frequency, const int32_t* axis, int32_t pairs, uint64_t* table) {
  if (pairs < 0 || pairs > t5k::ROTARY_MAX_DIM / 2) return bad("pairs must lie in 0 .. 256");
  if (pairs == 0) return T5H_OK;
  if (!frequency || !table) return bad("NULL buffer");
  for (int32_t i = 0; i < pairs; i++) {
    if (!isfinite(frequency[i])) return bad("frequencies must be finite");
    if (axis && (axis[i] < 0 || axis[i] >= t5k::ROTARY_MAX_AXES)) return bad("a pair's axis must lie in 0 .. 7");
  }
  for (int32_t i = 0; i < pairs; i++) {
    const long double turns = (long double)frequency[i] / 6.283185307179586476925286766559L;
    const long double part = turns - floorl(turns);  // 0 .. 1; 1 itself where a tiny negative rounds to it
    const uint64_t fixed = (uint64_t)llrintl(part * 0x1p61L) & (((uint64_t)1 << 61) - 1);
    table[i] = fixed << t5k::ROTARY_AXIS_BITS | (uint64_t)(axis ? axis[i] : 0);
  }
  return T5H_OK;
}

int t5h_rotary_device(const void* d_q, int64_t ldq, int32_t q_heads, const void* d_k, int64_t ldk, int32_t k_heads,
                      int32_t type, int32_t T, int32_t D, const float* d_q_gamma, const float* d_k_gamma, float eps,
                      const uint64_t* d_table, int32_t rot, int32_t pairing, const int32_t* d_pos, int32_t axes,
                      void* d_q_out, int64_t ldq_out, void* d_k_out, int64_t ldk_out, void* stream) {
  TRY(check_shape(q_heads, k_heads, type, T, D, eps, rot, pairing, axes));
  if (T == 0 || (q_heads == 0 && k_heads == 0)) return T5H_OK;
  const uint64_t size = type_bytes(type), qw = (uint64_t)q_heads * D, kw = (uint64_t)k_heads * D;
  const Rows q{(uintptr_t)d_q, qw * size, (uint64_t)ldq * size, "q"}, k{(uintptr_t)d_k, kw * size, (uint64_t)ldk * size, "k"};
  const Rows qo{(uintptr_t)d_q_out, qw * size, (uint64_t)ldq_out * size, "q_out"};
  const Rows ko{(uintptr_t)d_k_out, kw * size, (uint64_t)ldk_out * size, "k_out"};
  const char* shared = "an output overlaps a buffer without being its own input";
  if (q_heads) {
    TRY(check_rows(q, ldq, qw));
    TRY(check_rows(qo, ldq_out, qw));
    if (!(q.at == qo.at && q.stride == qo.stride) && overlap(q, qo, T)) return bad(shared);
  }
  if (k_heads) {
    TRY(check_rows(k, ldk, kw));
    TRY(check_rows(ko, ldk_out, kw));
    if (!(k.at == ko.at && k.stride == ko.stride) && overlap(k, ko, T)) return bad(shared);
  }
  if (q_heads && k_heads && (overlap(qo, ko, T) || overlap(qo, k, T) || overlap(ko, q, T))) return bad(shared);
  if (((uintptr_t)d_q_gamma | (uintptr_t)d_k_gamma | (uintptr_t)d_pos) % 4) return bad("gammas and positions must lie on 4 bytes");
  if (rot) {
    if (!d_table || !d_pos) return bad("NULL table or positions");
    if ((uintptr_t)d_table % 8) return bad("the table must lie on 8 bytes");
  }
  const t5k::RotaryArgs a{d_q, d_k, ldq, ldk, d_q_out, d_k_out, ldq_out, ldk_out, q_heads, k_heads, type, T, D,
                          q_heads ? d_q_gamma : nullptr, k_heads ? d_k_gamma : nullptr, eps, d_table, rot, d_pos, axes};
  HIP_OK(t5k::launch_rotary(a, pairing, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_rotary(int32_t hip_device, const void* q, int32_t q_heads, const void* k, int32_t k_heads, int32_t type,
               int32_t T, int32_t D, const float* q_gamma, const float* k_gamma, float eps, const uint64_t* table,
               int32_t rot, int32_t pairing, const int32_t* pos, int32_t axes, void* q_out, void* k_out) {
  TRY(check_shape(q_heads, k_heads, type, T, D, eps, rot, pairing, axes));
  if (T == 0 || (q_heads == 0 && k_heads == 0)) return T5H_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || (rot && (!table || !pos))) return bad("NULL buffer");
  HostCall d;
  const int64_t qw = (int64_t)q_heads * D, kw = (int64_t)k_heads * D;
  const size_t qb = (size_t)T * qw * type_bytes(type), kb = (size_t)T * kw * type_bytes(type), gb = (size_t)D * 4;
  const size_t tb = (size_t)rot / 2 * 8, pb = rot ? (size_t)axes * T * 4 : 0;
  const size_t dq = d.part(qb), dk = d.part(kb), dqg = d.part(gb), dkg = d.part(gb), dt = d.part(tb), dp = d.part(pb);
  TRY(d.open(hip_device));
  if (q_heads) TRY(d.up(dq, q, qb));
  if (k_heads) TRY(d.up(dk, k, kb));
  if (q_gamma) TRY(d.up(dqg, q_gamma, gb));
  if (k_gamma) TRY(d.up(dkg, k_gamma, gb));
  if (rot) {
    TRY(d.up(dt, table, tb));
    TRY(d.up(dp, pos, pb));
  }
  const t5k::RotaryArgs a{d.p + dq, d.p + dk, qw, kw, d.p + dq, d.p + dk, qw, kw, q_heads, k_heads, type, T, D,
                          q_gamma ? (const float*)(d.p + dqg) : nullptr, k_gamma ? (const float*)(d.p + dkg) : nullptr,
                          eps, (const uint64_t*)(d.p + dt), rot, (const int32_t*)(d.p + dp), axes};
  HIP_OK(t5k::launch_rotary(a, pairing, nullptr));
  HIP_OK(hipDeviceSynchronize());
  if (q_heads) TRY(d.down(q_out, dq, qb));
  if (k_heads) TRY(d.down(k_out, dk, kb));
  return T5H_OK;
}

}  // extern "C"
