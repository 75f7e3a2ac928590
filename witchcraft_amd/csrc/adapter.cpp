// adapter.cpp -- the C ABI entry points of the low-rank adapters: argument checks, and the host-buffer form around
// the launches of k_adapter.hip.
#include "adapter.hpp"
#include "abi.hpp"
#include "fp8.hpp"

namespace {

using t5h_detail::fail;
using t5h_detail::HostCall;
using t5h_detail::known_type;
using t5h_detail::overlap;
using t5h_detail::Rows;
using t5h_detail::type_bytes;

static_assert(T5H_TYPE_E4M3 == t5k::ADAPTER_E4M3, "the kernels take the ABI's type codes");

constexpr int32_t kMostRows = 1 << 30, kMostAdapters = 1 << 24, kMostCols = 1 << 24;
constexpr int64_t kMostStride = (int64_t)1 << 24;  // the kernels' offsets between a tile's rows have 32 bits

int bad(const std::string& what) { return fail(T5H_ERR_INVALID, "adapter: " + what); }

int check_inner(int32_t T, int32_t K, int32_t slices, int32_t R) {
  if (T < 0 || T > kMostRows) return bad("rows must lie in 0 .. 2^30");
  if (K < 16 || K % 16 || K > t5k::FP8_MAX_K) return bad("row length must be a multiple of 16 in 16 .. 2^21");
  if (slices < 1 || slices > t5k::ADAPTER_MAX_SLICES) return bad("slices must lie in 1 .. 4");
  if (R < 8 || R % 8 || R > t5k::ADAPTER_MAX_RANK) return bad("rank must be a multiple of 8 in 8 .. 128");
  return T5H_OK;
}
int check_shape(int32_t x_type, int32_t T, int32_t K, int32_t G, int32_t w_type, int32_t R, const int32_t* cols,
                int32_t slices, int32_t y_type, int64_t& N) {
  TRY(check_inner(T, K, slices, R));
  if (G < 0 || G > kMostAdapters) return bad("adapters must lie in 0 .. 2^24");
  if (w_type != T5H_TYPE_F16 && w_type != T5H_TYPE_BF16) return bad("adapters must be f16 or bf16");
  if (x_type != w_type && x_type != T5H_TYPE_E4M3) return bad("rows must be of the adapters' type, or e4m3 codes");
  if (!known_type(y_type)) return bad("unknown type of results");
  if (x_type == T5H_TYPE_E4M3 && (((uint64_t)K + t5k::FP8_BLOCK - 1) / t5k::FP8_BLOCK * t5k::fp8_scale_rows(T)) >> 31)
    return bad("scales of x of 2^31 bytes or more");
  if (!cols) return bad("NULL columns");
  N = 0;
  for (int32_t i = 0; i < slices; i++) {
    if (cols[i] < 16 || cols[i] % 16 || cols[i] > kMostCols) return bad("a slice's columns must be a multiple of 16 in 16 .. 2^24");
    N += cols[i];
  }
  return T5H_OK;
}
int check_buffer(const void* p, const char* name, size_t align) {
  if (!p) return bad(std::string("NULL ") + name);
  if ((uintptr_t)p % align) return bad(std::string(name) + " is not aligned to " + std::to_string(align) + " bytes");
  return T5H_OK;
}
int check_rows(const Rows& r, int64_t ld, int64_t least) {
  TRY(check_buffer((const void*)r.at, r.name, 16));
  if (ld < least || ld > kMostStride) return bad(std::string(r.name) + "'s rows must be as long as its values, up to 2^24 apart");
  if (r.stride % 16) return bad(std::string(r.name) + "'s rows must start on 16 bytes");
  return T5H_OK;
}
size_t x_bytes(int32_t x_type) { return x_type == T5H_TYPE_E4M3 ? 1 : 2; }

}  // namespace

extern "C" {

int t5h_adapter_workspace(int32_t T, int32_t K, int32_t slices, int32_t R, size_t* bytes) {
  TRY(check_inner(T, K, slices, R));
  if (!bytes) return bad("NULL bytes");
  *bytes = t5k::adapter_work_bytes(T, K, slices, R);
  return T5H_OK;
}

int t5h_adapter_add_device(const void* d_x, int32_t x_type, const uint8_t* d_x_scales, int64_t ldx, int32_t T, int32_t K,
                           const int32_t* d_ids, int32_t G, const void* d_a, const void* d_b, int32_t w_type,
                           const int32_t* d_ranks, const float* d_scales, int32_t R, const int32_t* cols, int32_t slices,
                           const void* d_y, int64_t ldy, void* d_out, int64_t ldo, int32_t y_type, void* d_work,
                           size_t work_bytes, void* stream) {
  int64_t N;
  TRY(check_shape(x_type, T, K, G, w_type, R, cols, slices, y_type, N));
  if (T == 0) return T5H_OK;
  const uint64_t xs = x_bytes(x_type), ys = type_bytes(y_type);
  const Rows x{(uintptr_t)d_x, K * xs, (uint64_t)ldx * xs, "x"}, y{(uintptr_t)d_y, N * ys, (uint64_t)ldy * ys, "y"};
  const Rows out{(uintptr_t)d_out, N * ys, (uint64_t)ldo * ys, "out"};
  TRY(check_rows(x, ldx, K));
  TRY(check_rows(y, ldy, N));
  TRY(check_rows(out, ldo, N));
  if (!(y.at == out.at && y.stride == out.stride) && overlap(y, out, T)) return bad("out overlaps y without being y");
  if (x_type == T5H_TYPE_E4M3) TRY(check_buffer(d_x_scales, "scales of x", 16));
  TRY(check_buffer(d_ids, "ids", 4));
  if (G) {
    TRY(check_buffer(d_a, "a", 16));
    TRY(check_buffer(d_b, "b", 16));
  }
  if (d_ranks) TRY(check_buffer(d_ranks, "ranks", 4));
  if (d_scales) TRY(check_buffer(d_scales, "scales", 4));
  TRY(check_buffer(d_work, "workspace", 16));
  if (work_bytes < t5k::adapter_work_bytes(T, K, slices, R)) return bad("the workspace is smaller than t5h_adapter_workspace says");
  t5k::AdapterArgs p{};
  p.x = d_x, p.x_scales = d_x_scales, p.ldx = ldx, p.x_type = x_type, p.T = T, p.K = K;
  p.ids = d_ids, p.G = G, p.a = d_a, p.b = d_b, p.w_type = w_type, p.ranks = d_ranks, p.scales = d_scales;
  p.R = R, p.S = slices, p.N = (int)N;
  for (int32_t i = 0; i < slices; i++) p.cols[i] = cols[i];
  p.y = d_y, p.out = d_out, p.ldy = ldy, p.ldo = ldo, p.y_type = y_type;
  p.h = d_work;
  HIP_OK(t5k::launch_adapter(p, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_adapter_add(int32_t hip_device, const void* x, int32_t x_type, const uint8_t* x_scales, int32_t T, int32_t K,
                    const int32_t* ids, int32_t G, const void* a, const void* b, int32_t w_type, const int32_t* ranks,
                    const float* scales, int32_t R, const int32_t* cols, int32_t slices, const void* y, void* out,
                    int32_t y_type) {
  int64_t N;
  TRY(check_shape(x_type, T, K, G, w_type, R, cols, slices, y_type, N));
  if (T == 0) return T5H_OK;
  if (!x || !ids || !y || !out || (G && (!a || !b)) || (x_type == T5H_TYPE_E4M3 && !x_scales)) return bad("NULL buffer");
  HostCall d;
  const size_t xb = (size_t)T * K * x_bytes(x_type), yb = (size_t)T * N * type_bytes(y_type);
  const size_t sb = x_type == T5H_TYPE_E4M3 ? ((size_t)K + t5k::FP8_BLOCK - 1) / t5k::FP8_BLOCK * t5k::fp8_scale_rows(T) : 0;
  const size_t ab = (size_t)G * slices * R * K * 2, bb = (size_t)G * N * R * 2, wb = t5k::adapter_work_bytes(T, K, slices, R);
  const size_t dx = d.part(xb), ds = d.part(sb), di = d.part((size_t)T * 4), da = d.part(ab), db = d.part(bb);
  const size_t dr = d.part((size_t)G * 4), df = d.part((size_t)G * 4), dy = d.part(yb), dw = d.part(wb);
  TRY(d.open(hip_device));
  TRY(d.up(dx, x, xb));
  if (sb) TRY(d.up(ds, x_scales, sb));
  TRY(d.up(di, ids, (size_t)T * 4));
  if (G) {
    TRY(d.up(da, a, ab));
    TRY(d.up(db, b, bb));
    if (ranks) TRY(d.up(dr, ranks, (size_t)G * 4));
    if (scales) TRY(d.up(df, scales, (size_t)G * 4));
  }
  TRY(d.up(dy, y, yb));
  TRY(t5h_adapter_add_device(d.p + dx, x_type, (const uint8_t*)d.p + ds, K, T, K, (const int32_t*)(d.p + di), G, d.p + da,
                             d.p + db, w_type, G && ranks ? (const int32_t*)(d.p + dr) : nullptr,
                             G && scales ? (const float*)(d.p + df) : nullptr, R, cols, slices, d.p + dy, N, d.p + dy, N,
                             y_type, d.p + dw, wb, nullptr));
  HIP_OK(hipDeviceSynchronize());
  return d.down(out, dy, yb);
}

}  // extern "C"
