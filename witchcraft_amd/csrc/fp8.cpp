// fp8.cpp -- the C ABI entry points of the 8-bit operators: argument checks, and the host-buffer forms
// around the launches of k_fp8.hip and k_fp8_gemm.hip.
#include <hip/hip_runtime.h>
#include <math.h>

#include <string>

#include "../../include/t5hip.h"
#include "fp8.hpp"

namespace t5h_detail {
int fail(int code, const std::string& msg);
}

namespace {

using t5h_detail::fail;

#define HIP_OK(expr)                                                                   \
  do {                                                                                 \
    hipError_t e_ = (expr);                                                            \
    if (e_ != hipSuccess)                                                              \
      return fail(T5H_ERR_HIP, std::string(#expr ": ") + hipGetErrorString(e_));       \
  } while (0)

static_assert(T5H_TYPE_F32 == t5k::FP8_IO_F32 && T5H_TYPE_F16 == t5k::FP8_IO_F16 && T5H_TYPE_BF16 == t5k::FP8_IO_BF16,
              "the kernels take the ABI's type codes");
static_assert(T5H_SCALE_E8M0 == t5k::FP8_E8M0 && T5H_SCALE_F32 == t5k::FP8_F32, "and its scale types");

constexpr int32_t kMostRows = 1 << 30;

size_t type_bytes(int32_t t) { return t == T5H_TYPE_F32 ? 4 : 2; }
bool known_type(int32_t t) { return t == T5H_TYPE_F32 || t == T5H_TYPE_F16 || t == T5H_TYPE_BF16; }
bool known_scale(int32_t t) { return t == T5H_SCALE_E8M0 || t == T5H_SCALE_F32; }
size_t blocks_of(int32_t n) { return ((size_t)n + t5k::FP8_BLOCK - 1) / t5k::FP8_BLOCK; }
size_t act_scale_bytes(int32_t M, int32_t K) { return blocks_of(K) * t5k::fp8_scale_rows(M); }
size_t weight_scale_bytes(int32_t N, int32_t K, int32_t scale_type) {
  return blocks_of(N) * blocks_of(K) * (scale_type == T5H_SCALE_F32 ? 4 : 1);
}

int bad(const char* what) { return fail(T5H_ERR_INVALID, std::string("fp8: ") + what); }

// Rows and the summed length of a call; the kernels index blocks of 128 in 31 bits.
int check_shape(int32_t rows, int32_t K) {
  if (rows < 0 || rows > kMostRows) return bad("rows must lie in 0 .. 2^30");
  if (K < 16 || K % 16 || K > t5k::FP8_MAX_K) return bad("row length must be a multiple of 16 in 16 .. 2^21");
  if (((uint64_t)rows * blocks_of(K)) >> 31) return bad("2^31 blocks or more");
  return T5H_OK;
}
int check_buffer(const void* p, const char* name, size_t align = 16) {
  if (!p) return fail(T5H_ERR_INVALID, std::string("fp8: NULL ") + name);
  if ((uintptr_t)p % align) return fail(T5H_ERR_INVALID, std::string("fp8: ") + name + " is not aligned to " + std::to_string(align) + " bytes");
  return T5H_OK;
}
// a is b itself, or the two share no byte.
bool same_or_apart(const void* a, size_t an, const void* b, size_t bn) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x == y || x + an <= y || y + bn <= x;
}

#define TRY(expr)                   \
  do {                              \
    if (int rc_ = (expr)) return rc_; \
  } while (0)

int check_quantize(const void* x, int32_t type, int32_t M, int32_t K, const void* codes, const void* scales) {
  TRY(check_shape(M, K));
  if (!known_type(type)) return bad("unknown type");
  if (M == 0) return T5H_OK;
  TRY(check_buffer(x, "input"));
  TRY(check_buffer(codes, "codes"));
  return check_buffer(scales, "scales");
}

int check_quantize_weights(const void* w, int32_t type, int32_t N, int32_t K, int32_t scale_type, const void* codes,
                           const void* scales) {
  TRY(check_shape(N, K));
  if (!known_type(type)) return bad("unknown type");
  if (!known_scale(scale_type)) return bad("unknown scale type");
  if (N == 0) return T5H_OK;
  TRY(check_buffer(w, "input"));
  TRY(check_buffer(codes, "codes"));
  return check_buffer(scales, "scales", scale_type == T5H_SCALE_F32 ? 4 : 1);
}

int check_rmsnorm(const void* x, int32_t x_type, const void* delta, int32_t delta_type, int32_t M, int32_t D,
                  const float* gamma, float eps, const void* sum, const void* codes, const void* scales) {
  TRY(check_shape(M, D));
  if (!known_type(x_type) || (delta && !known_type(delta_type))) return bad("unknown type");
  if (!(eps >= 0.f) || isinf(eps)) return bad("eps must be finite and not negative");
  if (sum && !delta) return bad("a sum needs a delta");
  if (M == 0) return T5H_OK;
  TRY(check_buffer(x, "x"));
  TRY(check_buffer(gamma, "gamma"));
  TRY(check_buffer(codes, "codes"));
  TRY(check_buffer(scales, "scales"));
  if (delta) TRY(check_buffer(delta, "delta"));
  if (sum) {
    TRY(check_buffer(sum, "sum"));
    const size_t xb = (size_t)M * D * type_bytes(x_type), db = (size_t)M * D * type_bytes(delta_type);
    if (!same_or_apart(sum, xb, x, xb)) return bad("sum overlaps x without being x");
    if (!same_or_apart(sum, xb, delta, db) || (sum == delta && type_bytes(x_type) != type_bytes(delta_type)))
      return bad("sum overlaps delta without being delta, of the same size");
  }
  return T5H_OK;
}

int check_product(const void* a, const void* a_scales, int32_t M, const void* w, const void* w_scales, int32_t N,
                  int32_t K, int32_t scale_type, const void* out) {
  TRY(check_shape(M, K));
  TRY(check_shape(N, K));
  if (!known_scale(scale_type)) return bad("unknown scale type");
  if (M == 0 || N == 0) return T5H_OK;
  TRY(check_buffer(a, "activations"));
  TRY(check_buffer(a_scales, "activation scales"));
  TRY(check_buffer(w, "weights"));
  TRY(check_buffer(w_scales, "weight scales", scale_type == T5H_SCALE_F32 ? 4 : 1));
  return check_buffer(out, "output");
}

int check_gated(const void* a, const void* a_scales, int32_t M, const void* w0, const void* w0_scales, const void* w1,
                const void* w1_scales, int32_t N, int32_t K, int32_t scale_type, const void* codes, const void* scales) {
  TRY(check_product(a, a_scales, M, w0, w0_scales, N, K, scale_type, codes));
  if (N % 16) return bad("the gated product's columns must be a multiple of 16");
  if (((uint64_t)M * blocks_of(N)) >> 31) return bad("2^31 blocks or more");
  if (M == 0 || N == 0) return T5H_OK;
  TRY(check_buffer(w1, "up weights"));
  TRY(check_buffer(w1_scales, "up weight scales", scale_type == T5H_SCALE_F32 ? 4 : 1));
  return check_buffer(scales, "scales");
}

// Device copies of a host call's buffers: one allocation, parts on 256-byte boundaries, freed on every
// path.  Outputs are cleared first, so that the scales' unused rows come back as zeros.
struct HostCall {
  char* p = nullptr;
  size_t used = 0;
  HostCall() = default;
  HostCall(const HostCall&) = delete;
  HostCall& operator=(const HostCall&) = delete;
  ~HostCall() {
    if (p) (void)hipFree(p);
  }
  size_t part(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~(size_t)255;
    return at;
  }
  int open(int32_t dev) {
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) return fail(T5H_ERR_NODEVICE, "no HIP device");
    HIP_OK(hipSetDevice(dev < 0 ? 0 : dev));
    if (hipMalloc((void**)&p, used) != hipSuccess) {
      p = nullptr;
      return fail(T5H_ERR_NOMEM, "fp8 buffers");
    }
    HIP_OK(hipMemset(p, 0, used));
    return T5H_OK;
  }
  int up(size_t at, const void* from, size_t bytes) {
    HIP_OK(hipMemcpy(p + at, from, bytes, hipMemcpyHostToDevice));
    return T5H_OK;
  }
  int down(void* to, size_t at, size_t bytes) {
    HIP_OK(hipMemcpy(to, p + at, bytes, hipMemcpyDeviceToHost));
    return T5H_OK;
  }
};

t5k::Fp8GemmArgs gemm_args(const void* a, const void* a_scales, int32_t M, const void* w, const void* w_scales, int32_t N,
                           int32_t K, int32_t scale_type, void* out) {
  t5k::Fp8GemmArgs g{};
  g.a = (const uint8_t*)a;
  g.a_scales = (const uint8_t*)a_scales;
  g.w = (const uint8_t*)w;
  g.w_scales = w_scales;
  g.M = M, g.N = N, g.K = K;
  g.scale_type = scale_type;
  g.out = out;
  return g;
}

}  // namespace

extern "C" {

int t5h_fp8_quantize_device(const void* d_x, int32_t type, int32_t M, int32_t K, uint8_t* d_codes, uint8_t* d_scales,
                            void* stream) {
  TRY(check_quantize(d_x, type, M, K, d_codes, d_scales));
  HIP_OK(t5k::launch_fp8_quantize(d_x, type, M, K, d_codes, d_scales, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_fp8_quantize(int32_t hip_device, const void* x, int32_t type, int32_t M, int32_t K, uint8_t* codes,
                     uint8_t* scales) {
  TRY(check_shape(M, K));
  if (!known_type(type)) return bad("unknown type");
  if (M == 0) return T5H_OK;
  if (!x || !codes || !scales) return bad("NULL buffer");
  HostCall d;
  const size_t xb = (size_t)M * K * type_bytes(type), cb = (size_t)M * K, sb = act_scale_bytes(M, K);
  const size_t dx = d.part(xb), dc = d.part(cb), ds = d.part(sb);
  TRY(d.open(hip_device));
  TRY(d.up(dx, x, xb));
  HIP_OK(t5k::launch_fp8_quantize(d.p + dx, type, M, K, (uint8_t*)d.p + dc, (uint8_t*)d.p + ds, nullptr));
  HIP_OK(hipDeviceSynchronize());
  TRY(d.down(codes, dc, cb));
  return d.down(scales, ds, sb);
}

int t5h_fp8_quantize_weights_device(const void* d_w, int32_t type, int32_t N, int32_t K, int32_t scale_type,
                                    uint8_t* d_codes, void* d_scales, void* stream) {
  TRY(check_quantize_weights(d_w, type, N, K, scale_type, d_codes, d_scales));
  HIP_OK(t5k::launch_fp8_quantize_weights(d_w, type, N, K, scale_type, d_codes, d_scales, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_fp8_quantize_weights(int32_t hip_device, const void* w, int32_t type, int32_t N, int32_t K, int32_t scale_type,
                             uint8_t* codes, void* scales) {
  TRY(check_shape(N, K));
  if (!known_type(type)) return bad("unknown type");
  if (!known_scale(scale_type)) return bad("unknown scale type");
  if (N == 0) return T5H_OK;
  if (!w || !codes || !scales) return bad("NULL buffer");
  HostCall d;
  const size_t wb = (size_t)N * K * type_bytes(type), cb = (size_t)N * K, sb = weight_scale_bytes(N, K, scale_type);
  const size_t dw = d.part(wb), dc = d.part(cb), ds = d.part(sb);
  TRY(d.open(hip_device));
  TRY(d.up(dw, w, wb));
  HIP_OK(t5k::launch_fp8_quantize_weights(d.p + dw, type, N, K, scale_type, (uint8_t*)d.p + dc, d.p + ds, nullptr));
  HIP_OK(hipDeviceSynchronize());
  TRY(d.down(codes, dc, cb));
  return d.down(scales, ds, sb);
}

int t5h_fp8_rmsnorm_device(const void* d_x, int32_t x_type, const void* d_delta, int32_t delta_type, int32_t M,
                           int32_t D, const float* d_gamma, float eps, void* d_sum, uint8_t* d_codes,
                           uint8_t* d_scales, void* stream) {
  TRY(check_rmsnorm(d_x, x_type, d_delta, delta_type, M, D, d_gamma, eps, d_sum, d_codes, d_scales));
  const t5k::Fp8NormArgs a{d_x, d_delta, d_sum, d_gamma, eps, M, D, x_type, delta_type, d_codes, d_scales};
  HIP_OK(t5k::launch_fp8_rmsnorm(a, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_fp8_rmsnorm(int32_t hip_device, const void* x, int32_t x_type, const void* delta, int32_t delta_type, int32_t M,
                    int32_t D, const float* gamma, float eps, void* sum, uint8_t* codes, uint8_t* scales) {
  TRY(check_shape(M, D));
  if (!known_type(x_type) || (delta && !known_type(delta_type))) return bad("unknown type");
  if (!(eps >= 0.f) || isinf(eps)) return bad("eps must be finite and not negative");
  if (sum && !delta) return bad("a sum needs a delta");
  if (M == 0) return T5H_OK;
  if (!x || !gamma || !codes || !scales) return bad("NULL buffer");
  HostCall d;
  const size_t n = (size_t)M * D, xb = n * type_bytes(x_type), db = delta ? n * type_bytes(delta_type) : 0;
  const size_t sb = act_scale_bytes(M, D);
  const size_t dx = d.part(xb), dd = d.part(db), dg = d.part((size_t)D * 4), dc = d.part(n), ds = d.part(sb);
  TRY(d.open(hip_device));
  TRY(d.up(dx, x, xb));
  if (delta) TRY(d.up(dd, delta, db));
  TRY(d.up(dg, gamma, (size_t)D * 4));
  const t5k::Fp8NormArgs a{d.p + dx, delta ? d.p + dd : nullptr, sum ? d.p + dx : nullptr, (const float*)(d.p + dg), eps,
                           M, D, x_type, delta_type, (uint8_t*)d.p + dc, (uint8_t*)d.p + ds};
  HIP_OK(t5k::launch_fp8_rmsnorm(a, nullptr));
  HIP_OK(hipDeviceSynchronize());
  if (sum) TRY(d.down(sum, dx, xb));
  TRY(d.down(codes, dc, n));
  return d.down(scales, ds, sb);
}

int t5h_fp8_matmul_device(const uint8_t* d_a, const uint8_t* d_a_scales, int32_t M, const uint8_t* d_w,
                          const void* d_w_scales, int32_t N, int32_t K, int32_t scale_type, void* d_c, int32_t c_type,
                          void* stream) {
  TRY(check_product(d_a, d_a_scales, M, d_w, d_w_scales, N, K, scale_type, d_c));
  if (!known_type(c_type)) return bad("unknown type");
  t5k::Fp8GemmArgs g = gemm_args(d_a, d_a_scales, M, d_w, d_w_scales, N, K, scale_type, d_c);
  g.out_type = c_type;
  HIP_OK(t5k::launch_fp8_matmul(g, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_fp8_matmul(int32_t hip_device, const uint8_t* a, const uint8_t* a_scales, int32_t M, const uint8_t* w,
                   const void* w_scales, int32_t N, int32_t K, int32_t scale_type, void* c, int32_t c_type) {
  TRY(check_shape(M, K));
  TRY(check_shape(N, K));
  if (!known_scale(scale_type)) return bad("unknown scale type");
  if (!known_type(c_type)) return bad("unknown type");
  if (M == 0 || N == 0) return T5H_OK;
  if (!a || !a_scales || !w || !w_scales || !c) return bad("NULL buffer");
  HostCall d;
  const size_t ab = (size_t)M * K, asb = act_scale_bytes(M, K), wb = (size_t)N * K;
  const size_t wsb = weight_scale_bytes(N, K, scale_type), cb = (size_t)M * N * type_bytes(c_type);
  const size_t da = d.part(ab), das = d.part(asb), dw = d.part(wb), dws = d.part(wsb), dc = d.part(cb);
  TRY(d.open(hip_device));
  TRY(d.up(da, a, ab));
  TRY(d.up(das, a_scales, asb));
  TRY(d.up(dw, w, wb));
  TRY(d.up(dws, w_scales, wsb));
  t5k::Fp8GemmArgs g = gemm_args(d.p + da, d.p + das, M, d.p + dw, d.p + dws, N, K, scale_type, d.p + dc);
  g.out_type = c_type;
  HIP_OK(t5k::launch_fp8_matmul(g, nullptr));
  HIP_OK(hipDeviceSynchronize());
  return d.down(c, dc, cb);
}

int t5h_fp8_gated_gelu_device(const uint8_t* d_a, const uint8_t* d_a_scales, int32_t M, const uint8_t* d_w0,
                              const void* d_w0_scales, const uint8_t* d_w1, const void* d_w1_scales, int32_t N,
                              int32_t K, int32_t scale_type, uint8_t* d_codes, uint8_t* d_scales, void* stream) {
  TRY(check_gated(d_a, d_a_scales, M, d_w0, d_w0_scales, d_w1, d_w1_scales, N, K, scale_type, d_codes, d_scales));
  t5k::Fp8GemmArgs g = gemm_args(d_a, d_a_scales, M, d_w0, d_w0_scales, N, K, scale_type, d_codes);
  g.w1 = d_w1;
  g.w1_scales = d_w1_scales;
  g.out_scales = d_scales;
  HIP_OK(t5k::launch_fp8_gated_gelu(g, (hipStream_t)stream));
  return T5H_OK;
}

int t5h_fp8_gated_gelu(int32_t hip_device, const uint8_t* a, const uint8_t* a_scales, int32_t M, const uint8_t* w0,
                       const void* w0_scales, const uint8_t* w1, const void* w1_scales, int32_t N, int32_t K,
                       int32_t scale_type, uint8_t* codes, uint8_t* scales) {
  TRY(check_shape(M, K));
  TRY(check_shape(N, K));
  if (N % 16) return bad("the gated product's columns must be a multiple of 16");
  if (((uint64_t)M * blocks_of(N)) >> 31) return bad("2^31 blocks or more");
  if (!known_scale(scale_type)) return bad("unknown scale type");
  if (M == 0 || N == 0) return T5H_OK;
  if (!a || !a_scales || !w0 || !w0_scales || !w1 || !w1_scales || !codes || !scales) return bad("NULL buffer");
  HostCall d;
  const size_t ab = (size_t)M * K, asb = act_scale_bytes(M, K), wb = (size_t)N * K;
  const size_t wsb = weight_scale_bytes(N, K, scale_type), cb = (size_t)M * N, sb = act_scale_bytes(M, N);
  const size_t da = d.part(ab), das = d.part(asb), dw0 = d.part(wb), dw0s = d.part(wsb), dw1 = d.part(wb);
  const size_t dw1s = d.part(wsb), dc = d.part(cb), ds = d.part(sb);
  TRY(d.open(hip_device));
  TRY(d.up(da, a, ab));
  TRY(d.up(das, a_scales, asb));
  TRY(d.up(dw0, w0, wb));
  TRY(d.up(dw0s, w0_scales, wsb));
  TRY(d.up(dw1, w1, wb));
  TRY(d.up(dw1s, w1_scales, wsb));
  t5k::Fp8GemmArgs g = gemm_args(d.p + da, d.p + das, M, d.p + dw0, d.p + dw0s, N, K, scale_type, d.p + dc);
  g.w1 = (const uint8_t*)d.p + dw1;
  g.w1_scales = d.p + dw1s;
  g.out_scales = (uint8_t*)d.p + ds;
  HIP_OK(t5k::launch_fp8_gated_gelu(g, nullptr));
  HIP_OK(hipDeviceSynchronize());
  TRY(d.down(codes, dc, cb));
  return d.down(scales, ds, sb);
}

}  // extern "C"
