// ops.cpp — entry points of the serving operators: the 8-bit product, the
// residual norm and cross attention (declared in needle_b200.h).
//
// No counterpart in the reference.  Every argument is checked before the
// first CUDA call, and no C++ exception leaves an entry point.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <string>
#include <utility>
#include <vector>

#include "../../include/needle_b200.h"
#include "capi_internal.h"
#include "ops.h"

using namespace ndl;

namespace {

bool fail(const std::string &msg) {
  capi_set_last_error(msg);
  return false;
}

// An error that is reported here must not come back as the result of a later
// call's launch.
bool ok(cudaError_t e) {
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess || fail(std::string("CUDA error: ") + cudaGetErrorString(e));
}

// Makes `device` current for a call and puts the caller's device back.  What an
// earlier call of the library left as the thread's last error is dropped.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    cudaGetLastError();
    good_ = ok(cudaGetDevice(&before_));
    if (good_ && before_ != device) {
      good_ = ok(cudaSetDevice(device));
      moved_ = good_;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(before_);
  }
  bool good() const { return good_; }

 private:
  int before_ = 0;
  bool good_ = false, moved_ = false;
};

// The device that holds p; false (error set) when p is not device memory.
bool device_of(const char *what, const void *p, int *device) {
  cudaPointerAttributes at{};
  if (!ok(cudaPointerGetAttributes(&at, p))) return false;
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
    return fail(std::string(what) + " is not device memory");
  *device = at.device;
  return true;
}

bool on_device(const char *what, const void *p, int device) {
  int d = 0;
  if (!p) return true;
  if (!device_of(what, p, &d)) return false;
  return d == device || fail(std::string(what) + " is on device " + std::to_string(d) + ", not on device " +
                             std::to_string(device));
}

bool all_on(int device, std::initializer_list<std::pair<const char *, const void *>> operands) {
  for (const auto &o : operands)
    if (!on_device(o.first, o.second, device)) return false;
  return true;
}

bool float_type(int t) { return t == NEEDLE_F32 || t == NEEDLE_F16 || t == NEEDLE_BF16; }

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Natural alignment of an operand of element type t.
bool natural(const void *p, int t) { return aligned(p, dtype_size(t)); }

constexpr size_t kMaxRows = 0x7fffff00;  // whole tiles of 256 rows still count in 31 bits
constexpr int64_t kMaxItems = 1 << 26;    // of a cross attention plan: 3 GB
constexpr size_t kMaxStride = (size_t)1 << 36;  // elements

// Runs f, turning a C++ exception into an error.
template <typename F>
bool guarded(F f) {
  try {
    capi_clear_last_error();
    return f();
  } catch (const std::exception &e) {
    try {
      capi_set_last_error(std::string("needle call failed: ") + e.what());
    } catch (...) {
    }
    return false;
  }
}

// Reads and clears a plan's flag of expired waits; synchronises the device.
bool check_flag(int device, int *flag, const char *what) {
  OnDevice on(device);
  int e = 0;
  if (!on.good() || !ok(cudaDeviceSynchronize()) || !ok(cudaMemcpy(&e, flag, sizeof e, cudaMemcpyDeviceToHost)))
    return false;
  if (!e) return true;
  cudaMemset(flag, 0, sizeof e);
  return fail(std::string(what) + ": a wait inside a launch timed out");
}

void free_buffer(int device, void *buf) {
  OnDevice on(device);
  if (!on.good()) return;
  cudaDeviceSynchronize();
  cudaFree(buf);
}

}  // namespace

struct NeedleInt8Plan {
  int device = 0;
  CUtensorMap w_map;
  const float *w_scales = nullptr;
  int K = 0, N = 0, max_m = 0;
  void *buf = nullptr;
  int8_t *q = nullptr;        // [max_m][row bytes]
  float *q_scales = nullptr;  // [max_m]
  int *flag = nullptr;
};

struct NeedleCrossAttnPlan {
  int device = 0;
  XAttnWork work;
  int64_t q_rows = 0;  // query rows end here
  void *buf = nullptr;
  int *flag = nullptr;
};

namespace {

bool int8_product(NeedleInt8Plan *p, const int8_t *q, const float *qs, size_t M, const float *bias, void *y, int y_dtype,
                  size_t ldy, bool pdl, cudaStream_t st) {
  Int8Args a{q, &p->w_map, qs, p->w_scales, bias, y, (int64_t)ldy, (int)M, p->N, p->K, y_dtype};
  return ok(int8_matmul(a, pdl, p->flag, st));
}

}  // namespace

extern "C" {

size_t needle_int8_row_bytes(size_t K) { return (K + 15) / 16 * 16; }

int needle_int8_quantize_tokens(const void *x, int x_dtype, size_t M, size_t K, size_t ldx, int8_t *q, float *scales,
                                void *stream) {
  return guarded([&] {
    if (!x || !q || !scales || !float_type(x_dtype) || M == 0 || K == 0 || M > kMaxRows || K > kMaxRows || ldx < K ||
        ldx > kMaxStride || !natural(x, x_dtype) || !aligned(q, 16) || !aligned(scales, 4))
      return fail("invalid quantize arguments");
    int device = 0;
    if (!device_of("x", x, &device) || !all_on(device, {{"q", q}, {"scales", scales}})) return false;
    OnDevice on(device);
    return on.good() && ok(int8_quantize_rows(x, x_dtype, (int64_t)M, (int64_t)K, (int64_t)ldx, q, scales,
                                              (cudaStream_t)stream));
  }) ? 0 : -1;
}

int needle_int8_quantize_weight(const void *w, int w_dtype, size_t K, size_t N, int8_t *data, float *scales,
                                void *stream) {
  return guarded([&] {
    if (!w || !data || !scales || !float_type(w_dtype) || K == 0 || N == 0 || K > kMaxRows || N > kMaxRows ||
        !natural(w, w_dtype) || !aligned(data, 16) || !aligned(scales, 4))
      return fail("invalid quantize arguments");
    int device = 0;
    if (!device_of("w", w, &device) || !all_on(device, {{"data", data}, {"scales", scales}})) return false;
    OnDevice on(device);
    return on.good() &&
           ok(int8_quantize_cols(w, w_dtype, (int64_t)K, (int64_t)N, data, scales, (cudaStream_t)stream));
  }) ? 0 : -1;
}

NeedleInt8Plan *needle_int8_plan_create(const int8_t *w, const float *s, size_t K, size_t N, size_t max_m,
                                        void *stream) {
  NeedleInt8Plan *plan = nullptr;
  const bool good = guarded([&] {
    if (!w || !s || K == 0 || N == 0 || max_m == 0 || N > kMaxRows || max_m > kMaxRows || !aligned(w, 16) ||
        !aligned(s, 4))
      return fail("invalid plan arguments");
    if (K > (size_t)kInt8MaxK)
      return fail("K = " + std::to_string(K) + " is above " + std::to_string(kInt8MaxK) +
                  ", where a 32-bit sum of 8-bit products can overflow");
    int device = 0;
    if (!device_of("w_data", w, &device) || !on_device("w_scales", s, device)) return false;
    OnDevice on(device);
    if (!on.good()) return false;
    plan = new NeedleInt8Plan();
    plan->device = device;
    if (!ok(int8_weight_map(&plan->w_map, w, (int64_t)N, (int)K))) return false;
    plan->w_scales = s;
    plan->K = (int)K;
    plan->N = (int)N;
    plan->max_m = (int)max_m;
    const size_t qb = (max_m * needle_int8_row_bytes(K) + 255) / 256 * 256, sb = (max_m * 4 + 255) / 256 * 256;
    if (!ok(cudaMalloc(&plan->buf, qb + sb + 256))) return false;
    plan->q = (int8_t *)plan->buf;
    plan->q_scales = (float *)((char *)plan->buf + qb);
    plan->flag = (int *)((char *)plan->buf + qb + sb);
    return ok(cudaMemsetAsync(plan->flag, 0, 256, (cudaStream_t)stream)) &&
           ok(cudaStreamSynchronize((cudaStream_t)stream));
  });
  if (good) return plan;
  needle_int8_plan_free(plan);
  return nullptr;
}

int needle_int8_plan_matmul(NeedleInt8Plan *p, const void *x, int x_dtype, size_t M, size_t ldx, const float *bias,
                            void *y, int y_dtype, size_t ldy, void *stream) {
  return guarded([&] {
    if (!p || !x || !y || M == 0 || M > (size_t)p->max_m || !float_type(x_dtype) || !float_type(y_dtype) ||
        ldx < (size_t)p->K || ldy < (size_t)p->N || ldx > kMaxStride || ldy > kMaxStride || !natural(x, x_dtype) ||
        !natural(y, y_dtype) || !aligned(bias, 4))
      return fail("invalid plan matmul arguments");
    OnDevice on(p->device);
    if (!on.good() || !all_on(p->device, {{"x", x}, {"y", y}, {"bias", bias}})) return false;
    cudaStream_t st = (cudaStream_t)stream;
    if (int8_matmul_fuses((int)M, p->N, p->K)) {
      Int8Args a{nullptr, &p->w_map, nullptr, p->w_scales, bias, y, (int64_t)ldy, (int)M, p->N, p->K, y_dtype};
      a.x = x;
      a.ldx = (int64_t)ldx;
      a.x_dtype = x_dtype;
      a.x_vec = aligned(x, 16) && ldx * dtype_size(x_dtype) % 16 == 0;
      return ok(int8_matmul(a, false, p->flag, st));
    }
    return ok(int8_quantize_rows(x, x_dtype, (int64_t)M, p->K, (int64_t)ldx, p->q, p->q_scales, st)) &&
           int8_product(p, p->q, p->q_scales, M, bias, y, y_dtype, ldy, true, st);
  }) ? 0 : -1;
}

int needle_int8_plan_matmul_quantized(NeedleInt8Plan *p, const int8_t *q, const float *q_scales, size_t M,
                                      const float *bias, void *y, int y_dtype, size_t ldy, void *stream) {
  return guarded([&] {
    if (!p || !q || !q_scales || !y || M == 0 || M > (size_t)p->max_m || !float_type(y_dtype) ||
        ldy < (size_t)p->N || ldy > kMaxStride || !aligned(q, 16) || !aligned(q_scales, 4) || !natural(y, y_dtype) ||
        !aligned(bias, 4))
      return fail("invalid plan matmul arguments");
    OnDevice on(p->device);
    if (!on.good() || !all_on(p->device, {{"q", q}, {"q_scales", q_scales}, {"y", y}, {"bias", bias}})) return false;
    return int8_product(p, q, q_scales, M, bias, y, y_dtype, ldy, false, (cudaStream_t)stream);
  }) ? 0 : -1;
}

int needle_int8_plan_status(NeedleInt8Plan *p) {
  return guarded([&] { return p ? check_flag(p->device, p->flag, "8-bit product") : fail("null plan"); }) ? 0 : -1;
}

void needle_int8_plan_free(NeedleInt8Plan *p) {
  if (!p) return;
  if (p->buf) free_buffer(p->device, p->buf);
  delete p;
}

int needle_residual_norm(const void *x, int x_dtype, size_t ldx, const void *y, int y_dtype, size_t ldy, size_t M,
                         size_t d, const float *post_scale, const void *gate, uint32_t gate_flags, size_t ldg,
                         float residual_scale, const float *pre_scale, void *r, size_t ldr, void *h, int h_dtype,
                         size_t ldh, float *h_scales, void *stream) {
  return guarded([&] {
    const uint32_t kind = gate_flags & 3u;
    if (!x || (!r && !h) || !float_type(x_dtype) || !float_type(y_dtype) || M == 0 || d == 0 || M > kMaxRows ||
        ldx < d || ldx > kMaxStride || (gate_flags & ~(3u | NEEDLE_GATE_SIGMOID)) || !natural(x, x_dtype) ||
        !natural(y, y_dtype) || !aligned(post_scale, 4) || !aligned(pre_scale, 4) || !natural(r, x_dtype) ||
        !aligned(h_scales, 4))
      return fail("invalid residual norm arguments");
    if (d > (size_t)kResidualNormMaxD)
      return fail("residual norm: d = " + std::to_string(d) + " is above " + std::to_string(kResidualNormMaxD));
    if (x_dtype != NEEDLE_F32 && x_dtype != y_dtype)
      return fail("residual norm: x must be f32 or of y's type");
    if (y ? !r : r != nullptr) return fail("residual norm: r is written exactly when there is a y");
    if (y ? ldy < d || ldy > kMaxStride || ldr < d || ldr > kMaxStride : post_scale || gate)
      return fail("residual norm: invalid strides, or a post norm or gate without y");
    if ((kind != 0) != (gate != nullptr) || (kind == 0 && gate_flags))
      return fail("residual norm: the gate and its flags disagree");
    if (kind && !natural(gate, kind == NEEDLE_GATE_TOKEN ? y_dtype : NEEDLE_F32))
      return fail("invalid residual norm arguments");
    if (kind == NEEDLE_GATE_TOKEN && (ldg < d || ldg > kMaxStride))
      return fail("residual norm: invalid gate stride");
    if ((h != nullptr) != (pre_scale != nullptr)) return fail("residual norm: h and pre_scale go together");
    const bool i8 = h && h_dtype == NEEDLE_I8;
    if (h && ((h_dtype != y_dtype && !i8) || ldh < (i8 ? needle_int8_row_bytes(d) : d) || ldh > kMaxStride ||
              (i8 ? !aligned(h, 16) || ldh % 16 : !natural(h, h_dtype))))
      return fail("residual norm: h must be of y's type, or 8-bit rows on 16-byte boundaries");
    if (i8 != (h_scales != nullptr)) return fail("residual norm: h_scales go with an 8-bit h");
    int device = 0;
    if (!device_of("x", x, &device) || !all_on(device, {{"y", y}, {"r", r}, {"h", h}, {"gate", gate},
                                                        {"post_scale", post_scale}, {"pre_scale", pre_scale},
                                                        {"h_scales", h_scales}}))
      return false;
    OnDevice on(device);
    if (!on.good()) return false;
    ResidualNormArgs a{};
    a.x = x;
    a.y = y;
    a.gate = gate;
    a.r = r;
    a.h = h;
    a.post = post_scale;
    a.pre = pre_scale;
    a.h_scales = h_scales;
    a.ldx = (int64_t)ldx;
    a.ldy = (int64_t)ldy;
    a.ldg = (int64_t)ldg;
    a.ldr = (int64_t)ldr;
    a.ldh = (int64_t)ldh;
    a.M = (int64_t)M;
    a.d = (int)d;
    a.x_dtype = x_dtype;
    a.y_dtype = y_dtype;
    a.h_dtype = h_dtype;
    a.gate_kind = (int)kind;
    a.sigmoid = (gate_flags & NEEDLE_GATE_SIGMOID) != 0;
    a.scale = residual_scale;
    return ok(residual_norm(a, (cudaStream_t)stream));
  }) ? 0 : -1;
}

NeedleCrossAttnPlan *needle_cross_attn_plan_create(const uint64_t *q_start, const uint64_t *q_len,
                                                   const uint64_t *k_start, const uint64_t *k_len, size_t n_seq,
                                                   size_t H, size_t KVH, size_t D, int dtype, void *stream) {
  NeedleCrossAttnPlan *plan = nullptr;
  const bool good = guarded([&] {
    if (!q_start || !q_len || !k_start || !k_len || n_seq == 0 || n_seq > (1u << 24))
      return fail("invalid cross attention plan arguments");
    if (dtype != NEEDLE_F16 && dtype != NEEDLE_BF16) return fail("cross attention takes f16 or bf16");
    if (D == 0 || D > 128 || D % 8) return fail("cross attention: head_dim must be a multiple of 8 up to 128");
    if (KVH == 0 || H == 0 || H % KVH || H > 4096)
      return fail("cross attention: num_heads must be a multiple of num_kv_heads, up to 4096");
    int64_t q_rows = 0, k_rows = 0, items = 0;
    std::vector<std::pair<uint64_t, uint64_t>> spans;
    for (size_t i = 0; i < n_seq; ++i) {
      if (q_start[i] > kMaxRows || q_len[i] > kMaxRows - q_start[i] || k_start[i] > kMaxRows ||
          k_len[i] > kMaxRows - k_start[i] || q_len[i] * (H / KVH) > kMaxRows)
        return fail("cross attention: request " + std::to_string(i) + " has rows past 2^31 - 256");
      items += cross_attn_items((int64_t)(q_len[i] * (H / KVH))) * (int64_t)KVH;
      if (items > kMaxItems) return fail("cross attention: too many rows and heads for one plan");
      if (q_len[i]) {
        spans.emplace_back(q_start[i], q_start[i] + q_len[i]);
        q_rows = std::max(q_rows, (int64_t)(q_start[i] + q_len[i]));
        if (k_len[i]) k_rows = std::max(k_rows, (int64_t)(k_start[i] + k_len[i]));
      }
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      if (spans[i].first < spans[i - 1].second) return fail("cross attention: two requests share a query row");
    plan = new NeedleCrossAttnPlan();
    plan->q_rows = q_rows;
    int sms = 0;
    if (!ok(cudaGetDevice(&plan->device)) ||
        !ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, plan->device)))
      return false;
    plan->work.s = XAttnShape{(int)H, (int)KVH, (int)D, dtype, k_rows};
    const XAttnSplit split = cross_attn_split(plan->work.s, q_start, q_len, k_start, k_len, n_seq, sms);
    const size_t ib = (split.items.size() * sizeof(XAttnItem) + 255) / 256 * 256;
    if (!ok(cudaMalloc(&plan->buf, ib + (size_t)split.ws_floats * sizeof(float) + 256))) return false;
    plan->flag = (int *)((char *)plan->buf + ib);
    plan->work.items = (const XAttnItem *)plan->buf;
    plan->work.ws = (float *)((char *)plan->flag + 256);
    plan->work.n_few = (int)split.n_few;
    plan->work.n_tile = (int)split.n_tile;
    plan->work.n_groups = (int)split.n_groups;
    plan->work.group_rows = split.group_rows;
    cudaStream_t st = (cudaStream_t)stream;
    return (split.items.empty() || ok(cudaMemcpyAsync(plan->buf, split.items.data(), split.items.size() * sizeof(XAttnItem),
                                                      cudaMemcpyHostToDevice, st))) &&
           ok(cudaMemsetAsync(plan->flag, 0, 256, st)) && ok(cudaStreamSynchronize(st));
  });
  if (good) return plan;
  needle_cross_attn_plan_free(plan);
  return nullptr;
}

int needle_cross_attn_plan_run(NeedleCrossAttnPlan *p, const void *q, size_t q_row, size_t q_head, const void *k,
                               size_t k_row, size_t k_head, const void *v, size_t v_row, size_t v_head,
                               const uint8_t *key_mask, float scale, void *out, size_t out_row, size_t out_head,
                               float *lse, void *stream) {
  return guarded([&] {
    // operands of no rows may be NULL, as an empty tensor's pointer is
    if (!p || (p->q_rows && (!q || !out)) || (p->work.s.k_rows && (!k || !v)) || !aligned(lse, 4))
      return fail("invalid cross attention arguments");
    if (!(scale > 0.0f) || std::isinf(scale)) return fail("cross attention: scale must be positive and finite");
    const size_t D = (size_t)p->work.s.D;
    for (const void *b : {q, k, v, (const void *)out})
      if (!aligned(b, 16)) return fail("cross attention: q, k, v and out must start on 16-byte boundaries");
    for (size_t s : {q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head})
      if (s < D || s % 8 || s > kMaxStride)
        return fail("cross attention: strides must be multiples of 8 elements and at least head_dim");
    const size_t H = (size_t)p->work.s.H, rows = (size_t)p->q_rows;
    if (rows > 0 && out_row < (H - 1) * out_head + D && out_head < (rows - 1) * out_row + D)
      return fail("cross attention: rows and heads of out overlap");
    OnDevice on(p->device);
    if (!on.good() || !all_on(p->device, {{"q", q}, {"k", k}, {"v", v}, {"out", out}, {"key_mask", key_mask},
                                          {"lse", lse}}))
      return false;
    if (p->work.s.k_rows == 0) k = v = q;  // any address: nothing is read from it
    XAttnCall c{q, k, v, key_mask, out, lse, (int64_t)q_row, (int64_t)q_head, (int64_t)k_row, (int64_t)k_head,
                (int64_t)v_row, (int64_t)v_head, (int64_t)out_row, (int64_t)out_head, scale};
    return ok(cross_attn(p->work, c, p->flag, (cudaStream_t)stream));
  }) ? 0 : -1;
}

int needle_cross_attn_plan_status(NeedleCrossAttnPlan *p) {
  return guarded([&] { return p ? check_flag(p->device, p->flag, "cross attention") : fail("null plan"); }) ? 0 : -1;
}

void needle_cross_attn_plan_free(NeedleCrossAttnPlan *p) {
  if (!p) return;
  if (p->buf) free_buffer(p->device, p->buf);
  delete p;
}

}  // extern "C"
