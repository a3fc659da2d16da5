// ops.h — launchers of the serving operators (int8_matmul.cu,
// residual_norm.cu, cross_attn.cu) behind the entry points in ops.cpp.
//
// All pointers are device pointers unless a name says host.  Launchers enqueue
// on `st` and return the launch status.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace ndl {

// Element types, numbered as NEEDLE_F32 .. NEEDLE_I8.
enum DType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2, DT_I8 = 3 };
inline size_t dtype_size(int t) { return t == DT_F32 ? 4 : t == DT_I8 ? 1 : 2; }

// ── 8-bit product ──
// Rows of quantised operands are int8_row_bytes(K) bytes long, so that each
// starts on a 16-byte boundary.
__host__ __device__ inline int64_t int8_row_bytes(int64_t K) { return (K + 15) / 16 * 16; }
constexpr int64_t kInt8MaxK = 131071;  // K * 128 * 128 < 2^31: the sum fits 32 bits

cudaError_t int8_quantize_rows(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, int8_t *q, float *scales,
                               cudaStream_t st);
cudaError_t int8_quantize_cols(const void *w, int dtype, int64_t K, int64_t N, int8_t *data, float *scales,
                               cudaStream_t st);
struct Int8Args {
  const int8_t *q;                   // [M][Kp], or NULL with x set
  const CUtensorMap *w_map;          // of the weight [N][Kp] (host)
  const float *q_scales, *w_scales;  // [M], [N]
  const float *bias;                 // [N] or NULL
  void *y;                           // [M][ldy] of y_dtype
  int64_t ldy;
  int M, N, K, y_dtype;
  // unrounded tokens [M][ldx] for the kernel that rounds them itself
  const void *x = nullptr;
  int64_t ldx = 0;
  int x_dtype = 0;
  bool x_vec = false;  // rows on 16-byte boundaries
};
// Whether int8_matmul takes unrounded tokens of these sizes (few of them).
bool int8_matmul_fuses(int M, int N, int K);
// TMA descriptor of a weight [N][Kp], 16-byte aligned.
cudaError_t int8_weight_map(CUtensorMap *map, const int8_t *w, int64_t N, int K);
// *err is set if a bounded wait inside the kernel expired.  pdl: the kernel
// before it in the stream is int8_quantize_rows of the same tokens, which it
// may overlap (programmatic dependent launch).
cudaError_t int8_matmul(const Int8Args &a, bool pdl, int *err, cudaStream_t st);

// ── residual norm ──
struct ResidualNormArgs {
  const void *x, *y, *gate;
  void *r, *h;
  const float *post, *pre;
  float *h_scales;
  int64_t ldx, ldy, ldg, ldr, ldh;
  int64_t M;
  int d;
  int x_dtype, y_dtype, h_dtype;
  int gate_kind;  // 0 none, 1 scalar, 2 channel, 3 token
  bool sigmoid;
  float scale;
};
constexpr int kResidualNormMaxD = 32768;
cudaError_t residual_norm(const ResidualNormArgs &a, cudaStream_t st);

// ── cross attention ──
// One unit of work: `rows` packed query rows of one request and KV head
// against keys [k0, k0 + klen).  Packed row r is query token r / G, head
// kvh * G + r % G of the request, G = H / KVH; the item's are r0 ..
struct XAttnItem {
  int64_t q0;         // first query row of the request
  int64_t k0;         // first key row
  int64_t ws;         // workspace (floats) of the items on these rows, when there are several
  int klen, r0, rows, kvh;
  int split, nsplit;  // this item among those on the same rows
};
struct XAttnShape {
  int H, KVH, D, dtype;
  int64_t k_rows;  // rows of K and V that any request reads end here
};
struct XAttnCall {
  const void *q, *k, *v;
  const uint8_t *mask;
  void *out;
  float *lse;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
  float scale;
};
// A plan's work (host): items of few rows, tiles of up to 128, then one entry
// for each group of items that share rows, to be joined.
struct XAttnSplit {
  std::vector<XAttnItem> items;
  int64_t n_few = 0, n_tile = 0, n_groups = 0;
  int64_t ws_floats = 0;
  int group_rows = 0;  // most rows of a group
};
// Items, before splits, of a KV head of a request with `rows` rows for each.
int64_t cross_attn_items(int64_t rows);
XAttnSplit cross_attn_split(const XAttnShape &s, const uint64_t *q_start, const uint64_t *q_len, const uint64_t *k_start,
                            const uint64_t *k_len, size_t n_seq, int sms);
// The same on the device, with its workspace.
struct XAttnWork {
  XAttnShape s;
  const XAttnItem *items = nullptr;
  float *ws = nullptr;
  int n_few = 0, n_tile = 0, n_groups = 0, group_rows = 0;
};
cudaError_t cross_attn(const XAttnWork &w, const XAttnCall &c, int *err, cudaStream_t st);

}  // namespace ndl
