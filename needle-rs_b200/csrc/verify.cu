// verify.cu — drafted tokens checked against the target's logits.
//
// verify_rows_kernel reads every row of logits once: largest value, its index and
// the sum of the exponentials, for pieces of a row (bound by the bytes).
// verify_pick_kernel, a cluster of blocks for each request, joins the pieces,
// takes drafts while u q < p, and draws the token behind them.
//
// The definition is in 64 bits: a token is where a cumulative sum passes a
// random number.  Both kernels work in f32 and know how far they may be off
// (kAccept, kDraw below); where a comparison falls within that bound, the cluster repeats
// the row with 64-bit exponentials (about one draw in ten over 131,072 entries, next to
// no draft), so that results are those of the definition.  All draws in 64 bits take twice
// the time of the second kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "ops.h"
#include "rowio.cuh"

namespace ndl {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVectors = 4;  // 16-byte pieces of a row that a thread of the first kernel holds
constexpr float kLog2e = 1.4426950408889634f;
// Relative error of a row's sum as the first kernel finds it: a weight's argument t (base 2) is rounded three times
// (3 |t| 2^-24), where the mean of |t| over a row is at most log2 of its entries (24); its exponential is
// off by 2^-22, the sum by a few units.
constexpr double kAccept = 1e-5;
// The same in the second kernel, which carries what the argument's roundings leave out: an exponential's 2^-22 and a few units.
constexpr double kDraw = 5e-7;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A request's rows and temperature.
struct Request {
  int first, n;  // its first draft, its drafts
  bool ok;
};
__device__ __forceinline__ Request request(const VerifyCall &c, int i) {
  const int a = c.start[i], e = c.start[i + 1];
  Request r{a, e - a, true};
  r.ok = a >= 0 && a <= e && e <= c.n_drafts && (int64_t)r.n + 1 <= c.ld_out;
  return r;
}
// Zero and below (and NaN): greedy, log-probabilities of temperature 1.
__device__ __forceinline__ bool is_greedy(const VerifyCall &c, int i) { return c.temperature && !(c.temperature[i] > 0.0f); }
__device__ __forceinline__ float temperature(const VerifyCall &c, int i) {
  return c.temperature && c.temperature[i] > 0.0f ? c.temperature[i] : 1.0f;
}

// 8 bits of a row's mask from entry v on (the row has `words` 64-bit words).
__device__ __forceinline__ uint32_t mask_bits(const uint64_t *mask, int v, int words) {
  if (!mask) return 0xffu;
  const int w = v >> 6, o = v & 63;
  uint64_t x = mask[w] >> o;
  if (o > 56 && w + 1 < words) x |= mask[w + 1] << (64 - o);
  return (uint32_t)x & 0xffu;
}

// A row as vectors: entries before the first 16-byte boundary, whole vectors, the rest.
template <typename T>
struct Row {
  static constexpr int E = 16 / (int)sizeof(T);
  const T *p;
  const uint64_t *mask;
  int V, words, lead, vectors;

  __device__ Row(const VerifyCall &c, const VerifyShape &s, int64_t row) {
    p = (const T *)c.logits + row * c.ldl;
    mask = c.mask ? c.mask + row * c.ld_mask : nullptr;
    V = s.V;
    words = (V + 63) >> 6;
    lead = min(V, (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)));
    vectors = (V - lead) / E;
  }
  // Value of entry v, minus infinity where it is masked.
  __device__ float at(int v) const {
    if (mask && !((mask[v >> 6] >> (v & 63)) & 1)) return -INFINITY;
    return (float)p[v];
  }
  // Entries of unit u of the row, in their order: the lead (u = 0), vector u - 1, the rest.
  __device__ int units() const { return vectors + 2; }
  __device__ int first(int u) const { return u == 0 ? 0 : lead + (u - 1) * E; }
  __device__ int count(int u) const { return u == 0 ? lead : u <= vectors ? E : V - lead - vectors * E; }
  __device__ void load(int u, float *x) const {
    const int n = count(u), v0 = first(u);
    if (n == E) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(p + v0);
      const T *e = reinterpret_cast<const T *>(&raw);
      const uint32_t open = mask_bits(mask, v0, words);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = (open >> i) & 1 ? (float)e[i] : -INFINITY;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = i < n ? at(v0 + i) : -INFINITY;
    }
  }
};

// The larger value; of equal ones the lower index, or the higher.
__device__ __forceinline__ void better(float &x, int &i, float y, int j, bool last) {
  if (y > x || (y == x && (last ? j > i : j < i))) x = y, i = j;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(VerifyCall c, VerifyShape s, VerifyWork w) {
  pdl_trigger();
  constexpr int E = Row<T>::E;
  __shared__ float tops[kWarps], sums[kWarps];
  __shared__ int bests[kWarps], owner;
  const int64_t row = blockIdx.x / w.pieces;
  const int piece = (int)(blockIdx.x % w.pieces), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> r(c, s, row);
  // every load at once; the row's request is looked up meanwhile
  float x[kVectors][E];
  const int u0 = piece * kThreads * kVectors;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    const int u = u0 + k * kThreads + tid;
    if (u < r.units()) {
      r.load(u, x[k]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[k][i] = -INFINITY;
    }
  }
  if (tid == 0) owner = -1;
  __syncthreads();
  for (int i = tid; i < c.n_seq; i += kThreads) {
    const Request q = request(c, i);
    if (q.ok && row >= (int64_t)q.first + i && row <= (int64_t)q.first + i + q.n) owner = i;
  }
  const bool last = c.flags & 1;
  float top = -INFINITY;
  int best = last ? -1 : s.V;
  bool broken = false;
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    const int u = u0 + k * kThreads + tid, v0 = r.first(u);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      broken = broken || !(x[k][i] < INFINITY);  // NaN or plus infinity
      if (x[k][i] > -INFINITY) better(top, best, x[k][i], v0 + i, last);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    better(top, best, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, best, o), last);
  if (lane == 0) tops[warp] = top, bests[warp] = best;
  broken = __syncthreads_or(broken);
  if (owner < 0) return;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) better(top, best, tops[k], bests[k], last);
  const float cc = kLog2e / temperature(c, owner), from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kVectors; ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) sum += ex2((x[k][i] - from) * cc);
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0f;
    for (int k = 0; k < kWarps; ++k) sum += sums[k];
    w.piece[blockIdx.x] = make_float4(broken ? __uint_as_float(0x7fc00000u) : top, sum, __int_as_float(best), 0.0f);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_there(double *p, uint32_t rank, double v) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(a), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(there), "d"(v) : "memory");
}

constexpr int kCluster = 8;  // blocks of a request, at most
constexpr int kSegments = kCluster * kWarps;

// The weights of a row's entries: of p (unnormalised), or of max(p - q, 0).
template <typename T>
struct Weights {
  const Row<T> &r;
  float top, c_hi, c_lo;
  double top64, inv_t, inv_w;  // of the 64-bit form
  float inv_w32;
  const float *q;  // NULL: none
  int hole;        // an entry of weight zero, or -1
  bool rest;       // max(p - q, 0)

  // Weights of unit u's entries in 32 or 64 bits; returns their sum.
  template <bool EXACT>
  __device__ __forceinline__ double unit(int u, double *y) const {
    constexpr int E = Row<T>::E;
    float x[E];
    r.load(u, x);
    const int v0 = r.first(u), n = r.count(u);
    double sum = 0.0;
    if (EXACT) {
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        double e = x[i] == -INFINITY ? 0.0 : exp(((double)x[i] - top64) * inv_t);
        if (rest) e = fmax(e * inv_w - (double)q[v0 + i], 0.0);
        if (v0 + i == hole) e = 0.0;
        sum += y[i] = e;
      }
      for (int i = n; i < E; ++i) y[i] = 0.0;
      return sum;
    }
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      // (x - top) * c as a sum of two f32: 2^(a + b) = 2^a (1 + b ln 2)
      const float d = x[i] - top, back = x[i] - d, rest_d = (x[i] - (d + back)) + (back - top);
      const float a = d * c_hi, b = fmaf(d, c_hi, -a) + fmaf(rest_d, c_hi, d * c_lo);
      float e = ex2(a);
      e = x[i] == -INFINITY ? 0.0f : fmaf(e, b * 0.6931471805599453f, e);
      if (rest) e = i < n ? fmaxf(fmaf(e, inv_w32, -q[v0 + i]), 0.0f) : 0.0f;
      if (v0 + i == hole) e = 0.0f;
      part += e;
      y[i] = e;
    }
    return (double)part;
  }
};

struct Shared {
  double seg[2][kSegments];  // sums of the segments, of two turns
  double top_of[kWarps];
  int token, sure;
  double logp;
};

// Sums of the cluster's segments of a row (a warp's units lie side by side), in
// their order, into sm.seg[turn]; returns the total.
template <bool EXACT, typename T>
__device__ double segment_sums(const Weights<T> &w, Shared &sm, int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, size = (int)cluster_size(), me = (int)cluster_rank();
  const int segments = size * kWarps, seg = me * kWarps + warp, units = w.r.units();
  const int u0 = (int)((int64_t)units * seg / segments), u1 = (int)((int64_t)units * (seg + 1) / segments);
  double sum = 0.0, y[Row<T>::E];
#pragma unroll 2
  for (int u = u0 + lane; u < u1; u += 32) sum += w.template unit<EXACT>(u, y);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane < size) store_there(&sm.seg[turn][seg], (uint32_t)lane, sum);
  cluster_meet();
  double total = 0.0;
  for (int k = 0; k < segments; ++k) total += sm.seg[turn][k];
  return total;
}

// The first entry at which the sum of the weights passes `want` (the last of
// any weight, if rounding leaves none), by the warp whose segment it is; the
// others learn nothing.  `off`: how far the sums may be off; *sure: the entry is further than that from
// its borders.
template <bool EXACT, typename T>
__device__ void find(const Weights<T> &w, Shared &sm, int turn, double want, double off, int *token, bool *sure) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, size = (int)cluster_size(), me = (int)cluster_rank();
  const int segments = size * kWarps, units = w.r.units();
  int seg = -1, some = -1;
  double before = 0.0;
  for (int k = 0; k < segments && seg < 0; ++k) {
    const double x = sm.seg[turn][k];
    if (x > 0.0) some = k;
    if (x > 0.0 && before + x > want) seg = k;
    else before += x;
  }
  *token = -1;
  *sure = true;
  if (seg < 0) {
    seg = some;  // rounding: the last entry of the last segment of any weight
    before = want;
    *sure = false;
  }
  if (seg != me * kWarps + warp) return;
  const int u0 = (int)((int64_t)units * seg / segments), u1 = (int)((int64_t)units * (seg + 1) / segments);
  int last = -1;
  for (int a = u0; a < u1; a += 32) {
    constexpr int E = Row<T>::E;
    const int u = a + lane;
    double y[E], own = u < u1 ? w.template unit<EXACT>(u, y) : 0.0, upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, own > 0.0), here = __ballot_sync(0xffffffffu, own > 0.0 && before + upto > want);
    const int from = here ? __ffs(here) - 1 : some ? 31 - __clz(some) : -1;
    int pick = -1;
    bool fine = false;
    if (lane == from) {
      double at = before + upto - own;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!(y[i] > 0.0) || (here && pick >= 0 && at > want)) continue;
        fine = want >= at + off && want < at + y[i] - off;
        at += y[i];
        pick = w.r.first(u) + i;
      }
    }
    if (from >= 0) {
      pick = __shfl_sync(0xffffffffu, pick, from);
      fine = __shfl_sync(0xffffffffu, (int)fine, from);
      last = pick;
      if (here) {
        *token = pick;
        *sure = *sure && fine;
        return;
      }
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  *token = last;
  *sure = false;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_pick_kernel(VerifyCall c, VerifyShape s, VerifyWork w) {
  __shared__ Shared sm;
  __shared__ float tops[kThreads], sums[kThreads];
  __shared__ int bests[kThreads], found;
  const int size = (int)cluster_size(), me = (int)cluster_rank(), i = blockIdx.x / size, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5;
  cluster_meet();  // every block of the cluster is there before its shared memory is written
  const Request rq = request(c, i);
  uint32_t *out = c.out_ids + (int64_t)i * c.ld_out;
  float *logp = c.logprobs ? c.logprobs + (int64_t)i * c.ld_out : nullptr;
  if (!rq.ok) {
    for (int64_t j = me * kThreads + tid; j < c.ld_out; j += size * kThreads) {
      out[j] = 0xffffffffu;
      if (logp) logp[j] = 0.0f;
    }
    if (me == 0 && tid == 0) *w.bad = 1, c.out_len[i] = 0;
    return;
  }
  const bool greedy = is_greedy(c, i), last = c.flags & 1;
  const float temp = temperature(c, i);
  const double inv_t = 1.0 / (double)temp;
  const float *probs = c.probs;
  pdl_wait();

  // rows in rounds of kThreads: a warp joins a row's pieces, a thread checks a draft
  int taken = 0;           // drafts taken before this round
  int len = -1;            // tokens, when the request has ended
  uint32_t token = 0xffffffffu;
  float row_top = 0.0f;
  bool draw = false;
  for (int base = 0; len < 0; base += kThreads) {
    const int rows = min(kThreads, rq.n + 1 - base);
    for (int j = warp; j < rows; j += kWarps) {
      const float4 *p = w.piece + ((int64_t)rq.first + i + base + j) * w.pieces;
      float top = -INFINITY, sum = 0.0f;
      int best = last ? -1 : s.V;
      bool broken = false;
      for (int k = lane; k < w.pieces; k += 32) {
        const float4 x = p[k];
        broken = broken || x.x != x.x;
        better(top, best, x.x, __float_as_int(x.z), last);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        better(top, best, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, best, o), last);
      const float cc = kLog2e / temp;
      if (top > -INFINITY)
        for (int k = lane; k < w.pieces; k += 32) {
          const float4 x = p[k];
          sum += x.y * ex2((x.x - top) * cc);
        }
      sum = warp_sum(sum);
      broken = __any_sync(0xffffffffu, broken);
      if (lane == 0) tops[j] = broken ? -INFINITY : top, sums[j] = sum, bests[j] = best;
    }
    if (tid == 0) found = rows;
    __syncthreads();
    // 0: taken, 1: not, 2: too close to tell, 3: a row without a token
    int verdict = 1;
    float u = 0.0f;
    double q = 1.0;
    float lp = 0.0f;
    uint32_t d = 0xffffffffu;
    const int j = tid;
    const int64_t row = (int64_t)rq.first + i + base + j;
    if (j < rows) {
      const int t = rq.first + base + j;
      const bool drafted = base + j < rq.n;
      if (drafted) d = c.ids[t];
      if (tops[j] == -INFINITY) {
        verdict = 3;
      } else if (drafted && d < (uint32_t)s.V) {
        if (greedy) {
          verdict = d == (uint32_t)bests[j] ? 0 : 1;
        } else {
          const Row<T> r(c, s, row);
          const float x = r.at((int)d);
          u = c.accept_u[t];
          if (probs) q = (double)probs[(int64_t)t * c.ldp + d];
          if (x > -INFINITY) {
            const double p = exp(((double)x - (double)tops[j]) * inv_t) / (double)sums[j], lhs = (double)u * q;
            verdict = fabs(lhs - p) <= kAccept * p ? 2 : lhs < p ? 0 : 1;
          }
        }
        if (verdict == 0 || verdict == 2)
          lp = (float)(((double)Row<T>(c, s, row).at((int)d) - (double)tops[j]) * inv_t - log((double)sums[j]));
      }
      if (verdict != 0) atomicMin(&found, j);
    }
    __syncthreads();
    // drafts too close to tell, in order: the row's sum in 64 bits
    for (;;) {
      const int f = found;
      if (tid == f && f < rows) sm.sure = verdict;
      __syncthreads();
      if (f >= rows || sm.sure != 2) break;
      const Row<T> r(c, s, (int64_t)rq.first + i + base + f);
      Weights<T> wt{r, 0.0f, 0.0f, 0.0f, (double)tops[f], inv_t, 0.0, 0.0f, nullptr, -1, false};
      const double W = segment_sums<true>(wt, sm, 0);
      if (tid == 0) found = rows;
      __syncthreads();
      if (tid == f) {
        const double p = exp(((double)r.at((int)d) - (double)tops[f]) * inv_t) / W;
        verdict = (double)u * q < p ? 0 : 1;
      }
      if (j < rows && verdict != 0) atomicMin(&found, j);
      cluster_meet();  // found is whole, and the segments may be written again
    }
    const int f = found;
    if (me == 0 && j < min(f, rows)) {
      out[base + j] = d;
      if (logp) logp[base + j] = lp;
    }
    if (f < rows) {
      taken = base + f;
      row_top = tops[f];
      token = (uint32_t)bests[f];
      len = sm.sure == 3 ? taken : taken + 1;
      draw = sm.sure != 3;
    }
    __syncthreads();
  }

  // the token behind the drafts
  if (draw) {
    const Row<T> r(c, s, (int64_t)rq.first + i + taken);
    const bool replaced = taken < rq.n;
    const int t = rq.first + taken;
    const double c64 = 1.4426950408889634074 * inv_t;
    Weights<T> wt{r, row_top, (float)c64, (float)(c64 - (double)(float)c64), (double)row_top, inv_t, 0.0, 0.0f, nullptr, -1, false};
    double W = 0.0;
    bool mine = false;
    if (greedy) {
      if (logp) W = segment_sums<false>(wt, sm, 0);
      mine = me == 0 && tid == 0;
    } else {
      const double u = (double)c.final_u[i];
      int pick = -1;
      bool sure = true;
      // in f32; again in 64 bits if that is too close to tell
      for (int exact = 0; exact < 2; ++exact) {
        wt.rest = false;
        wt.hole = -1;
        if (tid == 0) sm.top_of[0] = 0.0;
        W = exact ? segment_sums<true>(wt, sm, 0) : segment_sums<false>(wt, sm, 0);
        double total = W, off = exact ? 0.0 : 2.0 * kDraw * W;
        int turn = 0;
        bool close = false;
        if (replaced) {
          wt.rest = probs != nullptr;
          wt.q = probs ? probs + (int64_t)t * c.ldp : nullptr;
          wt.inv_w = 1.0 / W;
          wt.inv_w32 = (float)wt.inv_w;
          const uint32_t d = c.ids[t];
          wt.hole = probs ? -1 : d < (uint32_t)s.V ? (int)d : -1;
          const double left = exact ? segment_sums<true>(wt, sm, 1) : segment_sums<false>(wt, sm, 1);
          const double bound = probs ? 4.0 * kDraw : 2.0 * kDraw * W;  // p has the error of W as well
          close = !exact && left <= 2.0 * bound;
          if (left > 0.0) {
            turn = 1;
            total = left;
            off = exact ? 0.0 : bound;
          } else {  // nothing left over: p itself
            wt.rest = false;
            wt.hole = -1;
          }
        }
        if (exact) find<true>(wt, sm, turn, u * total, 0.0, &pick, &sure);
        else find<false>(wt, sm, turn, u * total, off, &pick, &sure);
        mine = pick >= 0 && lane == 0;
        if (exact) break;
        // one warp of the cluster knows: it tells all
        if (pick >= 0 && lane < size) store_there(&sm.top_of[0], (uint32_t)lane, sure && !close ? 1.0 : 0.0);
        cluster_meet();
        const bool good = sm.top_of[0] == 1.0;
        cluster_meet();  // sm.seg and the answer may be written again
        if (good) break;
        mine = false;
      }
      token = (uint32_t)pick;
    }
    if (mine) {
      out[taken] = token;
      if (logp) logp[taken] = (float)(((double)r.at((int)token) - (double)row_top) * inv_t - log(W));
    }
  }
  // behind the tokens
  for (int64_t j = len + me * kThreads + tid; j < c.ld_out; j += size * kThreads) {
    out[j] = 0xffffffffu;
    if (logp) logp[j] = 0.0f;
  }
  if (me == 0 && tid == 0) c.out_len[i] = (uint32_t)len;
}

template <typename T>
cudaError_t run(const VerifyShape &s, const VerifyCall &c, const VerifyWork &w, cudaStream_t st) {
  const int64_t rows = (int64_t)c.n_drafts + c.n_seq;
  verify_rows_kernel<T><<<(unsigned)(rows * w.pieces), kThreads, 0, st>>>(c, s, w);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int size = s.V <= 4096 ? 1 : s.V <= 16384 ? 2 : kCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(c.n_seq * size));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_pick_kernel<T>, c, s, w);
}

}  // namespace

// A row's units (vectors and two ends) over those of a block.
int verify_pieces(const VerifyShape &s) {
  const int e = s.dtype == DT_F32 ? 4 : 8;
  return (s.V / e + 2 + kThreads * kVectors - 1) / (kThreads * kVectors);
}

cudaError_t verify_drafts(const VerifyShape &s, const VerifyCall &c, const VerifyWork &w, cudaStream_t st) {
  if (s.dtype == DT_F32) return run<float>(s, c, w, st);
  return s.dtype == DT_F16 ? run<__half>(s, c, w, st) : run<__nv_bfloat16>(s, c, w, st);
}

}  // namespace ndl
