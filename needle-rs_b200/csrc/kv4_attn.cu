// kv4_attn.cu — attention of query rows to a cache of keys and values in 4
// bits:
//   s_j = scale * q . k_j     out = sum_j e^(s_j) v_j / sum_j e^(s_j)
// with k = m + s c and v = m + s c of each group of 32 dimensions.
//
// The query heads that share a KV head are rows of one matrix: row r of a
// request and KV head is token r / G, head kvh * G + r % G (G = H / KVH), so
// the cache is read once for all of them.
//
// A tile of 16 tokens comes as the operands of mma.sync.m16n8k16: keys by
// dimensions, and values transposed, on the 16 rows, up to 8 query rows on the
// columns.  Codes become f16 numbers in place: a nibble under a mask is c * 2^-24 (the
// low four bits of a half, a subnormal) or c * 2^-20 (the next four), which
// tensor cores multiply exactly.
//   K: q . k = sum over groups of s (q . c) + m (sum of q): products with the
//      codes, exact in f32, then two FMAs a group for each score.  No key is rounded.
//   V: 1024 + c (or 64 + c) by an OR, minus 1024, times s plus m on pairs of
//      f16: a value is rounded to f16 once.
// q is brought to a largest value of 2^10 .. 2^11 by a power of two for each row and
// taken as f16 (exact, but for values below 2^-24 of the row's largest).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kv4.cuh"
#include "ops.h"
#include "rowio.cuh"

namespace ndl {
namespace {

using namespace kv4;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kUnit = 64;  // keys of a unit of work

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 halves(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma(float *d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// How the units of a call fall to the blocks: request i has KVH heads x blocks
// of ROWS rows x units of 64 keys, block b of n takes units
// [total * b / n, total * (b + 1) / n) of all requests' in order.
struct Share {
  int64_t total, begin, end, base;  // base: units before request `seq`, the one that `begin` falls in
  int blocks, seq;
};
struct Units {
  Seq q;
  int row_blocks;
  int64_t keys;  // units of a row block and head

  __device__ int64_t all(int KVH) const { return (int64_t)row_blocks * KVH * keys; }
};
template <int ROWS>
__device__ __forceinline__ Units units_of(const Kv4Rows &b, const Kv4Shape &s, int i, bool causal, int *bad) {
  Units u;
  u.q = sequence(b, s, i, causal, bad);
  u.row_blocks = (int)(((int64_t)u.q.n * (s.H / s.KVH) + ROWS - 1) / ROWS);
  u.keys = max(1, (u.q.len + kUnit - 1) / kUnit);
  return u;
}

// Partial results of items that are cut between blocks: two slots a block (the
// item that it starts in the middle of, the one that it leaves unfinished) of
// ROWS x (DP + 2) floats, and a counter of arrivals for each block where such an item begins.
template <int ROWS, int DP>
__device__ __forceinline__ float *slot_of(const Kv4Work &w, int64_t block, int which) {
  return w.ws + (block * 2 + which) * (ROWS * (DP + 2));
}

template <int ROWS>
__device__ Share share_of(const Kv4Rows &b, const Kv4Shape &s, bool causal, const Kv4Work &w) {
  __shared__ int64_t sums[kWarps], items[kWarps];
  __shared__ int64_t found_base;
  __shared__ int found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (b.n_seq + kThreads - 1) / kThreads, i0 = min((int)threadIdx.x * per, b.n_seq), i1 = min(i0 + per, b.n_seq);
  int64_t mine = 0, n = 0;
  for (int i = i0; i < i1; ++i) {
    const Units u = units_of<ROWS>(b, s, i, causal, w.bad);
    mine += u.all(s.KVH);
    n += (int64_t)u.row_blocks * s.KVH;
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 31) sums[warp] = upto;
  if (lane == 0) items[warp] = n;
  __syncthreads();
  Share r;
  r.total = n = 0;
  for (int k = 0; k < kWarps; ++k) {
    if (k < warp) upto += sums[k];
    r.total += sums[k];
    n += items[k];
  }
  // an item is cut into 128 pieces at most, and a block has two units at least
  const int64_t blocks = min(min((int64_t)gridDim.x, (r.total + 1) / 2), n * 128);
  r.blocks = (int)blocks;
  if (blockIdx.x >= blocks) return r;
  r.begin = r.total * blockIdx.x / blocks;
  r.end = r.total * (blockIdx.x + 1) / blocks;
  if (upto - mine <= r.begin && r.begin < upto) {
    int64_t base = upto - mine;
    for (int i = i0;; ++i) {
      const int64_t x = units_of<ROWS>(b, s, i, causal, w.bad).all(s.KVH);
      if (r.begin < base + x) {
        found = i;
        found_base = base;
        break;
      }
      base += x;
    }
  }
  __syncthreads();
  r.seq = found;
  r.base = found_base;
  return r;
}

// Stages of a warp's ring, and blocks an SM.
__host__ __device__ constexpr int few_stages(int ng) { return ng == 4 ? 5 : ng == 3 ? 6 : 8; }
__host__ __device__ constexpr int few_blocks(int nb) { return nb == 1 ? 4 : nb == 2 ? 3 : 2; }
template <int NG, int NB>
constexpr int few_smem() {
  constexpr int ring = kWarps * few_stages(NG) * tile_bytes(NG), merge = kWarps * NB * 8 * (NG * 32 + 4 + 2) * 4;
  return ring > merge ? ring : merge;
}

template <typename T, int NG, int NB>
__global__ void __launch_bounds__(kThreads, few_blocks(NB))
    few_kernel(Kv4AttnCall c, Kv4Shape s, Kv4Rows b, Kv4Work w) {
  constexpr int ST = few_stages(NG), TB = tile_bytes(NG), ROWS = NB * 8, DP = NG * 32;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int last_one;
  const Share share = share_of<ROWS>(b, s, c.causal, w);
  if (blockIdx.x >= share.blocks) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q4 = lane & 3;
  const int G = s.H / s.KVH, D = s.D;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * ST * TB;

  int seq = share.seq;
  int64_t base = share.base, at = share.begin;
  Units un = units_of<ROWS>(b, s, seq, c.causal, w.bad);
  while (at < share.end) {
    if (at >= base + un.all(s.KVH)) {  // on to the next request with rows, 32 at a time
      base += un.all(s.KVH);
      for (;;) {
        const int i = seq + 1 + lane;
        const bool some = i < b.n_seq && units_of<ROWS>(b, s, min(i, b.n_seq - 1), c.causal, w.bad).row_blocks > 0;
        const uint32_t any = __ballot_sync(0xffffffffu, some);
        if (any) {
          seq += __ffs(any);
          break;
        }
        seq += 32;
      }
      un = units_of<ROWS>(b, s, seq, c.causal, w.bad);
    }
    const int64_t item = (at - base) / un.keys, first = base + item * un.keys;
    const int u0 = (int)(at - first), u1 = (int)min(un.keys, share.end - first);
    at = first + u1;
    const int kvh = (int)(item % s.KVH), r0 = (int)(item / s.KVH) * ROWS;
    const int rows = min(ROWS, un.q.n * G - r0), len = un.q.len;
    // keys that row x of the block sees
    auto limit = [&](int x) { return c.causal ? len - un.q.n + (r0 + min(x, rows - 1)) / G + 1 : len; };
    const int k_all = limit(0);                                         // every row sees these
    const int t0 = u0 * (kUnit / kTokens);
    const int t1 = min(u1 * (kUnit / kTokens), (limit(rows - 1) + kTokens - 1) / kTokens);
    const int mine = max(0, (t1 - t0 - warp + kWarps - 1) / kWarps);  // tiles of this warp

    // tiles' places in units of 128 bytes, of 32 of the warp's tiles (a lane each) and of the next 32
    auto places = [&](int n) {
      const int t = t0 + warp + (n + lane) * kWarps;
      if (n + lane >= mine) return kNoPlace;
      return place_of(b, s, seq, t, kvh, w.bad);
    };
    uint32_t window = places(0), ahead = places(32);
    auto issue = [&](int n, int stage) {
      if ((n & 31) == 0 && n > 0) {
        window = ahead;
        ahead = places(n + 32);
      }
      const uint32_t place = __shfl_sync(0xffffffffu, window, n & 31);
      if (place != kNoPlace) {
        const uint8_t *src = c.pages + (int64_t)place * 128;
#pragma unroll
        for (int i = 0; i < (TB / 16 + 31) / 32; ++i)
          if (i * 32 + lane < TB / 16) cp16(ring + stage * TB + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
      }
      return place != kNoPlace;
    };
    uint32_t there = 0;  // bit `stage`: its tile exists
#pragma unroll
    for (int n = 0; n < ST - 1; ++n) {
      if (n < mine && issue(n, n)) there |= 1u << n;
      asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q: lane 4 n + q4 has dimensions 32 g + 8 q4 .. of row n, as its column of the matrix product
    uint32_t qf[NB][NG][4];
    float qs[NB][NG][2], sc[NB][2];  // sums of a group (* 2^-24), and the score's factor, of rows 2 q4 and 2 q4 + 1
    int lim[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int x = nb * 8 + r, row = r0 + x;
      const bool have = x < rows;
      const T *q = (const T *)c.q + (un.q.row0 + row / G) * c.q_row + (int64_t)(kvh * G + row % G) * c.q_head;
      float v[NG][8], top = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int d = g * 32 + q4 * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[g][i] = 0.0f;
        if (have && d < D) load<8>(q + d, v[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[g][i])));
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
      }
      // 2^e brings the largest value to [2^10, 2^11); infinities and NaN make the row NaN
      const int e = min(100, 137 - (int)(__float_as_uint(top) >> 23));
      const float up = __uint_as_float((uint32_t)(e + 127) << 23);
      const float mul = top <= 3.402823466e38f ? up : __uint_as_float(0x7fc00000u);
      const float factor = c.scale * kLog2e * 16777216.0f * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 h = __floats2half2_rn(v[g][2 * i] * mul, v[g][2 * i + 1] * mul);
          const float2 f = __half22float2(h);
          sum += f.x + f.y;
          // pairs 1 and 3 meet codes that are 16 times as large
          qf[nb][g][i] = bits(i & 1 ? __hmul2(h, __float2half2_rn(0.0625f)) : h);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= 5.9604644775390625e-8f;  // 2^-24
        qs[nb][g][0] = __shfl_sync(0xffffffffu, sum, 8 * q4);
        qs[nb][g][1] = __shfl_sync(0xffffffffu, sum, 8 * q4 + 4);
      }
      sc[nb][0] = __shfl_sync(0xffffffffu, factor, 8 * q4);
      sc[nb][1] = __shfl_sync(0xffffffffu, factor, 8 * q4 + 4);
      lim[nb][0] = limit(nb * 8 + 2 * q4);
      lim[nb][1] = limit(nb * 8 + 2 * q4 + 1);
    }

    float o[NB][NG][8], m[NB][2], l[NB][2];  // m: in units of log2
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[nb][g][i] = 0.0f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.0f;
    }

    int stage = 0;
    for (int n = 0; n < mine; ++n) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();  // every lane's copies of this stage, and the reads of the stage refilled next
      if (n + ST - 1 < mine) {
        const int to = stage == 0 ? ST - 1 : stage - 1;
        there = issue(n + ST - 1, to) ? there | 1u << to : there & ~(1u << to);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      const uint8_t *tile = sm + (warp * ST + stage) * TB;
      const bool have = (there >> stage) & 1;
      if (++stage == ST) stage = 0;
      if (!have) continue;
      const int j = (t0 + warp + n * kWarps) * kTokens;
      __syncwarp();  // the products below take a whole warp

      // scores
      float x[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[nb][i] = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 k = *reinterpret_cast<const uint2 *>(tile + g * 256 + lane * 8);
        const float2 p0 = __half22float2(*reinterpret_cast<const __half2 *>(tile + k_params(NG) + (r * NG + g) * 4));
        const float2 p1 = __half22float2(*reinterpret_cast<const __half2 *>(tile + k_params(NG) + ((r + 8) * NG + g) * 4));
        const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, kx = k.x >> 8, ky = k.y >> 8;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma(a, k.x & lo, k.y & lo, k.x & hi, k.y & hi, qf[nb][g][0], qf[nb][g][1]);
          mma(a, kx & lo, ky & lo, kx & hi, ky & hi, qf[nb][g][2], qf[nb][g][3]);
          x[nb][0] = fmaf(p0.x, a[0], fmaf(p0.y, qs[nb][g][0], x[nb][0]));
          x[nb][1] = fmaf(p0.x, a[1], fmaf(p0.y, qs[nb][g][1], x[nb][1]));
          x[nb][2] = fmaf(p1.x, a[2], fmaf(p1.y, qs[nb][g][0], x[nb][2]));
          x[nb][3] = fmaf(p1.x, a[3], fmaf(p1.y, qs[nb][g][1], x[nb][3]));
        }
      }
      const bool cut = j + kTokens > k_all;
      const int ja = j + 4 * (r >> 1) + (r & 1);  // the token of the matrix's row r; that of r + 8 is 2 on
      bool move = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[nb][i] *= sc[nb][i & 1];
          if (cut && ja + (i & 2) >= lim[nb][i & 1]) x[nb][i] = -INFINITY;
          move = move || x[nb][i] > m[nb][i & 1] + 8.0f;
        }
      // m moves only when a score passes it by 2^8: a weight is at most 256
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(x[nb][h], x[nb][2 + h]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            if (top > m[nb][h]) {
              const float f = ex2(m[nb][h] - top);
              m[nb][h] = top;
              l[nb][h] *= f;
#pragma unroll
              for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int i = h; i < 8; i += 2) o[nb][g][i] *= f;
            }
          }
        __syncwarp();
      }
      uint32_t pf[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float b0 = m[nb][0] == -INFINITY ? 0.0f : m[nb][0], b1 = m[nb][1] == -INFINITY ? 0.0f : m[nb][1];
        const float w0 = ex2(x[nb][0] - b0), w1 = ex2(x[nb][1] - b1), w2 = ex2(x[nb][2] - b0), w3 = ex2(x[nb][3] - b1);
        l[nb][0] += w0 + w2;
        l[nb][1] += w1 + w3;
        // keys by rows -> rows by keys: the other operand of the product with V
        pf[nb][0] = transpose8(bits(__floats2half2_rn(w0, w1)));
        pf[nb][1] = transpose8(bits(__floats2half2_rn(w2, w3)));
      }

      // O^T += V^T P^T
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 v = *reinterpret_cast<const uint2 *>(tile + v_codes(NG) + g * 256 + lane * 8);
        uint4 p = *reinterpret_cast<const uint4 *>(tile + v_params(NG) + (g * 4 + q4) * 16);
        if (cut) {  // behind the last token the page may hold anything
          const int left = len - j - 4 * q4;
          p.x &= left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
          p.z &= left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
          p.y &= left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
          p.w &= left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
        }
        const __half2 s0 = halves(p.x), s1 = halves(p.y), m0 = halves(p.z), m1 = halves(p.w);
        const __half2 c1024 = halves(0x64006400u), c64 = halves(0x54005400u);
        auto low = [&](uint32_t u, __half2 sc, __half2 mi) {
          return bits(__hfma2(__hsub2(halves((u & 0x000f000fu) | 0x64006400u), c1024), sc, mi));
        };
        auto high = [&](uint32_t u, __half2 sc, __half2 mi) {
          return bits(__hfma2(__hsub2(halves((u & 0x00f000f0u) | 0x54005400u), c64), sc, mi));
        };
        const uint32_t a0 = low(v.x, s0, m0), a1 = high(v.x, s0, m0), a2 = low(v.y, s1, m1), a3 = high(v.y, s1, m1);
        const uint32_t vx = v.x >> 8, vy = v.y >> 8;
        const uint32_t b0 = low(vx, s0, m0), b1 = high(vx, s0, m0), b2 = low(vy, s1, m1), b3 = high(vy, s1, m1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma(o[nb][g], a0, a1, a2, a3, pf[nb][0], pf[nb][1]);
          mma(o[nb][g] + 4, b0, b1, b2, b3, pf[nb][0], pf[nb][1]);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the rings are free

    // the four warps' results meet in shared memory: sums [warp][row][DP + 4], m and l [warp][row]
    constexpr int LD = DP + 4;
    float *so = reinterpret_cast<float *>(sm), *smm = so + kWarps * ROWS * LD, *sl = smm + kWarps * ROWS;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float lr = l[nb][h];
        lr += __shfl_xor_sync(0xffffffffu, lr, 4);
        lr += __shfl_xor_sync(0xffffffffu, lr, 8);
        lr += __shfl_xor_sync(0xffffffffu, lr, 16);
        const int x = warp * ROWS + nb * 8 + 2 * q4 + h;
        if (r == 0) {
          smm[x] = m[nb][h];
          sl[x] = lr;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
          *reinterpret_cast<float4 *>(so + x * LD + g * 32 + r * 4) =
              make_float4(o[nb][g][h], o[nb][g][2 + h], o[nb][g][4 + h], o[nb][g][6 + h]);
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == un.keys;
    const int quads = D / 4;
    auto finish = [&](int x, int d, float4 v, float M, float L) {
      const int row = r0 + x, h = kvh * G + row % G;
      const int64_t at_row = un.q.row0 + row / G;
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // no key: zeros
      alignas(8) T out[4] = {from_f32<T>(v.x * inv), from_f32<T>(v.y * inv), from_f32<T>(v.z * inv), from_f32<T>(v.w * inv)};
      *reinterpret_cast<uint2 *>((T *)c.out + at_row * c.o_row + (int64_t)h * c.o_head + d) = *reinterpret_cast<uint2 *>(out);
      if (d == 0 && c.lse) c.lse[at_row * s.H + h] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
    };
    float *slot = slot_of<ROWS, DP>(w, blockIdx.x, u0 == 0 ? 1 : 0);
    for (int u = threadIdx.x; u < rows * quads; u += kThreads) {
      const int x = u / quads, d = u % quads * 4;
      float mw[kWarps], M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int a = 0; a < kWarps; ++a) M = fmaxf(M, mw[a] = smm[a * ROWS + x]);
      const float from = M == -INFINITY ? 0.0f : M;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int a = 0; a < kWarps; ++a) {
        const float f = ex2(mw[a] - from);
        const float4 y = *reinterpret_cast<const float4 *>(so + (a * ROWS + x) * LD + d);
        L += f * sl[a * ROWS + x];
        v.x += f * y.x;
        v.y += f * y.y;
        v.z += f * y.z;
        v.w += f * y.w;
      }
      if (whole) {
        finish(x, d, v, M, L);
      } else {
        __stcg(reinterpret_cast<float4 *>(slot + x * DP + d), v);
        if (d == 0) {
          __stcg(slot + ROWS * DP + x, M);
          __stcg(slot + ROWS * (DP + 1) + x, L);
        }
      }
    }
    if (!whole) {
      // the blocks that hold parts of this item; the last to arrive joins them in their order
      auto block_of = [&](int64_t unit) { return ((unit + 1) * share.blocks - 1) / share.total; };
      const int64_t b0 = block_of(first), b1 = block_of(first + un.keys - 1);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int arrived = atomicAdd(w.counters + b0, 1);
        last_one = arrived == (int)(b1 - b0);
        if (last_one) w.counters[b0] = 0;
        __threadfence();
      }
      __syncthreads();
      if (last_one) {
        const int parts = (int)(b1 - b0) + 1;
        auto part = [&](int p) { return slot_of<ROWS, DP>(w, b0 + p, p == 0 ? 1 : 0); };
        for (int u = threadIdx.x; u < rows * quads; u += kThreads) {
          const int x = u / quads, d = u % quads * 4;
          float M = -INFINITY, L = 0.0f;
          for (int p = 0; p < parts; ++p) M = fmaxf(M, __ldcg(part(p) + ROWS * DP + x));
          const float from = M == -INFINITY ? 0.0f : M;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
          for (int p = 0; p < parts; ++p) {
            const float *sp = part(p);
            const float f = ex2(__ldcg(sp + ROWS * DP + x) - from);
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(sp + x * DP + d));
            L += f * __ldcg(sp + ROWS * (DP + 1) + x);
            v.x += f * y.x;
            v.y += f * y.y;
            v.z += f * y.z;
            v.w += f * y.w;
          }
          finish(x, d, v, M, L);
        }
      }
    }
    __syncthreads();  // shared memory becomes the rings again
  }
}

template <typename T, int NG, int NB>
cudaError_t launch_few(const Kv4Shape &s, const Kv4Rows &b, const Kv4AttnCall &c, const Kv4Work &w, cudaStream_t st) {
  constexpr int smem = few_smem<NG, NB>();
  auto *kernel = few_kernel<T, NG, NB>;
  static thread_local int ready = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && ready != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) ready = dev;
  }
  if (e != cudaSuccess) return e;
  kernel<<<w.sms * few_blocks(NB), kThreads, smem, st>>>(c, s, b, w);
  return cudaGetLastError();
}

template <typename T, int NG>
cudaError_t run(const Kv4Shape &s, const Kv4Rows &b, const Kv4AttnCall &c, const Kv4Work &w, cudaStream_t st) {
  const int64_t rows = (int64_t)b.max_new * (s.H / s.KVH);
  if (rows <= 8) return launch_few<T, NG, 1>(s, b, c, w, st);
  if (rows <= 16) return launch_few<T, NG, 2>(s, b, c, w, st);
  return launch_few<T, NG, 4>(s, b, c, w, st);
}

template <typename T>
cudaError_t run(const Kv4Shape &s, const Kv4Rows &b, const Kv4AttnCall &c, const Kv4Work &w, cudaStream_t st) {
  switch (s.ng) {
    case 1: return run<T, 1>(s, b, c, w, st);
    case 2: return run<T, 2>(s, b, c, w, st);
    case 3: return run<T, 3>(s, b, c, w, st);
    default: return run<T, 4>(s, b, c, w, st);
  }
}

}  // namespace

int64_t kv4_attn_blocks(int sms) { return (int64_t)sms * few_blocks(1); }

int64_t kv4_attn_floats(const Kv4Shape &s, int sms) {
  int64_t most = 0;
  for (int nb : {1, 2, 4}) most = std::max(most, (int64_t)sms * few_blocks(nb) * 2 * nb * 8 * (s.ng * 32 + 2));
  return most;
}

cudaError_t kv4_attn(const Kv4Shape &s, const Kv4Rows &b, const Kv4AttnCall &c, const Kv4Work &w, cudaStream_t st) {
  if (b.rows == 0) return cudaSuccess;
  return s.dtype == DT_F16 ? run<__half>(s, b, c, w, st) : run<__nv_bfloat16>(s, b, c, w, st);
}

}  // namespace ndl
