// kv4_share.cuh — how the work of an attention to the 4-bit cache falls to the
// blocks of a launch.
//
// Lengths are in device memory, so the blocks find their shares themselves.  A
// request's work is a row of items (query rows of a KV head), each a number of
// units of 64 keys; block b of n takes units [total * b / n, total * (b + 1) / n) of all
// requests' in order.  A border inside a short item moves to that item's nearer end:
// such items stay whole; longer ones are cut, and their parts joined by the last block to arrive.
// An item's first units stand for its start and end and hold no keys.
#pragma once
#include "kv4.cuh"

namespace ndl {
namespace kv4 {

constexpr int kUnit = 64;  // keys of a unit of work

struct Share {
  uint32_t total, begin, end, base;  // base: units before request `seq`, the one that `begin` falls in
  int blocks, seq;
  Seq q;  // request `seq`
};

// P: all(q): a request's units; item(q, at, &first, &units): the item of unit `at` of a request; snap(share): units of the
// longest item that stays whole; kLeast: units of a block at least.  A call of 2^31 units or more (2^37 keys) does nothing but say so.
template <class P, int W>
__device__ __forceinline__ void share_of(const P &p, const Kv4Rows &b, const Kv4Shape &s, bool causal, int *bad, Share *share) {
  constexpr int kThreads = W * 32;
  __shared__ uint64_t sums[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (b.n_seq + kThreads - 1) / kThreads, i0 = min((int)threadIdx.x * per, b.n_seq), i1 = min(i0 + per, b.n_seq);
  uint64_t own = 0;
  Seq q{0, 0, 0};
  for (int i = i0; i < i1; ++i) {
    q = sequence(b, s, i, causal, bad);
    own += min(p.all(q), (uint64_t)1 << 40);  // 2^20 requests' sum stays in 64 bits, whatever their numbers say
  }
  uint64_t sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  uint64_t in_all = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (k < warp) sum += sums[k];
    in_all += sums[k];
  }
  if (in_all >> 31) {
    *bad = 1;
    in_all = 0;
  }
  const uint32_t total = (uint32_t)in_all, upto = (uint32_t)sum, mine = (uint32_t)own;
  const uint32_t blocks = min(gridDim.x, (total + P::kLeast - 1) / P::kLeast), me = blockIdx.x;
  if (threadIdx.x == 0) {
    share->total = total;
    share->blocks = (int)blocks;
    share->end = total;
  }
  __syncthreads();
  if (me >= blocks) return;
  const uint32_t whole = total / blocks, rest = total - whole * blocks;
  const uint32_t lo = whole * me + rest * me / blocks, hi = whole * (me + 1) + rest * (me + 1) / blocks;
  const uint32_t before = upto - mine;
  if (before <= hi && lo < upto) {
    uint32_t base = before;
    for (int i = i0; i < i1; ++i) {
      if (per > 1) q = sequence(b, s, i, causal, bad);
      const uint32_t next = base + (uint32_t)p.all(q);
      auto border = [&](uint32_t x) {
        uint32_t first, n;
        p.item(q, x - base, &first, &n);
        const uint32_t in = x - base - first;
        return n > p.snap(whole) ? x : in * 2 < n ? x - in : x - in + n;
      };
      if (base <= lo && lo < next) {
        share->begin = border(lo);
        share->base = base;
        share->seq = i;
        share->q = q;
      }
      if (base <= hi && hi < next) share->end = border(hi);
      base = next;
    }
  }
  __syncthreads();
}
// The block that holds a unit of a cut item.
__device__ __forceinline__ int block_of(const Share &s, uint32_t unit) {
  return (int)((((uint64_t)unit + 1) * s.blocks - 1) / s.total);
}

// The next request with work behind `seq`, 32 at a time (the whole warp calls it); n_seq: none.
template <class P>
__device__ __forceinline__ int next_request(const P &p, const Kv4Rows &b, const Kv4Shape &s, int seq, bool causal, int *bad, Seq *q) {
  const int lane = threadIdx.x & 31;
  for (++seq; seq < b.n_seq; seq += 32) {
    const Seq next = sequence(b, s, min(seq + lane, b.n_seq - 1), causal, bad);
    const uint32_t any = __ballot_sync(0xffffffffu, seq + lane < b.n_seq && p.all(next) > 0);
    if (any) {
      const int from = __ffs(any) - 1;
      q->row0 = __shfl_sync(0xffffffffu, next.row0, from);
      q->n = __shfl_sync(0xffffffffu, next.n, from);
      q->len = __shfl_sync(0xffffffffu, next.len, from);
      return seq + from;
    }
  }
  return b.n_seq;
}

}  // namespace kv4
}  // namespace ndl
