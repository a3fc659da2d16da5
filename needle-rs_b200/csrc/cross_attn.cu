// cross_attn.cu — attention of ragged query rows to encoder states of other
// lengths:
//   s_j = scale * q . k_j     out = sum_j e^(s_j) v_j / sum_j e^(s_j)
// over a request's keys, masked ones left out.
//
// The query heads that share a KV head are rows of one matrix: row r of a
// request and KV head is token r / G, head kvh * G + r % G (G = H / KVH), so K
// and V are read once for all of them.  One pass over the keys keeps a running
// maximum m and sum l for each row (f32); weights are e^(s - m), rounded to the
// operands' type for the product with V, whose sums are f32.
//
// Two kernels.  Up to 16 rows read K and V from HBM faster than any tensor
// core needs them: xattn_few_kernel streams them through a ring for each warp
// and multiplies with mma.sync.  More rows are bound by the
// exponentials and the products: xattn_tile_kernel runs both on tcgen05 with
// 128-row tiles in TMEM.
//
// Long key ranges are cut so that all SMs work; the cuts' partial results
// (unnormalised sums, m in units of log2, l) meet in xattn_join_kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "attn_tile.cuh"
#include "common.cuh"
#include "ops.h"
#include "rowio.cuh"
#include "tc_common.cuh"
#include "tma_encode.h"

namespace ndl {
namespace {

using namespace tc;

// Partial results of split `s` of an item's rows: [rows][DP] sums, then m and
// l of each row, in a piece of rows * (DP + 4) floats (16-byte multiples).
__device__ __forceinline__ float *partial(const XAttnWork &w, const XAttnItem &it, int s, int DP) {
  return w.ws + it.ws + (int64_t)s * it.rows * (DP + 4);
}

// ── few rows ────────────────────────────────────────────────────────────────

constexpr int kFewWarps = 4, kFewKeys = 16;
// Rows of an item: what one MMA takes.  Two MMAs' rows (17 to 32) were up to a quarter
// slower than a tile of 128 that is mostly empty (24 requests of 16 tokens x 2 heads of 128
// over 512 keys: 16.6 us, tile 12.5; 256 of 16 x 2 heads of 64 over 64 to 512: 32.6 and 29.5;
// 8 of 12 x 2 heads of 64 over 8k to 20k: 35 and 38), two items of 32 half as fast
// (64 requests of 32 x 2 heads of 64 over 2000 keys: 68 and 37).
constexpr int kFewRows = 16;
// Stages of a warp's ring: two, and 5 CTAs an SM, where registers allow that
// many (256 decode requests: 16.6 us, with three 17.7), else three.  LONE, a CTA an SM
// at most: five, since nothing else covers a load's latency (8 heads of 64 over 512 keys:
// one request 7.4 us for 8.5, 32 requests 8.0 for 9.4; four stages and six the same).
template <int DP, bool LONE>
constexpr int kFewStages = LONE ? 5 : DP == 64 ? 2 : 3;
template <int DP, bool LONE>
constexpr int kFewCtas = LONE ? 1 : DP == 64 ? 5 : 2;

template <int DP>
constexpr int kFewStageBytes = 2 * kFewKeys * DP * 2;  // K and V rows of 16 keys
template <int DP, bool LONE>
constexpr int kFewSmem = kFewWarps * kFewStages<DP, LONE> * (kFewStageBytes<DP> + 4);

__device__ __forceinline__ void ldm4(uint32_t *r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t *r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Up to 16 rows of one request and KV head.  Each of four warps takes
// every fourth block of 16 keys through its own ring of cp.async stages, with
// its own running maxima: no barrier until the warps' results meet in shared
// memory at the end.  Rows of masked keys, of keys past the item and dimensions
// past D are written as zeros by the copies themselves, so nothing that they
// hold can reach a product.  Ring rows are swizzled (16-byte chunk c of row r
// at c ^ (r & 7)): ldmatrix reads them without bank conflicts.
template <typename T, int DP, bool LONE>
__global__ void __launch_bounds__(kFewWarps * 32, kFewCtas<DP, LONE>)
    xattn_few_kernel(const XAttnItem *items, XAttnWork w, XAttnCall c) {
  constexpr int ST = kFewStages<DP, LONE>, CH = DP / 8, KS = DP / 16;  // 16-byte chunks of a row, MMA steps over the dimensions
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t *live_of = reinterpret_cast<uint32_t *>(sm + kFewWarps * ST * kFewStageBytes<DP>);
  pdl_trigger();
  const XAttnItem it = items[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int G = w.s.H / w.s.KVH, D = w.s.D;
  const int nblk = (it.klen + kFewKeys - 1) / kFewKeys;
  const uint8_t *mask = c.mask ? c.mask + it.k0 : nullptr;
  const uint32_t ring = smem_u32(sm) + warp * ST * kFewStageBytes<DP>;
  // this lane's 16-byte chunk of the first rows of the warp's next block: the
  // other rows follow RS rows apart, the next block 64 rows on
  constexpr int RS = 32 / CH;
  const int ch0 = lane % CH, row0 = lane / CH;
  const T *kp = (const T *)c.k + (it.k0 + warp * kFewKeys + row0) * c.k_row + (int64_t)it.kvh * c.k_head + ch0 * 8;
  const T *vp = (const T *)c.v + (it.k0 + warp * kFewKeys + row0) * c.v_row + (int64_t)it.kvh * c.v_head + ch0 * 8;
  const int64_t k_step = RS * c.k_row, v_step = RS * c.v_row;
  const bool have = ch0 * 8 < D;

  // The 16 attended bits of the warp's n-th block, from a window of 32 blocks
  // (lane i holds block i's): the mask's bytes are fetched for 32 blocks at once, all
  // loads in flight together.
  uint32_t window = 0;
  auto live_block = [&](int n) -> uint32_t {
    if ((n & 31) == 0) {
      const int j = ((n + lane) * kFewWarps + warp) * kFewKeys, left = min(max(it.klen - j, 0), kFewKeys);
      window = (1u << left) - 1;
      if (mask) {
        uint32_t seen = 0;
#pragma unroll
        for (int i = 0; i < kFewKeys; ++i)
          if (i < left) seen |= (mask[j + i] != 0 ? 1u : 0u) << i;
        window = seen;
      }
    }
    return __shfl_sync(0xffffffffu, window, n & 31);
  };
  auto issue = [&](int n, int stage) {  // the warp's n-th block, in order
    const uint32_t live = live_block(n);
    if (lane == 0) live_of[warp * ST + stage] = live;
    const uint32_t dst = ring + stage * kFewStageBytes<DP>;
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
      const int row = row0 + RS * i;
      const bool take = ((live >> row) & 1) && have;
      const uint32_t at = dst + row * (DP * 2) + ((ch0 ^ (row & 7)) << 4);
      cp16(at, take ? kp + i * k_step : (const T *)c.k, take);
      cp16(at + kFewKeys * DP * 2, take ? vp + i * v_step : (const T *)c.v, take);
    }
    kp += kFewWarps * kFewKeys * c.k_row;
    vp += kFewWarps * kFewKeys * c.v_row;
  };
  const int mine = (nblk - warp + kFewWarps - 1) / kFewWarps;  // blocks of this warp

#pragma unroll
  for (int n = 0; n < ST - 1; ++n) {
    if (n < mine) issue(n, n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // Q as MMA fragments (rows g and g + 8)
  uint32_t qf[KS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = h * 8 + g, r = it.r0 + i;
      const T *q = (const T *)c.q + (it.q0 + r / G) * c.q_row + (int64_t)(it.kvh * G + r % G) * c.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = ks * 16 + u * 8 + 2 * t;
          qf[ks][2 * u + h] = i < it.rows && d < D ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
        }
    }

  const float sc = c.scale * kLog2e;
  float o[2 * KS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

  int stage = 0;
  for (int n = 0; n < mine; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncwarp();  // every lane's copies of this stage, and the reads of the stage refilled next
    if (n + ST - 1 < mine) issue(n + ST - 1, stage == 0 ? ST - 1 : stage - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    __syncwarp();  // the matrix loads below take a whole warp
    const uint32_t live = live_of[warp * ST + stage];
    const uint32_t K = ring + stage * kFewStageBytes<DP>, V = K + kFewKeys * DP * 2;
    if (++stage == ST) stage = 0;
    if (!live) continue;
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t kf[4];
      const int row = (lane >> 4) * 8 + (lane & 7), ch = 2 * ks + ((lane >> 3) & 1);
      ldm4(kf, K + row * (DP * 2) + ((ch ^ (row & 7)) << 4));
      mma16<T>(s[0], qf[ks], kf[0], kf[1]);
      mma16<T>(s[1], qf[ks], kf[2], kf[3]);
    }
    uint32_t pf[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // row g, then g + 8
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float &x = s[n][2 * h + u];
          if (!((live >> (n * 8 + 2 * t + u)) & 1)) x = -INFINITY;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (mx > m[h]) {
        const float f = ex2((m[h] - mx) * sc);
        m[h] = mx;
        l[h] *= f;
#pragma unroll
        for (int n = 0; n < 2 * KS; ++n) {
          o[n][2 * h] *= f;
          o[n][2 * h + 1] *= f;
        }
      }
      const float base = m[h] == -INFINITY ? 0.0f : m[h] * sc;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = ex2(fmaf(s[n][2 * h], sc, -base)), p1 = ex2(fmaf(s[n][2 * h + 1], sc, -base));
        l[h] += p0 + p1;
        pf[2 * n + h] = pack2<T>(p0, p1);
      }
    }
    __syncwarp();
#pragma unroll
    for (int nb = 0; nb < KS; ++nb) {
      uint32_t vf[4];
      const int row = ((lane >> 3) & 1) * 8 + (lane & 7), ch = 2 * nb + (lane >> 4);
      ldm4t(vf, V + row * (DP * 2) + ((ch ^ (row & 7)) << 4));
      mma16<T>(o[2 * nb], pf, vf[0], vf[1]);
      mma16<T>(o[2 * nb + 1], pf, vf[2], vf[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the rings are free

  // the four warps' results: sums [warp][row][DP] (rows 8 floats apart in banks:
  // a quarter of a warp's stores meet no other's), m and l [warp][row]
  constexpr int R = kFewRows, LD = DP + 8;
  float *so = reinterpret_cast<float *>(sm), *smm = so + kFewWarps * R * LD, *sl = smm + kFewWarps * R;
  static_assert(kFewWarps * R * (LD + 2) * 4 <= kFewWarps * ST * kFewStageBytes<DP>, "the rings hold the results");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 8 + g;
    float lr = l[h];
    lr += __shfl_xor_sync(0xffffffffu, lr, 1);
    lr += __shfl_xor_sync(0xffffffffu, lr, 2);
    if (i >= it.rows) continue;
    if (t == 0) {
      smm[warp * R + i] = m[h] * sc;
      sl[warp * R + i] = lr;
    }
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n)
      *reinterpret_cast<float2 *>(so + (warp * R + i) * LD + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  const int quads = D / 4;  // 4 dimensions a thread
  for (int u = threadIdx.x; u < it.rows * quads; u += kFewWarps * 32) {
    const int i = u / quads, d = u % quads * 4;
    float mw[kFewWarps], M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int a = 0; a < kFewWarps; ++a) M = fmaxf(M, mw[a] = smm[a * R + i]);
    const float base = M == -INFINITY ? 0.0f : M;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int a = 0; a < kFewWarps; ++a) {
      const float f = ex2(mw[a] - base);
      const float4 v = *reinterpret_cast<const float4 *>(so + (a * R + i) * LD + d);
      L += f * sl[a * R + i];
      x.x += f * v.x;
      x.y += f * v.y;
      x.z += f * v.z;
      x.w += f * v.w;
    }
    if (it.nsplit > 1) {
      float *p = partial(w, it, it.split, DP);
      *reinterpret_cast<float4 *>(p + i * DP + d) = x;
      if (d == 0) {
        p[it.rows * DP + i] = M;
        p[it.rows * (DP + 1) + i] = L;
      }
      continue;
    }
    const int r = it.r0 + i, h = it.kvh * G + r % G;
    const int64_t row = it.q0 + r / G;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // no key: zeros
    *reinterpret_cast<uint2 *>((T *)c.out + row * c.o_row + (int64_t)h * c.o_head + d) =
        make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
    if (d == 0 && c.lse) c.lse[row * w.s.H + h] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
  }
}

// ── many rows ───────────────────────────────────────────────────────────────

constexpr int kRows = 128, kKeys = 64, kTileThreads = 256;

template <int DP>
struct Tile {
  static constexpr int kAtoms = DP / 64;  // 64-dimension parts of a row (128 bytes each)
  static constexpr int kQAtom = kRows * 128, kAtom = kKeys * 128, kQBytes = kAtoms * kQAtom, kBytes = kAtoms * kAtom;
  static constexpr int kStages = DP == 64 ? 4 : 2;  // K tiles, and V tiles, in flight
  static constexpr int kQ = 0, kK = kQBytes, kV = kK + kStages * kBytes, kBar = kV + kStages * kBytes;
  static constexpr int kSmem = kBar + 256 + 1024;
  // TMEM columns: two S (P over each), then O
  static constexpr int kO = 2 * kKeys, kCols = 256;
  static_assert(kO + DP <= kCols, "S and O fit half of TMEM");
};

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Which keys of tile j of an item are attended to: bit i of word i / 32 (the
// whole warp calls it).
struct Live {
  uint32_t w[kKeys / 32];
};
struct LiveBytes {  // on their way, a lane's
  uint8_t b[kKeys / 32];
};
__device__ __forceinline__ LiveBytes live_load(const uint8_t *mask, int klen, int j, int lane) {
  LiveBytes v;
#pragma unroll
  for (int q = 0; q < kKeys / 32; ++q) {
    const int i = j * kKeys + 32 * q + lane;
    v.b[q] = i >= klen ? 0 : mask ? mask[i] : 1;
  }
  return v;
}
__device__ __forceinline__ Live live_bits(const LiveBytes &b) {
  Live v;
#pragma unroll
  for (int q = 0; q < kKeys / 32; ++q) v.w[q] = __ballot_sync(0xffffffffu, b.b[q] != 0);
  return v;
}
__device__ __forceinline__ bool all_live(const Live &v) {
  uint32_t a = 0xffffffffu;
#pragma unroll
  for (int q = 0; q < kKeys / 32; ++q) a &= v.w[q];
  return a == 0xffffffffu;
}

// Up to 128 rows of one request and KV head, tiles of 64 keys.  Warp 0 loads K
// and V (TMA, a ring each), warps 1 and 3 issue the MMAs of S and of O (in one warp
// their waits delay each other: 157 us on 16 x 1024 x 2048 targets, 146 in two), warp 2
// (only with a mask) zeroes the V rows of keys that are not attended to (their weights
// are zero, but zero times NaN is not; without a mask warp 3 does that for the last tile;
// its mask bytes come a tile ahead and its stores are predicated, not looped over: with
// half of 1024 to 2048 keys masked 171 us for 220),
// and warps 4-7 turn scores into weights, a thread a row.  For tile j:
//   S(j) = Q K_j^T    M128 N64, both K-major in shared memory
//   P(j) = weights    TMEM, 16 bits, over S(j)
//   O += P(j) V_j     M128 N DP, P from TMEM, V MN-major
// S has two buffers: S(j+1) is multiplied while the softmax works on S(j).  m
// moves only when a row's maximum passes it by 2^8, and O is rescaled then: a
// weight is at most 256.
//
// The exponentials bind (4 a clock on each SM partition).  Half of TMEM and of
// the registers make two CTAs an SM: one loads, reduces or ends while the other
// is at its exponentials.  CTAs are persistent: K and V tiles keep coming across
// items, and the next item's Q is fetched while O is waited for and its first S
// multiplied while O is stored.  Against a CTA for each item: 31 us for 44 on 64 requests
// of 256 to 512 x 64 to 128 keys (8 heads), 141 for 148 on 16 of 512 to 1024 x 1024 to
// 2048 (16 heads, 64 dimensions), 62 for 70 on 8 of 1024 x 1500 (8 heads, 128).  Items
// come longest first and are dealt in snake order.  Barriers of S, P and O count tiles
// through all items.
template <typename T, int DP>
__global__ void __launch_bounds__(kTileThreads, 2)
    xattn_tile_kernel(const XAttnItem *items, int n_items, const __grid_constant__ CUtensorMap mk,
                      const __grid_constant__ CUtensorMap mv, XAttnWork w, XAttnCall c, int *err) {
  using L = Tile<DP>;
  constexpr int ST = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *sm = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t *k_full = (uint64_t *)(sm + L::kBar), *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
  uint64_t *v_ok = v_empty + ST, *q_full = v_ok + ST, *o_free = q_full + 1, *s_full = o_free + 1, *p_full = s_full + 2,
           *pv_done = p_full + 2, *done = pv_done + 2;  // done: of a warp's MMAs in flight, after a wait that ran out
  uint32_t *tmem_slot = (uint32_t *)(done + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = w.s.H / w.s.KVH, D = w.s.D;
  // this CTA's item of a round; n_items or more: none
  auto item_of = [&](int round) {
    return round * (int)gridDim.x + (int)(round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  };
  auto tiles = [](int klen) { return (klen + kKeys - 1) / kKeys; };
  // keys of tile j that the MMAs cover: a multiple of 16
  auto covered = [](int klen, int j) { return min(kKeys, (klen - j * kKeys + 15) & ~15); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&v_ok[s], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(o_free, 4);
    for (int b = 0; b < 2; ++b) {  // of even and odd tiles: a wait never lags by two phases
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);
      mbar_init(&pv_done[b], 1);
      mbar_init(&done[b], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *(volatile uint32_t *)tmem_slot;
  // not before TMEM is held: a kernel behind this one could take it and wait for this one's end
  pdl_trigger();
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, k_done = 0, v_done = 0;  // tiles requested, up to ST
      uint32_t ph = 0;
      for (int round = 0, i; ok && (i = item_of(round)) < n_items; ++round) {
        const int kvh = items[i].kvh, nt = tiles(items[i].klen), row0 = (int)items[i].k0;
        for (int j = 0; j < nt; ++j) {
          const int row = row0 + j * kKeys;
          if (!(ok = mbar_sleep_wait(&k_empty[s], ph ^ 1, err))) break;
          mbar_expect_tx(&k_full[s], L::kBytes);
          for (int a = 0; a < L::kAtoms; ++a)
            tma_load_3d(sm + L::kK + s * L::kBytes + a * L::kAtom, &mk, &k_full[s], 64 * a, kvh, row);
          k_done = min(k_done + 1, ST);
          if (!(ok = mbar_sleep_wait(&v_empty[s], ph ^ 1, err))) {
            mbar_drain(&k_full[s], ph);
            k_done = min(k_done, ST - 1);
            break;
          }
          mbar_expect_tx(&v_full[s], L::kBytes);
          for (int a = 0; a < L::kAtoms; ++a)
            tma_load_3d(sm + L::kV + s * L::kBytes + a * L::kAtom, &mv, &v_full[s], 64 * a, kvh, row);
          v_done = min(v_done + 1, ST);
          if (++s == ST) s = 0, ph ^= 1;
        }
      }
      // no copy may be in flight when the CTA leaves
      for (int u = 0; u < ST; ++u) {
        if (s-- == 0) s = ST - 1, ph ^= 1;
        if (u < k_done) mbar_drain(&k_full[s], ph);
        if (u < v_done) mbar_drain(&v_full[s], ph);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // S(t), where P(t-2) was.  Descriptors share their high word; the low one is
    // the address / 16 (and, MN-major, the distance of the 64-dimension parts).
    const uint32_t s16 = smem_u32(sm) >> 4, q16 = (s16 + (uint32_t)(L::kQ >> 4)) | (1u << 16);
    const uint64_t hi = umma_desc(sm) & 0xFFFFFFFF00000000ull;
    const int steps = (D + 15) / 16;
    int t = 0, seen = 0;  // tiles, items with keys
    for (int round = 0, i; ok && (i = item_of(round)) < n_items; ++round) {
      const int klen = items[i].klen, nt = tiles(klen);
      if (nt == 0) continue;
      ok = warp_wait(q_full, (uint32_t)seen++ & 1, err);
      for (int j = 0; j < nt && ok; ++j, ++t) {
        const int s = t % ST;
        if (!(ok = warp_wait(&k_full[s], (uint32_t)(t / ST) & 1, err))) break;
        if (t >= 2 && !(ok = warp_wait(&pv_done[t & 1], (uint32_t)((t - 2) >> 1) & 1, err))) break;
        tc_after();
        const uint32_t k = (s16 + (uint32_t)((L::kK + s * L::kBytes) >> 4)) | (1u << 16);
        const uint32_t id = f16_idesc<T>(covered(klen, j), false), d = tmem + (uint32_t)((t & 1) * kKeys);
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) {
          const uint32_t in = (uint32_t)((u & 3) * 2), qa = (u >> 2) * (L::kQAtom >> 4) + in, ka = (u >> 2) * (L::kAtom >> 4) + in;
          if (u < steps) umma_bf16_e(d, hi | (q16 + qa), hi | (k + ka), id, u ? 1u : 0u);
        }
        umma_commit_e(&s_full[t & 1]);
        umma_commit_e(&k_empty[s]);
      }
    }
    if (!ok) {
      umma_commit_e(&done[0]);
      mbar_drain(&done[0], 0);
    }
  } else if (warp == 3) {
    // O += P(t) V_j
    const uint32_t s16 = smem_u32(sm) >> 4;
    const uint64_t hi = umma_desc(sm) & 0xFFFFFFFF00000000ull;
    const uint32_t id = f16_idesc<T>(DP, true);
    int t = 0, seen = 0;
    for (int round = 0, i; ok && (i = item_of(round)) < n_items; ++round) {
      const int klen = items[i].klen, nt = tiles(klen);
      for (int j = 0; j < nt && ok; ++j, ++t) {
        const int s = t % ST, n = covered(klen, j) >> 4;
        if (!(ok = warp_wait(c.mask ? &v_ok[s] : &v_full[s], (uint32_t)(t / ST) & 1, err))) break;
        if (!c.mask && (j + 1) * kKeys > klen) {  // the last tile's rows past the item
          const int r0 = klen - j * kKeys;
          for (int u = lane; u < (16 * n - r0) * 8 * L::kAtoms; u += 32)
            *reinterpret_cast<uint4 *>(sm + L::kV + s * L::kBytes + u / 8 % L::kAtoms * L::kAtom +
                                       (r0 + u / (8 * L::kAtoms)) * 128 + u % 8 * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
        }
        if (!(ok = warp_wait(&p_full[t & 1], (uint32_t)(t >> 1) & 1, err))) break;
        // the last item's O has been read
        if (j == 0 && seen++ > 0 && !(ok = warp_wait(o_free, (uint32_t)seen & 1, err))) break;
        tc_after();
        const uint32_t v = (s16 + (uint32_t)((L::kV + s * L::kBytes) >> 4)) | ((uint32_t)(L::kAtom >> 4) << 16);
#pragma unroll
        for (int u = 0; u < kKeys / 16; ++u)
          if (u < n)
            umma_bf16_ts_e(tmem + L::kO, tmem + (uint32_t)((t & 1) * kKeys + 8 * u), hi | (v + 128 * u), id, (j | u) ? 1u : 0u);
        umma_commit_e(&pv_done[t & 1]);
        umma_commit_e(&v_empty[s]);
      }
    }
    if (!ok) {
      umma_commit_e(&done[1]);
      mbar_drain(&done[1], 0);
    }
  } else if (warp == 2 && c.mask) {
    int t = 0;
    for (int round = 0, i; ok && (i = item_of(round)) < n_items; ++round) {
      const int klen = items[i].klen, nt = tiles(klen);
      const uint8_t *mask = c.mask + items[i].k0;
      LiveBytes ahead = live_load(mask, klen, 0, lane);
      for (int j = 0; j < nt && ok; ++j, ++t) {
        const int s = t % ST;
        const Live live = live_bits(ahead);
        ahead = live_load(mask, klen, j + 1, lane);
        if (!(ok = warp_wait(&v_full[s], (uint32_t)(t / ST) & 1, err))) break;
        if (!all_live(live)) {  // 8 lanes a row, 4 rows at a time
          uint8_t *to = sm + L::kV + s * L::kBytes + lane * 16;
#pragma unroll
          for (int q = 0; q < kKeys / 32; ++q) {
            const uint32_t bits = live.w[q] >> (lane >> 3);
#pragma unroll
            for (int r = 0; r < 32; r += 4)
              if (!((bits >> r) & 1))
#pragma unroll
                for (int a = 0; a < L::kAtoms; ++a)
                  *reinterpret_cast<uint4 *>(to + a * L::kAtom + (32 * q + r) * 128) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[s]);
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, i = quarter * 32 + lane;  // this thread's row of an item
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tO = tmem + lanes + (uint32_t)L::kO;
    const float sc = c.scale * kLog2e;
    // an item's row of Q on its way to shared memory, K-major with the 128-byte swizzle
    const uint32_t q_to = smem_u32(sm + L::kQ) + i * 128;
    auto fetch_q = [&](const XAttnItem *it) {
      const int r = it->r0 + i;
      const bool mine = i < it->rows;
      const T *q = (const T *)c.q + (it->q0 + r / G) * c.q_row + (int64_t)(it->kvh * G + r % G) * c.q_head;
#pragma unroll
      for (int ch = 0; ch < DP / 8; ++ch) {
        const bool take = mine && ch * 8 < D;
        cp16(q_to + (ch >> 3) * L::kQAtom + (((ch & 7) ^ (lane & 7)) << 4), take ? q + ch * 8 : (const T *)c.q, take);
      }
    };
    auto have_q = [&] {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    if (item_of(0) < n_items && items[item_of(0)].klen > 0) {
      fetch_q(items + item_of(0));
      have_q();
    }
    int t = 0;
    for (int round = 0, at; ok && (at = item_of(round)) < n_items; ++round) {
      const int klen = items[at].klen, nt = tiles(klen), next = item_of(round + 1);
      const uint8_t *mask = c.mask ? c.mask + items[at].k0 : nullptr;
      float m = -INFINITY, l = 0.0f;
      // the bytes of a tile's mask are fetched a tile ahead
      Live live = live_bits(live_load(mask, klen, 0, lane));
      for (int j = 0; j < nt; ++j, ++t) {
        const bool whole = all_live(live);
        const LiveBytes ahead = live_load(mask, klen, j + 1, lane);
        if (!(ok = warp_wait(&s_full[t & 1], (uint32_t)(t >> 1) & 1, err))) break;
        tc_after();
        const uint32_t tS = tmem + lanes + (uint32_t)((t & 1) * kKeys);
        uint32_t s[kKeys];
        tmem_ld32_raw(tS, s);
        tmem_ld32_raw(tS + 32, s + 32);
        tmem_wait_ld();
        if (!whole) {
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (!((live.w[e >> 5] >> (e & 31)) & 1)) s[e] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kKeys; e += 2)
          mx[(e >> 1) & 3] = fmax3(mx[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool move = (top - m) * sc > 8.0f;  // also at the first attended key (m = -inf)
        float f = 1.0f;
        if (move) {
          f = ex2((m - top) * sc);
          m = top;
          l *= f;
        }
        if (j > 0 && __any_sync(0xffffffffu, move)) {
          if (!(ok = warp_wait(&pv_done[(t - 1) & 1], (uint32_t)((t - 1) >> 1) & 1, err))) break;
          tc_after();
#pragma unroll 1
          for (int q = 0; q < DP / 16; ++q) {
            uint32_t o[16];
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]),
                  "=r"(o[8]), "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                : "r"(tO + 16 * q));
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(tO + 16 * q, o);
          }
        }
        const float mc = m == -INFINITY ? 0.0f : m * sc;
        const uint64_t cc = f2pack(sc, sc), nm = f2pack(-mc, -mc);
        uint64_t sum[2] = {f2pack(0.0f, 0.0f), f2pack(0.0f, 0.0f)};
        __syncwarp();  // TMEM is read and written by whole warps
#pragma unroll
        for (int q = 0; q < kKeys / 32; ++q) {
          uint32_t pw[16];
          weights<T>(s + 32 * q, cc, nm, pw, sum);
          tmem_st16(tS + 16 * q, pw);
        }
        float l0, l1;
        f2unpack(fadd2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
        tmem_wait_st();
        tc_before();
        live = live_bits(ahead);
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t & 1]);
      }
      if (!ok) break;
      // every S of this item is done: the next one's Q may take its place
      const bool more = next < n_items && items[next].klen > 0;
      if (more) fetch_q(items + next);
      if (nt > 0 && !(ok = warp_wait(&pv_done[(t - 1) & 1], (uint32_t)((t - 1) >> 1) & 1, err))) break;
      tc_after();
      if (more) have_q();
      const XAttnItem *it = items + at;
      const int r = it->r0 + i, h = it->kvh * G + r % G, nsplit = it->nsplit, rows = it->rows;
      const int64_t row = it->q0 + r / G;
      const bool mine = i < rows;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
      T *out = (T *)c.out + row * c.o_row + (int64_t)h * c.o_head;
      float *p = partial(w, *it, it->split, DP);
#pragma unroll
      for (int q = 0; q < DP / 32; ++q) {
        uint32_t o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
        __syncwarp();  // rows past the item's left the last turn early
        if (nt > 0) {
          tmem_ld32_raw(tO + 32 * q, o);
          tmem_wait_ld();
          if (q == DP / 32 - 1) {
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
          }
        }
        if (!mine) continue;
        if (nsplit > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4 *>(p + (int64_t)i * DP + 32 * q + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (32 * q + e >= D) break;
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              u[k] = pack2<T>(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4 *>(out + 32 * q + e) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
      if (mine) {
        if (nsplit > 1) {
          p[rows * DP + i] = m * sc;
          p[rows * (DP + 1) + i] = l;
        } else if (c.lse) {
          c.lse[row * w.s.H + h] = l == 0.0f ? -INFINITY : fmaf(m * sc, kLn2, logf(l));
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  if (warp == 1) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kCols));
  }
}

// ── joining split ranges ────────────────────────────────────────────────────

// A warp for each row of a group (blockIdx.x) of items on the same rows:
// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, in the order of the splits.
template <typename T>
__global__ void xattn_join_kernel(const XAttnItem *groups, XAttnWork w, XAttnCall c, int DP) {
  pdl_wait();
  const XAttnItem it = groups[blockIdx.x];
  const int lane = threadIdx.x & 31, i = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= it.rows) return;
  const int G = w.s.H / w.s.KVH, D = w.s.D, r = it.r0 + i, h = it.kvh * G + r % G;
  const int64_t row = it.q0 + r / G, stride = (int64_t)it.rows * (DP + 4);
  const float *p = partial(w, it, 0, DP), *pm = p + it.rows * DP + i, *pl = pm + it.rows;
  // lane s holds split s's m and l of 32 splits at a time; their sums are fetched 8 at once
  float M = -INFINITY;
  for (int s = lane; s < it.nsplit; s += 32) M = fmaxf(M, pm[s * stride]);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.0f : M;
  float L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const bool own = 4 * lane < D;
  const float *po = p + (int64_t)i * DP + (own ? 4 * lane : 0);
  for (int s0 = 0; s0 < it.nsplit; s0 += 32) {
    const int n = min(32, it.nsplit - s0);
    const float f = lane < n ? ex2(pm[(s0 + lane) * stride] - base) : 0.0f;
    L += warp_sum(lane < n ? f * pl[(s0 + lane) * stride] : 0.0f);
    for (int s1 = 0; s1 < n; s1 += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = s1 + u < n ? *reinterpret_cast<const float4 *>(po + (s0 + s1 + u) * stride) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __shfl_sync(0xffffffffu, f, s1 + u);
        o[0] += w * v[u].x;
        o[1] += w * v[u].y;
        o[2] += w * v[u].z;
        o[3] += w * v[u].w;
      }
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  if (own)
    *reinterpret_cast<uint2 *>((T *)c.out + row * c.o_row + (int64_t)h * c.o_head + 4 * lane) =
        make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  if (lane == 0 && c.lse) c.lse[row * w.s.H + h] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
}

// ── launches ────────────────────────────────────────────────────────────────

template <typename T, int DP, bool LONE>
cudaError_t launch_few(const XAttnItem *items, const XAttnWork &w, const XAttnCall &c, int dev, cudaStream_t st) {
  constexpr int kSmem = kFewSmem<DP, LONE>;
  auto *kernel = xattn_few_kernel<T, DP, LONE>;
  static thread_local int ready = -1;
  if (ready != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    ready = dev;
  }
  kernel<<<w.n_few, kFewWarps * 32, kSmem, st>>>(items, w, c);
  return cudaGetLastError();
}
template <typename T, int DP>
cudaError_t few_rows(const XAttnItem *items, const XAttnWork &w, const XAttnCall &c, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  return w.n_few <= sms ? launch_few<T, DP, true>(items, w, c, dev, st) : launch_few<T, DP, false>(items, w, c, dev, st);
}

cudaError_t kv_map(CUtensorMap *map, const void *p, const XAttnShape &s, int64_t row, int64_t head) {
  const uint64_t dims[3] = {(uint64_t)s.D, (uint64_t)s.KVH, (uint64_t)s.k_rows};
  const uint64_t strides[2] = {(uint64_t)head * 2, (uint64_t)row * 2};
  const uint32_t box[3] = {64, 1, kKeys};
  return tma_map_tiled(map, s.dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p,
                       dims, strides, box);
}

template <typename T, int DP>
cudaError_t launch_tile(const XAttnItem *items, int n, const XAttnWork &w, const XAttnCall &c, int *err, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  auto *kernel = xattn_tile_kernel<T, DP>;
  static thread_local int ready = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && ready != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<DP>::kSmem);
    if (e == cudaSuccess) ready = dev;
  }
  CUtensorMap mk, mv;
  XAttnShape s = w.s;
  s.k_rows = std::max<int64_t>(s.k_rows, 1);  // no keys at all: nothing is loaded
  if (e == cudaSuccess) e = kv_map(&mk, c.k, s, c.k_row, c.k_head);
  if (e == cudaSuccess) e = kv_map(&mv, c.v, s, c.v_row, c.v_head);
  if (e != cudaSuccess) return e;
  int sms = 0;
  e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  kernel<<<std::min(n, 2 * sms), kTileThreads, Tile<DP>::kSmem, st>>>(items, n, mk, mv, w, c, err);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t run(const XAttnWork &w, const XAttnCall &c, int *err, cudaStream_t st) {
  const XAttnItem *few = w.items, *tile = few + w.n_few, *groups = tile + w.n_tile;
  cudaError_t e = launch_tile<T, DP>(tile, w.n_tile, w, c, err, st);
  if (e == cudaSuccess && w.n_few) e = few_rows<T, DP>(few, w, c, st);
  if (e != cudaSuccess || w.n_groups == 0) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)w.n_groups, (unsigned)((w.group_rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, xattn_join_kernel<T>, groups, w, c, DP);
}

// Keys of an item (a multiple of `unit`) for ranges of `keys` each, run by
// `slots` CTAs at a time: the length with the least estimated finish.  An item costs
// its units and `fixed` more; with no more items than slots the longest
// decides, else the sum over the slots and half an item of imbalance.  Splitting
// costs the join.
int64_t choose_chunk(const std::vector<int64_t> &keys, int unit, double fixed, double join, int slots) {
  int64_t longest = 1, total = 0;
  std::vector<int64_t> units;
  for (int64_t k : keys) {
    units.push_back(std::max<int64_t>(1, (k + unit - 1) / unit));
    longest = std::max(longest, units.back());
    total += units.back();
  }
  double best = 1e300;
  int64_t chunk = longest;
  for (int64_t c = longest;; c = std::min(c - 1, c * 9 / 10)) {
    if (c < 2 && c != longest) break;
    int64_t n = 0;
    for (int64_t u : units) n += (u + c - 1) / c;
    double t = (double)c + fixed;
    if (n > slots) t = std::max(t, (total + n * fixed) / slots + t / 2);
    if (c < longest) t += join;
    if (t < best) best = t, chunk = c;
    if (c <= 1 || n > 8 * (int64_t)slots + (int64_t)units.size()) break;
  }
  return std::min<int64_t>(chunk * unit, 1 << 24);  // an item's key arithmetic is 32-bit
}

}  // namespace

int64_t cross_attn_items(int64_t rows) { return (rows + kRows - 1) / kRows; }

XAttnSplit cross_attn_split(const XAttnShape &s, const uint64_t *q_start, const uint64_t *q_len, const uint64_t *k_start,
                            const uint64_t *k_len, size_t n_seq, int sms) {
  const int G = s.H / s.KVH, DP = s.D <= 64 ? 64 : 128;
  std::vector<XAttnItem> whole[2];  // few rows, tiles
  XAttnSplit out;
  // Requests of few rows beside others join them in tiles, which saves a launch that would
  // wait for theirs, while that adds at most 25 tiles of 64 keys (about as many
  // microseconds, an item's start and end counted as 4) to each of the CTAs.  24 requests of 1
  // to 17 tokens x 3 heads of 80 dimensions, up to 511 keys (2 tiles a CTA): 12.6 us, apart
  // 22.8; nine in ten of 1 token x 2 heads of 64, else 16: 100 requests of 64 to 511 keys (10)
  // 16.6 and 21.7, 200 (20) 24.4 and 26.8, 400 (41) 43 and 35; 100 of 64 to 4000 (44) 61 and 53.
  int64_t tiles = 0, added = 0;
  for (size_t i = 0; i < n_seq; ++i) {
    const int64_t rows = (int64_t)q_len[i] * G;
    if (rows > kFewRows) tiles += s.KVH;
    else if (rows > 0) added += s.KVH * (((int64_t)k_len[i] + kKeys - 1) / kKeys + 4);
  }
  const int64_t few_rows = tiles > 0 && added <= 25 * 2 * (int64_t)sms ? 0 : kFewRows;
  for (size_t i = 0; i < n_seq; ++i) {
    const int64_t rows = (int64_t)q_len[i] * G;
    const int kind = rows <= few_rows ? 0 : 1, step = kind == 0 ? kFewRows : kRows;
    for (int64_t r0 = 0; r0 < rows; r0 += step)
      for (int g = 0; g < s.KVH; ++g) {
        XAttnItem it{};
        it.q0 = (int64_t)q_start[i];
        it.k0 = (int64_t)k_start[i];
        it.klen = (int)k_len[i];
        it.r0 = (int)r0;
        it.rows = (int)std::min<int64_t>(step, rows - r0);
        it.kvh = g;
        it.nsplit = 1;
        whole[kind].push_back(it);
      }
  }
  std::vector<XAttnItem> groups;
  for (int kind = 0; kind < 2; ++kind) {
    std::vector<int64_t> keys;
    for (const XAttnItem &it : whole[kind]) keys.push_back(it.klen);
    std::vector<XAttnItem> items;
    if (!keys.empty()) {
      // few rows: a unit is 64 keys (16 a warp); a CTA's start and end cost
      // about as much as 8 of them, a join as 8.  Tiles: 4 of 64 keys, a join 6.
      const int occ = DP == 64 ? 5 : 2;
      const int64_t chunk = kind == 0 ? choose_chunk(keys, 64, 8.0, 8.0, sms * occ) : choose_chunk(keys, kKeys, 4.0, 6.0, sms * 2);
      for (XAttnItem it : whole[kind]) {
        const int klen = it.klen, unit = 64;
        it.nsplit = (int)std::max<int64_t>(1, (klen + chunk - 1) / chunk);
        if (it.nsplit > 1) {
          it.ws = out.ws_floats;
          out.ws_floats += (int64_t)it.nsplit * it.rows * (DP + 4);
          groups.push_back(it);
          out.group_rows = std::max(out.group_rows, it.rows);
        }
        const int64_t units = (klen + unit - 1) / unit, k0 = it.k0;
        for (int q = 0; q < it.nsplit; ++q) {
          const int64_t a = units * q / it.nsplit * unit, b = std::min<int64_t>(units * (q + 1) / it.nsplit * unit, klen);
          it.split = q;
          it.k0 = k0 + a;
          it.klen = (int)(b - a);
          items.push_back(it);
        }
      }
      // the longest first
      std::stable_sort(items.begin(), items.end(), [](const XAttnItem &a, const XAttnItem &b) {
        return a.klen > b.klen;
      });
    }
    (kind == 0 ? out.n_few : out.n_tile) = (int64_t)items.size();
    out.items.insert(out.items.end(), items.begin(), items.end());
  }
  out.n_groups = (int64_t)groups.size();
  out.items.insert(out.items.end(), groups.begin(), groups.end());
  return out;
}

cudaError_t cross_attn(const XAttnWork &w, const XAttnCall &c, int *err, cudaStream_t st) {
  if (w.s.dtype == DT_F16) return w.s.D <= 64 ? run<__half, 64>(w, c, err, st) : run<__half, 128>(w, c, err, st);
  return w.s.D <= 64 ? run<__nv_bfloat16, 64>(w, c, err, st) : run<__nv_bfloat16, 128>(w, c, err, st);
}

}  // namespace ndl
