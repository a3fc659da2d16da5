"""The 4-bit cache and the verification of drafts without a GPU: refusals come
before any CUDA call (the pointers are numbers that nothing may read), and the
checks that kernels make of a batch's numbers run here on the CPU."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, load_pkg

nb = load_pkg()
P = 1 << 20  # stands for an aligned device pointer


def refused(match, call, *a, **k):
    with pytest.raises(nb.NeedleError, match=match):
        call(*a, **k)


def test_page_bytes():
    assert nb.kv4_page_bytes(1, 128, 16) == 2560 and nb.kv4_page_bytes(4, 64, 64) == 4 * 4 * 1280
    assert nb.kv4_page_bytes(2, 80, 32) == 2 * 2 * 1920 and nb.kv4_page_bytes(1, 8, 16) == 640


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=nb.F32), "f16 or bf16"), (dict(dtype=nb.I8), "f16 or bf16"), (dict(D=0), "head_dim"), (dict(D=60), "head_dim"),
    (dict(D=136), "head_dim"), (dict(H=6), "num_heads"), (dict(H=0), "num_heads"), (dict(KVH=0), "num_heads"), (dict(H=8192), "num_heads"),
    (dict(page=0), "page_tokens"), (dict(page=24), "page_tokens"), (dict(page=65552), "page_tokens"), (dict(pages=0), "invalid number"),
    (dict(pages=1 << 31), "invalid number"), (dict(seqs=0), "invalid number"), (dict(seqs=(1 << 20) + 1), "invalid number"),
    (dict(page=65536, pages=100000), "512 GiB"), (dict(rows=0), "invalid number"), (dict(rows=1 << 31), "invalid number"),
])
def test_kv4_plan_refuses(bad, match):
    a = dict(H=8, KVH=4, D=64, page=16, pages=10, seqs=4, rows=64, dtype=nb.BF16)
    a.update(bad)
    refused(match, nb.Kv4Plan, a["H"], a["KVH"], a["D"], a["page"], a["pages"], a["seqs"], a["rows"], a["dtype"])


def test_null_plans():
    L = nb.lib()
    b = nb.Kv4Batch(P, P, P, 1, 1, 1)
    assert L.needle_kv4_append(None, P, b._ref, P, 64, 64, P, 64, 64, None) == -1
    assert L.needle_kv4_read(None, P, b._ref, P, 64, 64, P, 64, 64, None) == -1
    assert L.needle_kv4_attn(None, P, b._ref, P, 64, 64, 1.0, 0, P, 64, 64, None, None) == -1
    assert L.needle_kv4_plan_status(None) == -1 and nb.last_error() == "null plan"
    assert L.needle_verify_plan_run(None, P, 8, None, 1, P, P, None, 8, None, P, P, 1, 1, 0, P, None, 2, P, None) == -1
    assert L.needle_verify_plan_status(None) == -1 and nb.last_error() == "null plan"
    L.needle_kv4_plan_free(None)
    L.needle_verify_plan_free(None)


@pytest.mark.parametrize("bad,match", [(dict(V=0), "invalid verification plan"), (dict(V=(1 << 24) + 1), "invalid verification plan"),
                                       (dict(seqs=0), "invalid verification plan"), (dict(drafts=1 << 31), "invalid verification plan"),
                                       (dict(dtype=nb.I8), "f32, f16 or bf16"), (dict(dtype=9), "f32, f16 or bf16")])
def test_verify_plan_refuses(bad, match):
    a = dict(V=100, seqs=2, drafts=8, dtype=nb.F32)
    a.update(bad)
    refused(match, nb.VerifyPlan, a["V"], a["seqs"], a["drafts"], a["dtype"])


HARNESS = r"""
#include <cstdio>
#include <cstdint>
#include <set>
#include <vector>
#include "kv4.cuh"
using namespace ndl;
using namespace ndl::kv4;

static int fails = 0;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); ++fails; } } while (0)

int main() {
  // every token's bytes of a tile are inside it, no two tokens share one, and together they fill it
  for (int ng = 1; ng <= 4; ++ng) {
    std::vector<int> owner(tile_bytes(ng), -1);
    auto claim = [&](int at, int n, int t) {
      for (int i = 0; i < n; ++i) {
        CHECK(at + i >= 0 && at + i < tile_bytes(ng));
        CHECK(owner[at + i] == -1);
        owner[at + i] = t;
      }
    };
    for (int t = 0; t < kTokens; ++t)
      for (int g = 0; g < ng; ++g) {
        for (int q = 0; q < 4; ++q) claim(k_word(t, g, q), 4, t);
        for (int r = 0; r < 8; ++r) claim(v_half(ng, t, g, r), 2, t);
        for (int w = 0; w < 2; ++w) claim(k_param(ng, t, g, w), 2, t), claim(v_param(ng, t, g, w), 2, t);
        CHECK(k_word(t, g, 0) % 4 == 0 && v_half(ng, t, g, 0) % 2 == 0 && k_param(ng, t, g, 0) % 2 == 0);
      }
    for (int b : owner) CHECK(b >= 0);
  }

  // the division of a tile's number by a page's tiles
  for (int per = 1; per <= 4096; per += per < 70 ? 1 : 61) {
    Kv4Shape d{1, 1, 32, 1, per * 16, 1, 1, 640 * per, kv4_inverse(per * 16)};
    std::vector<int32_t> one(1 << 20);
    Kv4Rows e{nullptr, nullptr, one.data(), 1, 1 << 20, 1, 1};
    for (int64_t t : {0ll, 1ll, per - 1ll, (long long)per, per + 1ll, 1000ll * per - 1, 1000ll * per, (1ll << 26) / per * per - 1, (1ll << 26) - 1})
      if (t >= 0 && t / per < (1 << 20) && t < 1 << 26) CHECK(page_of(e, d, 0, (int)t).in == t % per);
    for (uint64_t t : {(1ull << 26) - 1, (1ull << 26) / per * per - 1, (1ull << 25) + 7}) CHECK((t * d.per_inverse) >> 38 == t / per);
  }

  // numbers that do not fit give a request without rows and tokens
  Kv4Shape s{8, 4, 64, 2, 32, 1, 10, 4 * 2 * 1280, kv4_inverse(32)};
  const int32_t start[] = {0, 3, 3, 2, 9, 12, -1, 5, 2147483647}, len[] = {64, 10, 10, 10, 97, -1, 10, 10};
  std::vector<int32_t> table(8 * 3, 0);
  Kv4Rows b{start, len, table.data(), 8, 3, 11, 7};
  struct { int i; bool inside; int n, len, bad; } want[] = {
      {0, true, 3, 64, 0}, {0, false, 3, 64, 0}, {1, true, 0, 10, 0}, {2, true, 0, 0, 1} /* falls */, {3, true, 7, 10, 0},
      {4, true, 0, 0, 1} /* 97 tokens in 3 pages of 32, and row 12 of 11 */, {5, false, 0, 0, 1} /* falls, length -1 */,
      {6, true, 0, 0, 1} /* starts at -1 */, {7, true, 0, 0, 1} /* row 2^31 - 1 */};
  for (auto &w : want) {
    int bad = 0;
    const Seq q = sequence(b, s, w.i, w.inside, &bad);
    CHECK(q.n == w.n && q.len == w.len && bad == w.bad);
    CHECK(q.row0 >= 0 && q.row0 + q.n <= b.rows);
  }
  const int32_t few[] = {2, 10};
  const int32_t two[] = {0, 3, 6};
  Kv4Rows c{two, few, table.data(), 2, 3, 6, 6};
  int bad = 0;
  CHECK(sequence(c, s, 0, true, &bad).n == 0 && bad == 1);  // three rows among two tokens
  bad = 0;
  CHECK(sequence(c, s, 0, false, &bad).n == 3 && bad == 0);

  c.max_new = 2;
  CHECK(sequence(c, s, 0, false, &bad).n == 0 && bad == 1);  // three rows where two are the most

  // pages outside the array are not addressed
  for (int32_t page : {-1, 10, 2147483647, (int32_t)0x80000000}) {
    table[4] = page;
    bad = 0;
    CHECK(tile_at((uint8_t *)4096, b, s, 1, 2, 0, &bad) == nullptr && bad == 1);
    CHECK(tile_at((uint8_t *)4096, b, s, 1, 3, 3, &bad) == nullptr);
    bad = 0;
    CHECK(tile_at((uint8_t *)4096, b, s, 1, 1, 3, &bad) != nullptr && bad == 0);
  }
  std::set<uint8_t *> tiles;
  for (int page = 0; page < 10; ++page)
    for (int t = 0; t < 2; ++t)
      for (int h = 0; h < 4; ++h) {
        table[0] = page;
        uint8_t *p = tile_at((uint8_t *)4096, b, s, 0, t, h, &bad);
        CHECK(p >= (uint8_t *)4096 && p + tile_bytes(2) <= (uint8_t *)4096 + 10 * s.page_bytes);
        CHECK(((uintptr_t)p & 127) == 0);
        CHECK(tiles.insert(p).second);
      }
  CHECK(bad == 0);
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_layout_and_checks_of_a_batch_on_the_cpu(tmp_path):
    nvcc = os.environ.get("NVCC", "nvcc")
    if not shutil.which(nvcc):
        pytest.skip("no nvcc")
    src = tmp_path / "harness.cu"
    src.write_text(HARNESS)
    exe = tmp_path / "harness"
    subprocess.run([nvcc, "-std=c++17", "-I" + os.path.join(PKG_DIR, "csrc"), str(src), "-o", str(exe), "-gencode",
                    "arch=compute_100a,code=sm_100a"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
