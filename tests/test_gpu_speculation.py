"""Speculative decoding over the 4-bit cache: a step's tokens (the last one and its drafts) go through 8-bit products, into
the cache, to attention, to logits, and the drafts are checked; what was not taken is written over by the next step.

Each stage is held against 64-bit arithmetic on what the stage before it wrote."""
import numpy as np
import pytest

from conftest import load_pkg
from test_gpu_int8 import check, expected, quantized, random_weight
from test_gpu_verify import reference as verify_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import kv4_ref as ref  # noqa: E402

nb = load_pkg()


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


class Decoder:
    """One layer: embedding rows -> q, k, v (8-bit products) -> cache -> attention -> logits (8-bit product) -> verification."""

    def __init__(self, B, n_max, max_len, d, H, KVH, D, page, V, greedy):
        self.B, self.n_max, self.d, self.H, self.KVH, self.D, self.page, self.V = B, n_max, d, H, KVH, D, page, V
        self.R = R = B * (n_max + 1)
        self.width = -(-max_len // page)
        n_pages = B * self.width
        g = torch.Generator().manual_seed(5)
        self.w = {n: random_weight(*shape, s) for s, (n, shape) in enumerate((("q", (H * D, d)), ("k", (KVH * D, d)), ("v", (KVH * D, d)), ("o", (V, H * D))))}
        self.wd = {n: (a.cuda(), (s * (1.0 if n == "o" else 0.06)).cuda()) for n, (a, s) in self.w.items()}
        self.proj = {n: nb.Int8Plan(a.data_ptr(), s.data_ptr(), H * D if n == "o" else d, a.shape[0], R) for n, (a, s) in self.wd.items()}
        self.cache = nb.Kv4Plan(H, KVH, D, page, n_pages, B, R, nb.BF16)
        self.verify = nb.VerifyPlan(V, B, B * n_max, nb.BF16)
        self.pages = torch.full((n_pages * nb.kv4_page_bytes(KVH, D, page),), 0xff, dtype=torch.uint8, device="cuda")
        self.table = torch.randperm(n_pages, generator=g).to(torch.int32).view(B, self.width).cuda()
        self.emb = torch.randn((V, d), generator=g).bfloat16().cuda()
        e = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.tokens, self.row_start, self.kv_len, self.draft_start, self.drafts = i(R), i(B + 1), i(B), i(B + 1), i(B * n_max)
        self.x, self.q, self.k, self.v, self.a, self.logits = e(R, d), e(R, H, D), e(R, KVH, D), e(R, KVH, D), e(R, H, D), e(R, V)
        self.u, self.final, self.T = e(B * n_max, t=torch.float32), e(B, t=torch.float32), e(B, t=torch.float32)
        self.T.copy_(torch.tensor([0.0 if n % 3 == greedy else 0.8 for n in range(B)]))
        self.out, self.logp, self.len = i(B, n_max + 1), e(B, n_max + 1, t=torch.float32), i(B)
        self.batch = nb.Kv4Batch(self.row_start.data_ptr(), self.kv_len.data_ptr(), self.table.data_ptr(), B, R, self.width, n_max + 1)

    def step(self, st=None):
        p = lambda t: t.data_ptr()  # noqa: E731
        torch.index_select(self.emb, 0, self.tokens.long(), out=self.x)
        for n, to in (("q", self.q), ("k", self.k), ("v", self.v)):
            self.proj[n].matmul(p(self.x), self.R, p(to), nb.BF16, nb.BF16, stream=st)
        self.cache.append(p(self.pages), self.batch, p(self.k), p(self.v), stream=st)
        self.cache.attn(p(self.pages), self.batch, p(self.q), p(self.a), self.D ** -0.5, stream=st)
        self.proj["o"].matmul(p(self.a), self.R, p(self.logits), nb.BF16, nb.BF16, stream=st)
        self.verify.run(p(self.logits), p(self.draft_start), p(self.drafts), p(self.u), p(self.final), p(self.out), p(self.len), self.B,
                        self.B * self.n_max, self.n_max + 1, None, p(self.T), None, p(self.logp), stream=st)

    def results(self):
        return [t.clone() for t in (self.a, self.logits, self.out, self.len, self.logp, self.pages)]


def feed(m, rng, last, held, n):
    """The next step's tokens: each request's last one and n[i] drafts, its cache holding held[i] tokens."""
    start = np.cumsum([0] + [a + 1 for a in n])
    ds = np.cumsum([0] + n)
    drafts = rng.integers(0, m.V, ds[-1])
    tokens = np.zeros(m.R, np.int64)
    for i in range(m.B):
        tokens[start[i]:start[i + 1]] = [last[i], *drafts[ds[i]:ds[i + 1]]]
    lens = [held[i] + n[i] + 1 for i in range(m.B)]
    for t, v in ((m.tokens, tokens), (m.row_start, start), (m.kv_len, lens), (m.draft_start, ds)):
        t.copy_(torch.tensor(np.asarray(v), dtype=torch.int32))
    m.drafts[:ds[-1]] = torch.tensor(drafts, dtype=torch.int32)
    m.u.copy_(torch.tensor(rng.random(m.u.numel()) * 1e-3, dtype=torch.float32))  # many drafts pass
    m.final.copy_(torch.tensor(rng.random(m.B), dtype=torch.float32))
    return start, ds, drafts, lens


def verify_step(m, keys, values, held, start, ds, drafts, lens):
    """Every stage of a step against 64 bits; the cache's tokens are kept in keys and values."""
    for plan in (*m.proj.values(), m.cache, m.verify):
        plan.status()
    n = start[-1]
    c = lambda t: t.cpu()  # noqa: E731

    def product(x, name, got):
        q8, qs = quantized(c(x))
        check(got, *expected(torch.from_numpy(q8), torch.from_numpy(qs), m.w[name][0], c(m.wd[name][1]), None, x.shape[1]), nb.BF16)

    for name, got in (("q", m.q), ("k", m.k), ("v", m.v)):
        product(m.x, name, got.view(m.R, -1))
    for i in range(m.B):
        keys[i] = torch.cat([keys[i][:held[i]], m.k[start[i]:start[i + 1]]])
        values[i] = torch.cat([values[i][:held[i]], m.v[start[i]:start[i + 1]]])
    rows = [(int(start[i]), int(start[i + 1] - start[i])) for i in range(m.B)]
    want, _, eo, _ = ref.attention(m.q, [ref.stored(k, v) for k, v in zip(keys, values)], rows, lens, m.D ** -0.5, True)
    f = torch.finfo(torch.bfloat16)
    tol = eo + f.eps / 2 * (want.abs() + eo) + f.tiny * f.eps / 2
    assert ((m.a.double() - want).abs() <= tol)[:n].all()
    product(m.a.view(m.R, -1)[:n], "o", m.logits[:n])
    out, ln, logp = verify_reference(c(m.logits[:n]), None, [int(a) for a in ds], torch.tensor(drafts), None, c(m.T), c(m.u), c(m.final), False,
                                     m.n_max + 1)
    assert np.array_equal(c(m.out).numpy(), out) and np.array_equal(c(m.len).numpy(), ln)
    # f32 exponentials and sums of logits whose size is below 2^6 / 0.8
    assert np.abs(c(m.logp).double().numpy() - logp).max() <= 2.0 ** -24 * (16 + 4 * float(m.logits[:n].abs().max()) / 0.8 + 2 * np.abs(logp).max())
    return out, ln


@pytest.mark.parametrize("B,n_max,d,H,KVH,D,page,V,prompt", [(6, 4, 256, 8, 4, 64, 16, 1000, 40), (3, 7, 192, 12, 4, 80, 32, 777, 300), (1, 3, 512, 8, 2, 128, 64, 4100, 1)])
def test_steps_of_speculative_decoding(B, n_max, d, H, KVH, D, page, V, prompt):
    rng = np.random.default_rng(B)
    m = Decoder(B, n_max, prompt + 60, d, H, KVH, D, page, V, 0)
    twin = Decoder(B, n_max, prompt + 60, d, H, KVH, D, page, V, 0)  # replays a graph of the same step
    graph = torch.cuda.CUDAGraph()
    for p in (*twin.proj.values(), twin.cache, twin.verify):
        p.status()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        twin.step(torch.cuda.current_stream().cuda_stream)
    keys, values = ([torch.zeros((0, KVH, D), dtype=torch.bfloat16, device="cuda")] * B for _ in range(2))
    held, last, taken = [0] * B, list(rng.integers(0, V, B)), 0
    # the prompts come as runs of drafts that all count as taken
    prompts = [[int(t) for t in rng.integers(0, V, int(rng.integers(1, prompt + 1)))] for _ in range(B)]
    for turn in range(200):
        forced = [max(0, len(prompts[i]) - held[i]) for i in range(B)]
        n = [min(n_max, f - 1) if f else int(rng.integers(0, n_max + 1)) for f in forced]
        state = rng.bit_generator.state
        start, ds, drafts, lens = feed(m, rng, last, held, n)
        for i in range(B):
            if forced[i]:
                run = prompts[i][held[i]:held[i] + n[i] + 1]
                m.tokens[int(start[i]):int(start[i + 1])] = torch.tensor(run, dtype=torch.int32)
                m.drafts[int(ds[i]):int(ds[i + 1])] = torch.tensor(run[1:], dtype=torch.int32)
                drafts[ds[i]:ds[i + 1]] = run[1:]
        rng.bit_generator.state = state
        feed(twin, rng, last, held, n)
        twin.tokens.copy_(m.tokens)
        twin.drafts.copy_(m.drafts)
        m.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(m.results(), twin.results()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        if turn < 2 or not any(forced):
            out, ln = verify_step(m, keys, values, held, start, ds, drafts, lens)
        else:
            out, ln = m.out.cpu().numpy(), m.len.cpu().numpy()
            for i in range(B):
                keys[i] = torch.cat([keys[i][:held[i]], m.k[start[i]:start[i + 1]]])
                values[i] = torch.cat([values[i][:held[i]], m.v[start[i]:start[i + 1]]])
        for i in range(B):
            if forced[i]:
                held[i] += n[i] + 1
                last[i] = int(out[i, int(ln[i]) - 1]) if int(ln[i]) == n[i] + 1 else 1
            else:
                taken += int(ln[i]) - 1
                held[i] += int(ln[i])
                last[i] = int(out[i, int(ln[i]) - 1])
        if not any(forced) and turn > 3 and (min(held) > prompt + 20 or max(held) > prompt + 60 - n_max - 2):
            break
    assert taken > 0 or not bool((m.T > 0).any())  # random drafts are hardly ever the largest logit
