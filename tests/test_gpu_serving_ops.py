"""The serving operators one behind the other, as a decoder layer's cross
attention uses them, eager and replayed from a graph.

Each step is held against 64-bit arithmetic on what the step before it wrote,
with that operator's own tolerance."""
import pytest

from conftest import load_pkg
from test_gpu_cross_attn import close as attn_close, reference as attn_reference
from test_gpu_int8 import check, expected, quantized, random_weight
from test_gpu_residual_norm import close, reference as norm_reference, rounded

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

nb = load_pkg()
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


class Layer:
    """x + gate * self-attention's y, its norm in 8 bits; q from that; attention to
    the encoder's keys and values; the output product; the second residual norm."""

    def __init__(self, ql, kl, d, H, KVH, D, with_mask):
        self.ql, self.kl, self.d, self.H, self.KVH, self.D = ql, kl, d, H, KVH, D
        self.M, self.R = sum(ql), sum(kl)
        self.qs, self.ks = ([sum(n[:i]) for i in range(len(n))] for n in (ql, kl))
        self.w = {n: random_weight(*shape, seed) for n, shape, seed in (("kv", (2 * KVH * D, d), 1), ("q", (H * D, d), 2), ("o", (d, H * D), 3))}
        self.wd = {n: (a.cuda(), (s / 16).cuda()) for n, (a, s) in self.w.items()}
        self.plan = {n: nb.Int8Plan(a.data_ptr(), s.data_ptr(), H * D if n == "o" else d, a.shape[0], self.R if n == "kv" else self.M)
                     for n, (a, s) in self.wd.items()}
        self.attn = nb.CrossAttnPlan(self.qs, ql, self.ks, kl, H, KVH, D, nb.BF16)
        e = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        M, R = self.M, self.R
        self.x, self.y, self.enc = e(M, d, t=torch.float32), e(M, d), e(R, d)
        g = torch.Generator().manual_seed(9)
        self.pre, self.pre2, self.post, self.chan = ((torch.randn(d, generator=g) * 0.1).cuda() for _ in range(4))
        self.gate = torch.tensor([0.3], device="cuda")
        self.mask = (torch.rand(R, generator=g) < 0.8).to(torch.uint8).cuda() if with_mask else None
        self.r, self.h8, self.hs = e(M, d, t=torch.float32), e(M, nb.int8_row_bytes(d), t=torch.int8), e(M, t=torch.float32)
        self.kv, self.q, self.a, self.o = e(R, 2, KVH, D), e(M, H, D), e(M, H, D), e(M, d)
        self.r2, self.h2 = e(M, d, t=torch.float32), e(M, d)
        self.scale = D ** -0.5

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        for t in (self.x, self.y, self.enc):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))

    def run(self, st):
        p = lambda t: t.data_ptr()  # noqa: E731
        self.plan["kv"].matmul(p(self.enc), self.R, p(self.kv), nb.BF16, nb.BF16, stream=st)
        nb.residual_norm(p(self.x), nb.F32, p(self.y), nb.BF16, self.M, self.d, p(self.pre), p(self.r), p(self.h8), nb.I8,
                         gate_ptr=p(self.gate), gate_flags=nb.GATE_SCALAR | nb.GATE_SIGMOID, h_scales_ptr=p(self.hs), stream=st)
        self.plan["q"].matmul_quantized(p(self.h8), p(self.hs), self.M, p(self.q), nb.BF16, stream=st)
        s = (2 * self.KVH * self.D, self.D)
        self.attn.run(p(self.q), p(self.kv), p(self.kv[:, 1]), p(self.a), self.scale, None, s, s,
                      key_mask_ptr=None if self.mask is None else p(self.mask), stream=st)
        self.plan["o"].matmul(p(self.a), self.M, p(self.o), nb.BF16, nb.BF16, stream=st)
        nb.residual_norm(p(self.r), nb.F32, p(self.o), nb.BF16, self.M, self.d, p(self.pre2), p(self.r2), p(self.h2), nb.BF16,
                         post_scale_ptr=p(self.post), gate_ptr=p(self.chan), gate_flags=nb.GATE_CHANNEL, stream=st)

    def results(self):
        return [t.clone() for t in (self.kv, self.r, self.h8, self.hs, self.q, self.a, self.o, self.r2, self.h2)]

    def verify(self):
        for p in [*self.plan.values(), self.attn]:
            p.status()
        c = lambda t: None if t is None else t.cpu()  # noqa: E731
        M, R, d, H, D = self.M, self.R, self.d, self.H, self.D

        def product(x, name, got):
            q, qs = quantized(x.cpu()) if not isinstance(x, tuple) else (c(x[0]).numpy(), c(x[1]).numpy())
            K = H * D if name == "o" else d
            check(got, *expected(torch.from_numpy(q), torch.from_numpy(qs), self.w[name][0], self.wd[name][1].cpu(), None, K), nb.BF16)

        product(self.enc, "kv", self.kv.view(R, -1))
        r, h, er, eh = norm_reference(c(self.x), c(self.y), None, c(self.gate), True, 1.0, c(self.pre))
        close(self.r, r, rounded(er, r, nb.F32))
        s, top = self.hs.double().cpu()[:, None], eh.amax(1, keepdim=True)
        # half a step of 8 bits, and two roundings of a quotient of up to 127 steps
        close(self.h8[:, :d] * self.hs[:, None].double(), h, eh + s * (0.5 + 4 * 127 * U) + top)
        product((self.h8, self.hs), "q", self.q.view(M, -1))
        out, _, eo, _ = attn_reference(c(self.q), c(self.kv[:, 0]), c(self.kv[:, 1]), c(self.mask), self.qs, self.ql, self.ks, self.kl, self.scale)
        attn_close(self.a, out, eo, nb.BF16)
        product(self.a.view(M, -1), "o", self.o)
        r, h, er, eh = norm_reference(c(self.r), c(self.o), c(self.post), c(self.chan), False, 1.0, c(self.pre2))
        close(self.r2, r, rounded(er, r, nb.F32))
        close(self.h2, h, rounded(eh, h, nb.BF16))


LAYERS = [([1] * 12, [64, 500, 1, 0, 33, 512, 100, 7, 300, 64, 65, 1000], 512, 8, 4, 64, False), ([1], [77], 512, 8, 4, 64, False),
          ([3, 0, 17, 130], [90, 5, 200, 700], 264, 6, 2, 40, True), ([40, 41], [129, 300], 1000, 4, 1, 128, True)]


@pytest.mark.parametrize("i", range(len(LAYERS)))
def test_a_decoder_layers_cross_attention(i):
    layer = Layer(*LAYERS[i])
    layer.fill(1)
    layer.run(None)
    torch.cuda.synchronize()
    layer.verify()


def test_a_captured_layer_replays_on_new_states():
    layer = Layer(*LAYERS[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        layer.run(torch.cuda.current_stream().cuda_stream)
    for seed in (2, 3):
        layer.fill(seed)
        g.replay()
        torch.cuda.synchronize()
        layer.verify()
        replayed = layer.results()
        layer.run(None)  # the same bits without the graph
        torch.cuda.synchronize()
        for a, b in zip(replayed, layer.results()):
            assert torch.equal(a, b)


def test_two_layers_on_two_streams():
    """Plans of their own: no order between the streams is needed."""
    layers = [Layer(*LAYERS[0]), Layer(*LAYERS[2])]
    want = []
    for n, layer in enumerate(layers):
        layer.fill(n + 5)
        layer.run(None)
        torch.cuda.synchronize()
        want.append(layer.results())
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for layer, st in zip(layers, streams):
            layer.run(st.cuda_stream)
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        layer.verify()
        for a, b in zip(w, layer.results()):
            assert torch.equal(a, b)


def test_an_error_is_reported_once():
    """A failed allocation is not the next call's result."""
    w, s = torch.zeros((16, 1 << 17), dtype=torch.int8, device="cuda"), torch.zeros(16, device="cuda")
    x, pre, h = torch.ones((2, 64), device="cuda"), torch.zeros(64, device="cuda"), torch.empty((2, 64), device="cuda")
    for _ in range(2):
        with pytest.raises(nb.NeedleError, match="CUDA error"):
            nb.Int8Plan(w.data_ptr(), s.data_ptr(), 131071, 16, 1 << 30)  # 128 TiB of rows
        nb.residual_norm(x.data_ptr(), nb.F32, None, nb.F32, 2, 64, pre.data_ptr(), None, h.data_ptr(), nb.F32)
    torch.cuda.synchronize()
    assert torch.isfinite(h).all()


@pytest.mark.parametrize("ql,kl,H,KVH,D", [([1] * 9, [400, 31, 0, 512, 7, 300, 1000, 64, 65], 8, 4, 64), ([3, 130], [700, 2500], 6, 2, 40)])
def test_attention_behind_norms_of_heads(ql, kl, H, KVH, D):
    """As the shipped model has it: query heads and key heads are normed between their product and the attention,
    by the residual norm without a block's output on a row for each token and head."""
    d, M, R = 512, sum(ql), sum(kl)
    qs, ks = ([sum(n[:i]) for i in range(len(n))] for n in (ql, kl))
    g = torch.Generator().manual_seed(D)
    p = lambda t: t.data_ptr()  # noqa: E731
    e = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    h, enc = (torch.randn(n, d, generator=g).bfloat16().cuda() for n in (M, R))
    q_scale, k_scale = ((torch.randn(D, generator=g) * 0.1).cuda() for _ in range(2))
    w = {n: random_weight(heads * D, d, seed) for n, heads, seed in (("q", H, 1), ("k", KVH, 2), ("v", KVH, 3))}
    wd = {n: (a.cuda(), (s / 16).cuda()) for n, (a, s) in w.items()}
    plan = {n: nb.Int8Plan(p(a), p(s), d, a.shape[0], M if n == "q" else R) for n, (a, s) in wd.items()}
    attn = nb.CrossAttnPlan(qs, ql, ks, kl, H, KVH, D, nb.BF16)
    q, qn, a, k, kn, v = e(M, H, D), e(M, H, D), e(M, H, D), e(R, KVH, D), e(R, KVH, D), e(R, KVH, D)
    plan["k"].matmul(p(enc), R, p(k), nb.BF16, nb.BF16)  # once a prompt
    plan["v"].matmul(p(enc), R, p(v), nb.BF16, nb.BF16)
    nb.residual_norm(p(k), nb.BF16, None, nb.BF16, R * KVH, D, p(k_scale), None, p(kn), nb.BF16)
    plan["q"].matmul(p(h), M, p(q), nb.BF16, nb.BF16)
    nb.residual_norm(p(q), nb.BF16, None, nb.BF16, M * H, D, p(q_scale), None, p(qn), nb.BF16)
    attn.run(p(qn), p(kn), p(v), p(a), D ** -0.5)
    for plan_ in [*plan.values(), attn]:
        plan_.status()
    for n, x, got in (("q", h, q), ("k", enc, k), ("v", enc, v)):
        x8, xs = quantized(x.cpu())
        check(got.view(got.shape[0], -1), *expected(torch.from_numpy(x8), torch.from_numpy(xs), w[n][0], wd[n][1].cpu(), None, d), nb.BF16)
    for x, s, got in ((q, q_scale, qn), (k, k_scale, kn)):
        _, want, _, err = norm_reference(x.view(-1, D).cpu(), None, None, None, False, 1.0, s.cpu())
        close(got.view(-1, D), want, rounded(err, want, nb.BF16))
    out, _, eo, _ = attn_reference(qn.cpu(), kn.cpu(), v.cpu(), None, qs, ql, ks, kl, D ** -0.5)
    attn_close(a, out, eo, nb.BF16)
