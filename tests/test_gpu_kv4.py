"""The 4-bit cache of keys and values on the GPU against 64-bit arithmetic."""
import itertools

import numpy as np
import pytest

from conftest import load_pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import kv4_ref as ref  # noqa: E402

nb = load_pkg()
TYPES = {nb.F16: torch.float16, nb.BF16: torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """Pages that start as NaN everywhere, handed to requests in a shuffled order, and what each
    request's tokens were."""

    def __init__(self, B, max_len, H, KVH, D, page, dtype, seed=0, max_rows=None, spare=3, plan=None):
        self.B, self.H, self.KVH, self.D, self.page, self.dtype, self.t = B, H, KVH, D, page, dtype, TYPES[dtype]
        self.width = max(1, -(-max_len // page))
        self.n_pages = B * self.width + spare
        self.page_bytes = nb.kv4_page_bytes(KVH, D, page)
        self.pages = torch.full((self.n_pages, self.page_bytes), 0xff, dtype=torch.uint8, device="cuda")
        self.g = torch.Generator().manual_seed(seed)
        self.order = torch.randperm(self.n_pages, generator=self.g)[:B * self.width].view(B, self.width)
        self.table = self.order.to(torch.int32).cuda()
        self.plan = plan or nb.Kv4Plan(H, KVH, D, page, self.n_pages, B, max_rows or max(1, B * max_len), dtype)
        e = torch.zeros((0, KVH, D), dtype=self.t)
        self.k, self.v = [e] * B, [e] * B

    def rows(self, n, gap=0):
        return [int(a) for a in np.cumsum([0] + [m + gap for m in n])]

    def batch(self, start, lens, rows):
        self.held = i32(start), i32(lens)
        return nb.Kv4Batch(self.held[0].data_ptr(), self.held[1].data_ptr(), self.table.data_ptr(), self.B, rows, self.width)

    def make(self, shape, width=1.0):
        chan = torch.exp(torch.randn(shape[1:], generator=self.g) * 0.5)
        return ((torch.randn(shape, generator=self.g) * chan + torch.randn(shape[1:], generator=self.g)) * width).to(self.t)

    def append(self, n, k=None, v=None, fused=False, keep=None, stream=None):
        """n[i] more tokens for request i, of which it holds keep[i] before."""
        start = self.rows(n)
        R = max(start[-1], 1)
        k = self.make((R, self.KVH, self.D)) if k is None else k
        v = self.make((R, self.KVH, self.D)) if v is None else v
        for i in range(self.B):
            old = len(self.k[i]) if keep is None else keep[i]
            self.k[i] = torch.cat([self.k[i][:old], k[start[i]:start[i + 1]]])
            self.v[i] = torch.cat([self.v[i][:old], v[start[i]:start[i + 1]]])
        if fused:  # the parts of a wider row
            wide = torch.full((R, 3, self.KVH, self.D + 8), 7.0, dtype=self.t, device="cuda")
            wide[:, 1, :, :self.D], wide[:, 2, :, :self.D] = k.cuda(), v.cuda()
            kd, vd = wide[:, 1, :, :self.D], wide[:, 2, :, :self.D]
        else:
            kd, vd = k.cuda(), v.cuda()
        b = self.batch(start, self.lens(), start[-1])
        self.plan.append(self.pages.data_ptr(), b, kd.data_ptr(), vd.data_ptr(), kd.stride()[:2], vd.stride()[:2], stream=stream)
        torch.cuda.synchronize()

    def lens(self):
        return [len(k) for k in self.k]

    def stored(self):
        return [ref.stored(k.cuda(), v.cuda()) for k, v in zip(self.k, self.v)]

    def check_read(self, n=None, heads_first=False, parts="kv"):
        """The last n[i] tokens of each request, into rows with some of no request between."""
        n = self.lens() if n is None else n
        start = self.rows(n)
        R = start[-1] + 2
        shape = (self.KVH, R, self.D) if heads_first else (R, self.KVH, self.D + 8)
        out = [torch.full(shape, 5.0, dtype=self.t, device="cuda") for _ in range(2)]
        view = [o.transpose(0, 1) if heads_first else o[..., :self.D] for o in out]
        b = self.batch(start, self.lens(), R)
        ptr = [o.data_ptr() if c in parts else None for o, c in zip(view, "kv")]
        self.plan.read(self.pages.data_ptr(), b, *ptr, view[0].stride()[:2], view[1].stride()[:2])
        self.plan.status()
        fin = torch.finfo(self.t)
        for o, c, which in zip(view, "kv", range(2)):
            assert (o[start[-1]:] == 5).all()
            if c not in parts:
                assert (o == 5).all()
                continue
            for i, s in enumerate(self.stored()):
                got, want = o[start[i]:start[i + 1]].double(), s[which][len(self.k[i]) - n[i]:]
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                # rounded once to the type, of a sum that f32 holds to 2^-24
                tol = want.abs() * (fin.eps / 2 * (1 + 2.0 ** -10)) + fin.tiny * fin.eps / 2
                assert ((got - want).abs() <= tol)[~torch.isnan(want)].all()
        if not heads_first:
            assert (out[0][..., self.D:] == 5).all() and (out[1][..., self.D:] == 5).all()

    def untouched(self):
        """Pages that no request holds, and those behind a request's tokens, are as they were."""
        used = torch.zeros(self.n_pages, dtype=torch.bool)
        for i, n in enumerate(self.lens()):
            used[self.order[i, :-(-n // self.page)]] = True
        assert (self.pages[~used.cuda()] == 0xff).all()


STORES = [
    ([1], 1, 64, 16, nb.BF16), ([65] * 4, 4, 64, 64, nb.BF16), ([16, 32, 48], 2, 128, 16, nb.F16), ([0, 1, 0, 15, 17, 0], 3, 80, 32, nb.F16),
    ([200, 3, 77], 1, 8, 16, nb.BF16), ([33, 31], 5, 40, 48, nb.F16), ([500, 1], 8, 128, 256, nb.BF16), ([100, 260], 2, 96, 128, nb.BF16),
    ([70], 3, 72, 16, nb.F16), ([129] * 3, 1, 32, 64, nb.F16), ([20], 130, 16, 16, nb.BF16),
]


@pytest.mark.parametrize("i", range(len(STORES)))
def test_tokens_come_back_as_their_four_bits(i):
    lens, KVH, D, page, dtype = STORES[i]
    c = Cache(len(lens), max(lens) + 40, KVH, KVH, D, page, dtype, i)
    c.append(lens, fused=i % 2 == 1)
    c.check_read()
    c.untouched()
    c.append([3 * (j % 3) for j in range(len(lens))])  # onto any token of a tile
    for _ in range(3):
        c.append([1] * len(lens))
    c.check_read(heads_first=True)
    c.check_read([min(5, n) for n in c.lens()])
    c.untouched()
    # drafts that were not taken are written over
    c.append([4] * len(lens), keep=[max(0, n - 3) for n in c.lens()])
    c.append([1] * len(lens), keep=[max(0, n - 2) for n in c.lens()])
    c.check_read(parts="k")
    c.check_read(parts="v")


def test_codes_at_every_boundary():
    """Groups whose values sit on codes, between them and next to the middle; equal values; tiny and large ones."""
    D, KVH = 64, 2
    x = torch.zeros((24, KVH, D))
    for i in range(16):
        x[i, :, :32] = torch.arange(32) * 0.5 * 2.0 ** (i - 8) - 3.0 * (i % 3)
    x[16] = 1.2345
    x[17] = -32768.0
    x[17, :, ::2] = 32768.0
    x[18] = torch.linspace(-6e-5, 6e-5, D)
    x[19] = 1e-7
    x[20] = 1000.0 + torch.linspace(0, 1, D)
    x[21, 0] = -0.0
    x[22] = torch.linspace(-1, 1, D) * 2.0 ** -20
    for dtype in TYPES:
        c = Cache(1, 32, KVH, KVH, D, 16, dtype)
        c.append([24], x.to(c.t), x.flip(-1).to(c.t))
        c.check_read()


def test_a_token_that_does_not_fit_is_nan_and_no_other():
    D, KVH = 80, 3
    for dtype in TYPES:
        c = Cache(1, 64, KVH, KVH, D, 16, dtype)
        k, v = c.make((40, KVH, D)), c.make((40, KVH, D))
        k[3, 0, 79] = float("inf")
        k[9, 1, 0] = float("nan")
        v[20, 2, 40] = -float("inf")
        v[21, 0, 5] = 40000.0
        v[33, 1, 31] = float("nan")
        c.append([40], k, v)
        assert sum(int(torch.isnan(s).any(-1).sum()) for s in c.stored()[0][:2]) == 10
        c.check_read()


def test_numbers_of_a_batch_that_do_not_fit_are_reported():
    """The other requests of the call are right, and nothing is touched behind the pages' ends."""
    c = Cache(4, 64, 4, 2, 64, 16, nb.BF16, spare=2)
    c.append([20, 30, 40, 50])
    good = c.table.clone()
    k = c.make((4, 2, 64)).cuda()
    q = c.make((4, 4, 64)).cuda()
    out, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)

    def calls(start, lens):
        b = c.batch(start, lens, 4)
        p = c.pages.data_ptr()
        return [lambda: c.plan.append(p, b, k.data_ptr(), k.data_ptr()), lambda: c.plan.read(p, b, ko.data_ptr(), vo.data_ptr()),
                lambda: c.plan.attn(p, b, q.data_ptr(), out.data_ptr(), 0.1)]

    for start, lens in (([0, 1, 2, 3, 5], [20, 30, 40, 50]), ([0, 1, 3, 2, 4], [20, 30, 40, 50]), ([0, 1, 2, 3, 4], [20, -1, 40, 50]),
                        ([0, 1, 2, 3, 4], [20, 30, 65, 50]), ([-1, 1, 2, 3, 4], [20, 30, 40, 50]), ([0, 1, 2, 3, 4], [20, 0, 40, 50])):
        for f in calls(start, lens):
            f()
            with pytest.raises(nb.NeedleError, match="out of range"):
                c.plan.status()
            c.plan.status()  # reported once
    for page in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        c.table.copy_(good)
        c.table[2, 2] = page  # of token 39
        for f in calls([0, 1, 2, 3, 4], [20, 30, 40, 50]):
            f()
            with pytest.raises(nb.NeedleError, match="out of range"):
                c.plan.status()
        c.table[2, 2] = good[2, 2]
        c.table[2, 3] = page  # behind the tokens: not read
        for f in calls([0, 1, 2, 3, 4], [20, 30, 40, 50]):
            f()
        c.plan.status()


class Attn:
    def __init__(self, cache, new, seed=1, width=1.0, gap=0, layout="token"):
        self.c, self.new = cache, new
        self.start = cache.rows(new)
        self.R = self.start[-1] + gap
        g = torch.Generator().manual_seed(seed)
        H, D = cache.H, cache.D
        q = (torch.randn((self.R, H, D), generator=g) * width).to(cache.t).cuda()
        if layout == "head":
            self.q = q.transpose(0, 1).contiguous().transpose(0, 1)
            self.out = torch.full((H, self.R, D), 7.0, dtype=cache.t, device="cuda").transpose(0, 1)
        elif layout == "fused":
            self.q = torch.full((self.R, 2, H, D + 8), 3.0, dtype=cache.t, device="cuda")[:, 1, :, :D]
            self.q.copy_(q)
            self.out = torch.full((self.R, H, D + 8), 7.0, dtype=cache.t, device="cuda")[..., :D]
        else:
            self.q, self.out = q, torch.full((self.R, H, D), 7.0, dtype=cache.t, device="cuda")
        self.lse = torch.full((self.R, H), 7.0, device="cuda")
        self.lens = cache.lens()
        self.held = i32(self.start), i32(self.lens)
        self.batch = nb.Kv4Batch(self.held[0].data_ptr(), self.held[1].data_ptr(), cache.table.data_ptr(), cache.B, self.R, cache.width,
                                 max(new))

    def run(self, scale, causal, stream=None, plan=None):
        (plan or self.c.plan).attn(self.c.pages.data_ptr(), self.batch, self.q.data_ptr(), self.out.data_ptr(), scale, causal,
                                   self.q.stride()[:2], self.out.stride()[:2], self.lse.data_ptr(), stream=stream)

    def check(self, scale, causal):
        self.c.plan.status()
        n = self.start[-1]
        rows = [(self.start[i], self.new[i]) for i in range(self.c.B)]
        out, lse, eo, el = ref.attention(self.q, self.c.stored(), rows, self.lens, scale, causal)
        f = torch.finfo(self.c.t)
        got = self.out.double()
        assert (got[n:] == 7).all() and (self.lse[n:] == 7).all()
        got, out, lse, eo, el, gl = got[:n], out[:n], lse[:n], eo[:n], el[:n], self.lse[:n].double()
        nan = torch.isnan(out)
        assert torch.equal(torch.isnan(got), nan)
        tol = eo + f.eps / 2 * (out.abs() + eo) + f.tiny * f.eps / 2
        assert ((got - out).abs() <= tol)[~nan].all(), float(((got - out).abs() / tol)[~nan].max())
        assert torch.equal(torch.isnan(gl), torch.isnan(lse)) and torch.equal(gl == -np.inf, lse == -np.inf)
        fin = torch.isfinite(lse)
        assert ((gl - lse).abs() <= el)[fin].all(), float(((gl - lse).abs() / el)[fin].max())


def attend(new, lens, H, KVH, D, page, dtype, causal, layout="token", width=1.0, scale=None, seed=0):
    c = Cache(len(lens), max(lens), H, KVH, D, page, dtype, seed, max_rows=max(sum(lens), sum(new) + 2, 1))
    c.append(lens)
    a = Attn(c, new, seed + 1, width, 2, layout)
    scale = D ** -0.5 if scale is None else scale
    a.run(scale, causal)
    a.check(scale, causal)
    first = a.out.clone()
    a.run(scale, causal)  # the same bits again
    c.plan.status()
    assert torch.equal(first.view(torch.int16), a.out.view(torch.int16))
    return c, a


SHAPES = [
    # requests' rows, tokens, heads, KV heads, dimensions, page, type, causal
    ([1], [1], 1, 1, 64, 16, nb.BF16, True), ([1], [0], 2, 1, 64, 16, nb.F16, False), ([1], [17], 4, 4, 32, 16, nb.F16, True),
    ([1] * 12, [64, 500, 1, 0, 33, 512, 100, 7, 300, 64, 65, 1000], 8, 4, 64, 64, nb.BF16, False),
    ([1] * 7, [16, 15, 31, 32, 33, 128, 129], 6, 2, 128, 16, nb.BF16, True),
    ([3, 0, 1, 9, 5], [3, 70, 1, 200, 1500], 12, 4, 80, 16, nb.F16, True),
    ([5, 0, 8], [700, 90, 64], 32, 4, 96, 32, nb.BF16, True), ([4, 4], [5, 20000], 4, 1, 128, 128, nb.F16, True),
    ([1], [40000], 8, 1, 64, 256, nb.BF16, True), ([17, 40], [17, 333], 8, 8, 40, 48, nb.F16, True),
    ([130, 1, 60], [130, 600, 61], 6, 3, 64, 16, nb.BF16, True), ([200], [1000], 16, 2, 128, 64, nb.F16, True),
    ([100, 0, 50], [0, 30, 700], 4, 2, 72, 16, nb.BF16, False), ([33], [33], 20, 1, 8, 16, nb.BF16, True),
    ([2, 2, 2], [50, 51, 52], 24, 1, 16, 16, nb.F16, True), ([70, 300], [2000, 4000], 16, 8, 128, 64, nb.BF16, True),
    ([1] * 40, [37 * i % 611 + 1 for i in range(40)], 64, 2, 112, 32, nb.F16, True),
    ([7] * 30, [90 + 53 * i % 700 for i in range(30)], 9, 3, 48, 16, nb.BF16, True),
    ([257], [300], 2, 1, 128, 16, nb.F16, True), ([300, 7], [301, 2000], 64, 2, 64, 32, nb.BF16, True), ([64, 64], [64, 128], 2, 2, 24, 16, nb.F16, False),
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(i):
    attend(*SHAPES[i], layout=("token", "head", "fused")[i % 3], seed=i)


@pytest.mark.parametrize("G,D,n", list(itertools.product((1, 2, 3, 5, 7, 8, 12, 16, 33, 128), (32, 64, 96, 128), (1, 2, 4))))
def test_attention_of_few_rows(G, D, n):
    """Every count of rows that share a KV head, on ranges that end anywhere in a tile."""
    attend([n] * 3, [n, 100 + G, 530 + D], 2 * G, 2, D, 32, (nb.F16, nb.BF16)[(G + n) % 2], True, seed=G * n)


@pytest.mark.parametrize("D", (24, 40, 64, 80, 128))
@pytest.mark.parametrize("n", (20, 65, 128, 129, 300))
def test_attention_of_many_rows(n, D):
    attend([n, n // 2, 1], [n, 513, 1025], 4, 2, D, 64, nb.BF16, True, seed=n)
    attend([n, n // 2, 0], [777, 1, 40], 3, 1, D, 16, nb.F16, False, seed=n)


@pytest.mark.parametrize("G,D,new,lens,page,dtype,causal", [
    (4, 128, [1024], [1024], 64, nb.BF16, True), (4, 64, [300, 1, 0, 257], [4000, 1, 17, 257], 16, nb.F16, True),
    (1, 96, [400, 129], [400, 2050], 32, nb.BF16, True), (8, 32, [64, 65, 33], [64, 65, 700], 48, nb.F16, True),
    (3, 80, [200, 90], [200, 5000], 16, nb.BF16, True), (2, 128, [600, 0, 5], [0, 70, 333], 128, nb.F16, False),
    (16, 40, [17, 100, 16], [17, 100, 3000], 256, nb.F16, True), (5, 112, [90] * 7, [90 + 131 * i for i in range(7)], 64, nb.BF16, True),
    (2, 16, [1000], [1030], 16, nb.F16, True), (4, 72, [257, 63], [63, 2111], 32, nb.BF16, False),
])
def test_attention_of_whole_chunks(G, D, new, lens, page, dtype, causal):
    """Enough rows and heads for the tensor cores' tiles, items cut between blocks and joined among them."""
    attend(new, lens, 8 * G, 8, D, page, dtype, causal, layout=("token", "head", "fused")[D // 8 % 3], seed=D)


@pytest.mark.parametrize("width,scale", [(30.0, 0.3), (1e-4, 1.0), (1e4, 1e-5), (0.0, 1.0)])
@pytest.mark.parametrize("new", [[1, 2], [40, 130], [300, 290]])
def test_sharp_flat_and_scaled_rows(new, width, scale):
    """Weights that fall on one key, on all, and q far from one."""
    for dtype in TYPES:
        attend(new, [300, 2500], 8, 2, 64, 64, dtype, True, width=width, scale=scale)


@pytest.mark.parametrize("new,heads", [([3, 5], 4), ([40, 70], 4), ([200, 90], 32)])
def test_tokens_that_do_not_fit_reach_only_rows_that_see_them(new, heads):
    """A draft's infinity is behind the rows before it; the page behind the last token holds NaN from the start."""
    lens = [203, 90]
    c = Cache(2, 256, heads, 2, 64, 16, nb.F16)
    n = sum(lens)
    k, v = c.make((n, 2, 64)), c.make((n, 2, 64))
    k[lens[0] - 1, 0, 3] = float("nan")  # only the last row sees it
    v[n - 2, 1, 60] = float("inf")  # the last two
    c.append(lens, k, v)
    a = Attn(c, new)
    a.run(0.125, True)
    a.check(0.125, True)
    assert 0 < int(torch.isnan(a.out).any(-1).sum()) == heads // 2 * (1 + 2)


def test_offsets_past_32_bits():
    """Pages whose bytes are numbered past 2^32."""
    H, KVH, D, page = 8, 8, 128, 256
    n_pages = (1 << 32) // nb.kv4_page_bytes(KVH, D, page) + 40
    c = Cache(2, 600, H, KVH, D, page, nb.BF16, spare=0)
    c.pages = torch.empty((n_pages, c.page_bytes), dtype=torch.uint8, device="cuda")
    c.n_pages = n_pages
    c.plan = nb.Kv4Plan(H, KVH, D, page, n_pages, 2, 1200, nb.BF16)
    c.table = (n_pages - 1 - torch.arange(6, dtype=torch.int32, device="cuda") * 6).view(2, 3)
    c.append([600, 333])
    c.check_read()
    for new in ([1, 1], [70, 30], [600, 333]):
        a = Attn(c, new)
        a.run(0.1, True)
        a.check(0.1, True)


def test_a_captured_step_replays_on_other_lengths():
    """Append, attention and read in one graph; lengths, pages and rows change between replays."""
    B, H, KVH, D = 5, 8, 2, 64
    c = Cache(B, 400, H, KVH, D, 16, nb.BF16, max_rows=2000)
    c.append([100, 3, 250, 0, 31])
    n = [1, 4, 2, 3, 6]
    start = c.rows(n)
    R = start[-1]
    k, v, q = (torch.empty((R, h, D), dtype=c.t, device="cuda") for h in (KVH, KVH, H))
    out, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    lse = torch.zeros((R, H), device="cuda")
    st, ln = i32(start), i32(c.lens())
    b = nb.Kv4Batch(st.data_ptr(), ln.data_ptr(), c.table.data_ptr(), B, R, c.width)

    def step(s):
        c.plan.append(c.pages.data_ptr(), b, k.data_ptr(), v.data_ptr(), stream=s)
        c.plan.attn(c.pages.data_ptr(), b, q.data_ptr(), out.data_ptr(), 0.125, lse_ptr=lse.data_ptr(), stream=s)
        c.plan.read(c.pages.data_ptr(), b, ko.data_ptr(), vo.data_ptr(), stream=s)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        step(torch.cuda.current_stream().cuda_stream)
    for turn, n in enumerate(([1, 4, 2, 3, 6], [1, 1, 1, 1, 1], [0, 9, 0, 0, 7], [0] * 5)):
        start = c.rows(n)
        st.copy_(i32(start))
        kk, vv = c.make((R, KVH, D)), c.make((R, KVH, D))
        for i in range(B):
            c.k[i], c.v[i] = torch.cat([c.k[i], kk[start[i]:start[i + 1]]]), torch.cat([c.v[i], vv[start[i]:start[i + 1]]])
        ln.copy_(i32(c.lens()))
        k.copy_(kk)
        v.copy_(vv)
        q.copy_(c.make((R, H, D)))
        for t in (out, ko, vo, lse):
            t.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        a = Attn.__new__(Attn)
        a.c, a.new, a.start, a.R, a.lens, a.q, a.out, a.lse = c, n, start, R, c.lens(), q, out, lse
        a.check(0.125, True)
        for o, which in ((ko, 0), (vo, 1)):
            assert (o[start[-1]:] == 7).all()
            for i, s in enumerate(c.stored()):
                want = s[which][len(c.k[i]) - n[i]:]
                assert ((o[start[i]:start[i + 1]].double() - want).abs() <= want.abs() * 2.0 ** -8).all()
        replayed = [t.clone() for t in (out, ko, vo, lse)]
        step(None)
        torch.cuda.synchronize()
        for x, y in zip(replayed, (out, ko, vo, lse)):
            assert torch.equal(x, y)


def test_two_plans_on_two_streams():
    parts, want = [], []
    for i, (new, lens) in enumerate((([1] * 6, [900, 5000, 30, 1, 77, 2048]), ([390, 400], [400, 1000]))):
        c = Cache(len(lens), max(lens), 8, 2, 128, 64, nb.F16, i, max_rows=sum(lens))
        c.append(lens)
        a = Attn(c, new)
        a.run(0.09, True)
        a.check(0.09, True)
        parts.append(a)
        want.append(a.out.clone())
    streams = [torch.cuda.Stream() for _ in parts]
    for _ in range(20):
        for a, s in zip(parts, streams):
            a.run(0.09, True, s.cuda_stream)
    torch.cuda.synchronize()
    for a, w in zip(parts, want):
        a.c.plan.status()
        assert torch.equal(a.out, w)


def test_parts_that_are_not_there():
    """Without a bound of rows, and outputs that are NULL with strides of 0."""
    c = Cache(2, 64, 4, 2, 64, 16, nb.F16)
    c.append([20, 33])
    a = Attn(c, [3, 5])
    a.batch.max_new = 0
    a.run(0.125, True)
    a.check(0.125, True)
    L, o = nb.lib(), torch.zeros((8, 2, 64), dtype=c.t, device="cuda")
    assert L.needle_kv4_read(c.plan._h, c.pages.data_ptr(), a.batch._ref, None, 0, 0, o.data_ptr(), 128, 64, None) == 0
    assert L.needle_kv4_read(c.plan._h, c.pages.data_ptr(), a.batch._ref, None, 0, 0, None, 0, 0, None) == -1
    c.plan.status()
    assert torch.equal(o[:3].double(), c.stored()[0][1][-3:].half().double())


def test_requests_that_share_pages():
    """A prefix of several requests in the same pages."""
    c = Cache(3, 128, 4, 2, 64, 16, nb.BF16)
    c.append([64, 0, 0])
    c.table[1, :4] = c.table[0, :4]
    c.table[2, :4] = c.table[0, :4]
    for i in (1, 2):
        c.k[i], c.v[i] = c.k[0], c.v[0]
    c.append([7, 20, 33])
    a = Attn(c, [7, 20, 1])
    a.run(0.125, True)
    a.check(0.125, True)


def test_requests_that_share_rows_do_nothing():
    # row starts that rise and fall: 131,073 requests of the same 65,536 rows, 2^32 tiles and more
    R, n = 65536, 2 * 131073
    plan = nb.Kv4Plan(8, 8, 8, R, 1, n, R, nb.F16)
    pages = torch.full((nb.kv4_page_bytes(8, 8, R),), 0xff, dtype=torch.uint8, device="cuda")
    start, lens, table = i32([0, R] * (n // 2) + [0]), i32([R] * n), i32([0] * n)
    b = nb.Kv4Batch(start.data_ptr(), lens.data_ptr(), table.data_ptr(), n, R, 1)
    x = torch.ones((R, 8, 8), dtype=torch.float16, device="cuda")
    out, ko, vo = (torch.full_like(x, 7.0) for _ in range(3))
    for f in (lambda: plan.append(pages.data_ptr(), b, x.data_ptr(), x.data_ptr()),
              lambda: plan.read(pages.data_ptr(), b, ko.data_ptr(), vo.data_ptr()),
              lambda: plan.attn(pages.data_ptr(), b, x.data_ptr(), out.data_ptr(), 0.1)):
        f()
        with pytest.raises(nb.NeedleError, match="out of range"):
            plan.status()
    assert (pages == 0xff).all() and all((t == 7.0).all() for t in (out, ko, vo))
