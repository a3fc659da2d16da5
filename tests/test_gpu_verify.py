"""Verification of drafts on the GPU against 64-bit arithmetic."""
import math

import numpy as np
import pytest

from conftest import load_pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

nb = load_pkg()
TYPES = {nb.F32: torch.float32, nb.F16: torch.float16, nb.BF16: torch.bfloat16}
NONE = -1  # 0xffffffff as int32


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


def reference(logits, ok, start, ids, probs, T, u, final, last_tie, width):
    """(ids, lengths, log-probabilities); logits [rows][V] and ok [rows][V] on the CPU."""
    B = len(start) - 1
    out, logp, lens = np.full((B, width), NONE, np.int64), np.zeros((B, width)), []
    V = logits.shape[1]
    for i in range(B):
        n, at, j = start[i + 1] - start[i], start[i] + i, 0
        while j <= n:
            z = logits[at + j].double().numpy()
            if ok is not None:
                z = np.where(ok[at + j].numpy(), z, -np.inf)
            if np.isnan(z).any() or (z == np.inf).any() or (z == -np.inf).all():
                break
            temp = float(T[i])
            z = z if temp <= 0 else z / temp
            top = z.max()
            w = np.exp(z - top)
            p = w / w.sum()
            d = int(ids[start[i] + j]) if j < n else -1
            known = 0 <= d < V
            best = np.flatnonzero(z == top)[-1 if last_tie else 0]
            if temp <= 0:
                take, token = j < n and d == best, best
            else:
                q = (probs[start[i] + j].double().numpy() if probs is not None else np.eye(1, V, d)[0] if known else np.zeros(V)) if j < n else None
                take = j < n and known and float(u[start[i] + j]) * q[d] < p[d]
                rest = p
                if j < n and np.maximum(p - q, 0).sum() > 0:
                    rest = np.maximum(p - q, 0)
                c = np.cumsum(rest)
                past = np.flatnonzero((c > float(final[i]) * c[-1]) & (rest > 0))
                token = past[0] if len(past) else np.flatnonzero(rest > 0)[-1]
            token = d if take else int(token)
            out[i, j], logp[i, j] = token, z[token] - top - math.log(w.sum())
            j += 1
            if not take:
                break
        lens.append(j)
    return out, np.array(lens), logp


def pack(ok, words):
    """Bits as 64-bit words, bit v % 64 of word v / 64."""
    a = np.zeros((ok.shape[0], words * 64), np.uint8)
    a[:, :ok.shape[1]] = ok.numpy()
    return torch.from_numpy(np.packbits(a, axis=1, bitorder="little").view(np.int64).copy())


class Case:
    def __init__(self, n, V, dtype, seed, probs=True, keep=None, temps=(1.0,), spread=2.0, noise=0.7):
        self.n, self.V, self.dtype = n, V, dtype
        g = torch.Generator().manual_seed(seed)
        self.start = [int(a) for a in np.cumsum([0] + n)]
        rows, self.total, B = self.start[-1] + len(n), self.start[-1], len(n)
        self.logits = (torch.randn((rows, V), generator=g) * spread).to(TYPES[dtype])
        self.ok = None if keep is None else torch.rand((rows, V), generator=g) < keep
        if self.ok is not None:
            self.ok.scatter_(1, torch.randint(0, V, (rows, 1), generator=g), True)
        of = [self.start[i] + i + j for i in range(B) for j in range(n[i])]
        d = self.logits[of].float() + noise * torch.randn((self.total, V), generator=g)
        if self.ok is not None:
            d = d.masked_fill(~self.ok[of], -np.inf)
        self.probs = torch.softmax(d, -1) if probs else None
        self.ids = (torch.multinomial(self.probs, 1, generator=g)[:, 0] if probs and self.total else d.argmax(-1)).to(torch.int64)
        self.u, self.final = torch.rand(self.total, generator=g), torch.rand(B, generator=g)
        self.T = torch.tensor([temps[i % len(temps)] for i in range(B)])
        self.width = max(n) + 1

    def place(self, pad=0):
        """On the GPU; rows `pad` elements longer than they need to be."""
        def rows(t, extra, fill):
            w = torch.full((t.shape[0], t.shape[1] + extra), fill, dtype=t.dtype, device="cuda")
            w[:, :t.shape[1]] = t.cuda()
            return w
        self.dl = rows(self.logits, pad, float("nan"))
        self.dm = None if self.ok is None else rows(pack(self.ok, (self.V + 63) // 64), pad, -1)
        self.dp = None if self.probs is None or not self.total else rows(self.probs, pad, float("nan"))
        self.ds, self.di = torch.tensor(self.start, dtype=torch.int32, device="cuda"), self.ids.to(torch.int32).cuda()
        self.du, self.df, self.dt = self.u.cuda(), self.final.cuda(), self.T.cuda()
        B = len(self.n)
        self.out = torch.full((B, self.width + pad), 77, dtype=torch.int32, device="cuda")
        self.logp, self.len = torch.full((B, self.width + pad), 7.0, device="cuda"), torch.full((B,), 77, dtype=torch.int32, device="cuda")
        self.pad = pad

    def run(self, plan, stream=None, flags=0, logp=True, temps=True):
        p = lambda t: t.data_ptr() if t is not None and t.numel() else None  # noqa: E731
        plan.run(p(self.dl), p(self.ds), p(self.di), p(self.du), p(self.df), p(self.out), p(self.len), len(self.n), self.total,
                 self.width + self.pad, p(self.dp), p(self.dt) if temps else None, p(self.dm), p(self.logp) if logp else None,
                 self.V + self.pad, self.V + self.pad, (self.V + 63) // 64 + self.pad, flags, stream)

    def check(self, last_tie=False, temps=True, logp=True):
        T = self.T if temps else torch.ones_like(self.T)
        out, lens, lp = reference(self.logits, self.ok, self.start, self.ids, self.probs, T, self.u, self.final, last_tie, self.width)
        w = self.width
        assert np.array_equal(self.len.cpu().numpy(), lens)
        assert np.array_equal(self.out.cpu().numpy()[:, :w], out) and (self.out[:, w:] == NONE).all()
        if logp:
            # z and the largest are exact or rounded once each to f32 at most, their difference and the logarithm of
            # the sum too; the sum's terms are f32 exponentials (4 units and one for each unit of the argument, of
            # which a weight's decay leaves less than one)
            U = 2.0 ** -24
            got = self.logp.cpu().double().numpy()
            zs = np.abs(self.logits.float().numpy())
            top = np.where(np.isfinite(zs), zs, 0).max() / min([t for t in T.tolist() if t > 0] + [1.0])
            assert (np.abs(got[:, :w] - lp) <= U * (16 + 4 * top + 2 * np.abs(lp))).all(), np.abs(got[:, :w] - lp).max()
            assert (got[:, w:] == 0).all()
        return lens

    def go(self, pad=0, **k):
        plan = nb.VerifyPlan(self.V, len(self.n), self.total, self.dtype)
        self.place(pad)
        self.run(plan, **k)
        plan.status()
        lens = self.check(bool(k.get("flags")), k.get("temps", True))
        return lens


CASES = [
    dict(n=[4], V=8192, dtype=nb.F32, keep=0.05), dict(n=[0], V=100, dtype=nb.F32), dict(n=[0, 0, 3], V=1, dtype=nb.F16),
    dict(n=[5, 0, 2, 1, 7], V=32003, dtype=nb.F16, temps=(0.7, 0.0, 1.3)), dict(n=[3] * 20, V=1000, dtype=nb.BF16, probs=False),
    dict(n=[1, 2] * 20, V=4099, dtype=nb.BF16, temps=(0.0,)), dict(n=[4] * 9, V=131072, dtype=nb.BF16),
    dict(n=[2, 3, 0, 1] * 16, V=777, dtype=nb.F32, keep=0.5, probs=False, temps=(0.5, 1.0, 0.0)),
    dict(n=[8] * 40, V=65, dtype=nb.F32, keep=0.1), dict(n=[3] * 30, V=64, dtype=nb.F16, spread=8.0), dict(n=[2] * 50, V=7, dtype=nb.F32),
    dict(n=[1] * 130, V=5000, dtype=nb.F32, noise=3.0), dict(n=[63], V=2049, dtype=nb.BF16, noise=0.1), dict(n=[4], V=200001, dtype=nb.F32),
    dict(n=[3, 3], V=1000003, dtype=nb.F16, keep=0.3), dict(n=[4] * 6, V=50257, dtype=nb.F32, spread=0.01),
]


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("pad", (0, 3))
def test_drafts(i, pad):
    Case(seed=i, **CASES[i]).go(pad)


def test_both_outcomes_occur():
    """Over many requests drafts are taken and replaced, at every place."""
    lens = Case([4] * 200, 500, nb.F32, 3).go()
    assert set(lens.tolist()) == {1, 2, 3, 4, 5}


def test_without_temperatures_and_log_probabilities():
    c = Case([3, 1] * 10, 300, nb.F32, 5, temps=(0.3, 0.0))
    c.go(temps=False)
    plan = nb.VerifyPlan(300, 20, c.total, nb.F32)
    c.place()
    c.run(plan, logp=False)
    c.check(logp=False)
    assert (c.logp == 7).all()


def test_ties():
    """Equal largest logits: the lowest index, or with the flag the highest."""
    for dtype in TYPES:
        c = Case([2] * 16, 4097, dtype, 1, probs=False, temps=(0.0,))
        c.logits.clamp_(max=4.0)
        for v in (5, 2048, 4096):
            c.logits[:, v] = 4.0
        c.ids = torch.tensor([5, 4096] * 16)
        c.go()
        c.go(flags=nb.VERIFY_LAST_TIE)


def test_final_numbers_at_the_ends():
    """The first and the last entry of weight, whatever is masked around them."""
    V = 3001
    for u in (0.0, 1.0 - 2.0 ** -24):
        c = Case([0] * 8 + [2] * 8, V, nb.F32, 2, keep=0.2, spread=1.0)
        c.final[:] = u
        c.go()


@pytest.mark.parametrize("temps", [(1e-30, 1e-6, 0.01), (3e38, float("inf"), 1e4)])
def test_temperatures_far_from_one(temps):
    for probs in (True, False):
        Case([3, 0, 2] * 8, 700, nb.F32, 11, probs=probs, temps=temps).go()
        Case([2] * 9, 4099, nb.BF16, 12, probs=probs, temps=temps, spread=30.0).go()


def test_residuals():
    """The drafter's distribution is the target's (nothing is left over but rounding), a single entry, or far off."""
    V = 600
    c = Case([1] * 24, V, nb.F32, 4)
    rows = [2 * i for i in range(24)]
    p = torch.softmax(c.logits[rows].double(), -1)
    c.probs = p.float() * 2  # twice as large everywhere: a rejected draft leaves nothing, and p takes its place
    c.probs[1::3] = 0.0
    for i in range(1, 24, 3):
        c.probs[i, c.ids[i]] = 1.0
    c.probs[2::3] = 1.0 / V
    c.u[:] = 0.999
    c.u[::4] = 0.0
    lens = c.go()
    assert {1, 2} == set(lens.tolist())


def test_certain_drafts():
    """A one-entry mask with the draft on it, then the draft off it; drafts outside the vocabulary."""
    c = Case([3] * 6, 130, nb.F32, 6, keep=0.5, probs=False, temps=(1.0, 0.0))
    c.ok[:] = False
    rows = torch.arange(c.ok.shape[0])
    c.ok[rows, rows % 130] = True
    at = [i * 4 + j for i in range(6) for j in range(3)]
    c.ids = torch.tensor([a % 130 for a in at])
    c.ids[4] = 77
    c.ids[8] = 130
    c.ids[13] = 2 ** 31 - 1
    c.ids[17] = -1
    lens = c.go()
    assert lens.tolist() == [4, 2, 3, 4, 2, 3]


def test_rows_that_leave_nothing_end_their_request():
    V = 500
    for probs in (True, False):
        for dtype in TYPES:
            c = Case([2] * 12, V, dtype, 7, keep=0.5, probs=probs, temps=(1.0, 0.0, 0.7))
            bad = float("nan")
            lo = torch.finfo(TYPES[dtype]).min
            c.ok[1] = False  # request 0, token 1
            c.logits[3][c.ok[3]] = -np.inf
            c.logits[6, int(c.ok[6].nonzero()[3])] = bad
            c.logits[9, int(c.ok[9].nonzero()[0])] = np.inf
            for r in (12, 15, 18):  # masked places hold anything
                c.logits[r][~c.ok[r]] = bad
                c.logits[r, int((~c.ok[r]).nonzero()[1])] = np.inf
            c.logits[21][c.ok[21]] = lo  # the type's lowest value is a value
            c.logits[24] = -np.inf
            c.logits[24, 400] = -3.0
            c.ok[24, 400] = True
            c.go()


def test_numbers_that_do_not_fit_are_reported():
    c = Case([2] * 5, 300, nb.F32, 8)
    plan = nb.VerifyPlan(300, 5, c.total, nb.F32)
    for start, lost in (([0, 2, 4, 6, 8, 11], [4]), ([-1, 2, 4, 6, 8, 10], [0]), ([0, 2, 4, 3, 8, 10], [2, 3]), ([0, 2, 4, 6, 10, 10], [3])):
        c.place()
        c.ds.copy_(torch.tensor(start, dtype=torch.int32))
        c.run(plan)
        with pytest.raises(nb.NeedleError, match="out of range"):
            plan.status()
        plan.status()
        n = c.len.tolist()
        assert all(n[i] == 0 for i in lost) and all(n[i] > 0 for i in range(5) if i not in lost and start[i + 1] - start[i] <= 2)
        assert all((c.out[i] == NONE).all() for i in lost)


def test_captured_and_on_other_streams():
    c = Case([3, 0, 5, 2] * 8, 9001, nb.BF16, 9, temps=(1.0, 0.0))
    plan = nb.VerifyPlan(9001, 32, c.total, nb.BF16)
    c.place()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        c.run(plan, torch.cuda.current_stream().cuda_stream)
    for seed in (10, 11):
        d = Case([3, 0, 5, 2] * 8, 9001, nb.BF16, seed, temps=(1.0, 0.0))
        for name in ("logits", "probs", "ids", "u", "final"):
            setattr(c, name, getattr(d, name))
        c.dl.copy_(c.logits), c.dp.copy_(c.probs), c.di.copy_(c.ids), c.du.copy_(c.u), c.df.copy_(c.final)
        g.replay()
        plan.status()
        c.check()
        kept = [t.clone() for t in (c.out, c.len, c.logp)]
        c.run(plan, torch.cuda.Stream().cuda_stream)
        torch.cuda.synchronize()
        for a, b in zip(kept, (c.out, c.len, c.logp)):
            assert torch.equal(a, b)


def test_overlapping_outputs_are_refused():
    c = Case([4], 100, nb.F32, 12)
    plan = nb.VerifyPlan(100, 1, c.total, nb.F32)
    c.place()
    out, logp, lens = c.out, c.logp, c.len
    kept = [t.clone() for t in (out, logp, lens, c.di, c.dl)]
    for name, other in (("out", c.di), ("out", c.du), ("len", c.ds), ("len", c.df), ("logp", c.dt), ("logp", c.dp), ("out", c.dl[2:])):
        setattr(c, name, other)
        with pytest.raises(nb.NeedleError, match="output overlaps an input"):
            c.run(plan)
        c.out, c.logp, c.len = out, logp, lens
    for name, other in (("out", c.logp), ("len", c.out[0, 4:])):
        setattr(c, name, other)
        with pytest.raises(nb.NeedleError, match="outputs overlap"):
            c.run(plan)
        c.out, c.logp, c.len = out, logp, lens
    plan.status()
    assert all(torch.equal(a, b) for a, b in zip(kept, (out, logp, lens, c.di, c.dl)))
    c.run(plan)
    c.check()
