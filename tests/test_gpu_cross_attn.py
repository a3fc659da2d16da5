"""Cross attention of ragged rows on the GPU against 64-bit arithmetic."""
import numpy as np
import pytest

from conftest import load_pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

nb = load_pkg()
TYPES = {nb.F16: torch.float16, nb.BF16: torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


def reference(q, k, v, mask, qs, ql, ks, kl, scale):
    """(out, lse, tolerance of out before its rounding, tolerance of lse) in
    64 bits, on the GPU's f64 units; q [rows][H][D], k and v [rows][KVH][D].

    A score is a sum of D products kept in f32 (at most D + 8 roundings, each
    within 2 U of the sum of magnitudes) and then scaled; its exponential adds
    8 U and U for each unit of its argument; a weight is rounded to the type
    (half a step relative; below f16's normal range half of its smallest
    step), and sums over n keys add n U.  Numerator and denominator both
    carry these errors.  A weight is at most 1/e^8 below the one its row
    is normalised by when the row's running maximum is not the final
    one; the smallest step is therefore taken against the row's sum of at
    least 2^-9."""
    H, KVH, D = q.shape[1], k.shape[1], q.shape[2]
    eps = torch.finfo(q.dtype).eps
    tiny = 2.0 ** -25 * 512 if q.dtype == torch.float16 else 0.0
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -np.inf, dtype=torch.float64)
    eo, el = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    for a, n, b, m in zip(qs, ql, ks, kl):
        seen = torch.arange(b, b + m)
        if mask is not None:
            seen = seen[mask[b:b + m] != 0]
        if not n or not seen.numel():
            continue
        kk, vv = (t[seen].double().cuda().repeat_interleave(H // KVH, dim=1) for t in (k, v))
        qq = q[a:a + n].double().cuda()
        s = torch.einsum("qhd,khd->hqk", qq, kk) * scale
        es = torch.einsum("qhd,khd->hqk", qq.abs(), kk.abs()) * (scale * 2 * (D + 8) * U)
        pr = torch.softmax(s, -1)
        top = s.amax(-1, keepdim=True)
        ep = es + (8 + (s - top).abs() * 2) * U
        rel = (pr * ep).sum(-1) + seen.numel() * U
        o = torch.einsum("hqk,khd->qhd", pr, vv)
        mag = torch.einsum("hqk,khd->qhd", pr * (ep + eps / 2 * (1 + eps)), vv.abs())
        mag = mag + torch.einsum("hqk,khd->qhd", pr, vv.abs()) * (rel.t()[..., None] + 4 * U)
        l = torch.exp(s - top).sum(-1)
        mag = mag + tiny * (vv.abs().sum(0)[None] / l.t()[..., None]).clamp(max=vv.abs().max())
        out[a:a + n], eo[a:a + n] = o.cpu(), mag.cpu()
        ls = torch.logsumexp(s, -1).t()
        lse[a:a + n], el[a:a + n] = ls.cpu(), (rel.t() + es.amax(-1).t() + 4 * U * (1 + ls.abs() + top[..., 0].t().abs())).cpu()
    return out, lse, eo, el


def close(got, want, e, dtype):
    f = torch.finfo(TYPES[dtype])
    tol = e + f.eps / 2 * (want.abs() + e) + f.tiny * f.eps / 2
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def make(ql, kl, H, KVH, D, dtype, seed, keep=1.0, gap=0, width=1.0):
    """Ragged rows with `gap` rows that no request owns behind each request's."""
    g = torch.Generator().manual_seed(seed)
    qs = np.cumsum([0] + [n + gap for n in ql])
    ks = np.cumsum([0] + [n + gap for n in kl])
    t = TYPES[dtype]
    q = (torch.randn((max(int(qs[-1]), 1), H, D), generator=g) * width).to(t)
    k, v = (torch.randn((max(int(ks[-1]), 1), KVH, D), generator=g).to(t) for _ in range(2))
    mask = (torch.rand(k.shape[0], generator=g) < keep).to(torch.uint8) if keep < 1 else None
    return q, k, v, mask, [int(a) for a in qs[:-1]], [int(a) for a in ks[:-1]]


def run(q, k, v, mask, qs, ql, ks, kl, dtype, scale, layout="token", lse=True, check=True):
    H, KVH, D = q.shape[1], k.shape[1], q.shape[2]
    plan = nb.CrossAttnPlan(qs, ql, ks, kl, H, KVH, D, dtype)
    if layout == "token":
        qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
        od = torch.full_like(qd, 7.0)
    elif layout == "head":
        qd, kd, vd = (t.transpose(0, 1).contiguous().cuda().transpose(0, 1) for t in (q, k, v))
        od = torch.full((H, q.shape[0], D), 7.0, dtype=q.dtype, device="cuda").transpose(0, 1)
    else:  # parts of fused rows
        wide = torch.full((q.shape[0], H, D + 8), 3.0, dtype=q.dtype, device="cuda")
        wide[:, :, :D] = q.cuda()
        qd = wide[:, :, :D]
        kv = torch.stack([k, v], dim=2).cuda()  # [rows][KVH][2][D]
        kd, vd = kv[:, :, 0], kv[:, :, 1]
        od = torch.full((q.shape[0], H, D + 8), 7.0, dtype=q.dtype, device="cuda")[:, :, :D]
    md = None if mask is None else mask.cuda()
    ld = torch.full((q.shape[0], H), 7.0, device="cuda") if lse else None
    st = lambda t: (t.stride(0), t.stride(1))  # noqa: E731
    call = lambda: plan.run(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), od.data_ptr(), scale, st(qd), st(kd), st(vd), st(od),  # noqa: E731
                            None if md is None else md.data_ptr(), None if ld is None else ld.data_ptr())
    call()
    plan.status()
    first = od.clone()
    call()  # the plan's workspace is as it was: the same bits again
    plan.status()
    assert torch.equal(first.view(torch.int16), od.view(torch.int16))
    if check:
        owned = torch.zeros(q.shape[0], dtype=torch.bool)
        for a, n in zip(qs, ql):
            owned[a:a + n] = True
        out, ls, eo, el = reference(q, k, v, mask, qs, ql, ks, kl, scale)
        close(od.cpu()[owned], out[owned], eo[owned], dtype)
        assert (od.cpu()[~owned] == 7).all()
        if lse:
            got, want = ld.cpu().double()[owned], ls[owned]
            none = torch.isinf(want)
            assert torch.equal(none, torch.isinf(got)) and (got[none] < 0).all()
            assert ((got - want).abs()[~none] <= el[owned][~none]).all()
            assert (ld.cpu()[~owned] == 7).all()
    plan.close()
    return od, ld


SHAPES = [
    # query lengths, key lengths, H, KVH, D
    ([1], [1], 1, 1, 8), ([1], [256], 8, 4, 64), ([1, 1, 1], [64, 511, 300], 8, 4, 64), ([1] * 5, [0, 1, 127, 128, 129], 4, 1, 128),
    ([3], [33], 2, 2, 32), ([0, 2, 17, 0, 5], [9, 0, 200, 77, 63], 12, 4, 80), ([16, 1, 4], [1000, 64, 65], 6, 2, 96),
    ([130], [70], 4, 4, 64), ([1, 257], [513, 640], 8, 2, 64), ([128], [128], 2, 1, 128), ([129, 300], [1, 385], 3, 1, 72),
    ([64], [2000], 16, 2, 128), ([700], [900], 2, 2, 40), ([1], [20000], 8, 8, 128), ([1, 1], [9000, 5], 64, 8, 64),
    ([2], [4097], 1, 1, 16), ([31, 33], [8192, 100], 4, 2, 64), ([260], [5000], 2, 1, 128), ([1], [33], 40, 1, 64)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_against_64_bits(i, dtype):
    ql, kl, H, KVH, D = SHAPES[i]
    layout = ("token", "head", "fused")[(i + dtype) % 3]
    keep = (1.0, 0.7)[(i // 2 + dtype) % 2]
    q, k, v, mask, qs, ks = make(ql, kl, H, KVH, D, dtype, i, keep, gap=i % 3)
    run(q, k, v, mask, qs, ql, ks, kl, dtype, D ** -0.5, layout)


@pytest.mark.parametrize("mask", ["none", "random", "padding"])
@pytest.mark.parametrize("D", [64, 128])
def test_more_tiles_of_rows_than_fit_at_once(D, mask):
    """Hundreds of tiles of 128 rows, so that each CTA works through several: of
    different lengths, some without keys, some wholly masked."""
    ql = [150 + 7 * i % 90 for i in range(40)]
    kl = [0 if i % 11 == 3 else (37 * i) % 400 + 1 for i in range(40)]
    dtype = nb.F16 if D == 64 else nb.BF16
    q, k, v, m, qs, ks = make(ql, kl, 16, 4, D, dtype, D, 0.6 if mask == "random" else 1.0, gap=2)
    if mask == "padding":  # what is behind a document's end inside its row, from none of it to all
        m = torch.ones(k.shape[0], dtype=torch.uint8)
        for i, (b, n) in enumerate(zip(ks, kl)):
            m[b + n * (i % 6) // 5:b + n] = 0
        v[m == 0] = float("nan")
        k[m == 0] = float("inf")
    od, ld = run(q, k, torch.nan_to_num(v), m, qs, ql, ks, kl, dtype, D ** -0.5)
    if mask == "padding":
        again, _ = run(q, k, v, m, qs, ql, ks, kl, dtype, D ** -0.5, check=False)
        assert torch.equal(again.view(torch.int16), od.view(torch.int16))


@pytest.mark.parametrize("n,D", [(6, 64), (6, 80), (70, 64), (70, 128)])
def test_single_tokens_beside_longer_queries(n, D):
    """Requests of few rows and of many in one plan: few requests, whose tiles fit
    the GPU at once, and more."""
    ql = [(1, 40, 3, 0, 9, 130)[i % 6] for i in range(n)]
    kl = [(53 * i) % 300 for i in range(n)]
    dtype = nb.BF16 if D == 64 else nb.F16
    q, k, v, mask, qs, ks = make(ql, kl, 8, 4, D, dtype, n + D, 0.7, gap=1)
    run(q, k, v, mask, qs, ql, ks, kl, dtype, D ** -0.5)


@pytest.mark.parametrize("n", [1, 40])
def test_what_is_masked_changes_nothing(n):
    """NaN, infinities and the lowest value in masked keys, in the rows between requests and behind the last."""
    ql, kl, H, KVH, D, dtype = [n, n, n], [100, 130, 257], 4, 2, 64, nb.BF16
    q, k, v, mask, qs, ks = make(ql, kl, H, KVH, D, dtype, 3, 0.5, gap=5)
    clean, cl = run(q, k, v, mask, qs, ql, ks, kl, dtype, 0.125)
    unseen = mask == 0
    for a, m in zip(ks, kl):
        unseen[a + m:a + m + 5] = True
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min):
        k2, v2 = k.clone(), v.clone()
        k2[unseen], v2[unseen] = bad, bad
        got, gl = run(q, k2, v2, mask, qs, ql, ks, kl, dtype, 0.125, check=False)
        assert torch.equal(got, clean) and torch.equal(gl, cl)


@pytest.mark.parametrize("n", [1, 5, 150])
def test_rows_without_keys(n):
    ql, kl, H, KVH, D, dtype = [n, n, n], [300, 0, 40], 4, 4, 64, nb.F16
    q, k, v, mask, qs, ks = make(ql, kl, H, KVH, D, dtype, 4, 0.5)
    mask[:300] = 0
    mask[300] = 1
    od, ld = run(q, k, v, mask, qs, ql, ks, kl, dtype, 0.125)
    assert (od[:2 * n] == 0).all() and torch.isinf(ld[:2 * n]).all()
    mask[:] = 0
    od, ld = run(q, k, v, mask, qs, ql, ks, kl, dtype, 0.125)
    assert (od == 0).all() and torch.isinf(ld).all()


@pytest.mark.parametrize("n", [1, 130])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_growing_and_large_scores(n, dtype):
    """Scores that rise along the keys (the running maximum moves at every tile), and scores whose exponentials span the type."""
    H, KVH, D, m = 2, 1, 64, 900
    q, k, v, _, qs, ks = make([n], [m], H, KVH, D, dtype, 6)
    k = (k.float() * 0.1 + torch.linspace(-4, 4, m)[:, None, None] * torch.sign(q[0, 0].float())[None, None]).to(TYPES[dtype])
    run(q, k, v, None, qs, [n], ks, [m], dtype, 0.5)
    run(q, k.flip(0).contiguous(), v, None, qs, [n], ks, [m], dtype, 0.5)


def test_shared_keys():
    """Several drafts over one prompt: the same key range for each."""
    ql, kl, H, KVH, D, dtype = [1, 3, 2, 140], [500, 500, 321, 500], 8, 4, 64, nb.BF16
    q, k, v, mask, qs, _ = make(ql, [500], H, KVH, D, dtype, 7, 0.9)
    run(q, k, v, mask, qs, ql, [0, 0, 100, 0], [500, 500, 321, 500], dtype, 0.125)


def test_no_queries_at_all():
    q, k, v, mask, qs, ks = make([0, 0], [5, 6], 2, 1, 32, nb.F16, 1, gap=1)
    od, ld = run(q, k, v, None, qs, [0, 0], ks, [5, 6], nb.F16, 0.2)
    assert (od == 7).all() and (ld == 7).all()


def test_nan_in_a_seen_key_reaches_its_rows_alone():
    ql, kl, dtype = [2, 2], [90, 90], nb.BF16
    q, k, v, _, qs, ks = make(ql, kl, 2, 2, 64, dtype, 2)
    v[10, 0, 3] = float("nan")
    od, _ = run(q, k, v, None, qs, ql, ks, kl, dtype, 0.125, check=False)
    bad = torch.isnan(od.cpu())
    want = torch.zeros_like(bad)
    want[:2, 0, 3] = True
    assert torch.equal(bad, want)


def test_far_rows():
    """Rows whose element offset passes 32 bits."""
    H = KVH = 1
    D, dtype, stride = 64, nb.BF16, 1 << 21
    rows = 1100
    if torch.cuda.mem_get_info()[0] < 3 * rows * stride * 2:
        pytest.skip("too little memory")
    base = torch.zeros((rows, stride), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((rows, 1, D), generator=g).to(torch.bfloat16) for _ in range(3))
    for i, t in enumerate((q, k, v)):
        base[:, i * D:(i + 1) * D] = t[:, 0].cuda()
    qs, ql, ks, kl = [1080, 0], [20, 1], [1030, 1090], [70, 3]
    plan = nb.CrossAttnPlan(qs, ql, ks, kl, H, KVH, D, dtype)
    s, at = (stride, D), base.data_ptr()
    plan.run(at, at + 2 * D, at + 4 * D, at + 6 * D, 0.125, s, s, s, s)
    plan.status()
    out, _, eo, _ = reference(q, k, v, None, qs, ql, ks, kl, 0.125)
    got = base[:, 3 * D:4 * D].reshape(rows, 1, D)
    for a, n in zip(qs, ql):
        close(got[a:a + n], out[a:a + n], eo[a:a + n], dtype)


def test_graph_replays_on_new_states():
    ql, kl, H, KVH, D, dtype = [1] * 6 + [40], [64, 200, 3000, 1, 0, 512, 700], 8, 4, 64, nb.BF16
    q, k, v, _, qs, ks = make(ql, kl, H, KVH, D, dtype, 11)
    plan = nb.CrossAttnPlan(qs, ql, ks, kl, H, KVH, D, dtype)
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    od = torch.zeros_like(qd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        plan.run(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), od.data_ptr(), 0.125, stream=torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        q, k, v, _, _, _ = make(ql, kl, H, KVH, D, dtype, seed)
        qd.copy_(q), kd.copy_(k), vd.copy_(v)
        g.replay()
        out, _, eo, _ = reference(q, k, v, None, qs, ql, ks, kl, 0.125)
        close(od, out, eo, dtype)
    plan.status()


def test_run_refuses():
    plan = nb.CrossAttnPlan([0], [4], [0], [9], 4, 2, 64, nb.F16)
    t = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    p = t.data_ptr()
    bad = [(dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q_ptr=None), "invalid"),
           (dict(k_ptr=p + 2), "16-byte"), (dict(k_strides=(128, 60)), "strides"), (dict(v_strides=(129, 64)), "strides"),
           (dict(out_strides=(64, 64)), "overlap"), (dict(lse_ptr=p + 2), "invalid")]
    for b, match in bad:
        a = dict(q_ptr=p, k_ptr=p, v_ptr=p, out_ptr=p, scale=0.125)
        a.update(b)
        with pytest.raises(nb.NeedleError, match=match):
            plan.run(**a)
    host = np.zeros(4096, np.float16)
    at = (host.ctypes.data + 15) // 16 * 16
    with pytest.raises(nb.NeedleError, match="device memory|CUDA error"):
        plan.run(at, p, p, p, 0.125)


@pytest.mark.parametrize("layout", ["token", "head", "fused"])
def test_no_queries_in_any_layout(layout):
    q, k, v, _, qs, ks = make([0, 0], [5, 6], 4, 2, 32, nb.F16, 1, gap=1)
    od, ld = run(q, k, v, None, qs, [0, 0], ks, [5, 6], nb.F16, 0.2, layout)
    assert (od == 7).all() and (ld == 7).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ql", [[1, 2], [3, 150], [0, 0]])
def test_operands_of_no_rows_may_be_null(ql, D):
    """The pointer of an empty tensor: K and V where no request has keys, q and out where none has queries."""
    H, KVH, rows = 4, 2, sum(ql)
    plan = nb.CrossAttnPlan([0, ql[0]], ql, [0, 0], [0, 0], H, KVH, D, nb.BF16)
    q = torch.randn((rows, H, D), device="cuda").bfloat16()
    empty = torch.empty((0, KVH, D), dtype=torch.bfloat16, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((rows, H), 7.0, device="cuda")
    assert empty.data_ptr() == 0 and (rows or q.data_ptr() == 0)
    plan.run(q.data_ptr(), empty.data_ptr(), empty.data_ptr(), out.data_ptr(), 0.125, lse_ptr=lse.data_ptr())
    plan.status()
    assert (out == 0).all() and (lse == -float("inf")).all()
    one = nb.CrossAttnPlan([0], [1], [0], [1], H, KVH, D, nb.BF16)
    p = torch.zeros((1, H, D), dtype=torch.bfloat16, device="cuda").data_ptr()
    for a in ((None, p, p, p), (p, None, p, p), (p, p, None, p), (p, p, p, None)):
        with pytest.raises(nb.NeedleError, match="invalid"):
            one.run(*a, 0.125)


VISIBLE = [([1], [20000], 8, 4, 64), ([1, 3], [9000, 70], 4, 4, 64), ([2], [4097], 2, 1, 128), ([40], [5000], 4, 2, 64),
           ([130, 1], [3001, 641], 2, 2, 128), ([300, 17], [700, 385], 4, 2, 80), ([1] * 40, [500 + 13 * i for i in range(40)], 4, 2, 64)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(VISIBLE)))
def test_every_block_of_keys_is_seen_by_itself(i, dtype, masked):
    """Each column of V is zero but for one block of 64 keys, with a value of its own for each key of it, so that an
    output is that block's share of the weights: a key that is left out, taken twice or from elsewhere, in a tile, in the last
    part of one or where a range is cut, moves it by about a sixty-fourth.  Scores are small, so that every block has a share.

    Relative to a share: the errors of the scores and exponentials (as above), half a step of the type for each
    weight, n + 4 U of the sums, and the row's sum with the same but for the step.  A row's sum is at least 1 in units of
    its largest weight, and no weight was rounded in smaller units than that (a running maximum is never above
    the final one), so f16 adds at most half of its smallest step, 2^-25, for each key of the block."""
    ql, kl, H, KVH, D = VISIBLE[i]
    q, k, _, mask, qs, ks = make(ql, kl, H, KVH, D, dtype, 100 + i, 0.7 if masked else 1.0, gap=1, width=0.3)
    t, scale, eps = TYPES[dtype], D ** -0.5, torch.finfo(TYPES[dtype]).eps
    tiny = 2.0 ** -25 if dtype == nb.F16 else 0.0
    cols = KVH * D
    plan = nb.CrossAttnPlan(qs, ql, ks, kl, H, KVH, D, dtype)
    qd, kd, md = q.cuda(), k.cuda(), None if mask is None else mask.cuda()
    od = torch.empty_like(qd)
    for first in range(0, (max(kl) + 63) // 64, cols):
        v = torch.zeros((k.shape[0], cols), dtype=t)
        for b, m in zip(ks, kl):
            j = torch.arange(m)
            at = j // 64 - first
            ok = (at >= 0) & (at < cols)
            v[b + j[ok], at[ok]] = (1 + (j[ok] % 64) / 64).to(t)  # exact in 8 bits
        vd = v.view(-1, KVH, D).cuda()
        plan.run(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), od.data_ptr(), scale, key_mask_ptr=None if md is None else md.data_ptr())
        plan.status()
        for a, n, b, m in zip(qs, ql, ks, kl):
            seen = torch.arange(b, b + m, device="cuda")
            if md is not None:
                seen = seen[md[b:b + m] != 0]
            kk, vv = (x[seen].double().repeat_interleave(H // KVH, dim=1) for x in (kd, vd))
            qq = qd[a:a + n].double()
            s = torch.einsum("qhd,khd->hqk", qq, kk) * scale
            es = torch.einsum("qhd,khd->hqk", qq.abs(), kk.abs()) * (scale * 2 * (D + 8) * U)
            pr = torch.softmax(s, -1)
            top = s.amax(-1, keepdim=True)
            ep = es + (8 + (s - top).abs() * 2) * U
            rel = ((pr * ep).sum(-1) + (seen.numel() + 4) * U).t()[..., None]
            want = torch.einsum("hqk,khd->qhd", pr, vv)
            e = torch.einsum("hqk,khd->qhd", pr * (ep + eps / 2 * (1 + eps)), vv) + want * (rel + (seen.numel() + 4) * U)
            e = e + tiny * (vv.sum(0)[None] / torch.exp(s - top).sum(-1).t()[..., None])
            close(od[a:a + n], want.cpu(), e.cpu(), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 40, 200])
def test_values_of_one(n, dtype):
    """All values 1: an output is the sum of the rounded weights over the sum of the weights."""
    m, H, KVH, D = 7001, 4, 2, 64
    q, k, v, mask, qs, ks = make([n], [m], H, KVH, D, dtype, n, 0.9)
    od, _ = run(q, k, torch.ones_like(v), mask, qs, [n], ks, [m], dtype, 0.125, check=False)
    half = torch.finfo(TYPES[dtype]).eps / 2
    tiny = 2.0 ** -25 * m if dtype == nb.F16 else 0.0
    assert ((od.double() - 1).abs() <= half + tiny + 2 * (m + 4) * U + half * (1 + 2 * half)).all()
