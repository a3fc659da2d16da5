"""The residual norm on the GPU against 64-bit arithmetic."""
import pytest

from conftest import load_pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

nb = load_pkg()
TYPES = {nb.F32: torch.float32, nb.F16: torch.float16, nb.BF16: torch.bfloat16}
U = 2.0 ** -24
KINDS = {"none": 0, "scalar": nb.GATE_SCALAR, "channel": nb.GATE_CHANNEL, "token": nb.GATE_TOKEN}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


def reference(x, y, post, gate, sigmoid, scale, pre):
    """(r, h, tolerance of r, tolerance of h) before rounding to a type.

    A statistic sums d squares: a thread up to 32 of them one after another,
    then 10 levels of a tree, so it is off by at most 45 U relative and the
    factor 1/sqrt by half of that and 4 roundings; gates and products add
    under 12.  r: 40 U of each summand.  h: r's error times the factor, the
    factor's own error (from r's errors and from its sum), 4 roundings."""
    x = x.double()
    if y is None:
        r, er = scale * x, 2 * U * (scale * x).abs()
    else:
        y = y.double()
        if post is not None:
            y = (1 + post.double()) * y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6)
        if gate is not None:
            g = gate.double()
            y = y * (torch.sigmoid(g) if sigmoid else g)
        r = scale * x + y
        er = 40 * U * ((scale * x).abs() + y.abs())
    if pre is None:
        return r, None, er, None
    inv = 1 / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + 1e-6)
    h = (1 + pre.double()) * r * inv
    off = torch.sqrt(er.pow(2).mean(-1, keepdim=True)) * inv
    eh = er * (1 + pre.double()).abs() * inv + h.abs() * (off + 40 * U)
    return r, h, er, eh


def rounded(e, v, dtype):
    f = torch.finfo(TYPES[dtype])
    return e + f.eps / 2 * (v.abs() + e) + f.tiny * f.eps / 2


def close(got, want, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def inputs(M, d, tx, ty, gate, post, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, y = (rnd(M, d) * 2).to(TYPES[tx]), (rnd(M, d) * 0.7).to(TYPES[ty])
    gates = {"none": None, "scalar": rnd(1), "channel": rnd(d), "token": rnd(M, d).to(TYPES[ty])}[gate]
    return x, y, gates, rnd(d) * 0.1 if post else None, rnd(d) * 0.1


def cuda(*a):
    return [None if t is None else t.cuda() for t in a]


def p(t):
    return None if t is None else t.data_ptr()


CASES = [(1, 512, nb.F32, nb.F32, "scalar", True, False, 1.0), (1, 1, nb.F32, nb.BF16, "none", False, True, 1.0),
         (5, 7, nb.F16, nb.F16, "token", True, True, 0.5), (9, 33, nb.BF16, nb.BF16, "channel", False, True, 1.0),
         (17, 256, nb.F32, nb.F16, "token", False, False, 0.7), (3, 264, nb.F32, nb.F32, "channel", True, True, -1.5),
         (4, 1000, nb.F32, nb.BF16, "channel", True, True, 1.0), (2, 1531, nb.F16, nb.F16, "scalar", False, True, 1.0),
         (6, 2048, nb.BF16, nb.BF16, "none", False, False, 1.0), (3, 4096, nb.F32, nb.BF16, "token", True, True, 0.5),
         (2, 4104, nb.F32, nb.F32, "token", True, True, 1.0), (2, 8191, nb.BF16, nb.BF16, "token", False, True, 1.0),
         (2, 16384, nb.F32, nb.F16, "channel", True, True, 1.0), (1, 32768, nb.F32, nb.F32, "none", False, True, 1.0),
         (1, 32767, nb.F16, nb.F16, "token", True, True, 1.0), (1000, 512, nb.F32, nb.F32, "scalar", True, True, 1.0)]


@pytest.mark.parametrize("M,d,tx,ty,gate,sigmoid,post,scale", CASES)
def test_against_64_bits(M, d, tx, ty, gate, sigmoid, post, scale):
    x, y, g, ps, pre = inputs(M, d, tx, ty, gate, post, M + d)
    r, h, er, eh = reference(x, y, ps, g, sigmoid, scale, pre)
    flags = KINDS[gate] | (nb.GATE_SIGMOID if gate != "none" and sigmoid else 0)
    xd, yd, gd, pd, prd = cuda(x, y, g, ps, pre)
    rd, hd = torch.full_like(xd, float("nan")), torch.full_like(yd, float("nan"))
    common = dict(post_scale_ptr=p(pd), gate_ptr=p(gd), gate_flags=flags, residual_scale=scale)
    nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(rd), p(hd), ty, **common)
    close(rd, r, rounded(er, r, tx))
    close(hd, h, rounded(eh, h, ty))
    # 8-bit rows: the scale is max|h| / 127, each value within half a step
    Kp = nb.int8_row_bytes(d)
    q, s = torch.full((M, Kp), 9, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    r2 = torch.empty_like(rd)
    nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(r2), p(q), nb.I8, h_scales_ptr=p(s), **common)
    assert torch.equal(r2, rd) and not q[:, d:].any()
    s, q = s.double().cpu(), q[:, :d].double().cpu()
    top = h.abs().max(dim=1).values
    etop = eh.max(dim=1).values
    assert ((s - top / 127).abs() <= etop / 127 + 2 * U * s).all()
    # the quotient is rounded to f32 twice (127 / top and the product), up to 127 steps from zero
    close(q * s[:, None], h, eh + s[:, None] * (0.5 + 4 * 127 * U) + etop[:, None])
    assert (q.abs().max(dim=1).values == 127).all()
    # r alone, in place; h in the place of y
    nb.residual_norm(p(xd), tx, p(yd), ty, M, d, None, p(xd), None, ty, **common)
    assert torch.equal(xd, rd)
    xd = x.cuda()
    nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(xd), p(yd), ty, **common)
    assert torch.equal(xd, rd) and torch.equal(yd, hd)


@pytest.mark.parametrize("M,d,tx,ty", [(3, 512, nb.F32, nb.BF16), (2, 77, nb.F32, nb.F32), (1, 8200, nb.F16, nb.F16)])
def test_norm_before_the_first_block(M, d, tx, ty):
    x, _, _, _, pre = inputs(M, d, tx, ty, "none", False, 3)
    _, h, _, eh = reference(x, None, None, None, False, 0.25, pre)
    xd, prd = cuda(x, pre)
    hd = torch.empty((M, d), dtype=TYPES[ty], device="cuda")
    nb.residual_norm(p(xd), tx, None, ty, M, d, p(prd), None, p(hd), ty, residual_scale=0.25)
    close(hd, h, rounded(eh, h, ty))


@pytest.mark.parametrize("d", [40, 1000, 37])
@pytest.mark.parametrize("off", [0, 1])
def test_strides_and_alignment(d, off):
    """Rows inside wider rows, on and off 16-byte boundaries; what lies between them stays."""
    M, ty = 6, nb.BF16
    x, y, g, ps, pre = inputs(M, d, nb.F32, ty, "token", True, d)
    r, h, er, eh = reference(x, y, ps, g, True, 1.0, pre)
    ld = (d + 7) // 8 * 8 + 8 * (1 - off) + 3 * off

    def wide(t, dtype):
        b = torch.full((M * ld + 16,), 5.0, dtype=TYPES[dtype], device="cuda")
        v = b[off:off + M * ld].view(M, ld)
        if t is not None:
            v[:, :d] = t.cuda()
        return v

    xd, yd, gd, rd, hd = wide(x, nb.F32), wide(y, ty), wide(g, ty), wide(None, nb.F32), wide(None, ty)
    pd, prd = cuda(ps, pre)
    nb.residual_norm(p(xd), nb.F32, p(yd), ty, M, d, p(prd), p(rd), p(hd), ty, post_scale_ptr=p(pd), gate_ptr=p(gd),
                     gate_flags=nb.GATE_TOKEN | nb.GATE_SIGMOID, ldx=ld, ldy=ld, ldg=ld, ldr=ld, ldh=ld)
    close(rd[:, :d], r, rounded(er, r, nb.F32))
    close(hd[:, :d], h, rounded(eh, h, ty))
    assert (rd[:, d:] == 5).all() and (hd[:, d:] == 5).all()


MANY = [(20000, 33), (20000, 64), (9000, 264), (9000, 257), (9001, 512), (8000, 777), (6000, 1000), (5000, 1024), (4001, 2048),
        (3000, 2054), (2500, 4096), (2000, 4099), (1500, 4360), (1500, 6738), (1300, 8192), (1200, 8191), (20000, 131), (15000, 255)]


@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "token", "no block"])
@pytest.mark.parametrize("M,d", MANY)
def test_many_rows(M, d, gate):
    """Enough rows for every block to take several, in whole vectors and off 16-byte boundaries; every row is checked."""
    k = MANY.index((M, d)) + ["none", "scalar", "channel", "token", "no block"].index(gate)
    ty = (nb.BF16, nb.F16, nb.F32)[k % 3]
    tx = nb.F32 if k % 2 else ty
    sigmoid, post, i8 = k % 4 != 1, k % 5 != 2, k % 2 == 0
    x, y, g, ps, pre = inputs(M, d, tx, ty, "none" if gate == "no block" else gate, post, k)
    xd, prd = cuda(x, pre)
    Kp = nb.int8_row_bytes(d)
    hd = torch.full((M + 1, Kp), 9, dtype=torch.int8, device="cuda") if i8 else torch.full((M + 1, d), 7.0, dtype=TYPES[ty], device="cuda")
    hs = torch.full((M + 1,), 7.0, device="cuda") if i8 else None
    if gate == "no block":
        r, h, er, eh = reference(x, None, None, None, False, 0.75, pre)
        nb.residual_norm(p(xd), tx, None, ty, M, d, p(prd), None, p(hd), nb.I8 if i8 else ty, residual_scale=0.75, h_scales_ptr=p(hs))
    else:
        r, h, er, eh = reference(x, y, ps, g, sigmoid, 0.75, pre)
        yd, gd, pd = cuda(y, g, ps)
        rd = torch.full((M + 1, d), 7.0, dtype=TYPES[tx], device="cuda")
        flags = KINDS[gate] | (nb.GATE_SIGMOID if gate != "none" and sigmoid else 0)
        nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(rd), p(hd), nb.I8 if i8 else ty, post_scale_ptr=p(pd), gate_ptr=p(gd),
                         gate_flags=flags, residual_scale=0.75, h_scales_ptr=p(hs))
        close(rd[:M], r, rounded(er, r, tx))
        assert (rd[M] == 7).all()
    if i8:
        s, q, etop = hs[:M].double().cpu(), hd[:M].double().cpu(), eh.max(dim=1).values
        assert (q[:, d:] == 0).all() and (hd[M] == 9).all() and hs[M] == 7
        assert ((s - h.abs().max(dim=1).values / 127).abs() <= etop / 127 + 2 * U * s).all()
        close(q[:, :d] * s[:, None], h, eh + s[:, None] * (0.5 + 4 * 127 * U) + etop[:, None])
    else:
        close(hd[:M], h, rounded(eh, h, ty))
        assert (hd[M] == 7).all()


@pytest.mark.parametrize("M,d,tx,ty,gate", [(20000, 33, nb.F16, nb.F16, "channel"), (9000, 257, nb.F32, nb.BF16, "token"),
                                            (9000, 512, nb.BF16, nb.BF16, "none"), (5000, 1024, nb.F16, nb.F16, "token"),
                                            (2500, 4096, nb.F32, nb.BF16, "token"), (1500, 6738, nb.BF16, nb.BF16, "scalar")])
def test_many_rows_in_place(M, d, tx, ty, gate):
    """r in the place of x and h in that of y, where rows are fetched ahead and pieces of 16 bytes hold parts of two rows."""
    x, y, g, ps, pre = inputs(M, d, tx, ty, gate, True, 3)
    xd, yd, gd, pd, prd = cuda(x, y, g, ps, pre)
    rd, hd = torch.empty_like(xd), torch.empty_like(yd)
    call = lambda r, h: nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(r), p(h), ty, post_scale_ptr=p(pd), gate_ptr=p(gd),  # noqa: E731
                                         gate_flags=KINDS[gate])
    call(rd, hd)
    call(xd, yd)
    assert torch.equal(rd, xd) and torch.equal(hd, yd)


def test_zero_rows_infinities_and_nan():
    M, d = 4, 96
    x, y, _, ps, pre = inputs(M, d, nb.F32, nb.F32, "none", True, 1)
    x[0], y[0] = 0, 0
    x[1, 4], y[2, 7] = float("inf"), float("nan")
    xd, yd, pd, prd = cuda(x, y, ps, pre)
    rd, q, s = torch.empty_like(xd), torch.empty((M, 96), dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    nb.residual_norm(p(xd), nb.F32, p(yd), nb.F32, M, d, p(prd), p(rd), p(q), nb.I8, post_scale_ptr=p(pd), h_scales_ptr=p(s))
    s, q = s.cpu(), q.cpu()
    assert s[0] == 0 and not q[0].any() and torch.isnan(s[1]) and torch.isnan(s[2]) and s[3] > 0
    assert not q[1].any() and not q[2].any()


def test_graph_on_another_stream():
    M, d = 33, 512
    x, y, g, ps, pre = inputs(M, d, nb.F32, nb.BF16, "scalar", True, 8)
    xd, yd, gd, pd, prd = cuda(x, y, g, ps, pre)
    rd, hd = torch.empty_like(xd), torch.empty_like(yd)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=torch.cuda.Stream()):
        nb.residual_norm(p(xd), nb.F32, p(yd), nb.BF16, M, d, p(prd), p(rd), p(hd), nb.BF16, post_scale_ptr=p(pd), gate_ptr=p(gd),
                         gate_flags=nb.GATE_SCALAR | nb.GATE_SIGMOID, stream=torch.cuda.current_stream().cuda_stream)
    x2 = x + 1
    xd.copy_(x2)
    gr.replay()
    r, h, er, eh = reference(x2, y, ps, g, True, 1.0, pre)
    close(rd, r, rounded(er, r, nb.F32))
    close(hd, h, rounded(eh, h, nb.BF16))


@pytest.mark.parametrize("M,d,tx,ty", [(1, 512, nb.F32, nb.F32), (7, 2048, nb.F32, nb.BF16), (9000, 512, nb.BF16, nb.BF16), (2500, 4096, nb.F16, nb.F16)])
def test_a_scalar_gate_lies_anywhere(M, d, tx, ty):
    """One of an array of gates, a layer each: its address changes nothing, nor does the stride of an h that is not written."""
    x, y, g, ps, pre = inputs(M, d, tx, ty, "scalar", True, M + d)
    gates = torch.zeros(8, device="cuda")
    xd, yd, pd, prd = cuda(x, y, ps, pre)
    got = []
    for at in (0, 1, 2, 3):
        gates.fill_(float("nan"))
        gates[at] = g[0]
        rd, hd, r2 = torch.empty_like(xd), torch.empty_like(yd), torch.empty_like(xd)
        common = dict(post_scale_ptr=p(pd), gate_ptr=p(gates[at:]), gate_flags=nb.GATE_SCALAR | nb.GATE_SIGMOID)
        nb.residual_norm(p(xd), tx, p(yd), ty, M, d, p(prd), p(rd), p(hd), ty, **common)
        nb.residual_norm(p(xd), tx, p(yd), ty, M, d, None, p(r2), None, ty, ldh=d + at, **common)
        got.append((rd, hd, r2))
    r, h, er, eh = reference(x, y, ps, g, True, 1.0, pre)
    close(got[1][0], r, rounded(er, r, tx))
    close(got[1][1], h, rounded(eh, h, ty))
    for t in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(t, got[0]))


@pytest.mark.parametrize("M,d", [(3, 512), (3, 131), (9000, 512), (9000, 257), (20000, 33), (2500, 2051), (1500, 4099), (1300, 8191)])
def test_wide_f32_gates(M, d):
    """The logistic function of f32 gates from -90 to 90: a few roundings, however far it is from 1.  x is zero, so
    that r is the gated y alone; h follows the largest of a row.  (At -90 the function is below the normal range, where
    exp(90) is infinite: 0 or its value, both within 2^-126.)"""
    g = torch.Generator().manual_seed(d)
    x, y = torch.zeros(M, d), torch.randn(M, d, generator=g)
    gate = (torch.rand(d, generator=g) * 2 - 1) * 90
    gate[:5] = torch.tensor([-90.0, -87.0, -20.0, 20.0, 90.0])
    xd, yd, gd = cuda(x, y, gate)
    rd = torch.empty_like(xd)
    nb.residual_norm(p(xd), nb.F32, p(yd), nb.F32, M, d, None, p(rd), None, nb.F32, gate_ptr=p(gd), gate_flags=nb.GATE_CHANNEL | nb.GATE_SIGMOID)
    want = y.double() * torch.sigmoid(gate.double())
    # exp within 2 units, a unit being 2 U (and its own share of the sum), the sum, the quotient and the product half a unit each
    close(rd, want, (2 * 2 + 3) * U * (1 + U) ** 8 * want.abs() + y.double().abs() * 2.0 ** -126)


@pytest.mark.parametrize("M,d", [(5, 257), (9000, 257), (20000, 33), (9000, 512)])
@pytest.mark.parametrize("where", ["gate", "post"])
def test_an_infinite_factor_stays_in_its_column(where, M, d):
    """r is infinite in the last column alone; the row's mean is then infinite, and h = r / sqrt(infinity) is 0
    in the other columns and NaN (infinity * 0) in that one."""
    g = torch.Generator().manual_seed(d)
    x, y, one = torch.randn(M, d, generator=g), torch.randn(M, d, generator=g), torch.zeros(d)
    far = torch.zeros(d)
    far[-1] = float("inf")
    xd, yd, fd, od = cuda(x, y, far if where == "post" else far + 1, one)
    rd, hd = torch.empty_like(xd), torch.empty_like(yd)
    a = dict(post_scale_ptr=p(fd)) if where == "post" else dict(gate_ptr=p(fd), gate_flags=nb.GATE_CHANNEL)
    nb.residual_norm(p(xd), nb.F32, p(yd), nb.F32, M, d, p(od), p(rd), p(hd), nb.F32, **a)
    assert torch.isfinite(rd[:, :-1]).all() and torch.isinf(rd[:, -1]).all()
    assert (hd[:, :-1] == 0).all() and torch.isnan(hd[:, -1]).all()
