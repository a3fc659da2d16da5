"""The 8-bit product on the GPU: quantised values bit for bit, and the product
against 64-bit arithmetic."""
import numpy as np
import pytest

from conftest import load_pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

nb = load_pkg()
TYPES = {nb.F32: torch.float32, nb.F16: torch.float16, nb.BF16: torch.bfloat16}
U = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


def rows(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(TYPES[dtype])


def quantized(x):
    """(values, scales) of f32 rows by the documented formula, each step rounded to f32."""
    x = x.float().numpy()
    with np.errstate(all="ignore"):
        top = np.abs(x).max(axis=1).astype(np.float32)
        bad = ~np.isfinite(x).all(axis=1)
        some = ~bad & (top >= np.float32(127.0 * 2.0 ** -126))
        scale = np.where(some, top / np.float32(127), np.float32(0)).astype(np.float32)
        inv = np.where(some, np.float32(127) / top, np.float32(0)).astype(np.float32)
        q = np.where(some[:, None], np.rint(x * inv[:, None]), 0).astype(np.int8)
    scale[bad] = np.nan
    return q, scale


def random_weight(N, K, seed):
    g = torch.Generator().manual_seed(seed)
    Kp = nb.int8_row_bytes(K)
    w = torch.zeros((N, Kp), dtype=torch.int8)
    w[:, :K] = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    return w, torch.rand(N, generator=g) * 0.02 + 0.001


def expected(q, qs, w, ws, bias, K):
    """(product, result) in 64 bits."""
    acc = q[:, :K].double() @ w[:, :K].double().t()
    prod = acc * (qs.double()[:, None] * ws.double()[None])
    return prod, prod if bias is None else prod + bias.double()


def check(got, prod, want, dtype):
    # roundings to f32: the sum, the scales' product, the product, the bias; then one to the type
    e = torch.finfo(TYPES[dtype])
    tol = 4 * U * (prod.abs() + want.abs()) + e.eps / 2 * want.abs() * (1 + 8 * U) + e.tiny * e.eps / 2
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,pad", [(1, 1, 0), (1, 512, 0), (3, 17, 5), (8, 1000, 0), (65, 130, 2), (5, 4096, 8), (2, 33000, 0)])
def test_quantize_tokens(M, K, pad, dtype):
    x = rows((M, K + pad), dtype, M * K, 3.0)
    want, ws = quantized(x[:, :K])
    Kp = nb.int8_row_bytes(K)
    xd, q, s = x.cuda(), torch.full((M, Kp), 99, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    nb.int8_quantize_tokens(xd.data_ptr(), M, K, q.data_ptr(), s.data_ptr(), dtype, K + pad)
    q = q.cpu().numpy()
    assert np.array_equal(q[:, :K], want) and np.array_equal(s.cpu().numpy(), ws) and not q[:, K:].any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K", [(20001, 40), (20000, 72), (9000, 512), (6000, 1000), (4000, 2056), (3001, 4096), (2500, 4104), (1300, 8192),
                                 (3000, 617), (70000, 8), (1000, 20001)])
def test_quantize_many_tokens(M, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + K)
    x = (torch.randn((M, K), generator=g, device="cuda") * torch.exp(torch.randn((M, 1), generator=g, device="cuda"))).to(TYPES[dtype])
    Kp = nb.int8_row_bytes(K)
    q, s = torch.full((M + 1, Kp), 99, dtype=torch.int8, device="cuda"), torch.full((M + 1,), 5.0, device="cuda")
    nb.int8_quantize_tokens(x.data_ptr(), M, K, q.data_ptr(), s.data_ptr(), dtype)
    want, ws = quantized(x.cpu())
    q = q.cpu().numpy()
    assert np.array_equal(q[:M, :K], want) and not q[:M, K:].any() and (q[M] == 99).all()
    assert np.array_equal(s.cpu().numpy()[:M], ws) and s[M] == 5


def test_quantize_odd_rows():
    # zeros, subnormals, the largest values, ties, an infinity and NaN
    x = torch.zeros((8, 40))
    x[1] = 1e-40
    x[2] = 3.0e38
    x[2, 3] = -3.4e38
    x[3] = torch.arange(40) - 20 + 0.5
    x[3, 0] = 127.0
    x[4, 7] = float("inf")
    x[5, 39] = float("nan")
    x[6, 1] = -1e-36
    x[7, 2] = 127 * 2.0 ** -126
    want, ws = quantized(x)
    xd = x.cuda()
    for off in (0, 1):  # the second pass from rows that are not 16-byte aligned
        src = torch.zeros(8 * 41 + 4, device="cuda")
        ld = 40 + off
        view = src[off:off + 8 * ld].view(8, ld)[:, :40]
        view.copy_(xd)
        q, s = torch.empty((8, 48), dtype=torch.int8, device="cuda"), torch.empty(8, device="cuda")
        nb.int8_quantize_tokens(view.data_ptr(), 8, 40, q.data_ptr(), s.data_ptr(), nb.F32, ld)
        assert np.array_equal(q.cpu().numpy()[:, :40], want)
        assert np.array_equal(s.cpu().numpy(), ws, equal_nan=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,N", [(1, 1), (17, 33), (512, 64), (1000, 31), (64, 1523)])
def test_quantize_weight(K, N, dtype):
    w = rows((K, N), dtype, K + N)
    want, ws = quantized(w.t().contiguous())
    d, s = torch.full((N, nb.int8_row_bytes(K)), 7, dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda")
    wd = w.cuda()
    nb.int8_quantize_weight(wd.data_ptr(), K, N, d.data_ptr(), s.data_ptr(), dtype)
    assert np.array_equal(d.cpu().numpy()[:, :K], want) and np.array_equal(s.cpu().numpy(), ws)


SIZES = [(1, 1, 1), (1, 16, 16), (1, 512, 2048), (2, 17, 130), (7, 1000, 129), (8, 4096, 64), (9, 96, 512), (16, 512, 8192),
         (17, 31, 33), (33, 513, 257), (64, 2048, 512), (65, 160, 1), (100, 128, 384), (127, 4097, 200), (128, 128, 128),
         (129, 129, 129), (200, 1000, 1523), (256, 512, 2048), (257, 300, 700), (300, 64, 5000), (1025, 640, 320), (4097, 144, 72)]


@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(M, K, N):
    x_dtype, y_dtype = (M + N) % 3, (M + K) % 3
    with_bias = (M + K + N) % 2 == 0
    w, ws = random_weight(N, K, M + K + N)
    x = rows((M, K), x_dtype, 5 * M + N)
    bias = rows((N,), nb.F32, 3) if with_bias else None
    q, qs = quantized(x)
    prod, want = expected(torch.from_numpy(q), torch.from_numpy(qs), w, ws, bias, K)
    wd, wsd, xd = w.cuda(), ws.cuda(), x.cuda()
    bd = bias.cuda() if with_bias else None
    plan = nb.Int8Plan(wd.data_ptr(), wsd.data_ptr(), K, N, M)
    # rows of y two elements apart from each other, which stay as they were
    y = torch.full((M + 1, N + 2), 7.0, dtype=TYPES[y_dtype], device="cuda")
    plan.matmul(xd.data_ptr(), M, y.data_ptr(), x_dtype, y_dtype, ldy=N + 2, bias_ptr=bd.data_ptr() if with_bias else None)
    plan.status()
    check(y[:M, :N], prod, want, y_dtype)
    assert (y[M] == 7).all() and (y[:M, N:] == 7).all()
    # the same from rows quantised beforehand, and again: the same bits
    qp = torch.zeros((M, nb.int8_row_bytes(K)), dtype=torch.int8)
    qp[:, :K] = torch.from_numpy(q)
    qp[:, K:] = 55  # never read
    qd, qsd = qp.cuda(), torch.from_numpy(qs).cuda()
    for _ in range(2):
        y2 = torch.full((M, N), float("nan"), dtype=TYPES[y_dtype], device="cuda")
        plan.matmul_quantized(qd.data_ptr(), qsd.data_ptr(), M, y2.data_ptr(), y_dtype, bias_ptr=bd.data_ptr() if with_bias else None)
        assert torch.equal(y2, y[:M, :N])
    plan.close()


def test_weight_pad_is_never_read():
    M, K, N = 40, 100, 64
    w, ws = random_weight(N, K, 1)
    x = rows((M, K), nb.F32, 2)
    ys = []
    for pad in (0, 77):
        w[:, K:] = pad
        wd, wsd, xd, y = w.cuda(), ws.cuda(), x.cuda(), torch.empty((M, N), device="cuda")
        for m in (1, M):
            nb.Int8Plan(wd.data_ptr(), wsd.data_ptr(), K, N, M).matmul(xd.data_ptr(), m, y.data_ptr())
        ys.append(y.cpu())
    assert torch.equal(*ys)


def test_largest_sum():
    # the largest K with every product at its extreme: the sum needs all 31 bits
    K, M, N = 131071, 2, 20
    Kp = nb.int8_row_bytes(K)
    w = torch.full((N, Kp), -128, dtype=torch.int8, device="cuda")
    q = torch.full((M, Kp), -128, dtype=torch.int8, device="cuda")
    q[1] = 127
    one = torch.ones(N, device="cuda")
    y = torch.empty((M, N), device="cuda")
    nb.Int8Plan(w.data_ptr(), one.data_ptr(), K, N, M).matmul_quantized(q.data_ptr(), one.data_ptr(), M, y.data_ptr())
    want = torch.tensor([[K * 16384.0], [-K * 127.0 * 128.0]], dtype=torch.float64)
    assert ((y.cpu().double() - want).abs() <= U * want.abs()).all()


def test_bad_rows_give_nan_and_leave_the_others():
    M, K, N = 70, 256, 300
    w, ws = random_weight(N, K, 9)
    x = rows((M, K), nb.BF16, 1)
    x[3, 5], x[40, 0] = float("nan"), float("inf")
    x[41] = 0
    wd, wsd, xd, y = w.cuda(), ws.cuda(), x.cuda(), torch.zeros((M, N), device="cuda")
    nb.Int8Plan(wd.data_ptr(), wsd.data_ptr(), K, N, M).matmul(xd.data_ptr(), M, y.data_ptr(), nb.BF16)
    y = y.cpu()
    bad = torch.zeros(M, dtype=torch.bool)
    bad[3] = bad[40] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all() and (y[41] == 0).all()


def test_graph_and_stream():
    # captured on a side stream and replayed on new tokens; fewer rows than the plan's
    M, K, N = 24, 512, 1000
    w, ws = random_weight(N, K, 4)
    wd, wsd = w.cuda(), ws.cuda()
    x, y = torch.zeros((M, K), device="cuda"), torch.zeros((M, N), device="cuda")
    plan = nb.Int8Plan(wd.data_ptr(), wsd.data_ptr(), K, N, 64)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        plan.matmul(x.data_ptr(), M, y.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        new = rows((M, K), nb.F32, seed)
        x.copy_(new)
        g.replay()
        q, qs = quantized(new)
        check(y, *expected(torch.from_numpy(q), torch.from_numpy(qs), w, ws, None, K), nb.F32)
    plan.status()


def test_plan_refuses():
    w, ws = torch.zeros((32, 64), dtype=torch.int8, device="cuda"), torch.zeros(32, device="cuda")
    x = torch.zeros((9, 64), device="cuda")
    plan = nb.Int8Plan(w.data_ptr(), ws.data_ptr(), 64, 32, 8)
    p = x.data_ptr()
    for a, k in [((p, 9, p), {}), ((p, 0, p), {}), ((None, 1, p), {}), ((p, 1, p, nb.I8), {}), ((p, 1, p), dict(ldx=63)),
                 ((p, 1, p), dict(ldy=31)), ((p + 2, 1, p), {}), ((p, 1, p + 2), {}), ((p, 1, p), dict(bias_ptr=p + 1))]:
        with pytest.raises(nb.NeedleError, match="invalid plan matmul"):
            plan.matmul(*a, **k)
    host = np.zeros(4096, np.float32)
    with pytest.raises(nb.NeedleError, match="device memory|CUDA error"):
        plan.matmul(host.ctypes.data, 1, p)
    with pytest.raises(nb.NeedleError, match="invalid plan matmul"):
        plan.matmul_quantized(p + 4, p, 1, p)


def launched(call):
    """Names of the kernels that call(stream) launches, in order, from a graph that captures it."""
    driver = pytest.importorskip("cuda.bindings.driver")
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        call(torch.cuda.current_stream().cuda_stream)
    graph = driver.CUgraph(g.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(graph)
    err, nodes, n = driver.cuGraphGetNodes(graph, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    names = []
    for node in nodes[:n]:
        if driver.cuGraphNodeGetType(node)[1] != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        err, params = driver.cuGraphKernelNodeGetParams(node)
        assert err == driver.CUresult.CUDA_SUCCESS
        err, name = driver.cuFuncGetName(params.func) if int(params.func) else driver.cuKernelGetName(params.kern)
        assert err == driver.CUresult.CUDA_SUCCESS
        names.append(name.decode())
    return names


# M, K, N and the kernel of the product: tiles of 16 to 256 tokens, and pairs of CTAs with 256 x 256 tiles, whose last
# tiles have few or odd channels, tokens and values of K; 153 tiles on 74 pairs use both accumulators again
FORMS = [(1, 512, 2048, "int8_tc_kernelILi16E"), (16, 2048, 2048, "int8_tc_kernelILi16E"), (31, 4096, 4096, "int8_tc_kernelILi32E"),
         (64, 4096, 4096, "int8_tc_kernelILi64E"), (200, 2050, 5001, "int8_tc_kernelILi128E"), (2100, 70, 8200, "int8_tc_kernelILi256E"),
         (1025, 2050, 3001, "int8_pair_kernel"), (2049, 2050, 3001, "int8_pair_kernel"), (2049, 1100, 4099, "int8_pair_kernel"),
         (4096, 512, 4096, "int8_pair_kernel"), (2305, 4097, 2304, "int8_pair_kernel")]


@pytest.mark.parametrize("y_dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N,form", FORMS)
def test_every_form_of_the_product(M, K, N, form, y_dtype):
    g = torch.Generator(device="cuda").manual_seed(M + K + N)
    Kp = nb.int8_row_bytes(K)
    w = torch.full((N, Kp), 99, dtype=torch.int8, device="cuda")  # past K: never read
    w[:, :K] = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device="cuda")
    ws = torch.rand(N, generator=g, device="cuda") * 0.02 + 0.001
    bias = torch.randn(N, generator=g, device="cuda")
    x_dtype = (M + y_dtype) % 3
    x = torch.randn((M, K + 8), generator=g, device="cuda").to(TYPES[x_dtype])
    q, qs = quantized(x[:, :K].cpu())
    qd = torch.full((M, Kp), 55, dtype=torch.int8, device="cuda")
    qd[:, :K] = torch.from_numpy(q).cuda()
    qsd = torch.from_numpy(qs).cuda()
    # exact in 64 bits: the sums stay below 2^53
    prod = (qd[:, :K].double() @ w[:, :K].double().t()) * (qsd.double()[:, None] * ws.double()[None])
    want = (prod + bias.double()).cpu()
    plan = nb.Int8Plan(w.data_ptr(), ws.data_ptr(), K, N, M + 3)
    y = torch.full((M + 1, N + 3), 7.0, dtype=TYPES[y_dtype], device="cuda")

    def call(st):
        plan.matmul(x.data_ptr(), M, y.data_ptr(), x_dtype, y_dtype, ldx=K + 8, ldy=N + 3, bias_ptr=bias.data_ptr(), stream=st)

    call(None)
    plan.status()
    check(y[:M, :N], prod.cpu(), want, y_dtype)
    assert (y[M] == 7).all() and (y[:M, N:] == 7).all()
    y2 = torch.full((M, N), float("nan"), dtype=TYPES[y_dtype], device="cuda")
    plan.matmul_quantized(qd.data_ptr(), qsd.data_ptr(), M, y2.data_ptr(), y_dtype, bias_ptr=bias.data_ptr())
    plan.status()
    assert torch.equal(y2, y[:M, :N])
    assert form in launched(call)[-1], launched(call)
