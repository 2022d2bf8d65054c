"""The dense FP8 linear map against its definition in 64 bits.

Codes and scales are compared bit for bit with the FP32 definition.  A product is held to
    |y - exact| <= half a step of the output type * |exact| + (K-blocks + 16) * 2^-23 * S,      S = sum |terms|
The second part counts FP32 roundings, each at most 2^-24 of a partial sum that S bounds (doubled, since the tensor core's
rounding is not specified): one per K-block for the promotion, two for the scale, up to 8 for joining the parts of a split,
and four accumulations plus an alignment inside a K-block of the tensor core."""
import pytest
import torch

from netra_kernel_b200 import abi, balance, dense

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def blocks(n):
    return -(-n // 128)


def quantize_definition(x):
    """FP32 definition on the CPU, one rounding at a time."""
    m, k = x.shape
    pad = torch.zeros(m, blocks(k) * 128)
    pad[:, :k] = x.detach().cpu().float()
    b = pad.view(m, blocks(k), 128)
    scale = b.abs().amax(dim=2).clamp_min(1e-10) * torch.tensor(1.0 / 448.0, dtype=torch.float32)
    q = (b * (1.0 / scale)[:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(m, -1)[:, :k]
    return q, scale


def make_weight(n, k, seed, pitch=None):
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.exp(torch.randn(blocks(n), blocks(k), generator=g)) * 1e-3
    if pitch is None:
        pitch = -(-k // 16) * 16
    full = torch.full((n, pitch), 0x7f, dtype=torch.uint8)          # NaN behind the rows: it must not be read into a sum
    full[:, :k] = codes.view(torch.uint8)
    w = full.cuda().view(torch.float8_e4m3fn)[:, :k]
    return w, scale.cuda()


def exact_product(q, s, w, ws, transposed):
    """(sum, sum of magnitudes) in 64 bits from the codes' values."""
    n, k = w.shape
    wv = w.cpu().float().double() * ws.cpu().double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:n, :k]
    av = q.cpu().float().double() * s.cpu().double().repeat_interleave(128, 1)[:, :q.shape[1]]
    wv = wv if transposed else wv.T
    return av @ wv, av.abs() @ wv.abs()


def check_product(y, q, s, w, ws, transposed=False):
    want, size = exact_product(q, s, w, ws, transposed)
    kb = s.shape[1]
    tol = torch.finfo(y.dtype).eps / 2 * want.abs() + (kb + 16) * 2.0 ** -23 * size
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                       # half a subnormal step
    err = (y.cpu().double() - want).abs()
    assert y.shape == want.shape
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))


SIZES = [(1, 16, 16), (1, 2048, 4096), (2, 1, 128), (3, 129, 112), (7, 64, 144), (8, 300, 1040), (9, 65, 128), (12, 512, 2048),
         (16, 127, 256), (17, 128, 384), (31, 1043, 272), (33, 96, 4112), (64, 256, 512), (100, 63, 640), (127, 192, 128), (128, 128, 128),
         (129, 257, 2064), (200, 2048, 512), (257, 512, 1024), (300, 80, 16), (777, 1043, 2064), (1024, 640, 384), (1500, 1280, 256),
         (1, 1, 1), (4, 1, 260), (5, 33, 77), (20, 200, 131), (140, 97, 1001), (64, 2048, 2048), (40, 130, 16400), (130, 1, 4100)]


@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 7), (5, 130), (16, 1000), (33, 2048), (257, 144), (64, 4112), (2000, 640)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_bit_for_bit(m, k, dtype):
    g = torch.Generator().manual_seed(m * 1000 + k)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g) * 3)).to(dtype)
    x[0, : min(k, 128)] = 0                                          # a block of zeros takes the smallest scale
    x[-1, -1] = 3e-12 if dtype == torch.float32 else 0.0
    codes, scale = dense.quantize_rows(x.cuda())
    want, want_scale = quantize_definition(x)
    assert codes.shape == (m, k) and scale.shape == (m, blocks(k)) and codes.dtype == torch.float8_e4m3fn
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(codes.cpu().view(torch.uint8) & 0xff, want.view(torch.uint8) & 0xff)


def test_quantize_rows_strides_and_extremes():
    g = torch.Generator().manual_seed(3)
    base = torch.randn(40, 700, generator=g).to(torch.bfloat16)
    for view in (lambda t: t[::2, 3:500], lambda t: t[5:6, 1:130], lambda t: t[:, :384], lambda t: t.t()[10:200, :]):
        codes, scale = dense.quantize_rows(view(base.cuda()))
        want, want_scale = quantize_definition(view(base))
        assert torch.equal(scale.cpu(), want_scale) and torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))
    codes, scale = dense.quantize_rows(base.cuda()[:1, :256].expand(5, 256))          # rows that share memory
    assert torch.equal(codes[4].view(torch.uint8), codes[0].view(torch.uint8))
    codes, scale = dense.quantize_rows(base.cuda().view(5, 8, 700))
    assert codes.shape == (40, 700)
    assert dense.quantize_rows(base.cuda()[:0])[0].shape == (0, 700)
    big = torch.tensor([[3.3e38, -1e38, 1.0, 0.0], [1e-38, 1e-45, -2e-12, 0.0]])
    codes, scale = dense.quantize_rows(big.cuda())
    want, want_scale = quantize_definition(big)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))
    bad = torch.zeros(3, 256)
    bad[0, 5], bad[1, 200], bad[2, 0] = float("nan"), float("inf"), 1.0
    codes, scale = dense.quantize_rows(bad.cuda())
    values = codes.float().cpu()
    assert bool(values[0, 5].isnan()) and bool(torch.isfinite(values[0, 128:]).all()) and scale[1, 1].item() == float("inf")
    y = dense.fp8_linear(bad.cuda(), *make_weight(16, 256, 1))
    assert bool(y[0].isnan().all()) and bool(y[1].isnan().all()) and bool(torch.isfinite(y[2]).all())


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_against_64_bits(m, n, k):
    dtype = TYPES[(m + n + k) % 3]
    g = torch.Generator().manual_seed(m + 7 * n + 13 * k)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    w, ws = make_weight(n, k, n + k)
    y = dense.fp8_linear(x.cuda(), w, ws)
    assert y.dtype == dtype
    check_product(y, *quantize_definition(x), w, ws)
    codes, scale = dense.quantize_rows(x.cuda())
    for out_dtype in TYPES:
        check_product(dense.block_scaled_matmul(codes, scale, w, ws, out_dtype=out_dtype), *quantize_definition(x), w, ws)
    dense.check_status()


# outputs of many tiles: whole and ragged in every direction, one K-block and several, each element type and pitch
LARGE = [(2500, 2312, 400, torch.bfloat16), (700, 8200, 144, torch.float16), (4097, 1043, 272, torch.float32), (2305, 2305, 16, torch.bfloat16),
         (2048, 2560, 1024, torch.float32), (9000, 520, 528, torch.float16)]


@pytest.mark.parametrize("m,n,k,dtype", LARGE)
def test_large_products_against_64_bits(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + n)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    w, ws = make_weight(n, k, n + k)
    frame = torch.full((m + 1, n + 3), 7.0, device="cuda", dtype=dtype)
    check_product(dense.fp8_linear(x.cuda(), w, ws), *quantize_definition(x), w, ws)
    codes, scale = dense.quantize_rows(x.cuda())
    y = dense.block_scaled_matmul(codes, scale, w, ws, out=frame[:-1, 2:-1])
    check_product(y, *quantize_definition(x), w, ws)
    assert bool((frame[-1] == 7.0).all()) and bool((frame[:, :2] == 7.0).all()) and bool((frame[:, -1] == 7.0).all())
    # the same sizes with the weight as stored: [m, k] codes times [k, n]
    w, ws = make_weight(k, n, n)
    y = dense.block_scaled_matmul(codes, scale, w, ws, transpose_weight=True, out_dtype=dtype)
    check_product(y, *quantize_definition(x), w, ws, True)
    dense.check_status()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_transposed_product_against_64_bits(m, n, k):
    """The gradient form: [m, n] codes times the weight [n, k] as stored."""
    g = torch.Generator().manual_seed(m + 7 * n + 13 * k)
    x = torch.randn(m, n, generator=g).to(TYPES[(m + k) % 3])
    w, ws = make_weight(n, k, n + k)
    codes, scale = dense.quantize_rows(x.cuda())
    for out_dtype in TYPES:
        y = dense.block_scaled_matmul(codes, scale, w, ws, transpose_weight=True, out_dtype=out_dtype)
        check_product(y, *quantize_definition(x), w, ws, True)
    dense.check_status()


def test_operand_layouts():
    """Row pitches, row-major scales, an output that is part of a larger matrix, weights whose scales are a view."""
    g = torch.Generator().manual_seed(5)
    m, n, k = 45, 200, 400
    x = torch.randn(m, k, generator=g)
    w, ws = make_weight(n, k, 2, pitch=448)
    wide = torch.zeros(blocks(n), 9, device="cuda")
    wide[:, 3:3 + blocks(k)] = ws
    codes, scale = dense.quantize_rows(x.cuda())
    padded = torch.full((m, 512), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :k]
    padded.view(torch.uint8).copy_(codes.view(torch.uint8))
    frame = torch.full((m + 2, n + 5), 7.0, device="cuda")
    y = dense.block_scaled_matmul(padded, scale.contiguous(), w, wide[:, 3:3 + blocks(k)], out=frame[1:-1, 2:-3])
    check_product(y, *quantize_definition(x), w, ws)
    inner = frame.clone()
    inner[1:-1, 2:-3] = 7.0
    assert bool((inner == 7.0).all())                                # nothing beside the output was written
    lead = dense.fp8_linear(x.cuda().view(5, 9, k), w, ws)
    assert lead.shape == (5, 9, n) and torch.equal(lead.view(m, n), dense.fp8_linear(x.cuda(), w, ws))
    assert dense.fp8_linear(x.cuda()[:0], w, ws).shape == (0, n)
    assert dense.fp8_linear(x.cuda()[:, :, None], w[:, :1], ws[:, :1]).shape == (m, k, n)
    assert torch.equal(dense.fp8_linear(x.cuda()[3], w, ws), dense.fp8_linear(x.cuda()[3:4], w, ws)[0])
    t = torch.zeros(k, m, device="cuda")
    t.copy_(x.t())
    assert torch.equal(dense.fp8_linear(t.t(), w, ws), dense.fp8_linear(x.cuda(), w, ws))


@pytest.mark.parametrize("m,k", [(1, 1040), (5, 264), (16, 640), (17, 640), (32, 272), (33, 1040)])
def test_alignment_of_the_activations_changes_nothing(m, k):
    """Rows on any boundary take other accesses (and, for few rows, a quantiser launch of their own) to the same bits."""
    g = torch.Generator().manual_seed(m)
    for dtype in TYPES:
        wide = torch.randn(m, k + 24, generator=g).to(dtype).cuda()
        w, ws = make_weight(80, k, 6)
        want = dense.fp8_linear(wide[:, 5:5 + k].clone(), w, ws)
        assert torch.equal(dense.fp8_linear(wide[:, 5:5 + k], w, ws), want)
        check_product(want, *quantize_definition(wide[:, 5:5 + k]), w, ws)


def test_runs_repeat_and_zero_rows_stay_zero():
    g = torch.Generator().manual_seed(6)
    for m in (5, 40, 300):
        x = torch.randn(m, 1040, generator=g).to(torch.bfloat16)
        x[m // 2] = 0
        w, ws = make_weight(520, 1040, 4)
        y = dense.fp8_linear(x.cuda(), w, ws)
        assert bool((y[m // 2] == 0).all())
        for _ in range(3):
            assert torch.equal(dense.fp8_linear(x.cuda(), w, ws), y)


@pytest.mark.parametrize("m,n,k", [(1, 32, 16), (4, 256, 512), (37, 144, 272), (300, 512, 640)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_is_the_formula(m, n, k, dtype):
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).to(dtype).cuda().requires_grad_()
    w, ws = make_weight(n, k, n)
    dy = (torch.randn(m, n, generator=g) * 0.3).to(dtype)
    y = dense.fp8_linear(x, w, ws)
    deep = x.detach().view(1, m, 1, k).requires_grad_()
    (deep_dx,) = torch.autograd.grad(dense.fp8_linear(deep, w, ws), deep, dy.cuda().view(1, m, 1, n))
    (none,) = torch.autograd.grad(dense.fp8_linear(x[:0], w, ws).sum(), x)
    assert bool((none == 0).all())
    (dx,) = torch.autograd.grad(y, x, dy.cuda())
    assert dx.dtype == dtype
    check_product(dx, *quantize_definition(dy), w, ws, True)
    assert deep_dx.shape == deep.shape and torch.equal(deep_dx.view(m, k), dx)
    (dx2,) = torch.autograd.grad(dense.fp8_linear(x, w, ws).sum(), x)        # an expanded gradient
    check_product(dx2, *quantize_definition(torch.ones(m, n).to(dtype)), w, ws, True)
    with torch.no_grad():
        assert not dense.fp8_linear(x, w, ws).requires_grad


def test_gradient_against_differences():
    """Rows whose values are codes (every block's largest magnitude 448, so the scale is 448 * fl(1/448)) move to other codes:
    the map is linear between them, so <dy, y(x + d) - y(x)> = <dx, d> up to FP32 rounding."""
    g = torch.Generator().manual_seed(8)
    m, n, k = 6, 256, 384
    def codes(cols):
        v = torch.randint(-15, 16, (m, cols), generator=g).float()
        v[:, ::128] = 448.0
        return v
    x, dy = codes(k), codes(n)
    d = torch.randint(-1, 2, (m, k), generator=g).float()
    d[:, ::128] = 0
    w, ws = make_weight(n, k, 3)
    xg = x.cuda().requires_grad_()
    y0 = dense.fp8_linear(xg, w, ws)
    (dx,) = torch.autograd.grad(y0, xg, dy.cuda())
    y1 = dense.fp8_linear((x + d).cuda(), w, ws)
    left = ((y1 - y0.detach()).cpu().double() * dy.double()).sum()
    right = (dx.cpu().double() * d.double()).sum()
    s448 = float(torch.tensor(448.0) * torch.tensor(1.0 / 448.0, dtype=torch.float32))
    assert abs(s448 - 1.0) <= 2.0 ** -24
    size = (y0.detach().abs() + y1.abs()).cpu().double().mul(dy.abs().double()).sum() + (dx.abs().cpu().double() * d.abs().double()).sum()
    _, big = exact_product(*quantize_definition(x), w, ws, False)
    tol = (3 + 16 + 8) * 2.0 ** -23 * (size + 2 * (big * dy.abs().double()).sum())
    assert abs(left - right) <= tol, (float(left), float(right), float(tol))


def test_streams_and_captured_graphs():
    g = torch.Generator().manual_seed(9)
    w, ws = make_weight(512, 640, 5)
    xs = [torch.randn(m, 640, generator=g).to(torch.bfloat16).cuda() for m in (3, 90, 260)]
    want = [dense.fp8_linear(x, w, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(20):                                              # calls that overlap share nothing
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense.fp8_linear(xs[i], w, ws))
    torch.cuda.synchronize()
    for i in range(len(xs)):
        assert all(torch.equal(y, want[i]) for y in got[i])
    static = xs[1].clone()
    graphs, outs = [], []
    for _ in range(2):                                               # two graphs of the same call
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(dense.fp8_linear(static, w, ws))
        graphs.append(graph)
    for trial in range(3):
        static.copy_(torch.randn(90, 640, generator=g).to(torch.bfloat16))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        y = dense.fp8_linear(static, w, ws)
        assert torch.equal(outs[0], y) and torch.equal(outs[1], y)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()          # a fork and a join inside one graph
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            left = dense.fp8_linear(static, w, ws)
        right = dense.fp8_linear(xs[2], w, ws)
        torch.cuda.current_stream().wait_stream(side)
        both = dense.fp8_linear(torch.cat([left, right])[:, :256].contiguous(), w[:, :256], ws[:, :2])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(left, dense.fp8_linear(static, w, ws)) and torch.equal(right, want[2])
    assert torch.equal(both, dense.fp8_linear(torch.cat([left, right])[:, :256].contiguous(), w[:, :256], ws[:, :2]))
    leaf = xs[1].clone().requires_grad_()
    dy = torch.randn(90, 512, generator=g).to(torch.bfloat16).cuda()
    (eager,) = torch.autograd.grad(dense.fp8_linear(leaf, w, ws), leaf, dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dx,) = torch.autograd.grad(dense.fp8_linear(leaf, w, ws), leaf, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, eager)
    dense.check_status()


@pytest.mark.parametrize("m", [3, 12, 20, 32, 200, 2600])
def test_chains_of_dependent_calls(m):
    """Each call reads what the one before it wrote, into memory that the allocator hands around, with nothing between them: the
    kernels start before their predecessors end and must not see what the memory held earlier."""
    n, depth = 512, 24
    w, ws = make_weight(n, n, 13)
    ws = ws / ws.mean() * 0.02
    xs = [torch.randn(m, n, device="cuda", dtype=torch.bfloat16, generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(4)]

    def chain(x, wait):
        for _ in range(depth):
            x = dense.fp8_linear(x, w, ws)
            if wait:
                torch.cuda.synchronize()
        return x

    want = [chain(x, True) for x in xs]
    for _ in range(20):
        for x, y in zip(xs, want):
            assert torch.equal(chain(x, False), y)
    static, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(static, False)
    for _ in range(5):
        for x, y in zip(xs, want):
            static.copy_(x)
            graph.replay()
            assert torch.equal(out, y)
    assert bool(torch.isfinite(want[0]).all()) and bool((want[0] != 0).any())
    dense.check_status()


def test_capture_beside_a_living_eager_graph_of_the_leaf_is_refused():
    """torch itself cannot capture this backward pass; the call says so while the capture can still be ended."""
    w, ws = make_weight(64, 128, 1)
    leaf = torch.randn(4, 128, device="cuda").requires_grad_()
    alive = dense.fp8_linear(leaf, w, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="eager graph"):
            dense.fp8_linear(leaf, w, ws)
        with pytest.raises(RuntimeError, match="eager graph"):
            balance.balance_loss(leaf, torch.ones(128, dtype=torch.int32, device="cuda"))
        plain = dense.fp8_linear(leaf.detach(), w, ws)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, alive.detach())
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = dense.fp8_linear(leaf, w, ws), dense.fp8_linear(leaf, w, ws)
        (dx,) = torch.autograd.grad(first.sum() + second.sum(), leaf)
    graph.replay()
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(dense.fp8_linear(leaf, w, ws).sum() * 2, leaf)
    assert torch.allclose(dx, want, rtol=2.0 ** -22, atol=0)


def test_second_derivatives_are_refused():
    w, ws = make_weight(32, 128, 1)
    x = torch.randn(3, 128, device="cuda").requires_grad_()
    dy = torch.ones(3, 32, device="cuda").requires_grad_()
    (dx,) = torch.autograd.grad(dense.fp8_linear(x, w, ws), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dx.sum().backward()
    counts = torch.ones(128, dtype=torch.int32, device="cuda")
    (dz,) = torch.autograd.grad(balance.balance_loss(x, counts), x, torch.ones((), device="cuda").requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dz.sum().backward()


def test_offsets_beyond_32_bits():
    """More than 2^31 activations and outputs: sampled rows against the same rows alone (whole rows are quantised and multiplied
    independently of their neighbours, through the same kernel only if the sizes say so: FP32 rounding apart, as derived above)."""
    m, n, k = 70001, 32784, 144
    w, ws = make_weight(n, k, 9)
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    y = dense.fp8_linear(x, w, ws)
    pick = torch.tensor([0, 1, 32767, 65535, 65536, 65537, 69999, 70000])
    check_product(y[pick.cuda()], *quantize_definition(x[pick.cuda()]), w, ws)
    codes, scale = dense.quantize_rows(y)                             # 2.3e9 elements
    want, want_scale = quantize_definition(y[pick.cuda()])
    assert torch.equal(scale[pick.cuda()].cpu(), want_scale)
    assert torch.equal(codes.view(torch.uint8)[pick.cuda()].cpu(), want.view(torch.uint8))
    dense.check_status()


def test_refusals():
    x = torch.zeros(4, 256, device="cuda")
    w, ws = make_weight(64, 256, 1)
    for call, why in [
        (lambda: dense.fp8_linear(x[:, :255], w, ws), "columns"),
        (lambda: dense.fp8_linear(x.double(), w, ws), "bfloat16"),
        (lambda: dense.fp8_linear(x, w.float(), ws), "float8"),
        (lambda: dense.fp8_linear(x, w, ws.t()), "weight_scale"),
        (lambda: dense.fp8_linear(x, w, ws.cpu()), "device"),
        (lambda: dense.fp8_linear(x, w[:, 8:], ws), "columns"),
        (lambda: dense.fp8_linear(x[:, 8:], w[:, 8:], ws), "16-byte"),
        (lambda: dense.quantize_rows(x.int()), "bfloat16"),
        (lambda: dense.quantize_rows(x[:, :0]), "column"),
    ]:
        with pytest.raises(ValueError, match=why):
            call()
    codes, scale = dense.quantize_rows(x)
    for call, why in [
        (lambda: dense.block_scaled_matmul(x, scale, w, ws), "float8"),
        (lambda: dense.block_scaled_matmul(codes, scale[:, :1], w, ws), "a_scale"),
        (lambda: dense.block_scaled_matmul(codes, scale, w, ws, transpose_weight=True), "reduces"),
        (lambda: dense.block_scaled_matmul(codes, scale, w, ws, out_dtype=torch.float64), "out_dtype"),
        (lambda: dense.block_scaled_matmul(codes, scale, w, ws, out=torch.zeros(4, 63, device="cuda")), "out"),
        (lambda: dense.block_scaled_matmul(codes, scale, w, ws, out=torch.zeros(64, 4, device="cuda").t()), "out"),
        (lambda: dense.block_scaled_matmul(codes[:, 8:], scale, w[:, 8:], ws), "16-byte"),
    ]:
        with pytest.raises(ValueError, match=why):
            call()


def test_router_fine_tuning_step():
    """A frozen FP8 projection, a BF16 router behind it, top-8 choices, counts and balance loss, back to the hidden states and
    the router weight; against the same chain in plain FP32 torch (straight-through quantisers)."""
    g = torch.Generator().manual_seed(21)
    t, k, n, e = 200, 512, 384, 64
    hidden = torch.randn(t, k, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    router = (torch.randn(e, n, generator=g) * 0.1).to(torch.bfloat16).cuda().requires_grad_()
    w, ws = make_weight(n, k, 11)
    mask = (torch.rand(t, generator=g) < 0.8).cuda()

    x = dense.fp8_linear(hidden, w, ws)
    logits = x @ router.t()
    ids = logits.detach().float().topk(8, dim=1).indices
    counts = balance.expert_counts(ids, e, mask)
    loss = balance.balance_loss(logits, counts, mask) * 0.01
    loss.backward()

    q, s = quantize_definition(hidden)
    want_x, _ = exact_product(q, s, w, ws, False)
    assert float((x.detach().cpu().double() - want_x).norm() / want_x.norm()) < 2.0 ** -8
    z = logits.detach().cpu().double().requires_grad_()
    kept = mask.cpu()
    hits = torch.bincount(ids.cpu()[kept].reshape(-1), minlength=e)
    assert torch.equal(counts.cpu().long(), hits)
    p = torch.softmax(z[kept], dim=1).mean(dim=0)
    want = 0.01 * e * (hits.double() / hits.sum() * p).sum()
    want.backward()
    assert abs(loss.item() - want.item()) < 1e-5 * want.item()
    dz = z.grad.to(torch.bfloat16)                                     # as the router's product receives it
    want_router = dz.double().T @ x.detach().cpu().double()
    dx = (dz.double() @ router.detach().cpu().double()).to(torch.bfloat16)
    gq, gs = quantize_definition(dx)
    want_hidden, _ = exact_product(gq, gs, w, ws, True)
    # BF16 gradients of the logits (2^-8 each) pass through two products, an FP8 rounding (2^-4 each) that a BF16 step may tip
    # over to the next code, and a last rounding; relative to the whole gradient 2 * 2^-8 and 2^-4 bound those
    assert float((router.grad.cpu().double() - want_router).norm() / want_router.norm()) < 2.0 ** -7
    assert float((hidden.grad.cpu().double() - want_hidden).norm() / want_hidden.norm()) < 2.0 ** -4
    assert bool((hidden.grad[~mask] == 0).all())
    assert abi.load().netra_moe_last_error() is not None


def test_second_derivatives_are_refused_in_every_call():
    """The loss's gradient depends on the logits themselves, so whatever the upstream gradient is, nothing that holds it can be
    differentiated again: neither back to all leaves nor to chosen ones, and not through a copy of strided logits."""
    from netra_kernel_b200 import torch_ops  # noqa: F401
    counts = torch.arange(16, dtype=torch.int32, device="cuda")
    scale = torch.full((), 2.0, device="cuda")
    for loss_of in (balance.balance_loss, torch.ops.netra.balance_loss):
        for base, view in ((torch.randn(5, 16), lambda t: t), (torch.randn(16, 5), lambda t: t.t())):
            for upstream in (None, scale, scale.clone().requires_grad_()):
                z = base.cuda().requires_grad_()
                loss = loss_of(view(z), counts)
                (dz,) = torch.autograd.grad(loss, z, upstream, create_graph=True)
                penalty = dz.pow(2).sum()
                for again in (lambda: (loss + penalty).backward(retain_graph=True), lambda: torch.autograd.grad(loss + penalty, z, retain_graph=True),
                              lambda: torch.autograd.grad(penalty, z, retain_graph=True)):
                    with pytest.raises(RuntimeError):
                        again()
            with pytest.raises(RuntimeError):
                torch.autograd.functional.hessian(lambda v: loss_of(view(v), counts), base.cuda())
            loss = loss_of(view(z), counts)                            # a first derivative stays a plain tensor
            (dz,) = torch.autograd.grad(loss, z)
            assert not dz.requires_grad
    w, ws = make_weight(32, 128, 1)
    for linear in (dense.fp8_linear, torch.ops.netra.fp8_linear):
        x = torch.randn(3, 128, device="cuda").requires_grad_()
        dy = torch.ones(3, 32, device="cuda").requires_grad_()
        y = linear(x, w, ws)
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        for again in (lambda: torch.autograd.grad(dx.sum() + dy.sum(), dy, retain_graph=True), lambda: (y.sum() + dx.pow(2).sum()).backward()):
            with pytest.raises(RuntimeError):
                again()
        (dx,) = torch.autograd.grad(linear(x, w, ws), x, dy.detach(), create_graph=True)       # depends on nothing that is differentiated
        assert torch.equal(dx, torch.autograd.grad(linear(x, w, ws), x, dy.detach())[0])


def test_forward_mode_is_refused():
    """No output without its tangent: neither for operands that require a gradient nor for those that do not, nor in a backward pass."""
    from torch.autograd import forward_ad
    from netra_kernel_b200 import torch_ops  # noqa: F401
    w, ws = make_weight(64, 256, 1)
    x, z = torch.randn(4, 256, device="cuda"), torch.randn(5, 16, device="cuda")
    counts, one = torch.ones(16, dtype=torch.int32, device="cuda"), torch.ones((), device="cuda")
    codes, scale = dense.quantize_rows(x)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))      # noqa: E731
        leaf, dz = x.clone().requires_grad_(), z.clone().requires_grad_()
        for call in (lambda: dense.fp8_linear(dual(x), w, ws), lambda: dense.fp8_linear(dual(leaf), w, ws), lambda: dense.fp8_linear(x, w, dual(ws)),
                     lambda: dense.fp8_linear(dual(x).t().contiguous().t(), w, ws), lambda: dense.fp8_linear(dual(x)[:0], w, ws),
                     lambda: dense.quantize_rows(dual(x)), lambda: dense.block_scaled_matmul(codes, dual(scale), w, ws),
                     lambda: dense.block_scaled_matmul(codes, scale, w, ws, out=dual(torch.zeros(4, 64, device="cuda"))),
                     lambda: torch.autograd.grad(dense.fp8_linear(leaf, w, ws), leaf, dual(torch.ones(4, 64, device="cuda"))),
                     lambda: balance.balance_loss(dual(z), counts), lambda: balance.balance_loss(dual(dz), counts),
                     lambda: balance.balance_loss_grad(one, dual(z), counts), lambda: balance.balance_loss_grad(dual(one), z, counts),
                     lambda: torch.autograd.grad(balance.balance_loss(dz, counts), dz, dual(one)),
                     lambda: torch.ops.netra.fp8_linear(dual(x), w, ws), lambda: torch.ops.netra.balance_loss(dual(z), counts)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        plain = dense.fp8_linear(x, w, ws)                                # nothing else changes inside a dual level
    assert torch.equal(plain, dense.fp8_linear(x, w, ws))


def test_a_given_output_counts_as_written():
    """A tensor that autograd keeps for a backward pass is not the same one after it has been an output."""
    w, ws = make_weight(64, 256, 1)
    codes, scale = dense.quantize_rows(torch.randn(4, 256, device="cuda"))
    frame, leaf = torch.ones(6, 64, device="cuda"), torch.ones(4, 64, device="cuda").requires_grad_()
    product = (leaf * frame[1:5]).sum()
    assert dense.block_scaled_matmul(codes, scale, w, ws, out=frame[1:5]).data_ptr() == frame[1:5].data_ptr()
    with pytest.raises(RuntimeError, match="inplace operation"):
        product.backward()
    before = frame._version
    dense.block_scaled_matmul(codes[:0], scale[:0], w, ws, out=frame[:0])
    assert frame._version == before                                   # nothing was written
    with torch.inference_mode():
        kept = torch.zeros(4, 64, device="cuda")
        dense.block_scaled_matmul(codes, scale, w, ws, out=kept)
    dense.block_scaled_matmul(codes, scale, w, ws, out=kept)
    assert torch.equal(kept, frame[1:5])


def test_status_waits_for_every_stream():
    """A product still running on a stream of its own has not reported yet."""
    w, ws = make_weight(64, 256, 1)
    x, side = torch.randn(300, 256, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)                                # about 0.2 s
        dense.fp8_linear(x, w, ws)
        done = side.record_event()
    dense.check_status()
    assert done.query()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dense.fp8_linear(x, w, ws)
        with pytest.raises(RuntimeError, match="captured"):
            dense.check_status()
    graph.replay()
    dense.check_status()
    assert torch.equal(y, dense.fp8_linear(x, w, ws))


def test_a_product_of_ready_codes_refuses_operands_that_require_a_gradient():
    w, ws = make_weight(64, 256, 1)
    codes, scale = dense.quantize_rows(torch.randn(4, 256, device="cuda").requires_grad_())
    assert not codes.requires_grad and not scale.requires_grad
    learned, learned_codes = scale.clone().requires_grad_(), codes.clone().requires_grad_()
    for a, s in ((codes, learned), (learned_codes, scale), (codes, learned * 2)):
        with pytest.raises(ValueError, match="gradient"):
            dense.block_scaled_matmul(a, s, w, ws)
        with torch.no_grad():
            y = dense.block_scaled_matmul(a, s, w, ws)
        assert not y.requires_grad and torch.equal(y, dense.block_scaled_matmul(a.detach(), s.detach(), w, ws))


def test_captured_backward_beside_a_living_eager_graph_of_a_leaf_behind_the_operand_is_refused():
    """The leaf may lie behind other operations, and the operators by name know it only in their backward step; what does not reach
    that leaf is captured as usual."""
    from netra_kernel_b200 import torch_ops  # noqa: F401
    w, ws = make_weight(64, 128, 1)
    x, router = torch.randn(4, 128, device="cuda"), torch.randn(64, 64, device="cuda").requires_grad_()
    counts = torch.arange(64, dtype=torch.int32, device="cuda")
    hidden = dense.fp8_linear(x, w, ws)
    warm = torch.zeros(4, 64, device="cuda").requires_grad_()          # torch sets up its matrix products, which a capture does not allow
    torch.autograd.grad((warm @ torch.ones_like(router)).sum(), warm)
    alive = hidden @ router                                            # an eager graph of the router
    leaf = x.clone().requires_grad_()
    alive_linear = leaf * 2
    fresh = torch.zeros(4, 64, device="cuda").requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for loss_of in (balance.balance_loss, torch.ops.netra.balance_loss):
            loss = loss_of(hidden @ router, counts)
            with pytest.raises(RuntimeError, match="eager graph"):
                torch.autograd.grad(loss, router)
            with pytest.raises(RuntimeError, match="eager graph"):
                loss_of(hidden @ router, counts).backward()
        for linear in (dense.fp8_linear, torch.ops.netra.fp8_linear):
            y = linear(leaf + 1, w, ws)
            with pytest.raises(RuntimeError, match="eager graph"):
                torch.autograd.grad(y.sum(), leaf)
        y = torch.ops.netra.fp8_linear(leaf, w, ws)
        with pytest.raises(RuntimeError, match="eager graph"):
            torch.autograd.grad(y.sum(), leaf)
        loss = balance.balance_loss((hidden + fresh) @ router, counts)
        (d_fresh,) = torch.autograd.grad(loss, fresh)
    graph.replay()
    torch.cuda.synchronize()
    again = torch.zeros(4, 64, device="cuda").requires_grad_()
    (want,) = torch.autograd.grad(balance.balance_loss((hidden + again) @ router, counts), again)
    assert torch.equal(d_fresh, want)
    del alive, alive_linear, y, loss
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(torch.ops.netra.balance_loss(hidden @ router, counts), router)
        (got_x,) = torch.autograd.grad(torch.ops.netra.fp8_linear(leaf, w, ws).sum(), leaf)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, torch.autograd.grad(balance.balance_loss(hidden @ router, counts), router)[0])
    assert torch.equal(got_x, torch.autograd.grad(dense.fp8_linear(leaf, w, ws).sum(), leaf)[0])


def test_an_output_in_an_operands_memory_is_refused():
    """Other blocks still read what the first ones would overwrite.  Neighbours in one buffer are fine."""
    w, ws = make_weight(64, 256, 1)
    codes, scale = dense.quantize_rows(torch.randn(4, 256, device="cuda"))
    wide, wide_scale = make_weight(256, 128, 2)
    tall = dense.quantize_rows(torch.randn(64, 128, device="cuda"))
    square_scale = torch.ones(4, 2, device="cuda")
    few, few_scale = make_weight(2, 256, 3)
    for call in (lambda: dense.block_scaled_matmul(codes, scale, w, ws, out=codes.view(torch.float32)),
                 lambda: dense.block_scaled_matmul(codes, square_scale, few, few_scale, out=square_scale),
                 lambda: dense.block_scaled_matmul(*tall, wide, wide_scale, out=wide.view(torch.bfloat16).view(64, 256))):
        with pytest.raises(ValueError, match="memory"):
            call()
    buffer = torch.zeros(2048, dtype=torch.uint8, device="cuda")
    near, out = buffer[:1024].view(torch.float8_e4m3fn).view(4, 256), buffer[1024:].view(torch.float32).view(4, 64)
    near.view(torch.uint8).copy_(codes.view(torch.uint8))
    assert torch.equal(dense.block_scaled_matmul(near, scale, w, ws, out=out), dense.block_scaled_matmul(codes, scale, w, ws, out_dtype=torch.float32))


def test_results_may_be_modified_in_place():
    """As any linear layer's: a bias or an activation on the spot, whatever the leading sizes, with gradients."""
    from netra_kernel_b200 import torch_ops  # noqa: F401
    w, ws = make_weight(48, 128, 1)
    bias, dy = torch.randn(48, device="cuda"), torch.randn(12, 48, device="cuda")
    flat = torch.randn(12, 128, device="cuda")
    for linear in (dense.fp8_linear, torch.ops.netra.fp8_linear):
        plain = flat.clone().requires_grad_()
        want = torch.relu(linear(plain, w, ws) + bias)
        (want_dx,) = torch.autograd.grad(want, plain, dy)
        for shape in ((12,), (2, 6), (3, 1, 4)):
            x = flat.view(*shape, 128).clone().requires_grad_()
            y = linear(x, w, ws)
            y += bias
            y.relu_()
            assert y.shape == (*shape, 48) and torch.equal(y.view(12, 48), want)
            (dx,) = torch.autograd.grad(y, x, dy.view(*shape, 48))
            assert torch.equal(dx.view(12, 128), want_dx)
    x = flat[0].clone().requires_grad_()
    y = dense.fp8_linear(x, w, ws)
    y += bias
    y.sum().backward()
    loss = balance.balance_loss(flat.clone().requires_grad_(), torch.ones(128, dtype=torch.int32, device="cuda"))
    loss *= 0.5
    loss.backward()


@pytest.mark.parametrize("m,n,dtype", [(19000, 40, torch.bfloat16), (20001, 64, torch.float32), (19500, 129, torch.float16)])
def test_tall_narrow_products_against_64_bits(m, n, dtype):
    """More row tiles than the device holds at once, and hardly a tile's width of columns."""
    k = 272
    g = torch.Generator().manual_seed(m + n)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    w, ws = make_weight(n, k, n)
    check_product(dense.fp8_linear(x.cuda(), w, ws), *quantize_definition(x), w, ws)
    w, ws = make_weight(k, n, n)
    codes, scale = dense.quantize_rows(x.cuda())
    check_product(dense.block_scaled_matmul(codes, scale, w, ws, transpose_weight=True, out_dtype=dtype), *quantize_definition(x), w, ws, True)
    dense.check_status()
