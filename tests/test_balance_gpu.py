"""Expert counts and balance loss against their formulas in 64 bits.

Counts are exact.  A probability carries a relative error of at most u = (E/32 + 16 + spread of the row's logits) * 2^-23:
the subtraction and the exponential (2 steps plus the rounded argument), E/32 additions per lane and five across lanes, the
division.  The loss is a mean of d_t = sum f p (FP64 across tokens), so it is held to 2u * loss + one FP32 step; a gradient
to 3u * (E/n) p (f + d) plus half a step of its type."""
import pytest
import torch

from netra_kernel_b200 import balance, synth
from netra_kernel_b200.moe import RoutedMoELayer

pytestmark = pytest.mark.gpu


def definition(z, counts, mask):
    z = z.detach().cpu().double()
    t, e = z.shape
    kept = torch.ones(t, dtype=torch.bool) if mask is None else mask.cpu()
    c = counts.cpu().double()
    f = c / c.sum() if c.sum() > 0 else torch.zeros(e, dtype=torch.float64)
    p = torch.softmax(z, dim=1)
    p = torch.where(torch.isinf(z).all(dim=1, keepdim=True) & (z < 0).all(dim=1, keepdim=True), torch.zeros_like(p), p)
    n = max(1, int(kept.sum()))
    d = p @ f
    loss = e / n * d[kept].sum()
    grad = torch.where(kept[:, None], e / n * p * (f - d[:, None]), torch.zeros_like(p))
    size = e / n * p * (f + d[:, None])
    finite = torch.where(torch.isinf(z), torch.zeros_like(z), z)
    spread = (finite.amax(dim=1) - finite.amin(dim=1)).clamp_max(110.0)      # exp(-110) is 0 in FP32
    u = ((e / 32 + 16) + spread) * 2.0 ** -23
    return loss, grad, size, u


def check(z, counts, mask, upstream=1.0):
    loss, grad, size, u = definition(z, counts, mask)
    leaf = z.detach().clone().requires_grad_()
    got = balance.balance_loss(leaf, counts, mask)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(got.item() - loss.item()) <= (2 * float(u.max()) + 2.0 ** -24) * abs(loss.item()) + 1e-37, (got.item(), loss.item())
    assert torch.equal(balance.balance_loss(z, counts, mask), got.detach())
    (dz,) = torch.autograd.grad(got * upstream, leaf)
    assert dz.dtype == z.dtype
    eps = torch.finfo(z.dtype)
    tol = 3 * u[:, None] * size * abs(upstream) + eps.eps / 2 * grad.abs() * abs(upstream) + max(eps.tiny * eps.eps, 1e-37)
    err = (dz.cpu().double() - grad * upstream).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    return got, dz


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (3, 256, 8), (7, 60, 4), (33, 33, 1), (64, 64, 6), (65, 65, 2), (256, 256, 8),
                                   (500, 257, 8), (1000, 512, 10), (2049, 160, 6), (300, 1024, 16), (5000, 16, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_counts_loss_and_gradient(t, e, k, dtype):
    g = torch.Generator().manual_seed(t + e)
    z = (torch.randn(t, e, generator=g) * 2 - torch.arange(e) * 0.01).to(dtype).cuda()
    ids = z.float().topk(min(k, e), dim=1).indices
    for mask in (None, (torch.rand(t, generator=g) < 0.6).cuda()):
        kept = slice(None) if mask is None else mask.cpu()
        want = torch.bincount(ids.cpu()[kept].reshape(-1), minlength=e)
        counts = balance.expert_counts(ids, e, mask)
        assert counts.dtype == torch.int32 and torch.equal(counts.cpu().long(), want)
        assert torch.equal(balance.expert_counts(ids.int(), e, mask), counts)
        check(z, counts, mask, upstream=0.25)


def test_counts_strides_foreign_ids_and_empty_calls():
    g = torch.Generator().manual_seed(1)
    wide = torch.randint(0, 64, (1000, 12), generator=g, dtype=torch.int32).cuda()
    for view in (wide[:, 2:9], wide[::3, :8], wide.t()[:12, :500], wide[4:5].expand(70, 12)):
        want = torch.bincount(view.cpu().reshape(-1).long(), minlength=64)
        assert torch.equal(balance.expert_counts(view, 64).cpu().long(), want)
    wild = wide[:, :8].clone()
    wild[::5, 1], wild[::7, 2], wild[3, 3], wild[4, 4] = -1, 64, 2 ** 31 - 1, -2 ** 31
    ok = wild.cpu()[(wild.cpu() >= 0) & (wild.cpu() < 64)].long()
    assert torch.equal(balance.expert_counts(wild, 64).cpu().long(), torch.bincount(ok, minlength=64))
    far = wild.long()
    far[9, 0] = 2 ** 40 + 3
    ok = far.cpu()[(far.cpu() >= 0) & (far.cpu() < 64)]
    assert torch.equal(balance.expert_counts(far, 64).cpu().long(), torch.bincount(ok, minlength=64))
    assert bool((balance.expert_counts(wide[:0], 64) == 0).all()) and bool((balance.expert_counts(wide[:, :0], 64) == 0).all())
    assert bool((balance.expert_counts(wide, 64, torch.zeros(1000, dtype=torch.bool, device="cuda")) == 0).all())
    same = torch.full((70000, 8), 5, dtype=torch.int32, device="cuda")                # every choice the same expert
    assert balance.expert_counts(same, 8).tolist() == [0, 0, 0, 0, 0, 560000, 0, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_experts_and_rows(dtype):
    g = torch.Generator().manual_seed(2)
    low = torch.finfo(dtype).min
    z = torch.randn(40, 96, generator=g).to(dtype)
    z[:, 10:20] = float("-inf")
    z[1], z[2] = float("-inf"), low                                   # nothing left; every logit the lowest value
    z[3, :] = low
    z[3, 7] = 1.0
    z[4] = torch.finfo(dtype).max
    counts = torch.randint(0, 50, (96,), generator=g, dtype=torch.int32).cuda()
    z = z.cuda()
    _, dz = check(z, counts, None)
    assert bool((dz[1] == 0).all()) and bool((dz[:, 10:20][5:] == 0).all())
    mask = torch.ones(40, dtype=torch.bool, device="cuda")
    mask[6:9] = False
    dirty = z.clone()
    dirty[6], dirty[7], dirty[8] = float("nan"), float("inf"), float("-inf")
    clean = z.clone()
    clean[6:9] = 0
    a, da = check(clean, counts, mask)
    leaf = dirty.requires_grad_()
    b = balance.balance_loss(leaf, counts, mask)
    (db,) = torch.autograd.grad(b, leaf)
    assert torch.equal(a.detach(), b.detach()) and torch.equal(da, db)                # uncounted rows are not read
    assert balance.balance_loss(dirty.detach(), counts).isnan()
    none = torch.zeros(40, dtype=torch.bool, device="cuda")
    loss, dz = check(z, counts, none)
    assert loss.item() == 0.0 and bool((dz == 0).all())
    loss, dz = check(z, torch.zeros(96, dtype=torch.int32, device="cuda"), None)
    assert loss.item() == 0.0 and bool((dz == 0).all())


def test_even_and_nearly_even_loads():
    """An even load has no gradient at all; one choice more or less gives a gradient as exact as the small difference it comes
    from (counts up to 2^24 are whole numbers in FP32)."""
    g = torch.Generator().manual_seed(6)
    z = torch.randn(50, 64, generator=g).cuda().requires_grad_()
    even = torch.full((64,), 123457, dtype=torch.int32, device="cuda")
    loss = balance.balance_loss(z, even)
    (grad,) = torch.autograd.grad(loss, z)
    assert abs(loss.item() - 1.0) <= 40 * 2.0 ** -23 and bool((grad == 0).all())
    even[3] += 1
    even[9] -= 2
    loss, grad, _, u = definition(z, even, None)
    (got,) = torch.autograd.grad(balance.balance_loss(z, even), z)
    c = even.cpu().double() - even.min().item()
    p = torch.softmax(z.detach().cpu().double(), dim=1)
    size = 64 / 50 * p * (c + (p @ c)[:, None]) / even.sum().item()
    assert bool(((got.cpu().double() - grad).abs() <= 3 * u[:, None] * size + 1e-37).all())


def test_layouts_and_empty_batches():
    g = torch.Generator().manual_seed(3)
    base = torch.randn(64, 300, generator=g).cuda()
    counts = torch.randint(0, 9, (60,), generator=g, dtype=torch.int32).cuda()
    for view in (lambda t: t[::2, 11:71], lambda t: t.t()[:60, :60], lambda t: t[3:4, :60].expand(9, 60)):
        leaf = base.clone().requires_grad_()
        loss = balance.balance_loss(view(leaf), counts)
        (grad,) = torch.autograd.grad(loss, leaf)
        plain = view(base).contiguous().requires_grad_()
        again = balance.balance_loss(plain, counts)
        assert torch.equal(loss.detach(), again.detach())
        (want,) = torch.autograd.grad(again, plain)
        full = torch.zeros_like(base).requires_grad_()
        (placed,) = torch.autograd.grad(view(full), full, want)
        assert torch.equal(grad, placed)
    empty = base[:0, :60].clone().requires_grad_()
    loss = balance.balance_loss(empty, counts)
    (grad,) = torch.autograd.grad(loss, empty)
    assert loss.item() == 0.0 and grad.shape == (0, 60)


def test_gradient_against_differences():
    """Central differences of the loss along a direction, step h = 2^-5 in logits of size 1: the third derivative of the loss is
    at most E (the loss of one expert's probability), so the curvature costs at most E h^2 / 6 per unit; FP32 rounding of two
    losses costs (2u + 2^-24) * loss / h."""
    g = torch.Generator().manual_seed(4)
    z = torch.randn(30, 24, generator=g).cuda()
    counts = torch.randint(0, 20, (24,), generator=g, dtype=torch.int32).cuda()
    d = torch.randn(30, 24, generator=g).cuda()
    d = d / d.abs().max()
    h = 2.0 ** -5
    leaf = z.clone().requires_grad_()
    loss = balance.balance_loss(leaf, counts)
    (grad,) = torch.autograd.grad(loss, leaf)
    up, down = balance.balance_loss(z + h * d, counts).item(), balance.balance_loss(z - h * d, counts).item()
    u = (24 / 32 + 16 + 12) * 2.0 ** -23
    slope = float((grad.double() * d.double()).sum())
    assert abs((up - down) / (2 * h) - slope) <= 24 * h * h / 6 + (2 * u + 2.0 ** -24) * loss.item() / h


def test_repeats_streams_and_captured_graphs():
    g = torch.Generator().manual_seed(5)
    z = torch.randn(3000, 256, generator=g).to(torch.bfloat16).cuda()
    ids = z.float().topk(8, dim=1).indices.int()
    mask = (torch.rand(3000, generator=g) < 0.9).cuda()

    def step(logits):
        counts = balance.expert_counts(ids, 256, mask)
        loss = balance.balance_loss(logits, counts, mask)
        return counts, loss.detach(), torch.autograd.grad(loss, logits)[0]

    want = step(z.clone().requires_grad_())
    streams = [torch.cuda.Stream() for _ in range(3)]
    leaves = [z.clone().requires_grad_() for _ in streams]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, leaf in zip(streams, leaves):
            with torch.cuda.stream(s):
                got.append(step(leaf))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))
    graph, leaf = torch.cuda.CUDAGraph(), z.clone().requires_grad_()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_counts_of_the_layers_own_routing():
    dev = torch.device("cuda", 0)
    hidden, router_w, bias = synth.make_activations(333, 1.2, seed=3)
    zeros = torch.zeros
    layer = RoutedMoELayer(router_w.to(dev), zeros(257, 1024, 2048, dtype=torch.uint8, device=dev), torch.ones(257, 8, 16, device=dev),
                           zeros(257, 2048, 512, dtype=torch.uint8, device=dev), torch.ones(257, 16, 4, device=dev), 333, bias.to(dev), tiled=False)
    x = hidden.to(dev)
    out = torch.empty_like(x)
    for stage in range(5):
        layer.launch_stage(stage, x, out)
    inter = layer.intermediates(333)
    counts = balance.expert_counts(inter["topk_ids"], 256)             # nine slots: the shared expert's is not counted
    assert torch.equal(counts, inter["counts"])
    check(inter["logits"].clone(), counts, None)
    layer.close()


def test_operators_by_name_are_the_modules():
    from netra_kernel_b200 import dense, torch_ops  # noqa: F401
    g = torch.Generator().manual_seed(8)
    z = torch.randn(70, 64, generator=g).cuda().requires_grad_()
    ids = z.detach().topk(4, dim=1).indices
    for mask in (None, (torch.rand(70, generator=g) < 0.5).cuda()):
        counts = torch.ops.netra.expert_counts(ids, 64, mask)
        assert torch.equal(counts, balance.expert_counts(ids, 64, mask))
        loss = torch.ops.netra.balance_loss(z, counts, mask)
        (dz,) = torch.autograd.grad(loss * 3, z)
        want = balance.balance_loss(z, counts, mask)
        assert torch.equal(loss, want) and torch.equal(dz, torch.autograd.grad(want * 3, z)[0])
    w = (torch.randn(96, 64, generator=g) * 50).to(torch.float8_e4m3fn).cuda()
    ws = torch.full((1, 1), 0.01, device="cuda")
    x = z.detach().view(2, 35, 64).requires_grad_()
    dy = torch.randn(2, 35, 96, generator=g).cuda()
    y, want = torch.ops.netra.fp8_linear(x, w, ws), dense.fp8_linear(x, w, ws)
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(want, x, dy)[0])


def test_refusals():
    z = torch.zeros(4, 16, device="cuda")
    counts = torch.ones(16, dtype=torch.int32, device="cuda")
    mask = torch.ones(4, dtype=torch.bool, device="cuda")
    for call, why in [
        (lambda: balance.balance_loss(z.double(), counts), "BF16"), (lambda: balance.balance_loss(z[0], counts), "matrix"),
        (lambda: balance.balance_loss(z[:, :0], counts), "experts"), (lambda: balance.balance_loss(torch.zeros(2, 1025, device="cuda"), counts), "experts"),
        (lambda: balance.balance_loss(z, counts.long()), "counts"), (lambda: balance.balance_loss(z, counts[:15]), "counts"),
        (lambda: balance.balance_loss(z, counts.cpu()), "counts"), (lambda: balance.balance_loss(z, counts, mask[:3]), "token_mask"),
        (lambda: balance.balance_loss(z, counts, mask.float()), "token_mask"), (lambda: balance.balance_loss(z, counts, mask.cpu()), "token_mask"),
        (lambda: balance.balance_loss_grad(mask.float(), z, counts), "upstream"), (lambda: balance.balance_loss_grad(z[0, 0], z, counts.long()), "counts"),
        (lambda: balance.expert_counts(z, 16), "topk_ids"), (lambda: balance.expert_counts(z.int()[0], 16), "topk_ids"),
        (lambda: balance.expert_counts(z.int(), 0), "num_experts"), (lambda: balance.expert_counts(z.int(), 1025), "num_experts"),
        (lambda: balance.expert_counts(z.int(), 16, mask[:2]), "token_mask"),
    ]:
        with pytest.raises(ValueError, match=why):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_improbable_experts_keep_their_precision(dtype):
    """Logits whose differences are exact, one likely expert without a choice, the others up to e^-80 as likely.  In units of 2^-24 a
    gradient is off by at most: 5 for its exponential (two steps of FP32 and a rounding) and 5 for the row's (all but the likely one,
    whose exponential is 1), 9 additions in the row's sum and as many in that of the counts, 2 quotients, 3 for f - d and the loss's
    factor, 5 products; 38 together, and half a step of its type.  The rounding of the exponent alone (gap * log2 e, half a step of
    up to 2^-17) would cost up to 90."""
    t, e = 300, 64
    gap = torch.randint(8, 640, (t, e), generator=torch.Generator().manual_seed(9)).double() / 8
    if dtype == torch.bfloat16:
        gap = gap.floor()                                            # whole numbers below 128 are BF16 values
    gap[:, 0] = 0
    counts = torch.full((e,), 1000, dtype=torch.int32)
    counts[0] = 0
    z = (-gap).to(dtype).cuda().requires_grad_()
    assert torch.equal(z.detach().cpu().double(), -gap)
    (grad,) = torch.autograd.grad(balance.balance_loss(z, counts.cuda()), z)
    p, f = torch.softmax(-gap, dim=1), counts.double() / counts.sum()
    want = e / t * p * (f - (p @ f)[:, None])
    tol = (38 * 2.0 ** -24 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0)) * want.abs()
    err = (grad.cpu().double() - want).abs()[:, 1:]
    assert bool((err <= tol[:, 1:]).all()), float((err / want.abs()[:, 1:]).max() * 2 ** 24)
