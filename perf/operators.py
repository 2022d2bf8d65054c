"""Cases and plain forms of the operators around the routed-MoE layer: the block-scaled FP8 linear map (with the row
quantiser that feeds it and the gradient to its input) and the router's balance loss with its per-expert counts.

Plain forms are elementary torch operations in 32 bits.  With ``own`` true, ``run`` calls the framework instead."""
import torch

own = False
BLOCK = 128
FLOOR = 1e-10          # smallest block amax the quantiser divides by
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the token rows of a prefill call on their way into an FP8 product (hidden width 2048)
        {"name": "quantize_8192x2048", "op": "quantize", "m": 8192, "k": 2048, "dtype": "bf16"},
        # an odd row count, a width that ends inside a block, FP32 activations
        {"name": "quantize_ragged", "op": "quantize", "m": 1021, "k": 4112, "dtype": "f32"},
        # one decode token through the dense projection of the compiler's contract (M x 2048 x 4096)
        {"name": "linear_m1", "op": "linear", "m": 1, "n": 2048, "k": 4096, "dtype": "bf16"},
        # the 12 draft tokens of one sequence being verified
        {"name": "linear_m12", "op": "linear", "m": 12, "n": 4096, "k": 2048, "dtype": "bf16"},
        # a decode batch of 256 tokens
        {"name": "linear_m256", "op": "linear", "m": 256, "n": 4096, "k": 2048, "dtype": "bf16"},
        # sizes that end inside every tile, FP16 in and out
        {"name": "linear_ragged", "op": "linear", "m": 777, "n": 1043, "k": 2064, "dtype": "f16"},
        # the tokens of one step of the 40-layer stack through one projection
        {"name": "linear_m16384", "op": "linear", "m": 16384, "n": 4096, "k": 2048, "dtype": "bf16"},
        # a short fine-tuning batch through a frozen FP8 projection: output and the gradient to its input
        {"name": "linear_train_m300", "op": "linear_train", "m": 300, "n": 2048, "k": 1040, "dtype": "f32"},
        # a full fine-tuning batch
        {"name": "linear_train_m8192", "op": "linear_train", "m": 8192, "n": 4096, "k": 2048, "dtype": "bf16"},
        # load and balance loss of one decode batch of the layer's router
        {"name": "balance_t256", "op": "balance", "t": 256, "e": 256, "topk": 8, "dtype": "bf16", "zipf": 0.0, "keep": 1.0},
        # skewed routing over a padded batch
        {"name": "balance_t16384", "op": "balance", "t": 16384, "e": 256, "topk": 8, "dtype": "bf16", "zipf": 0.27, "keep": 0.9},
        # a router of another size, FP32 logits
        {"name": "balance_ragged", "op": "balance", "t": 5001, "e": 60, "topk": 4, "dtype": "f32", "zipf": 0.5, "keep": 0.7},
    ]


def _log(rng, lo, hi, step=1):
    """A whole number from lo to hi, a multiple of step, spread over its logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "linear_train", "linear_train", "balance", "balance"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantize":
        return {"op": op, "m": _log(rng, 1, 16384), "k": _log(rng, 128, 4096, 16), "dtype": dtype}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 128, 4096), "k": _log(rng, 128, 4096, 16), "dtype": dtype}
    if op == "linear_train":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 128, 4096, 16), "k": _log(rng, 128, 4096, 16), "dtype": dtype}
    e = rng.choice([8, 16, 60, 64, 128, 160, 256, 384, 512])
    return {"op": op, "t": _log(rng, 1, 16384), "e": e, "topk": rng.choice([1, 2, 4, 6, 8]), "dtype": rng.choice(["bf16", "f32"]),
            "zipf": rng.choice([0.0, 0.3, 1.0]), "keep": rng.choice([1.0, 0.8, 0.3])}


# ------------------------------------------------------------------------------------------------------------ inputs
def _weights(n, k, g):
    """A frozen projection as a checkpoint holds it: E4M3 codes [n, k] and one scale per 128 x 128 block."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    w[:n, :k] = torch.randn(n, k, generator=g, device="cuda") * 0.02
    b = w.view(nb, BLOCK, kb, BLOCK)
    scale = b.abs().amax(dim=(1, 3)).clamp_min(FLOOR) / 448.0
    q = (b / scale[:, None, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)
    return q[:n, :k].contiguous(), scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "balance":
        t, e, k = case["t"], case["e"], case["topk"]
        logits = torch.randn(t, e, generator=g, device="cuda") * 0.9
        rank = torch.arange(1, e + 1, device="cuda", dtype=torch.float32)
        logits -= case["zipf"] * 1.1 * rank.log()
        logits = logits.to(dt)
        ids = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
        mask = None
        if case["keep"] < 1.0:
            mask = torch.rand(t, generator=g, device="cuda") < case["keep"]
        return {"case": case, "logits": logits.requires_grad_(), "ids": ids, "mask": mask}
    m, k = case["m"], case["k"]
    # normalised hidden states: a few channels much larger than the rest, token rows of unequal size
    channel = torch.exp(torch.randn(k, generator=g, device="cuda") * 0.5)
    row = torch.exp(torch.randn(m, 1, generator=g, device="cuda") * 0.3)
    x = (torch.randn(m, k, generator=g, device="cuda") * channel * row).to(dt)
    if case["op"] == "quantize":
        return {"case": case, "x": x}
    w, w_scale = _weights(case["n"], k, g)
    state = {"case": case, "x": x, "w": w, "w_scale": w_scale}
    if case["op"] == "linear_train":
        # gradients as a loss averaged over the batch sends them back
        state["dy"] = (torch.randn(m, case["n"], generator=g, device="cuda") * (row * 0.02)).to(dt)
        state["x"] = x.requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _pad_blocks(x):
    m, k = x.shape
    kb = -(-k // BLOCK)
    return torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)


def _quantize_plain(x):
    """codes = rne(x * (1 / scale)), scale = max(amax of the row's block of 128, 1e-10) * (1 / 448), all in FP32."""
    m, k = x.shape
    b = _pad_blocks(x.float())
    scale = b.abs().amax(dim=2).clamp_min(FLOOR) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=x.device)
    q = (b * (1.0 / scale)[:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(m, -1)[:, :k], scale


def _dequantize_plain(codes, scale):
    m, k = codes.shape
    return (_pad_blocks(codes.float()) * scale[:, :, None]).view(m, -1)[:, :k]


def _weight_plain(w, w_scale):
    n, k = w.shape
    full = w_scale.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    return w.float() * full[:n, :k]


def _linear_plain(x, w, w_scale):
    return (_dequantize_plain(*_quantize_plain(x)) @ _weight_plain(w, w_scale).T).to(x.dtype)


def _input_grad_plain(dy, w, w_scale):
    return (_dequantize_plain(*_quantize_plain(dy)) @ _weight_plain(w, w_scale)).to(dy.dtype)


def _balance_plain(logits, ids, mask):
    """loss = E * sum_e f_e P_e; f_e = share of the counted choices that went to e, P_e = mean probability of e over the
    counted tokens; the counts carry no gradient."""
    z = logits.detach().float()
    t, e = z.shape
    live = torch.ones(t, dtype=torch.float32, device=z.device) if mask is None else mask.float()
    hits = (ids[:, :, None] == torch.arange(e, device=z.device, dtype=ids.dtype)).sum(dim=1)
    counts = (hits * live.to(hits.dtype)[:, None]).sum(dim=0)
    tokens = live.sum().clamp_min(1.0)
    share = counts.float() / counts.sum().clamp_min(1).float()
    p = torch.exp(z - z.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    dot = p @ share
    loss = (dot * live).sum() * e / tokens
    grad = p * (share[None, :] - dot[:, None]) * (live[:, None] * (e / tokens))
    return loss, counts.to(torch.int32), grad.to(logits.dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        from netra_kernel_b200 import balance, dense
        if op == "quantize":
            return dense.quantize_rows(state["x"])
        if op == "linear":
            return dense.fp8_linear(state["x"], state["w"], state["w_scale"])
        if op == "linear_train":
            y = dense.fp8_linear(state["x"], state["w"], state["w_scale"])
            (dx,) = torch.autograd.grad(y, state["x"], state["dy"])
            return y.detach(), dx
        counts = balance.expert_counts(state["ids"], state["case"]["e"], state["mask"])
        loss = balance.balance_loss(state["logits"], counts, state["mask"])
        (grad,) = torch.autograd.grad(loss, state["logits"])
        return loss.detach(), counts, grad
    with torch.no_grad():
        if op == "quantize":
            return _quantize_plain(state["x"])
        if op == "linear":
            return _linear_plain(state["x"], state["w"], state["w_scale"])
        if op == "linear_train":
            return _linear_plain(state["x"], state["w"], state["w_scale"]), _input_grad_plain(state["dy"], state["w"], state["w_scale"])
        return _balance_plain(state["logits"], state["ids"], state["mask"])


# -------------------------------------------------------------------------------------------------------- work, exact
def work(case):
    if case["op"] == "balance":
        t, e, k, b = case["t"], case["e"], case["topk"], BYTES[case["dtype"]]
        mask = t if case["keep"] < 1.0 else 0
        return {"bytes": t * e * b * 2 + t * k * 4 + mask + e * 4 + 4, "flops": 12 * t * e}
    m, k, b = case["m"], case["k"], BYTES[case["dtype"]]
    if case["op"] == "quantize":
        return {"bytes": m * k * (b + 1) + m * -(-k // BLOCK) * 4, "flops": 3 * m * k}
    n = case["n"]
    weight = n * k + -(-n // BLOCK) * -(-k // BLOCK) * 4
    if case["op"] == "linear":
        return {"bytes": weight + (m * k + m * n) * b, "flops": 2 * m * n * k}
    return {"bytes": weight + 2 * (m * k + m * n) * b, "flops": 4 * m * n * k}


def _round_e4m3(v):
    """Nearest E4M3 value in 64 bits, ties to the even code, saturating at 448."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _to32(v):
    """The nearest FP32 number, as 64 bits."""
    return v.float().double()


def _quantize_exact(x):
    """The quantiser's definition names three FP32 numbers - the scale, its reciprocal and the scaled value - each the nearest
    to its 64-bit result here.  (Small ratios of BF16 numbers often fall on the border of two codes: with a scale kept in
    64 bits the border, and so the code, would be another operator's.)"""
    m, k = x.shape
    values, scales = torch.empty(m, k, dtype=torch.float64, device=x.device), []
    floor, step = (_to32(torch.tensor(v, dtype=torch.float64, device=x.device)) for v in (FLOOR, 1.0 / 448.0))
    for c in range(0, k, BLOCK):
        part = x[:, c:c + BLOCK].double()
        s = _to32(torch.maximum(part.abs().max(dim=1).values, floor) * step)
        values[:, c:c + BLOCK] = _round_e4m3(_to32(part * _to32(1.0 / s)[:, None]))
        scales.append(s)
    return values, torch.stack(scales, dim=1)


def _product_exact(x, w, w_scale, transposed):
    values, scales = _quantize_exact(x)
    w = w.double() if transposed else w.double().T        # [reduction, outputs]
    s = w_scale.double() if transposed else w_scale.double().T
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    spread = torch.arange(w.shape[1], device=x.device) // BLOCK
    for b in range(scales.shape[1]):
        cut = slice(b * BLOCK, (b + 1) * BLOCK)
        out += (values[:, cut] @ w[cut]) * scales[:, b:b + 1] * s[b][spread][None, :]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _quantize_exact(state["x"])
    if case["op"] == "linear":
        return _product_exact(state["x"], state["w"], state["w_scale"], False)
    if case["op"] == "linear_train":
        x = state["x"].detach()
        return _product_exact(x, state["w"], state["w_scale"], False), _product_exact(state["dy"], state["w"], state["w_scale"], True)
    z, ids, mask = state["logits"].detach().double(), state["ids"].long(), state["mask"]
    t, e = z.shape
    kept = torch.arange(t, device=z.device) if mask is None else mask.nonzero()[:, 0]
    counts = torch.bincount(ids[kept].reshape(-1), minlength=e)
    share = counts.double() / max(1, int(counts.sum()))
    logp = z[kept] - torch.logsumexp(z[kept], dim=1, keepdim=True)
    p = logp.exp()
    n = max(1, kept.numel())
    loss = e * (share * p.sum(dim=0) / n).sum()
    grad = torch.zeros(t, e, dtype=torch.float64, device=z.device)
    grad[kept] = e / n * p * (share[None, :] - (p * share).sum(dim=1, keepdim=True))
    return loss, counts, grad
