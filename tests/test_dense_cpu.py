"""The dense FP8 and balance-loss entry points refuse bad operands before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from netra_kernel_b200 import abi, balance, dense


def _fp8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        dense.quantize_rows(torch.zeros(2, 128))
    with pytest.raises(ValueError, match="CUDA"):
        dense.fp8_linear(torch.zeros(2, 128), _fp8(16, 128), torch.ones(1, 1))
    with pytest.raises(ValueError, match="CUDA"):
        dense.block_scaled_matmul(_fp8(2, 128), torch.ones(2, 1), _fp8(16, 128), torch.ones(1, 1))
    with pytest.raises(ValueError, match="CUDA"):
        balance.expert_counts(torch.zeros(2, 8, dtype=torch.int32), 256)
    with pytest.raises(ValueError, match="CUDA"):
        balance.balance_loss(torch.zeros(2, 8), torch.zeros(8, dtype=torch.int32))


def test_weight_checks():
    cpu = torch.device("cpu")
    ok, scale = _fp8(300, 272), torch.ones(3, 3)
    abi.torch_binding().check_weight(ok, scale, cpu)
    abi.torch_binding().check_weight(_fp8(300, 288)[:, :260], scale, cpu)                    # padded rows
    abi.torch_binding().check_weight(_fp8(1, 260), torch.ones(1, 3), cpu)                    # a single row has no pitch
    for weight, s, why in [
        (ok.view(torch.uint8), scale, "float8"), (_fp8(0, 128), torch.ones(0, 1), "float8"),
        (_fp8(300, 260), scale, "16-byte"), (ok.t(), torch.ones(3, 3), "16-byte"), (_fp8(301, 272).view(-1)[16 * 17 - 8:-8].view(300, 272), scale, "16-byte"),
        (ok, torch.ones(3, 2), "weight_scale"), (ok, scale.double(), "weight_scale"), (ok, torch.arange(9.0).view(3, 3).t(), "row-major"),
        (ok, torch.ones(3, 3, requires_grad=True), "frozen")]:
        with pytest.raises(ValueError, match=why):
            abi.torch_binding().check_weight(weight, s, cpu)


def test_c_entries_refuse_before_any_launch():
    lib = abi.load()
    p, odd = 4096, 4097                      # never dereferenced: every call below is refused on the host
    err = lambda: lib.netra_moe_last_error().decode()                      # noqa: E731
    quant = lambda codes=p, cp=128, s=p, x=p, dt=0, xp=128, m=2, k=128: lib.netra_dense_quantize_rows_launch(   # noqa: E731
        codes, cp, s, 1, 2, x, dt, xp, m, k, None)
    for kw, why in [(dict(codes=None), "null"), (dict(s=None), "null"), (dict(x=None), "null"), (dict(dt=3), "type"), (dict(m=0), "2^26"),
                    (dict(k=0), "2^26"), (dict(m=(1 << 26) + 1), "2^26"), (dict(xp=127), "pitch"), (dict(cp=100), "pitch"), (dict(x=odd), "aligned")]:
        assert quant(**kw) == -1 and why in err(), kw
    mm = lambda out=p, dt=0, op=64, a=p, ap=128, s=p, w=p, wp=128, ws=p, wsp=1, tr=0, m=2, r=64, c=128: lib.netra_dense_fp8_matmul_launch(   # noqa: E731
        out, dt, op, a, ap, s, 1, 2, w, wp, ws, wsp, tr, m, r, c, None)
    for kw, why in [(dict(out=None), "null"), (dict(a=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(s=None), "null"),
                    (dict(dt=7), "type"), (dict(tr=2), "transpose"), (dict(m=0), "2^26"), (dict(r=0), "2^26"), (dict(c=0), "2^26"),
                    (dict(a=p + 8), "16-byte"), (dict(w=p + 1), "16-byte"), (dict(ap=136), "16-byte"), (dict(wp=130), "16-byte"),
                    (dict(ap=112), "pitch"), (dict(wp=112), "pitch"), (dict(op=63), "pitch"), (dict(wsp=0), "pitch"), (dict(out=odd), "aligned")]:
        assert mm(**kw) == -1 and why in err(), kw
    size = lib.netra_dense_fp8_linear_workspace_bytes(3, 130)
    assert size >= 3 * 144 + 3 * 2 * 4
    lin = lambda ws=p, size=size: lib.netra_dense_fp8_linear_launch(p, 64, p, 0, 130, p, 144, p, 2, 0, 3, 64, 130, ws, size, None)      # noqa: E731
    for kw in (dict(ws=None), dict(ws=p + 8), dict(size=size - 1)):
        assert lin(**kw) == -1 and "workspace" in err(), kw
    needs = lambda x=p, dt=0, xp=128, tr=0, m=16, k=128: lib.netra_dense_fp8_linear_needs_workspace(x, dt, xp, tr, m, k)               # noqa: E731
    assert needs() == 0 and needs(m=1, dt=2) == 0
    for kw in (dict(m=17), dict(tr=1), dict(k=130), dict(x=p + 2), dict(xp=130), dict(dt=2)):
        assert needs(**kw) == 1, kw
    assert lib.netra_dense_status(None) == -1
    cnt = lambda c=p, ids=p, b=4, pitch=8, t=2, s=8, e=256: lib.netra_expert_counts_launch(c, ids, b, pitch, None, t, s, e, None)       # noqa: E731
    for kw, why in [(dict(c=None), "null"), (dict(ids=None), "null"), (dict(b=2), "bytes"), (dict(pitch=7), "pitch"), (dict(e=0), "1024"),
                    (dict(e=1025), "1024"), (dict(t=1 << 30), "2^31"), (dict(ids=4098), "aligned")]:
        assert cnt(**kw) == -1 and why in err(), kw
    assert lib.netra_balance_loss_workspace_bytes(2, 16) == 0            # small calls need none
    size = lib.netra_balance_loss_workspace_bytes(5000, 16)
    loss = lambda l=p, sc=p, z=p, dt=0, pitch=16, c=p, w=p, n=size, t=5000, e=16: lib.netra_balance_loss_launch(l, sc, z, dt, pitch, c, None, w, n, t, e, None)   # noqa: E731
    for kw, why in [(dict(l=None), "null"), (dict(sc=None), "null"), (dict(z=None), "null"), (dict(c=None), "null"), (dict(dt=3), "type"),
                    (dict(pitch=15), "pitch"), (dict(w=None), "workspace"), (dict(n=size - 1), "workspace"), (dict(w=p + 8), "workspace"),
                    (dict(t=0), "tokens"), (dict(e=0), "1024"), (dict(e=2000), "1024"), (dict(z=odd), "aligned")]:
        assert loss(**kw) == -1 and why in err(), kw
    grad = lambda g=p, gp=16, s=p, u=p: lib.netra_balance_loss_grad_launch(g, gp, p, 0, 16, p, None, s, u, 2, 16, None)                  # noqa: E731
    for kw, why in [(dict(g=None), "null"), (dict(s=None), "null"), (dict(u=None), "null"), (dict(gp=8), "pitch"), (dict(g=odd), "aligned")]:
        assert grad(**kw) == -1 and why in err(), kw
    assert isinstance(ctypes.c_uint64(size).value, int)


def test_operators_by_name_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from netra_kernel_b200 import torch_ops  # noqa: F401  (registers the operators)
    with FakeTensorMode():
        x = torch.empty(2, 5, 256, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(300, 256, dtype=torch.float8_e4m3fn, device="cuda")
        s = torch.empty(3, 2, device="cuda")
        y = torch.ops.netra.fp8_linear(x, w, s)
        assert y.shape == (2, 5, 300) and y.dtype == torch.bfloat16
        dx = torch.ops.netra.fp8_linear_input_grad(y, w, s)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        counts = torch.ops.netra.expert_counts(torch.empty(7, 8, dtype=torch.int32, device="cuda"), 60)
        assert counts.shape == (60,) and counts.dtype == torch.int32
        z = torch.empty(7, 60, device="cuda")
        loss = torch.ops.netra.balance_loss(z, counts)
        dz = torch.ops.netra.balance_loss_grad(loss, z, counts)
        assert loss.shape == () and loss.dtype == torch.float32 and dz.shape == z.shape


def test_c_entries_refuse_addresses_off_their_element():
    """Every address that a kernel reads or writes by whole elements; refused on the host, nothing is launched."""
    lib = abi.load()
    p = 4096                                 # never dereferenced
    size = lib.netra_balance_loss_workspace_bytes(5000, 16)
    quant = lambda s=p: lib.netra_dense_quantize_rows_launch(p, 128, s, 1, 2, p, 0, 128, 2, 128, None)                                   # noqa: E731
    matmul = lambda s=p, ws=p, out=p: lib.netra_dense_fp8_matmul_launch(out, 2, 64, p, 128, s, 1, 2, p, 128, ws, 1, 0, 2, 64, 128, None)   # noqa: E731
    cnt = lambda c=p, ids=p, b=8: lib.netra_expert_counts_launch(c, ids, b, 8, None, 2, 8, 256, None)                                    # noqa: E731
    loss = lambda l=p, sc=p, z=p, c=p, t=5000: lib.netra_balance_loss_launch(l, sc, z, 2, 16, c, None, p, size, t, 16, None)             # noqa: E731
    grad = lambda g=p, z=p, c=p, s=p, u=p: lib.netra_balance_loss_grad_launch(g, 16, z, 2, 16, c, None, s, u, 2, 16, None)               # noqa: E731
    for call, names in [(quant, ["s"]), (matmul, ["s", "ws", "out"]), (cnt, ["c", "ids"]), (loss, ["l", "sc", "z", "c"]), (grad, ["g", "z", "c", "s", "u"])]:
        for name in names:
            for off in (1, 2, 3):
                assert call(**{name: p + off}) == -1 and "aligned" in lib.netra_moe_last_error().decode(), (call, name, off)
    for off in (2, 6):
        assert loss(t=2, c=p + off) == -1 and "aligned" in lib.netra_moe_last_error().decode()      # the form without a workspace
