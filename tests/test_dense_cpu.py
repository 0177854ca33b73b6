"""The dense head without a GPU: host-side refusals of the C entry points (nothing is
launched), the custom operators' output shapes, and the tests' own 64-bit forms
against autograd and planted mistakes."""

import ctypes
import math
import os
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import dense_ref
from conftest import ROOT
from sft_amd import _native
from src.model.modules.dense import ops  # noqa: F401

P = ctypes.c_void_p(0x1000)  # never dereferenced: every call below must fail validation before any launch
HEADER = os.path.join(ROOT, "include", "sft_ft.h")


def _call(name, args):
    rc = getattr(_native.lib(), name)(*args)
    return rc, _native.last_error()


def test_constants_match_header():
    text = open(HEADER).read()
    for name in ("TYPE_F32", "TYPE_F16", "TYPE_BF16", "ACT_NONE", "ACT_RELU", "ACT_CRELU", "ACT_SCRELU", "ACT_SILU",
                 "ACT_GELU", "LINEAR_COPY", "BALANCE_MAX_EXPERTS", "DISTILL_MAX_K"):
        m = re.search(rf"#define SFT_{name} (0x[0-9a-f]+|\d+)", text)
        assert int(m.group(1), 0) == getattr(_native, "SFT_" + name), name


# dtype, x, ldx, w, ldw, bias, residual, ldr, y, ldy, deriv, M, K, N, act, ws, ws_bytes, stream
FWD = [1, P, 8, P, 8, P, None, 0, P, 16, None, 100, 8, 16, 0, None, 0, None]


@pytest.mark.parametrize("at,value,needle", [
    (0, 3, "type"), (0, -1, "type"), (14, 6, "activation"), (11, -1, "M must"), (12, 0, "K and N"), (13, 0, "K and N"),
    (13, (1 << 21) + 1, "K and N"), (11, 1 << 30, "too large"), (1, None, "null"), (3, None, "null"), (8, None, "null"),
    (2, 7, "stride"), (4, 7, "stride"), (9, 15, "stride"), (2, 1 << 40, "stride"), (1, ctypes.c_void_p(0x1001), "aligned"),
    (5, ctypes.c_void_p(0x1001), "aligned")])
def test_linear_fwd_refuses(at, value, needle):
    args = list(FWD)
    args[at] = value
    if (at, value) == (11, 1 << 30):
        args[12] = args[2] = args[4] = 1 << 20
    rc, why = _call("sft_linear_fwd", args)
    assert rc == -1 and needle in why


def test_linear_workspaces():
    n = ctypes.c_size_t(0)
    size = _native.lib().sft_linear_fwd_workspace_size
    assert size(1, 64, 333, 10, 1, ctypes.byref(n)) == 0 and n.value == 0  # few rows need none
    assert size(1, 5000, 1040, 4096, 0, ctypes.byref(n)) == 0 and n.value == 0  # read in place, no split
    assert size(1, 5000, 1040, 4096, 1, ctypes.byref(n)) == 0
    assert n.value >= (5000 + 4096) * 1040 * 2  # copies of both operands
    assert size(1, 5000, 1037, 4096, 0, ctypes.byref(n)) == 0
    assert n.value >= (5000 + 4096) * 1040 * 2  # rows that are no multiple of 16 bytes
    assert size(1, 10, 8, 8, 2, ctypes.byref(n)) == -1 and "flags" in _native.last_error()
    assert size(1, 10, 8, 8, 0, None) == -1
    bwd = _native.lib().sft_linear_bwd_workspace_size
    assert bwd(1, 0, 8, 8, 5, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert bwd(1, 5000, 1040, 4096, 5, 0, ctypes.byref(n)) == 0 and n.value >= 5000 * 4096 * 2  # dz
    # a call whose workspace is missing, too small or misaligned
    args = list(FWD)
    args[2], args[4] = 9, 9  # rows that are not 16-byte aligned are copied
    for ws, nbytes in ((None, 0), (P, 64), (ctypes.c_void_p(0x1010), 1 << 30)):
        args[15], args[16] = ws, nbytes
        rc, why = _call("sft_linear_fwd", args)
        assert rc == _native.SFT_EWORKSPACE and "sft_linear_fwd" in why


# dtype, dy, lddy, deriv, x, ldx, w, ldw, dx, dw, db, M, K, N, act, ws, ws_bytes, stream
BWD = [1, P, 16, P, P, 8, P, 8, P, P, P, 100, 8, 16, 5, None, 0, None]


@pytest.mark.parametrize("at,value,needle", [
    (0, 7, "type"), (1, None, "null"), (3, None, "null"), (4, None, "null"), (6, None, "null"), (2, 15, "stride"),
    (5, 7, "stride"), (7, 7, "stride"), (14, 9, "activation"), (8, ctypes.c_void_p(0x1001), "aligned")])
def test_linear_bwd_refuses(at, value, needle):
    args = list(BWD)
    args[at] = value
    rc, why = _call("sft_linear_bwd", args)
    assert rc == -1 and needle in why


@pytest.mark.parametrize("act", [0, 5])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("M,K,N", [(128, 1040, 1040), (1000, 1040, 520), (70, 24, 16), (20000, 136, 264)])
def test_linear_bwd_workspace_covers_any_grads(M, K, N, dtype, act):
    """The size is asked for before it is known which grads a step needs."""
    n = ctypes.c_size_t(0)
    assert _native.lib().sft_linear_bwd_workspace_size(dtype, M, K, N, act, 0, ctypes.byref(n)) == 0
    for grads in range(1, 8):
        dx, dw, db = (P if grads & bit else None for bit in (1, 2, 4))
        args = [dtype, P, N, P, P, K, P, K, dx, dw, db, M, K, N, act, ctypes.c_void_p(0x1010), 1 << 50, None]
        if act == 0 and not db:
            continue  # may need none, and then the call would not be refused
        rc, why = _call("sft_linear_bwd", args)  # refused: the workspace is not aligned
        assert rc == _native.SFT_EWORKSPACE
        assert int(re.search(r"needs (\d+) bytes", why).group(1)) <= n.value, grads


# dtype, logits, ld, mask, rows, experts, top_k, loss, counts, kept, ws, ws_bytes, stream
BALANCE = [0, P, 8, None, 10, 8, 1, P, P, P, None, 0, None]


@pytest.mark.parametrize("at,value,needle", [
    (0, 3, "type"), (4, -1, "rows"), (5, 0, "experts"), (5, 1025, "experts"), (6, 0, "top_k"), (6, 9, "top_k"),
    (2, 7, "stride"), (1, None, "null"), (7, None, "null"), (8, None, "null"), (9, None, "null"),
    (8, ctypes.c_void_p(0x1004), "aligned")])
def test_balance_refuses(at, value, needle):
    args = list(BALANCE)
    args[at] = value
    rc, why = _call("sft_balance_fwd", args)
    assert rc == -1 and needle in why
    rc, why = _call("sft_balance_fwd", BALANCE)
    assert rc == _native.SFT_EWORKSPACE
    assert _call("sft_balance_bwd", [0, P, 8, None, 10, 8, 1, P, P, None, P, None])[0] == -1
    assert _call("sft_balance_bwd", [0, None, 8, None, 0, 8, 1, None, None, None, None, None])[0] == 0


# dtype, student, lds, teacher dtype, teacher, indices, index bytes, rows, classes, k, T, weight, loss, grad, stream
DISTILL = [2, P, 50, 0, P, P, 4, 10, 50, 3, 1.0, None, P, P, None]


@pytest.mark.parametrize("at,value,needle", [
    (0, 5, "type"), (3, -1, "type"), (6, 2, "index_bytes"), (7, -1, "rows"), (8, 0, "classes"), (9, 0, "k must"),
    (9, 257, "k must"), (2, 49, "stride"), (10, 0.0, "temperature"), (10, -1.0, "temperature"),
    (10, math.inf, "temperature"), (10, math.nan, "temperature"), (1, None, "null"), (4, None, "null"),
    (5, None, "null"), (5, ctypes.c_void_p(0x1002), "aligned")])
def test_distill_refuses(at, value, needle):
    args = list(DISTILL)
    args[at] = value
    rc, why = _call("sft_distill", args)
    assert rc == -1 and needle in why
    args = list(DISTILL)
    args[12] = args[13] = None
    rc, why = _call("sft_distill", args)
    assert rc == -1 and "neither" in why


SHORTER = lambda t: t[:-1].contiguous()
NARROWER = lambda t: t[..., :-1].contiguous()


@pytest.mark.parametrize("call,at,wrong,needle", [
    ("linear_fwd", "w", NARROWER, "weight must be"), ("linear_fwd", "w", torch.Tensor.float, "weight must be"),
    ("linear_fwd", "bias", SHORTER, "bias must be"), ("linear_fwd", "bias", torch.Tensor.float, "bias must be"),
    ("linear_fwd", "residual", SHORTER, "residual must be"), ("linear_fwd", "residual", NARROWER, "residual must be"),
    ("linear_fwd", "y", SHORTER, "y must be"), ("linear_fwd", "deriv", torch.Tensor.half, "deriv must be"),
    ("linear_fwd", "x", torch.Tensor.double, "dtype"), ("linear_fwd", "x", torch.Tensor.flatten, "2 dimensions"),
    ("linear_fwd", "y", torch.Tensor.clone, "on a GPU"),
    ("linear_bwd", "dy", SHORTER, "grad_y must be"), ("linear_bwd", "dy", torch.Tensor.float, "grad_y must be"),
    ("linear_bwd", "deriv", SHORTER, "deriv must be"), ("linear_bwd", "dw", SHORTER, "dw must be"),
    ("linear_bwd", "db", SHORTER, "db must be"), ("linear_bwd", "dx", NARROWER, "dx must be"),
    ("linear_bwd", "dy", torch.Tensor.clone, "on a GPU"),
    ("balance_fwd", "mask", SHORTER, "mask must be"), ("balance_fwd", "mask", torch.Tensor.float, "mask must be"),
    ("balance_fwd", "counts", SHORTER, "counts must be"), ("balance_fwd", "loss", torch.Tensor.double, "loss must be"),
    ("balance_fwd", "mask", torch.Tensor.clone, "on a GPU"),
    ("balance_bwd", "mask", SHORTER, "mask must be"), ("balance_bwd", "grad_loss", torch.Tensor.half, "grad_loss must"),
    ("balance_bwd", "grad_logits", NARROWER, "grad_logits must"), ("balance_bwd", "mask", torch.Tensor.clone, "on a GPU"),
    ("distill", "teacher", SHORTER, "teacher logits must"), ("distill", "teacher", torch.Tensor.double, "dtype"),
    ("distill", "indices", NARROWER, "indices must"), ("distill", "indices", torch.Tensor.short, "indices must"),
    ("distill", "row_weight", SHORTER, "row_weight must"), ("distill", "row_weight", torch.Tensor.half, "row_weight must"),
    ("distill", "loss", SHORTER, "loss must"), ("distill", "grad_student", torch.Tensor.float, "grad_student must"),
    ("distill", "loss", torch.Tensor.clone, "on a GPU")])
def test_calls_refuse_tensors_that_do_not_fit(call, at, wrong, needle):
    """What traced programs reach: a tensor too short would be read past its end."""
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    n = lambda *s: torch.zeros(*s, dtype=torch.int64)
    good = {
        "linear_fwd": {"x": b(9, 5), "w": b(7, 5), "bias": b(7), "residual": b(9, 7), "y": b(9, 7),
                       "deriv": torch.zeros(9, 7, dtype=torch.int16), "act": 5},
        "linear_bwd": {"dy": b(9, 7), "deriv": torch.zeros(9, 7, dtype=torch.int16), "x": b(9, 5), "w": b(7, 5),
                       "dx": b(9, 5), "dw": b(7, 5), "db": b(7), "act": 5},
        "balance_fwd": {"logits": b(9, 6), "mask": torch.zeros(9, dtype=torch.bool), "top_k": 2,
                        "loss": torch.zeros(()), "counts": n(6), "kept": n(())},
        "balance_bwd": {"logits": b(9, 6), "mask": torch.zeros(9, dtype=torch.bool), "top_k": 2, "counts": n(6),
                        "kept": n(()), "grad_loss": torch.zeros(()), "grad_logits": b(9, 6)},
        "distill": {"student": b(9, 30), "teacher": torch.zeros(9, 2), "indices": n(9, 2), "temperature": 1.0,
                    "row_weight": torch.zeros(9), "loss": torch.zeros(9), "grad_student": b(9, 30)},
    }[call]
    args = dict(good)
    args[at] = wrong(args[at])
    with pytest.raises(ValueError, match=needle):
        getattr(_native, call)(*args.values())


def test_custom_op_shapes():
    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")
        y, d = torch.ops.sft.linear_fwd(e(9, 5), e(7, 5), e(7), None, 5, True)
        assert y.shape == (9, 7) and y.dtype == torch.bfloat16 and d.shape == (9, 7) and d.dtype == torch.int16
        assert torch.ops.sft.linear_fwd(e(9, 5), e(7, 5), None, None, 0, True)[1].shape == (0,)
        dx, dw, db = torch.ops.sft.linear_bwd(y, d, e(9, 5), e(7, 5), 5, True, False, True)
        assert dx.shape == (9, 5) and dw.shape == (0,) and db.shape == (7,)
        loss, counts, kept = torch.ops.sft.balance_fwd(e(9, 6), None, 2)
        assert loss.shape == () and loss.dtype == torch.float32
        assert counts.shape == (6,) and counts.dtype == kept.dtype == torch.int64
        assert torch.ops.sft.balance_bwd(e(9, 6), None, 2, counts, kept, loss).shape == (9, 6)
        t, i = e(9, 2, dtype=torch.float32), e(9, 2, dtype=torch.int32)
        assert torch.ops.sft.distill_loss(e(9, 30), t, i, 1.0).dtype == torch.float32
        loss, ds = torch.ops.sft.distill_loss_and_grad(e(9, 30), t, i, 1.0, None)
        assert loss.shape == (9,) and ds.shape == (9, 30) and ds.dtype == torch.bfloat16
        assert torch.ops.sft.distill_grad(e(9, 30), t, i, 1.0, loss).shape == (9, 30)


@pytest.mark.parametrize("name", list(dense_ref.SLOPE))
def test_linear_reference_against_autograd(name):
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*s, generator=g) for s in ((6, 5), (4, 5), (4,), (6, 4), (6, 4)))
    ref = dense_ref.linear(x, w, b, r, name, dy)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    z = leaves[0] @ leaves[1].t() + leaves[2]
    F = torch.nn.functional
    y = {"none": lambda: z, "relu": lambda: F.relu(z), "crelu": lambda: z.clamp(0, 1), "screlu": lambda: z.clamp(0, 1) ** 2,
         "silu": lambda: F.silu(z), "gelu": lambda: F.gelu(z)}[name]() + r.double()
    grads = torch.autograd.grad(y, leaves, dy.double())
    for got, n in zip((y, *grads), ("y", "dx", "dw", "db")):
        assert torch.allclose(got, ref[n][0], rtol=1e-12, atol=1e-12)
        assert dense_ref.worst(got.float(), ref[n]) <= 1.0
    wrong = ref["y"][0].float() + 1e-4  # a planted mistake is far outside the bounds
    assert dense_ref.worst(wrong, ref["y"]) > 1.0
    assert dense_ref.worst(ref["db"][0].float() * 1.001, ref["db"]) > 1.0


def test_balance_reference_against_autograd_and_planted_mistakes():
    g = torch.Generator().manual_seed(2)
    x, mask = torch.randn(40, 6, generator=g), torch.rand(40, generator=g) < 0.7
    (loss, lerr), counts, (d, derr) = dense_ref.balance(x, mask, 2, 0.3)
    leaf = x.double().requires_grad_()
    p = torch.softmax(leaf[mask], 1)
    f = counts.double() / (mask.sum() * 2)
    want = 6 * (f * p.mean(0)).sum()
    (grad,) = torch.autograd.grad(want * 0.3, [leaf])
    assert abs(loss - want).item() < 1e-12 and torch.allclose(d, grad, atol=1e-14)
    assert counts.sum().item() == 2 * mask.sum().item()
    assert dense_ref.worst(d.float(), (d, derr)) <= 1.0
    unmasked = dense_ref.balance(x, None, 2, 0.3)  # the mask forgotten
    assert dense_ref.worst(unmasked[2][0].float(), (d, derr)) > 1.0 and not torch.equal(unmasked[1], counts)


def test_distill_reference_against_autograd_and_planted_mistakes():
    g = torch.Generator().manual_seed(3)
    s, t, w = torch.randn(5, 20, generator=g), torch.randn(5, 4, generator=g), torch.rand(5, generator=g)
    i = torch.stack([torch.randperm(20, generator=g)[:4] for _ in range(5)])
    i[0] = -1
    (loss, lerr), (ds, derr) = dense_ref.distill(s, t, i, 2.0, w)
    leaf = s.double().requires_grad_()
    q = torch.softmax(t[1:].double() / 2, 1)
    logp = torch.log_softmax(leaf[1:] / 2, 1).gather(1, i[1:])
    each = 4 * (q * (q.log() - logp)).sum(1)
    (grad,) = torch.autograd.grad((each * w[1:].double()).sum(), [leaf])
    assert torch.allclose(loss[1:], each, atol=1e-12) and loss[0] == 0
    assert torch.allclose(ds, grad, atol=1e-14)
    for wrong in (loss / 2, loss + 1e-4):  # the temperature's factor, an offset
        assert dense_ref.worst(wrong.float(), (loss, lerr)) > 1.0
    assert dense_ref.worst((ds * 1.001).float(), (ds, derr)) > 1.0
