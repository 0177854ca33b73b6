"""fused_linear on the GPU against its 64-bit form, within bounds derived from
the sizes (tests/dense_ref.py): types, activations, odd and long sizes, strides
and alignments, empty batches, non-finite values, streams and graphs."""

import pytest
import torch

import dense_ref
from gpu_helpers import DEV, announce
from src.model.modules.dense import fused_linear

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
SMOOTH = ["none", "silu", "gelu"]
KINKS = ["relu", "crelu", "screlu"]


def _inputs(seed, M, K, N, dtype, kinks=False, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)

    if kinks:  # small multiples of powers of two: every pre-activation is exact, many lie on a kink
        x = torch.randint(-4, 5, (M, K), generator=g).to(dtype) / 2
        w = torch.randint(-4, 5, (N, K), generator=g).to(dtype) / 4
        b = torch.randint(-8, 9, (N,), generator=g).to(dtype) / 8
    else:
        x, w, b = normal(M, K), normal(N, K, scale=K ** -0.5), normal(N, scale=0.3)
    return x, w, b if bias else None, normal(M, N) if residual else None, normal(M, N)


def _check(x, w, b, r, dy, name, place=lambda t: t.to(DEV)):
    ref = dense_ref.linear(x, w, b, r, name, dy)
    leaves = [None if t is None else place(t).detach().requires_grad_() for t in (x, w, b, r)]
    y = fused_linear(*leaves, name)
    got = {"y": y}
    used = {n: t for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None}
    got |= dict(zip(used, torch.autograd.grad(y, list(used.values()), place(dy))))
    with torch.no_grad():
        again = fused_linear(*leaves, name)
    torch.cuda.synchronize()
    assert torch.equal(y, again)
    if r is not None:
        assert torch.equal(got.pop("dr").cpu(), dy)
    for n, v in got.items():
        assert dense_ref.worst(v, ref[n]) <= 1.0, n


SIZES = [(1, 1, 1), (1, 1040, 128), (2, 7, 3), (16, 8, 16), (17, 33, 31), (33, 64, 130), (64, 517, 301), (65, 129, 257),
         (128, 128, 128), (129, 136, 72), (200, 1040, 16), (300, 31, 1), (513, 1, 40), (1000, 264, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    announce(f"linear {size} {dtype}")
    n = sum(size)
    x, w, b, r, dy = _inputs(n, *size, dtype, bias=n % 3 != 0, residual=n % 2 == 0)
    _check(x, w, b, r, dy, SMOOTH[n % 3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", KINKS)
@pytest.mark.parametrize("size", [(5, 24, 40), (130, 33, 65), (257, 64, 128)])
def test_kinks(size, name, dtype):
    announce(f"linear kinks {size} {name} {dtype}")
    _check(*_inputs(sum(size), *size, dtype, kinks=True), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(70, 20000, 24), (9000, 136, 40), (4099, 517, 131), (72, 40, 9000)])
def test_long_sums(size, dtype):
    """Few tiles and a long sum in the forward, the weight grad or the input grad."""
    announce(f"linear long {size} {dtype}")
    _check(*_inputs(sum(size), *size, dtype), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 12000, 50), (16, 5761, 129), (40, 4104, 33), (64, 2049, 24)])
def test_few_rows_of_long_sums(size, dtype):
    """Few rows on both sides of the length from which k is split."""
    announce(f"linear few rows {size} {dtype}")
    _check(*_inputs(sum(size), *size, dtype), "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 8, 5), (70, 64, 300), (300, 136, 130), (700, 100, 129), (500, 1040, 264),
                                  (9000, 72, 40), (6000, 1040, 2050)])
def test_bias_grads_without_an_activation(size, dtype):
    """K with and without spare columns in the weight grad's last tiles, one part and many."""
    announce(f"linear bias grad {size} {dtype}")
    _check(*_inputs(sum(size), *size, dtype, residual=False), "none")


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_grad_alone(dtype):
    """Without the weight grad, and with non-finite gradients in one column."""
    announce(f"linear bias grad alone {dtype}")
    x, w, b, _, dy = _inputs(1, 200, 72, 40, dtype)
    dy[3, 7], dy[5, 9] = float("inf"), float("nan")
    xd, wd, bd = (t.to(DEV) for t in (x, w, b))
    bd.requires_grad_()
    alone, = torch.autograd.grad(fused_linear(xd, wd, bd), bd, dy.to(DEV))
    wd.requires_grad_()
    _, both = torch.autograd.grad(fused_linear(xd, wd, bd), (wd, bd), dy.to(DEV))
    value = dy.double().sum(0)
    bound = dense_ref.rounded((200 + 3) * dense_ref.U32 * dy.double().abs().sum(0), value, dtype)
    for got in (alone.cpu().double(), both.cpu().double()):
        assert torch.isinf(got[7]) and torch.isnan(got[9])
        rest = torch.isfinite(value)
        assert ((got - value).abs() <= bound)[rest].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(50, 64, 40), (300, 128, 136), (150, 72, 33)])
def test_strides(size, dtype):
    """Slices of wider rows, odd offsets, transposed weights: the values alone count."""
    announce(f"linear strides {size} {dtype}")
    x, w, b, r, dy = _inputs(sum(size), *size, dtype)

    def wide(t):  # a slice of a buffer 8 elements wider
        if t.dim() == 1:
            return t.to(DEV)
        buf = torch.full((t.shape[0], t.shape[1] + 8), float("nan"), dtype=dtype, device=DEV)
        buf[:, :t.shape[1]] = t.to(DEV)
        return buf[:, :t.shape[1]]

    def odd(t):  # one element past an allocation's start, rows an odd distance apart
        rows, cols = (1, t.shape[0]) if t.dim() == 1 else t.shape
        buf = torch.full((rows * (cols + 1) + 1 + (rows + cols) % 2,), float("nan"), dtype=dtype, device=DEV)
        v = buf[1:1 + rows * (cols + 1)].view(rows, cols + 1)[:, :cols]
        v.copy_(t.to(DEV).view(rows, cols))
        return v[0] if t.dim() == 1 else v

    def turned(t):  # column-major
        return t.to(DEV) if t.dim() == 1 else t.t().contiguous().to(DEV).t()

    for place in (wide, odd, turned):
        _check(x, w, b, r, dy, "gelu", place)


def test_leading_dimensions_and_expanded_grads():
    announce("linear leading dimensions")
    x, w, b, r, _ = _inputs(3, 30, 40, 24, torch.float32)
    x3, r3 = x.view(5, 6, 40).to(DEV).requires_grad_(), r.view(5, 6, 24).to(DEV).requires_grad_()
    y = fused_linear(x3, w.to(DEV), b.to(DEV), r3, "silu")
    assert y.shape == (5, 6, 24)
    dx, dr = torch.autograd.grad(y.sum(), [x3, r3])  # the incoming grad has stride 0
    ref = dense_ref.linear(x, w, b, r, "silu", torch.ones(30, 24))
    assert dense_ref.worst(y.view(30, 24), ref["y"]) <= 1.0
    assert dense_ref.worst(dx.view(30, 40), ref["dx"]) <= 1.0
    assert torch.equal(dr, torch.ones_like(dr))
    one = fused_linear(x3[0, 0], w.to(DEV))
    assert one.shape == (24,)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    announce(f"linear M=0 {dtype}")
    x = torch.empty(0, 13, dtype=dtype, device=DEV, requires_grad=True)
    w = torch.randn(7, 13, device=DEV).to(dtype).requires_grad_()
    b = torch.zeros(7, dtype=dtype, device=DEV, requires_grad=True)
    y = fused_linear(x, w, b, None, "gelu")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert y.shape == (0, 7) and dx.shape == (0, 13)
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [9, 300])
def test_non_finite_values_stay_in_their_rows(M, dtype):
    announce(f"linear non-finite M={M} {dtype}")
    x, w, b, r, _ = _inputs(11, M, 72, 40, dtype)
    clean = fused_linear(*(t.to(DEV) for t in (x, w, b, r)), "silu")
    bad = x.clone()
    bad[3, 5], bad[M - 1, 71], bad[7] = float("nan"), float("inf"), float("-inf")
    y = fused_linear(bad.to(DEV), *(t.to(DEV) for t in (w, b, r)), "silu")
    kept = [m for m in range(M) if m not in (3, 7, M - 1)]
    assert torch.equal(y[kept], clean[kept])
    assert torch.isnan(y[3]).all()
    assert not torch.isfinite(y[M - 1]).all()


def test_only_the_grads_asked_for():
    announce("linear partial grads")
    x, w, b, r, dy = _inputs(5, 90, 48, 56, torch.bfloat16)
    ref = dense_ref.linear(x, w, b, r, "gelu", dy)
    for names in (("dx",), ("dw",), ("db",), ("dx", "db")):
        leaves = {n: t.to(DEV).requires_grad_(n in names) for n, t in (("dx", x), ("dw", w), ("db", b))}
        y = fused_linear(*leaves.values(), r.to(DEV), "gelu")
        got = torch.autograd.grad(y, [leaves[n] for n in names], dy.to(DEV))
        for n, v in zip(names, got):
            assert dense_ref.worst(v, ref[n]) <= 1.0, n


@pytest.mark.parametrize("dtype", TYPES)
def test_a_bias_beside_a_frozen_weight(dtype):
    announce(f"linear frozen weight {dtype}")
    x, w, b, _, dy = _inputs(6, 128, 1040, 1040, dtype, residual=False)
    ref = dense_ref.linear(x, w, b, None, "none", dy)
    for need_x in (False, True):
        xd, bd = x.to(DEV).requires_grad_(need_x), b.to(DEV).requires_grad_()
        y = fused_linear(xd, w.to(DEV), bd)
        got = torch.autograd.grad(y, [bd, xd][:1 + need_x], dy.to(DEV))
        for n, v in zip(("db", "dx"), got):
            assert dense_ref.worst(v, ref[n]) <= 1.0, n


def test_grads_against_differences():
    """Central differences of the 32-bit forward along random directions: with step h the
    difference quotient is off by h^2 |f'''| / 6 and by the forward's rounding over h."""
    announce("linear differences")
    x, w, b, r, dy = (t.double() for t in _inputs(21, 20, 24, 16, torch.float32))
    f = lambda *t: (fused_linear(*(v.float().to(DEV) for v in t), r.float().to(DEV), "gelu").double().cpu() * dy).sum()
    leaves = [t.float().to(DEV).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fused_linear(*leaves, r.float().to(DEV), "gelu"), leaves, dy.float().to(DEV))
    g = torch.Generator().manual_seed(4)
    h = 2.0 ** -6
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=g).double()
        v /= v.norm()
        plus, minus = [x, w, b], [x, w, b]
        plus[i], minus[i] = plus[i] + h * v, minus[i] - h * v
        # the inputs' rounding, the outputs' rounding and the third-order term (|gelu'''| < 1.6), all summed over dy
        rows = dy.abs().sum().item()
        slack = rows * (64 * 2.0 ** -24 / h + h * h * 1.6 / 6 * (x.abs().max().item() + 1) ** 3)
        assert abs((f(*plus) - f(*minus)) / (2 * h) - (grads[i].double().cpu() * v).sum()).item() <= slack


def test_another_stream_and_graph_replays():
    announce("linear stream and graph")
    x, w, b, r, _ = (t.to(DEV) for t in _inputs(8, 300, 136, 72, torch.bfloat16))
    want = fused_linear(x, w, b, r, "crelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        got = fused_linear(x, w, b, r, "crelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static = x.clone()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fused_linear(static, w, b, r, "crelu")
        for i in range(3):
            static.copy_(x * (i + 1))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, fused_linear(static, w, b, r, "crelu"))


def test_refusals():
    announce("linear refusals")
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(3, 8, device=DEV)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    for args in [(x.cpu(), w.cpu()), (x.double(), w.double()), (x, w.half()), (x, w[:, :7]), (x, w[:0]),
                 (x, w, torch.zeros(4, device=DEV)), (x, w, None, torch.zeros(4, 4, device=DEV)),
                 (x, w, None, torch.zeros(3, device=DEV)), (x[:, :0], w[:, :0])]:
        with pytest.raises(AssertionError):
            fused_linear(*args)
