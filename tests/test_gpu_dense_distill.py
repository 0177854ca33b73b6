"""distill_loss and distill_loss_and_grad on the GPU against their 64-bit form,
within derived bounds (tests/dense_ref.py)."""

import math

import pytest
import torch

import dense_ref
from gpu_helpers import DEV, announce
from src.model.modules.dense import distill_loss, distill_loss_and_grad

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def _inputs(seed, R, V, k, dtype, ttype=torch.float32, itype=torch.int32, empty=True):
    g = torch.Generator().manual_seed(seed)
    s = (torch.randn(R, V, generator=g) * 2).to(dtype)
    t = torch.randn(R, k, generator=g).to(ttype)
    i = torch.stack([torch.randperm(V, generator=g)[:k] if V >= k else torch.randint(0, V, (k,), generator=g)
                     for _ in range(R)])
    if empty and R > 2:
        i[0] = -1  # no teacher
        i[1, k // 2:] = V  # past the classes
    return s, t, i.to(itype), torch.rand(R, generator=g) + 0.1


def _check(s, t, i, w, tau=1.0, place=lambda x: x.to(DEV)):
    loss_ref, ds_ref = dense_ref.distill(s, t, i, tau, w)
    td, idx = t.to(DEV), i.to(DEV)
    wd = None if w is None else w.to(DEV)
    loss, ds = distill_loss_and_grad(place(s), td, idx, wd, tau)
    leaf = place(s).detach().requires_grad_()
    each = distill_loss(leaf, td, idx, tau)
    (grad,) = torch.autograd.grad(each, [leaf], torch.ones_like(each) if wd is None else wd)
    torch.cuda.synchronize()
    assert loss.dtype == torch.float32 and ds.dtype == s.dtype
    assert torch.equal(each, loss) and torch.equal(grad, ds)
    assert dense_ref.worst(loss, loss_ref) <= 1.0
    assert dense_ref.worst(ds, ds_ref) <= 1.0


SIZES = [(1, 1, 1), (3, 2, 2), (4, 7, 3), (5, 33, 4), (600, 130, 3), (9, 1000, 64), (4, 2049, 65), (4, 4096, 32),
         (3, 5000, 100), (3, 9001, 130), (2, 20001, 256), (3, 33000, 9), (2, 70001, 33), (2, 140001, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    announce(f"distill {size} {dtype}")
    n = sum(size)
    s, t, i, w = _inputs(n, *size, dtype, TYPES[n % 3], (torch.int32, torch.int64)[n % 2])
    _check(s, t, i, w if n % 4 else None, (1.0, 2.0, 0.7)[n % 3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 4096, 10000, 140000])
def test_excluded_classes(V, dtype):
    """Illegal moves at -inf, rows with nothing left, slots without weight."""
    announce(f"distill excluded V={V} {dtype}")
    s, t, i, w = _inputs(V, 8, V, 6, dtype)
    taught = torch.zeros(8, V, dtype=torch.bool).scatter_(1, i.long().clamp(0, V - 1), True)
    s[(torch.rand(8, V, generator=torch.Generator().manual_seed(1)) < 0.8) & ~taught] = -INF
    s[2] = -INF  # no class left
    t[3, 1:] = -INF  # one slot with weight ...
    s[3, i[3, 2]] = -INF  # ... beside one whose class the student excludes
    t[4] = -INF  # slots without any weight
    _check(s, t, i, w, 2.0)
    s[torch.isinf(s)] = torch.finfo(dtype).min if dtype != torch.float32 else -1e30
    s[2] = 0.0
    s[3, i[3, 2]] = 0.0
    loss, ds = distill_loss_and_grad(s.to(DEV), t.to(DEV), i.to(DEV), w.to(DEV))
    assert torch.isfinite(loss).all() and torch.isfinite(ds).all()


def test_a_class_the_student_excludes_costs_infinitely_much():
    announce("distill infinite")
    s, t, i, w = _inputs(3, 4, 50, 5, torch.float32, empty=False)
    s[1, i[1, 0]] = -INF
    loss, ds = distill_loss_and_grad(s.to(DEV), t.to(DEV), i.to(DEV), w.to(DEV))
    assert loss[1].item() == INF and torch.isfinite(loss[[0, 2, 3]]).all()
    assert torch.isfinite(ds).all()  # the gradient has a value there: -q
    q = torch.softmax(t[1].double(), 0)[0] * w[1].double()
    assert abs(ds[1, i[1, 0]].item() + q.item()) <= 64 * dense_ref.U32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(146, 146), (5000, 256), (40000, 200)])
def test_logits_far_from_zero_and_teachers_that_agree(V, k, dtype):
    """The loss is a difference of logits: neither their common offset nor log-sums may show in its error."""
    announce(f"distill offset {V} {k} {dtype}")
    g = torch.Generator().manual_seed(V)
    s = (1000 + 2 * torch.randn(6, V, generator=g)).to(dtype)
    i = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(6)])
    t = s.float().gather(1, i) + 0.01 * torch.randn(6, k, generator=g)
    (loss_ref, _) = dense_ref.distill(s.float() - 1000, t - 1000, i, 2.0)  # exact differences
    loss, _ = distill_loss_and_grad(s.to(DEV), t.to(DEV), i.to(DEV), None, 2.0)
    assert dense_ref.worst(loss, loss_ref) <= 1.0


@pytest.mark.parametrize("dtype", TYPES)
def test_classes_named_twice(dtype):
    announce(f"distill repeated {dtype}")
    s, t, i, w = _inputs(4, 6, 90, 70, dtype, empty=False)
    i[1, 1:9] = i[1, 0]
    i[2] = 5
    i[3, 64:] = i[3, 0]
    i[4, ::2] = -1
    _check(s, t, i, w, 0.7)


@pytest.mark.parametrize("V", [5, 300, 5000, 20011])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_nan_are_not_taken_for_excluded_ones(V, dtype):
    announce(f"distill rows of NaN V={V} {dtype}")
    s, t, i, w = _inputs(5, 70, V, 4, dtype)
    i[1:] = i[1:].clamp(min=0)  # taught
    s[3], s[4], s[5] = float("nan"), -float("inf"), -float("inf")
    s[5, V - 1] = float("nan")
    loss, ds = distill_loss_and_grad(s.to(DEV), t.to(DEV), i.to(DEV), w.to(DEV))
    assert torch.isnan(loss[[3, 5]]).all() and torch.isnan(ds[[3, 5]]).all()
    assert loss[4].item() == 0.0 and torch.equal(ds[4], torch.zeros_like(ds[4]))
    kept = [r for r in range(70) if r not in (3, 5)]
    assert not torch.isnan(loss[kept]).any() and not torch.isnan(ds[kept]).any()


def test_nan_stays_in_its_row():
    announce("distill NaN")
    s, t, i, w = _inputs(5, 70, 300, 5, torch.bfloat16)
    clean = distill_loss_and_grad(s.to(DEV), t.to(DEV), i.to(DEV), w.to(DEV))
    bad = s.clone()
    bad[0, 3] = float("nan")  # a row without a teacher: still nothing
    bad[7, 299] = float("nan")
    t2 = t.clone()
    t2[0] = float("nan")  # empty slots
    got = distill_loss_and_grad(bad.to(DEV), t2.to(DEV), i.to(DEV), w.to(DEV))
    kept = [r for r in range(70) if r != 7]
    assert torch.equal(got[0][kept], clean[0][kept]) and torch.equal(got[1][kept], clean[1][kept])
    assert torch.isnan(got[0][7]) and torch.isnan(got[1][7]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [129, 4097, 70000])
def test_strides(V, dtype):
    announce(f"distill strides V={V} {dtype}")
    s, t, i, w = _inputs(V, 5, V, 7, dtype)

    def odd(x):
        buf = torch.full((5 * (V + 3) + 1,), float("nan"), dtype=dtype, device=DEV)
        v = buf[1:].view(5, V + 3)[:, 1:V + 1]
        v.copy_(x.to(DEV))
        return v

    _check(s, t, i, w, 1.0, odd)
    _check(s, t, i, w, 1.0, lambda x: x.t().contiguous().to(DEV).t())
    wide = distill_loss(s.to(DEV), t.to(DEV).t().contiguous().t(), i.to(DEV).t().contiguous().t())
    assert torch.equal(wide, distill_loss(s.to(DEV), t.to(DEV), i.to(DEV)))


def test_no_rows():
    announce("distill no rows")
    s = torch.empty(0, 9, device=DEV, requires_grad=True)
    t, i = torch.empty(0, 2, device=DEV), torch.empty(0, 2, dtype=torch.int64, device=DEV)
    loss = distill_loss(s, t, i)
    (ds,) = torch.autograd.grad(loss.sum(), [s])
    assert loss.shape == (0,) and ds.shape == (0, 9)


def test_grad_against_differences():
    """Central differences along random directions: h^2 / 6 of the third derivative (at most T^2 / T^3
    of a probability) and the loss's rounding over h."""
    announce("distill differences")
    s, t, i, _ = _inputs(6, 5, 40, 6, torch.float32, empty=False)
    leaf = s.to(DEV).requires_grad_()
    tau = 1.5
    (d,) = torch.autograd.grad(distill_loss(leaf, t.to(DEV), i.to(DEV), tau).sum(), [leaf])
    g = torch.Generator().manual_seed(7)
    h = 2.0 ** -5
    for _ in range(4):
        v = torch.randn(s.shape, generator=g)
        v /= v.abs().max()
        up, down = (distill_loss((s + x * h * v).to(DEV), t.to(DEV), i.to(DEV), tau).double().sum().item()
                    for x in (1, -1))
        slope = (d.double().cpu() * v).sum().item()
        assert abs((up - down) / (2 * h) - slope) <= 5 * (h * h + 256 * 2.0 ** -24 / h)


def test_another_stream_and_graph_replays():
    announce("distill stream and graph")
    s, t, i, w = (x.to(DEV) for x in _inputs(8, 40, 5000, 9, torch.bfloat16))
    want = distill_loss_and_grad(s, t, i, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = distill_loss_and_grad(s, t, i, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = s.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = distill_loss_and_grad(static, t, i, w)
    for n in range(3):
        static.copy_(s.flip(1) * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, distill_loss_and_grad(static, t, i, w)))


def test_refusals():
    announce("distill refusals")
    s, t, i = torch.zeros(3, 8, device=DEV), torch.zeros(3, 2, device=DEV), torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    for args in [(s.cpu(), t, i), (s.double(), t, i), (s[:2], t, i), (s, t[:, :1], i), (s, t, i.float()),
                 (s, t, i.cpu()), (s[:, :0], t, i), (s, t[:, :0], i[:, :0]),
                 (s, torch.zeros(3, 257, device=DEV), torch.zeros(3, 257, dtype=torch.int32, device=DEV))]:
        with pytest.raises(AssertionError):
            distill_loss(*args)
    for tau in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            distill_loss(s, t, i, tau)
    for w in (torch.zeros(2, device=DEV), torch.zeros(3, dtype=torch.float64, device=DEV), torch.zeros(3)):
        with pytest.raises(AssertionError):
            distill_loss_and_grad(s, t, i, w)
