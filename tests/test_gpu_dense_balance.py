"""expert_balance on the GPU against its 64-bit form: counts equal, loss and
gradient within derived bounds (tests/dense_ref.py)."""

import pytest
import torch

import dense_ref
from gpu_helpers import DEV, announce
from src.model.modules.dense import expert_balance

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _logits(seed, T, E, dtype):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, E, generator=g) * 1.5 + torch.randn(E, generator=g)).to(dtype)
    return x, torch.rand(T, generator=g) < 0.7


def _check(logits, mask, top_k, grad=0.37, place=lambda t: t.to(DEV)):
    grad = torch.tensor(grad).item()
    loss_ref, counts_ref, d_ref = dense_ref.balance(logits, mask, top_k, grad)
    leaf = place(logits).detach().requires_grad_()
    m = None if mask is None else mask.to(DEV)
    loss, counts = expert_balance(leaf, top_k, m)
    (d,) = torch.autograd.grad(loss, [leaf], torch.tensor(grad, device=DEV))
    again = expert_balance(leaf, top_k, m)
    torch.cuda.synchronize()
    assert torch.equal(counts.cpu(), counts_ref)
    assert loss.dtype == torch.float32 and counts.dtype == torch.int64 and d.dtype == logits.dtype
    assert dense_ref.worst(loss, loss_ref) <= 1.0
    assert dense_ref.worst(d, d_ref) <= 1.0
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)


SIZES = [(1, 1, 1), (1, 2, 1), (2, 5, 5), (5, 8, 1), (300, 8, 2), (257, 13, 3), (1000, 64, 2), (130, 100, 4),
         (64, 256, 1), (33, 511, 2), (20, 1000, 8), (20, 1024, 3), (9000, 24, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    announce(f"balance {size} {dtype}")
    T, E, k = size
    x, mask = _logits(sum(size), T, E, dtype)
    _check(x, mask if T % 2 == 0 else None, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lower_expert(dtype):
    announce(f"balance ties {dtype}")
    g = torch.Generator().manual_seed(1)
    for E, k in ((8, 3), (40, 5), (700, 4)):
        _check(torch.zeros(50, E, dtype=dtype), None, k)
        _check(torch.randint(0, 3, (90, E), generator=g).to(dtype), None, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [7, 64, 300])
def test_masks_and_excluded_experts(E, dtype):
    announce(f"balance masks E={E} {dtype}")
    x, mask = _logits(E, 200, E, dtype)
    x[torch.rand(200, E, generator=torch.Generator().manual_seed(2)) < 0.6] = -float("inf")
    x[5] = -float("inf")  # no expert left
    x[6, 1:] = -float("inf")  # one left, fewer than top_k
    mask[5:7] = True
    _check(x, mask, 3)
    _check(x, None, 3)
    x[torch.isinf(x)] = torch.finfo(dtype).min  # excluded by the type's lowest value
    _check(x, mask, 2)
    x[~mask] = float("nan")  # what is left out counts nowhere, whatever it holds
    x[(~mask).nonzero()[0, 0]] = float("inf")
    _check(x, mask, 2)
    loss, counts = expert_balance(x.to(DEV), 2, torch.zeros(200, dtype=torch.bool, device=DEV))
    assert loss.item() == 0.0 and counts.sum().item() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [1, 7, 64, 300])
def test_rows_of_nan_are_not_taken_for_excluded_ones(E, dtype):
    announce(f"balance rows of NaN E={E} {dtype}")
    x, _ = _logits(E, 200, E, dtype)
    x[3] = -float("inf")
    clean, counts = expert_balance(x.to(DEV), 1)
    x[7] = -float("inf")
    x[7, E - 1] = float("nan")
    leaf = x.to(DEV).requires_grad_()
    loss, bad = expert_balance(leaf, 1)
    (d,) = torch.autograd.grad(loss, [leaf])
    assert torch.isfinite(clean).item() and counts.sum().item() == 199
    assert torch.isnan(loss).item() and bad.sum().item() == 198  # nothing is chosen of such a row
    assert torch.isnan(d[7]).all() and torch.equal(d[3], torch.zeros_like(d[3]))


@pytest.mark.parametrize("dtype", TYPES)
def test_no_positions_and_all_masked(dtype):
    announce(f"balance empty {dtype}")
    for T in (0, 9):
        x = torch.randn(T, 6, device=DEV).to(dtype).requires_grad_()
        loss, counts = expert_balance(x, 2, torch.zeros(T, dtype=torch.bool, device=DEV))
        (d,) = torch.autograd.grad(loss, [x])
        assert loss.item() == 0.0 and torch.equal(counts, torch.zeros_like(counts))
        assert torch.equal(d, torch.zeros_like(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_leading_dimensions(dtype):
    announce(f"balance strides {dtype}")
    x, mask = _logits(4, 120, 24, dtype)

    def odd(t):
        buf = torch.full((120 * 27 + 1,), float("nan"), dtype=dtype, device=DEV)
        v = buf[1:].view(120, 27)[:, 2:26]
        v.copy_(t.to(DEV))
        return v

    _check(x, mask, 2, place=odd)
    _check(x, mask, 2, place=lambda t: t.t().contiguous().to(DEV).t())
    flat = expert_balance(x.to(DEV), 2, mask.to(DEV))
    lead = expert_balance(x.to(DEV).view(4, 30, 24), 2, mask.to(DEV).view(4, 30))
    assert torch.equal(flat[0], lead[0]) and torch.equal(flat[1], lead[1])


def test_grad_against_differences():
    """The counts do not move under small steps that change no choice; central differences with step h
    are off by h^2 / 6 times the third derivative (under 6 times the loss's scale) and by rounding over h."""
    announce("balance differences")
    x, _ = _logits(5, 60, 12, torch.float32)
    top = x.topk(3, 1).values
    x = x[(top[:, 1] - top[:, 2]) > 0.2]  # choices with a margin
    leaf = x.to(DEV).requires_grad_()
    loss, _ = expert_balance(leaf, 2)
    (d,) = torch.autograd.grad(loss, [leaf])
    g = torch.Generator().manual_seed(6)
    h = 2.0 ** -4
    for _ in range(4):
        v = torch.randn(x.shape, generator=g)
        v /= v.abs().max()
        step = [expert_balance((x + s * h * v).to(DEV), 2)[0].double().item() for s in (1, -1)]
        slope = (d.double().cpu() * v).sum().item()
        assert abs((step[0] - step[1]) / (2 * h) - slope) <= 12 * (h * h + 64 * 2.0 ** -24 / h) * loss.item()


def test_another_stream_and_graph_replays():
    announce("balance stream and graph")
    x, mask = (t.to(DEV) for t in _logits(8, 5000, 64, torch.bfloat16))
    want = expert_balance(x, 2, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = expert_balance(x, 2, mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = expert_balance(static, 2, mask)
    for i in range(3):
        static.copy_(x.flip(1) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        now = expert_balance(static, 2, mask)
        assert torch.equal(out[0], now[0]) and torch.equal(out[1], now[1])


def test_refusals():
    announce("balance refusals")
    x = torch.zeros(4, 8, device=DEV)
    for args in [(x.cpu(),), (x.double(),), (x, 0), (x, 9), (x, 1, torch.ones(4, device=DEV)),
                 (x, 1, torch.ones(5, dtype=torch.bool, device=DEV)), (torch.zeros(2, 1025, device=DEV),),
                 (x[:, :0],)]:
        with pytest.raises(AssertionError):
            expert_balance(*args)
