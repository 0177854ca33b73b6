"""MoveHead on the GPU, behind the feature transformer and by itself: a training step
and an evaluation through the dense operators against the same model in plain
torch operations in 64 bits, and compiled against eager."""

import pytest
import torch

from gpu_helpers import DEV, announce
from sft_amd import positions
from sft_amd.encode import encode_batch
from src.model.modules.dense import distill_loss, distill_loss_and_grad, expert_balance, fused_linear
from src.model.modules.features import get_feature_cls
from src.model.move_head import MoveHead
from src.model.transform_inputs import transform_inputs

pytestmark = pytest.mark.gpu


def _teacher(B, moves, k, seed):
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(moves, generator=g)[:k] for _ in range(B)])
    idx[1] = -1
    legal = torch.rand(B, moves, generator=g) < 0.1
    legal.scatter_(1, idx.clamp(min=0), True)
    return torch.randn(B, k, generator=g), idx, legal


def _plain(head, x, t, idx, legal, tau):
    """The head's loss in 64 bits from its parameters (leaves in, loss and leaves out)."""
    leaves = {n: p.detach().double().cpu().requires_grad_() for n, p in head.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    lin = lambda v, n: v @ leaves[n + ".weight"].t() + leaves[n + ".bias"]
    routes = lin(x, "router")
    p = torch.softmax(routes, 1)
    h = (lin(x, "expert").clamp(0, 1).view(-1, head.experts, head.width) * p.unsqueeze(2)).sum(1)
    for i in range(len(head.blocks)):
        h = h + torch.nn.functional.gelu(lin(h, f"blocks.{i}"))
    logits = lin(h, "moves").masked_fill(~legal, -float("inf"))
    taught = (idx >= 0).any(1)
    q = torch.softmax((t.double() / tau)[taught], 1)
    logp = torch.log_softmax(logits[taught] / tau, 1).gather(1, idx[taught])
    kl = tau * tau * (q * (q.log() - logp)).sum(1)
    chosen = torch.zeros_like(p).scatter_(1, routes.topk(head.top_k, 1).indices, 1.0)[taught]
    n = taught.sum()
    balance = head.experts * (chosen.sum(0) / (n * head.top_k) * p[taught].mean(0)).sum()
    loss = kl.mean() + head.balance_weight * balance
    return loss, x, leaves, chosen.sum(0).long()


def _rel(got, want):
    return ((got.detach().double().cpu() - want).norm() / want.norm()).item()


def test_training_step_behind_the_feature_transformer():
    announce("move head step")
    torch.manual_seed(3)
    boards, stm = positions.random_positions(192, seed=5)
    enc = encode_batch(torch.as_tensor(boards, device=DEV), torch.as_tensor(stm, device=DEV), "HalfKAv2_hm^")
    ft = get_feature_cls("HalfKAv2_hm^")(128 + 8).to(DEV)
    head = MoveHead(128, width=48, experts=6, blocks=2, moves=500, top_k=2, balance_weight=0.05, device=DEV)
    l0, _ = transform_inputs(ft, 128, enc["us"], enc["white"], enc["black"], enc["psqt_indices"])
    l0.retain_grad()
    t, idx, legal = _teacher(192, 500, 9, 1)
    loss, counts = head.loss(l0, t.to(DEV), idx.to(DEV), legal.to(DEV), 1.5)
    loss.backward()
    want, x, leaves, chosen = _plain(head, l0, t, idx, legal, 1.5)
    want.backward()
    torch.cuda.synchronize()
    assert torch.equal(counts.cpu(), chosen)
    # binary32 throughout: sums of up to 500 terms through four layers stay far within 2^-14
    assert abs(loss.item() - want.item()) <= 2.0 ** -14 * abs(want.item())
    assert _rel(l0.grad, x.grad) <= 2.0 ** -14
    for n, p in head.named_parameters():
        assert _rel(p.grad, leaves[n].grad) <= 2.0 ** -14, n
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in ft.parameters())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_mixed_precision_steps_learn(dtype):
    announce(f"move head {dtype}")
    torch.manual_seed(4)
    head = MoveHead(64, width=64, experts=4, blocks=1, moves=256, device=DEV, dtype=dtype)
    x = torch.rand(333, 64, device=DEV).to(dtype)
    t, idx, legal = (v.to(DEV) for v in _teacher(333, 256, 5, 2))
    opt = torch.optim.SGD(head.parameters(), lr=0.5)
    losses = []
    for _ in range(20):
        opt.zero_grad()
        loss, counts = head.loss(x, t, idx, legal)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert counts.sum().item() == 332  # one position has no teacher
    assert losses[-1] < losses[0]


def test_single_positions_agree_with_batches():
    announce("move head single rows")
    torch.manual_seed(5)
    head = MoveHead(72, width=40, experts=5, moves=130, device=DEV)
    x = torch.rand(90, 72, device=DEV)
    with torch.no_grad():
        whole, _ = head(x)
        for i in (0, 33, 89):
            one, _ = head(x[i:i + 1])
            assert (one - whole[i]).abs().max().item() <= 2.0 ** -16 * whole.abs().max().item()


def test_compiled_matches_eager():
    announce("move head compiled")
    torch.manual_seed(6)
    w = torch.randn(40, 72, device=DEV, requires_grad=True)
    b = torch.randn(40, device=DEV, requires_grad=True)
    x = torch.randn(130, 72, device=DEV, requires_grad=True)
    t, idx, _ = _teacher(130, 40, 4, 3)
    t, idx = t.to(DEV), idx.to(DEV)

    def step(x, w, b):
        y = fused_linear(x, w, b, None, "silu")
        balance, counts = expert_balance(y, 2)
        return distill_loss(y, t, idx, 2.0).mean() + balance, counts

    eager, counts = step(x, w, b)
    want = torch.autograd.grad(eager, [x, w, b])
    compiled, counts_c = torch.compile(step, fullgraph=True)(x, w, b)
    got = torch.autograd.grad(compiled, [x, w, b])
    assert torch.equal(counts, counts_c)
    assert abs(eager.item() - compiled.item()) <= 2.0 ** -20 * abs(eager.item())
    for a, c in zip(want, got):
        assert (a - c).abs().max().item() <= 2.0 ** -18 * a.abs().max().item()
    both = torch.compile(lambda s: distill_loss_and_grad(s, t, idx, None, 2.0), fullgraph=True)
    s = torch.randn(130, 40, device=DEV)
    assert all(torch.equal(a, c) for a, c in zip(both(s), distill_loss_and_grad(s, t, idx, None, 2.0)))


def test_second_derivatives_are_refused():
    announce("dense second derivative")
    x = torch.randn(70, 16, device=DEV, requires_grad=True)
    w = torch.randn(8, 16, device=DEV, requires_grad=True)
    t, idx = torch.randn(70, 2, device=DEV), torch.zeros(70, 2, dtype=torch.int64, device=DEV)
    for out in (fused_linear(x, w, activation="gelu").sum(), expert_balance(x, 1)[0], distill_loss(x, t, idx).sum()):
        (g,) = torch.autograd.grad(out, [x], create_graph=True)
        with pytest.raises(RuntimeError, match="once only"):
            g.sum().backward()
