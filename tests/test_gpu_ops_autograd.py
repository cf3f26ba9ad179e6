"""The training-step operators beside autograd: no gradient is lost without a word."""
import pytest
import torch

from msccl_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_backward_through_the_statistics_raises(score):
    x = torch.randn(40, 12, generator=gen(1), device="cuda")
    index = x.topk(3).indices
    want = ops.balance_stats(x, index, score=score)
    loss = ops.balance_loss(*want, 3, 0.1)
    leaf = x.clone().requires_grad_(True)
    counts, probs = ops.balance_stats(leaf, index, score=score)
    also = ops.balance_loss(counts, probs, 3, 0.1)
    assert torch.equal(counts, want[0]) and torch.equal(probs, want[1]) and torch.equal(also, loss)
    assert probs.requires_grad and also.requires_grad and not counts.requires_grad
    for out in (probs.sum(), also.sum(), leaf.square().sum() + also.sum()):
        with pytest.raises(RuntimeError, match="balance_backward"):
            out.backward(retain_graph=True)
    # as it is meant: the gradient added to what autograd brings to the logits
    up = ops.balance_backward(leaf, counts, 3, 0.1, score=score)
    assert not up.requires_grad
    leaf.grad = None
    torch.autograd.backward([leaf.square().sum(), leaf], [None, up])
    assert torch.equal(leaf.grad, 2 * x + up)
    with torch.no_grad():
        assert not ops.balance_stats(leaf, index, score=score)[1].requires_grad
    assert not ops.balance_loss(counts, probs.detach(), 3).requires_grad
    with pytest.raises(TypeError):
        ops.balance_stats(leaf, index[:10], score=score)


def refused(out):
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(retain_graph=True)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("views", [False, True])
def test_a_graph_refuses_weights_that_a_step_changed(bits, views):
    if views:
        flat = torch.randn(2048, generator=gen(2), device="cuda").to(torch.bfloat16)
        p = [flat[:1000], flat[1024:1324]]
    else:
        p = [torch.randn(n, generator=gen(n), device="cuda").to(torch.bfloat16).requires_grad_(True) for n in (1000, 300)]
    masters = [x.detach().float() for x in p]
    state = [ops.adamw_state(x, bits) for x in p]
    pick = lambda i: [s[i] for s in state]  # noqa: E731
    plan = ops.AdamW(p, [torch.ones_like(x.detach()) for x in p], pick(0), pick(1), torch.zeros(1, dtype=torch.int64, device="cuda"),
                     masters=masters, exp_avg_scales=pick(2) if bits == 8 else None,
                     exp_avg_sq_scales=pick(3) if bits == 8 else None, rounding="nearest" if bits == 8 else None)
    x = [torch.ones(t.numel(), device="cuda", dtype=torch.bfloat16, requires_grad=True) for t in p]
    held = [(a * b).sum() for a, b in zip(x, p)]
    also = [(a.float() * b).sum() for a, b in zip(x, masters)]
    old = [t._version for t in p + masters]
    plan.step(1e-3)
    assert all(t._version > v for t, v in zip(p + masters, old))
    for out in held + also:
        refused(out)
    (x[0] * p[0]).sum().backward()   # a graph of the new ones goes


def test_a_graph_refuses_other_tensors_that_are_written():
    x = torch.randn(20, 8, generator=gen(3), device="cuda")
    counts, _ = ops.balance_stats(x, x.topk(2).indices)
    w = torch.ones(20, 8, device="cuda", requires_grad=True)
    held = (w * x).sum()
    ops.balance_backward(x, counts, 2, out=x)   # in place of the logits
    refused(held)
    total = torch.zeros(1, dtype=torch.float64, device="cuda")
    v = torch.ones(1, dtype=torch.float64, device="cuda", requires_grad=True)
    held = (v * total).sum()
    ops.SquareSum([x])(out=total)
    refused(held)


def test_a_graph_refuses_what_a_sharded_step_and_a_reduction_wrote():
    import msccl_amd as M
    comms = M.Comm.init_all([0, 0])
    try:
        block = 512
        params = [torch.ones(2 * block, device="cuda") for _ in range(2)]
        shards = [torch.zeros(block, device="cuda") for _ in range(2)]
        plans, keep = [], []
        for r in range(2):
            p = params[r][r * block:(r + 1) * block]
            st = ops.adamw_state(p)
            keep.append(st)
            plans.append(ops.AdamW([p], [shards[r]], [st[0]], [st[1]], torch.zeros(1, dtype=torch.int64, device="cuda")))
        sums = [ops.SquareSum([s]) for s in shards]
        x = [torch.ones(2 * block, device="cuda", requires_grad=True) for _ in range(2)]
        held = [(a * b).sum() for a, b in zip(x, params)]
        ops.sharded_step(comms, [torch.ones(2 * block, device="cuda") for _ in range(2)], shards, params, plans, sums, 1e-3)
        counts = [torch.ones(9, dtype=torch.int64, device="cuda") for _ in range(2)]
        probs = [torch.ones(8, device="cuda") for _ in range(2)]
        held += [(a[:8] * b).sum() for a, b in zip(x, probs)]
        ops.balance_all_reduce(comms, counts, probs)
        torch.cuda.synchronize()
        for out in held:
            refused(out)
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()
