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
