"""Plans used on other streams than their tensors': what is dropped meanwhile is not used again too early."""
import pytest
import torch

from msccl_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def refill(sizes, value):
    """New tensors of these sizes, in memory that the allocator takes for free."""
    return [torch.full((n,), value, device="cuda") for n in sizes for _ in range(3)]


def test_a_square_sum_outlives_its_dropped_tensors():
    n = 1 << 24
    x = torch.randn(n, generator=gen(1), device="cuda")
    want = ops.SquareSum([x])()
    for made_on_side in (False, True):
        side = torch.cuda.Stream()
        y = x.clone()
        torch.cuda.synchronize()
        if made_on_side:
            with torch.cuda.stream(side):
                plan = ops.SquareSum([y])
        else:
            plan = ops.SquareSum([y])
        with torch.cuda.stream(side):
            got = [plan() for _ in range(100)]
        del plan, y
        junk = refill([n], 9.0)
        side.synchronize()
        assert all(torch.equal(g, want) for g in got)
        del junk, got


def test_steps_outlive_their_dropped_gradients():
    sizes = [1 << 22, 1 << 20, 5]
    make = lambda k: [torch.randn(n, generator=gen(10 * k + i), device="cuda") for i, n in enumerate(sizes)]  # noqa: E731

    def plan_of(grads):
        p = make(0)
        m, v = zip(*[ops.adamw_state(x) for x in p])
        return p, ops.AdamW(p, grads, m, v, torch.zeros(1, dtype=torch.int64, device="cuda"), weight_decay=0.1)
    want, plan = plan_of(make(1))
    for k in range(1, 5):
        plan.set_grads(make(k))
        for _ in range(10):
            plan.step(1e-2)
    side = torch.cuda.Stream()
    p, plan = plan_of(make(1))
    torch.cuda.synchronize()
    for k in range(1, 5):
        grads = make(k)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            plan.set_grads(grads)   # the ones before are no one's from here on
            for _ in range(10):
                plan.step(1e-2)
        del grads
        junk = refill(sizes, 1e3)
    del plan
    junk = refill(sizes, 1e3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p, want))
    del junk


def test_captured_gradients_live_as_long_as_the_plan():
    """Until the graph runs the table holds the gradients from before, and each replay sets the captured ones."""
    import gc
    import weakref
    n = 3000
    first, second, third = ([torch.randn(n, generator=gen(k), device="cuda")] for k in (1, 2, 3))
    values = [x[0].clone() for x in (first, second, third)]
    a, b = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    plans, grad = [], torch.zeros(n, device="cuda")
    for p, g in ((a, first), (b, [grad])):
        m, v = ops.adamw_state(p)
        plans.append(ops.AdamW([p], g, [m], [v], torch.zeros(1, dtype=torch.int64, device="cuda")))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plans[0].set_grads(second)
        plans[0].step(1e-2)
    alive = [weakref.ref(x[0]) for x in (first, second)]
    del first, second
    gc.collect()
    assert all(r() is not None for r in alive)

    def same(k):
        grad.copy_(values[k])
        plans[1].step(1e-2)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    plans[0].step(1e-2)      # not replayed yet: the first
    same(0)
    graph.replay()           # the second
    same(1)
    plans[0].set_grads(third)
    gc.collect()
    plans[0].step(1e-2)
    same(2)
    graph.replay()           # the second again, and from there on
    same(1)
    plans[0].step(1e-2)
    same(1)
    assert all(r() is not None for r in alive)
    torch.cuda.synchronize()
    plans[0].close()
    gc.collect()
    assert all(r() is None for r in alive)
