"""A sharded training step refuses what it refuses before its first collective."""
import pytest
import torch

import msccl_amd as M
from msccl_amd import ops

pytestmark = pytest.mark.gpu


class Ranks:
    def __init__(self, comms, dtype=torch.bfloat16, block=512):
        n = len(comms)
        self.comms, self.block = comms, block
        self.params = [torch.ones(n * block, dtype=dtype, device="cuda") for _ in range(n)]
        self.grads = [torch.ones(n * block, dtype=dtype, device="cuda") for _ in range(n)]
        self.shards = [torch.zeros(block, dtype=dtype, device="cuda") for _ in range(n)]
        self.plans, self.sums, self.state = [], [], []
        for r in range(n):
            plan, state = self.plan(r, self.params[r][r * block:(r + 1) * block], self.shards[r])
            self.plans.append(plan)
            self.state += state
            self.sums.append(ops.SquareSum([self.shards[r]]))

    def plan(self, r, p, g):
        m, v = ops.adamw_state(p)
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        return ops.AdamW([p], [g], [m], [v], step), [m, v, step]

    def go(self, **kw):
        args = dict(comms=self.comms, grads=self.grads, shards=self.shards, params=self.params, plans=self.plans, sums=self.sums, lr=1e-2)
        return ops.sharded_step(**(args | kw))


def test_nothing_has_run_when_a_step_is_refused(monkeypatch):
    comms = M.Comm.init_all([0, 0])
    try:
        k = Ranks(comms)
        lr = torch.full((1,), 1e-2, device="cuda")
        closed, _ = k.plan(1, k.params[1][512:], k.shards[1])
        closed.close()
        gone = ops.SquareSum([k.shards[1]])
        gone.close()
        half = k.shards[1].view(torch.float16)
        other_type, keep = k.plan(1, k.params[1][512:], half)
        other_weights, also = k.plan(1, k.params[1][512:].view(torch.float16), k.shards[1])
        called = []
        for name in ("reduce_scatter", "all_reduce", "all_gather"):
            real = getattr(M.Comm, name)
            monkeypatch.setattr(M.Comm, name, lambda *a, _r=real, _n=name, **kw: (called.append(_n), _r(*a, **kw))[1])
        bad = [dict(lr=[1e-2]), dict(lr=[lr] * 3), dict(lr=float("nan")), dict(lr=[1e-2, float("inf")]), dict(lr=lr.double()), dict(lr=[lr, lr.cpu()]),
               dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=-1.0), dict(max_norm=0.0), dict(max_norm=-1.0),
               dict(max_norm=float("nan")), dict(plans=[k.plans[0], closed]), dict(sums=[k.sums[0], gone]),
               dict(plans=[k.plans[0], other_type]), dict(sums=[k.sums[0], ops.SquareSum([half])]),
               dict(plans=[k.plans[0], other_weights])]
        old = [t.clone() for t in k.shards + k.params + k.state]
        for kw in bad:
            with pytest.raises((ValueError, TypeError, ops.NcclError)):
                k.go(**kw)
            torch.cuda.synchronize()
            assert called == [] and all(torch.equal(a, b) for a, b in zip(old, k.shards + k.params + k.state)), kw
        for kw in (dict(), dict(lr=[1e-2, 2e-2]), dict(lr=lr), dict(lr=(lr, lr), max_norm=1.0)):
            k.go(**kw)
        torch.cuda.synchronize()
        assert called == ["reduce_scatter", "reduce_scatter", "all_reduce", "all_reduce", "all_gather", "all_gather"] * 4
        assert [int(k.state[i]) for i in (2, 5)] == [4, 4] and torch.equal(k.params[0], k.params[1])
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def test_a_sharded_run_with_8_bit_states():
    """The documented chain (8-bit states rounded by chance, a 32-bit copy, clipping) against the same steps one
    by one: the shards' plans alone, fed with what the collectives should bring."""
    BF16 = torch.bfloat16
    n, block, sizes = 2, 4352, [1000, 3, 517, 2049]
    spans, at = [], 0
    for k in sizes:
        spans.append((at, k))
        at += -(-k // 256) * 256
    cut = lambda t: [t[a:a + k] for a, k in spans]  # noqa: E731
    start = torch.randn(n * block, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(BF16)

    def make(r, whole, shard):
        p = cut(whole[r * block:(r + 1) * block])
        w = [x.float() for x in p]
        m, v, ms, vs = zip(*[ops.adamw_state(x, bits=8) for x in p])
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        plan = ops.AdamW(p, cut(shard), m, v, step, masters=w, exp_avg_scales=ms, exp_avg_sq_scales=vs, weight_decay=[0.1, 0.0, 0.1, 0.0],
                         rounding="stochastic", seed=1)
        return plan, ops.SquareSum(cut(shard)), [step, *w, *m, *v, *ms, *vs]
    comms = M.Comm.init_all([0] * n)
    try:
        params = [start.clone() for _ in range(n)]
        shards = [torch.zeros(block, dtype=BF16, device="cuda") for _ in range(n)]
        plans, sums, states = (list(x) for x in zip(*[make(r, params[r], shards[r]) for r in range(n)]))
        alone = start.clone()
        parts = [torch.zeros(block, dtype=BF16, device="cuda") for _ in range(n)]
        ours, ourSums, ourStates = (list(x) for x in zip(*[make(r, alone, parts[r]) for r in range(n)]))
        for t in range(40):
            grads = [(torch.randn(n * block, generator=torch.Generator(device="cuda").manual_seed(100 * t + r), device="cuda") * 3).to(BF16)
                     for r in range(n)]
            totals = ops.sharded_step(comms, grads, shards, params, plans, sums, lr=1e-3, betas=(0.9, 0.999), max_norm=1.0)
            both = (grads[0].float() + grads[1].float()).to(BF16)   # added and rounded once
            for r in range(n):
                parts[r].copy_(both[r * block:(r + 1) * block])
            total = ourSums[0]() + ourSums[1]()
            assert all(torch.equal(x, total) for x in totals)
            for p in ours:
                p.step(1e-3, betas=(0.9, 0.999), grad_scale=0.5, grad_square_sum=total, max_norm=1.0)
            torch.cuda.synchronize()
            assert torch.equal(params[0], alone) and torch.equal(params[1], alone), t
            for a, b in zip(states, ourStates):
                assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b)), t
        assert not torch.equal(alone, start)
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def test_a_warning_that_is_an_error_comes_before_the_collectives(monkeypatch):
    import warnings
    comms = M.Comm.init_all([0, 0])
    try:
        k = Ranks(comms)
        plans = []
        for r in range(2):
            p = k.params[r][r * 512:(r + 1) * 512]
            m, v, ms, vs = ops.adamw_state(p, bits=8)
            k.state += [m, v, ms, vs]
            step = torch.zeros(1, dtype=torch.int64, device="cuda")
            plans.append(ops.AdamW([p], [k.shards[r]], [m], [v], step, exp_avg_scales=[ms], exp_avg_sq_scales=[vs]))
        called, real = [], M.Comm.reduce_scatter
        monkeypatch.setattr(M.Comm, "reduce_scatter", lambda *a, **kw: (called.append(1), real(*a, **kw))[1])
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            for _ in range(2):   # each of the plans says it once
                with pytest.raises(UserWarning):
                    k.go(plans=plans)
                assert called == []
            k.go(plans=plans)
        assert len(called) == 2
        torch.cuda.synchronize()
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()
