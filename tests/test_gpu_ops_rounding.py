"""AdamW's states of 8 bits rounded by chance: within a step against the definition, and over many steps
against the states in 64 bits."""
import math
import warnings

import pytest
import torch

from msccl_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Steps:
    """One tensor of n values with states of 8 bits, and its averages in 64 bits."""

    def __init__(self, n, param=F32, grad=F32, master=False, seed=1, rounding="stochastic", pieces=1):
        w = torch.randn(n, generator=gen(0), device="cuda")
        self.w = [x.clone() for x in w.tensor_split(pieces)]
        self.p = [x.to(param) for x in self.w]
        self.g = [torch.zeros(x.numel(), dtype=grad, device="cuda") for x in self.w]
        self.s = [ops.adamw_state(x, bits=8) for x in self.w]
        self.step = torch.zeros(1, dtype=torch.int64, device="cuda")
        m, v, ms, vs = (list(x) for x in zip(*self.s))
        self.plan = ops.AdamW(self.p, self.g, m, v, self.step, masters=self.w if master else None, exp_avg_scales=ms,
                              exp_avg_sq_scales=vs, rounding=rounding, seed=seed)
        self.m = torch.zeros(n, dtype=torch.float64, device="cuda")
        self.v = torch.zeros(n, dtype=torch.float64, device="cuda")

    def go(self, g, betas, lr=1e-4):
        at = 0
        for x in self.g:
            x.copy_(g[at:at + x.numel()])
            at += x.numel()
        self.plan.step(lr, betas=betas)
        g = torch.cat(self.g).double()
        self.m.mul_(betas[0]).add_(g, alpha=1 - betas[0])
        self.v.mul_(betas[1]).addcmul_(g, g, value=1 - betas[1])

    def got(self):
        return (torch.cat([ops.dequantize_state(s[0], s[2]) for s in self.s]).double(),
                torch.cat([ops.dequantize_state(s[1], s[3], second=True) for s in self.s]).double())

    def bits(self):
        return [t.view(torch.uint8).clone() for t in self.p + self.w + [x for s in self.s for x in s]]


KINDS = [(F32, F32, False), (BF16, BF16, False), (F16, BF16, True), (BF16, F32, True), (F16, F16, False)]


@pytest.mark.parametrize("param,grad,master", KINDS)
@pytest.mark.parametrize("runs", [5, 4096])   # one launch, two
def test_a_rounding_is_right_in_the_mean(param, grad, master, runs):
    """Every run the same 256 gradients, of sizes 2^20 apart: each code is one of the two next to its value,
    and over the runs their mean (of squares for v) is the value."""
    k = Steps(256 * runs, param, grad, master)
    size = torch.exp2(torch.linspace(-14, 6, 256, device="cuda")) * (1 + 0.3 * torch.rand(256, generator=gen(3), device="cuda"))
    sign = torch.where(torch.rand(256, generator=gen(4), device="cuda") < 0.5, -1.0, 1.0)
    k.go((size * sign).repeat(runs), (0.9, 0.999))
    m, v = (x.reshape(runs, 256) for x in k.got())
    for got, want, scale in ((m, k.m, k.s[0][2]), (v.sqrt(), k.v.sqrt(), k.s[0][3])):
        want = want.reshape(runs, 256)[0]
        unit = float(scale[0])
        # the codes' step at the value: 2^-3 of its power of two, 2^-9 of the unit at least
        step = torch.exp2(torch.floor(torch.log2(want.abs() / unit).clamp_min(-6.0)) - 3) * unit
        low = got.abs().amin(0)
        high = got.abs().amax(0)
        # (the value itself is off by 16 roundings, which may move it over a code)
        near = want.abs() * 16 * U
        root = got is not m
        if root:   # no second moment above zero has the zero code
            want = want.clamp_min(2.0 ** -9 * unit)
            assert bool((low > 0).all())
        assert bool((high <= want.abs() + step + near).all()) and bool((low >= want.abs() - step - near).all())
        assert runs < 100 or int((high > low).sum()) > 200   # (the codes differ from run to run)
        # Hoeffding: the mean of `runs` independent values from an interval of width a is further than
        # a sqrt(ln(2 / q) / (2 runs)) off with probability q; 512 means, q = 1e-12
        far = math.sqrt(math.log(2 / 1e-12) / (2 * runs))
        if root:
            width = (want + step) ** 2 - (want - step).clamp_min(0) ** 2
            off = ((got ** 2).mean(0) - want ** 2).abs()
            assert bool((off <= width / 2 * far + want ** 2 * 40 * U + step * near).all())
        else:
            off = (got * sign.double()).mean(0) - want.abs()
            assert bool((off.abs() <= step * far + near).all())


def grads_ramp(t, steps, n, noise=None):
    """One element of each run grows fivefold, the others stay."""
    g = torch.ones(n, device="cuda")
    g[::256] = 1.0 + 4.0 * min(1.0, 1.2 * t / steps)
    return g


def grads_turn(t, steps, n, noise):
    """Random gradients, of which a quarter falls to a quarter after a fifth of the steps and another rises fourfold."""
    size = torch.ones(256, device="cuda")
    if 5 * t > steps:
        size[:64], size[64:128] = 0.25, 4.0
    return torch.randn(n, generator=noise, device="cuda") * size.repeat(n // 256)


@pytest.mark.parametrize("grads", [grads_ramp, grads_turn])
@pytest.mark.parametrize("betas,steps", [((0.9, 0.95), 600), ((0.9, 0.999), 5000), ((0.97, 0.99), 2000)])
def test_averages_over_many_steps(grads, betas, steps):
    """Against the averages in 64 bits.  The roundings are right in the mean and the averages linear in what
    was rounded, so the mean over elements of state / average is one, but for the sample's own spread; of a
    run's largest element the scale holds all digits."""
    n = 256 * 128
    k = Steps(n, BF16, F32, True)
    noise = gen(77)
    for t in range(steps):
        k.go(grads(t, steps, n, noise), betas, lr=1e-6)
    m, v = k.got()
    ratio = (v / k.v).reshape(-1, 256)
    for part in (slice(1, 64), slice(64, 128), slice(128, 256)):
        x = ratio[:, part].reshape(-1)
        spread = float(x.std())
        # one standard deviation: the random walk of codes 1/16 to 1/8 apart against the averages' pull,
        # (1/2 to 1/4 of a code's step in the root)
        assert spread < 0.6, (part, spread)
        assert abs(float(x.mean()) - 1) <= 6 * spread / math.sqrt(x.numel()) + 1e-4, (part, float(x.mean()), spread)
    # m: the difference, in units of the run's own size
    size = k.v.sqrt().reshape(-1, 256)
    off = ((m - k.m).reshape(-1, 256) / size)[:, 1:].reshape(-1)
    assert float(off.std()) < 0.3 and abs(float(off.mean())) <= 6 * float(off.std()) / math.sqrt(off.numel()) + 1e-5


def test_weights_follow_those_of_32_bit_states():
    """Where a neighbour grows, the other weights step as far as with 32-bit states (to nearest: a fifth of it)."""
    n, steps = 256 * 16, 4000
    a = Steps(n, F32, F32)
    p = a.w[0].clone()
    m, v = ops.adamw_state(p)
    grad, step = a.g[0], torch.zeros(1, dtype=torch.int64, device="cuda")
    b = ops.AdamW([p], [grad], [m], [v], step)
    start = p.clone()
    for t in range(steps):
        if t == steps - 500:
            before, also = a.p[0].clone(), p.clone()
        a.go(grads_ramp(t, steps, n), (0.9, 0.999))
        b.step(1e-4)
    moved = ((a.p[0] - before) / (p - also)).reshape(-1, 256)[:, 1:].double()
    # the mean step: 1 / sqrt(v) of a v spread by s has 3 / 8 s^2 more; s < 0.3 with equal gradients, and m's own spread averages out
    assert abs(float(moved.mean()) - 1) < 0.04 and not torch.equal(start, p)


def test_same_bits_again_and_other_seeds():
    kinds = [dict(seed=3), dict(seed=3), dict(seed=4), dict(seed=(1 << 64) - 1)]
    for n, pieces in ((5000, 3), (3_000_001, 7)):
        many = [Steps(n, BF16, BF16, False, pieces=pieces, **kw) for kw in kinds]
        g = torch.randn(n, generator=gen(5), device="cuda")
        for t in range(3):
            for k in many:
                k.go(g * (1 + t), (0.9, 0.999))
        bits = [k.bits() for k in many]
        same = [all(torch.equal(x, y) for x, y in zip(bits[0], b)) for b in bits]
        assert same == [True, True, False, False]


def test_steps_and_neighbours_throw_their_own_dice():
    """Two elements, or one in two steps, go the same way half the time."""
    n = 256 * 4096
    k = Steps(n, F32, F32)
    codes = []
    for t in range(3):
        for s in k.s:
            for x in s:
                x.view(torch.uint8).zero_()
        k.step.fill_(t)
        g = torch.ones(n, device="cuda")
        g[1::2] = 1.3171   # m and sqrt(v) between two codes of the unit that the run's largest sets
        g[::256] = 7.0
        k.go(g, (0.9, 0.999))
        v = k.s[0][1].view(torch.uint8).reshape(-1, 256)[:, 1:].to(torch.int32)
        m = k.s[0][0].view(torch.uint8).reshape(-1, 256)[:, 1:].to(torch.int32)
        odd = v[:, ::2]
        codes.append((odd - odd.min()).double() - (odd - odd.min()).double().mean())
        one = m[:, ::2]
        codes.append((one - one.min()).double() - (one - one.min()).double().mean())
    assert all(float(c.std()) > 0.1 for c in codes)
    corr = lambda a, b: float((a * b).mean() / (a.std() * b.std()))  # noqa: E731
    limit = 6 / math.sqrt(codes[0].numel())   # of independent ones the correlation's deviation is one over that root
    for i in range(len(codes)):
        for j in range(i):
            assert abs(corr(codes[i], codes[j])) < limit, (i, j)
        for d in (1, 2, 3, 4, 8, 32, 64):
            assert abs(corr(codes[i][:, d:], codes[i][:, :-d])) < 4 * limit, (i, d)
        assert abs(corr(codes[i][1:], codes[i][:-1])) < limit and abs(corr(codes[i][8:], codes[i][:-8])) < limit


def test_captured_steps_are_the_eager_ones():
    a, b = (Steps(70_000, BF16, BF16, True, pieces=4) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.plan.step(1e-3, betas=(0.9, 0.999))
    for t in range(4):
        for x, y in zip(a.g, b.g):
            x.copy_(torch.randn(x.numel(), generator=gen(t), device="cuda"))
            y.copy_(x)
        graph.replay()
        b.plan.step(1e-3, betas=(0.9, 0.999))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a.bits(), b.bits())) and int(a.step) == t + 1


def test_runs_of_zeros_ends_and_values_that_are_not_finite():
    k = Steps(1000, F32, F32)
    g = torch.zeros(1000, device="cuda")
    k.go(g, (0.9, 0.999))
    m, v = k.got()
    assert float(m.abs().max()) == 0 and float(v.abs().max()) == 0
    g[999], g[300], g[0] = 3.0, float("nan"), -2.0
    k.go(g, (0.9, 0.999))
    m, v = k.got()
    assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
    for i in (0, 999):   # the largest of its run is exact, and nothing beside it
        assert abs(float(m[i] - k.m[i])) <= 6 * U * abs(float(k.m[i])) and abs(float(v[i] - k.v[i])) <= 12 * U * float(k.v[i])
    rest = torch.ones(1000, dtype=torch.bool, device="cuda")
    rest[256:512] = False
    rest[0] = rest[999] = False
    assert float(m[rest].abs().max()) == 0 and float(v[rest].abs().max()) == 0


def test_refusals_and_the_warning():
    x = torch.ones(10, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    m, v, ms, vs = ops.adamw_state(x, bits=8)
    make = lambda **kw: ops.AdamW([x], [x.clone()], [m], [v], step, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], **kw)  # noqa: E731
    for kw in (dict(rounding="up"), dict(rounding="stochastic", seed=-1), dict(rounding="stochastic", seed=1 << 64)):
        with pytest.raises(ValueError):
            make(**kw)
    m32, v32 = ops.adamw_state(x)
    with pytest.raises(ValueError):
        ops.AdamW([x], [x.clone()], [m32], [v32], step, rounding="stochastic")
    plan = ops.AdamW([x], [x.clone()], [m32], [v32], step, rounding="nearest")
    assert ops._lib().mscclAmdAdamWSetRounding(plan.handle, 1, 0) == 4
    plan = make()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        plan.step(1e-3, betas=(0.9, 0.9))          # (its averages move by more than half a code's step)
        make(rounding="nearest").step(1e-3)
        make(rounding="stochastic").step(1e-3)
        with pytest.raises(UserWarning):
            plan.step(1e-3)
        plan.step(1e-3)                             # said once
