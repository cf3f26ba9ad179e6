"""The training-step operators (msccl_amd/ops.py) against their definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of a 32-bit value; a value stored in 16 bits is off
by half a step more, HALF[type] of its size (float16 also by half its smallest step, 2^-25)."""
import math

import pytest
import torch

from msccl_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E4M3 = torch.float8_e4m3fn
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, want, bound, what):
    """Every element within its bound; what is not finite in one is the same in the other."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(torch.isnan(want), torch.isnan(got)), what
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()), float((got - want).abs()[fine].max()))


def carve(sizes, dtype, odd, fill=0.0):
    """Tensors of these sizes in one buffer, apart from each other, `odd` elements off 16-byte boundaries,
    and the buffer."""
    at, spans = 16, []
    for n in sizes:
        spans.append((at + odd, n))
        at += -(-(n + odd) // 16) * 16 + 16
    buf = torch.full((at + 32,), fill, dtype=F32, device="cuda").to(dtype)
    return [buf[a:a + n] for a, n in spans], buf, spans


def between(buf, spans):
    """What lies in the buffer beside the tensors."""
    keep = torch.ones(buf.numel(), dtype=torch.bool, device="cuda")
    for a, n in spans:
        keep[a:a + n] = False
    return buf.view(torch.uint8).reshape(buf.numel(), -1)[keep]


# ---- square sum ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,odd", [([1], 0), ([0], 0), ([7, 0, 9], 1), ([2048], 0), ([2049, 2047], 3), ([8191, 1, 0, 0, 4099], 5),
                                       ([1] * 70, 1), ([300] * 4100, 0), ([5_000_003, 17], 1)])
def test_square_sum(dtype, sizes, odd):
    ts, buf, _ = carve(sizes, dtype, odd, fill=3.0)
    g = gen(7)
    for t in ts:
        t.copy_(torch.randn(t.numel(), generator=g, device="cuda") * 3)
    plan = ops.SquareSum(ts)
    got = plan()
    want = sum(t.double().square().sum() for t in ts)
    # products of 24-bit values are exact in 53 bits; each of at most n positive additions is off by 2^-53
    assert abs(float(got) - float(want)) <= float(want) * sum(sizes) * 2 * 2.0 ** -53
    assert torch.equal(plan(), got)   # the same bits again


def test_square_sum_range_and_non_finite():
    x = torch.full((5000,), 1e30, device="cuda")
    plan = ops.SquareSum([x])
    one = float(x[0].double()) ** 2
    assert abs(float(plan()) - 5000 * one) <= 5000 * one * 5000 * 2.0 ** -52
    for bad, check in ((float("inf"), math.isinf), (float("nan"), math.isnan)):
        x[4999] = bad
        assert check(float(plan()))


def test_square_sum_streams_out_and_graph():
    xs = [torch.randn(n, generator=gen(n), device="cuda") for n in (100_000, 3)]
    plan = ops.SquareSum(xs)
    want = plan()
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    assert plan(out=out) is out and torch.equal(out, want)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(side[k % 2]):
            got.append(plan())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = plan()
    for k in range(4):
        xs[0].mul_(0.5)
        graph.replay()
        eager = plan()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)


def test_square_sum_refuses():
    x = torch.ones(8, device="cuda")
    with pytest.raises(TypeError):
        ops.SquareSum([x, x.bfloat16()])
    with pytest.raises(TypeError):
        ops.SquareSum([x.double()])
    with pytest.raises(ValueError):
        ops.SquareSum([torch.ones(4, 4, device="cuda").t()[:, :2]])
    plan = ops.SquareSum([x])
    with pytest.raises(TypeError):
        plan(out=torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.SquareSum([x])
    torch.cuda.synchronize()
    plan.close()
    with pytest.raises(ValueError):
        plan()


# ---- AdamW ---------------------------------------------------------------------------------------

class Model:
    """Tensors, states and a plan; `want` makes the next step in 64 bits from what the tensors hold now."""

    def __init__(self, sizes, param=F32, grad=F32, master=False, bits=32, odd=0, seed=1, t0=0, decay=0.1, rate=1.0, spread=1.0):
        g = gen(seed)
        rand = lambda n, s: torch.randn(n, generator=g, device="cuda") * s  # noqa: E731
        self.sizes, self.bits, self.param, self.bufs = sizes, bits, param, {}

        def make(name, dtype, per=1):
            ts, buf, spans = carve([-(-n // per) for n in sizes], dtype, odd, fill=2.0)
            self.bufs[name] = (buf, spans, between(buf, spans).clone())
            return ts
        self.p = make("param", param)
        self.g = make("grad", grad)
        self.w = make("master", F32) if master else None
        if bits == 32:
            self.m, self.v, self.ms, self.vs = make("m", F32), make("v", F32), None, None
        else:
            self.m, self.v = make("m", E4M3), make("v", E4M3)
            self.ms, self.vs = make("ms", F32, 256), make("vs", F32, 256)
        for i, n in enumerate(sizes):
            w = rand(n, 0.5)
            self.p[i].copy_(w)
            if master:
                self.w[i].copy_(w)
            for x in (self.m, self.v, self.ms, self.vs):
                if x is not None:
                    x[i].view(torch.uint8).zero_()
        self.rand, self.spread = rand, spread
        self.new_grads()
        self.step = torch.full((1,), t0, dtype=torch.int64, device="cuda")
        k = len(sizes)
        self.decay = decay if isinstance(decay, list) else [decay] * k
        self.rate = rate if isinstance(rate, list) else [rate] * k
        self.plan = ops.AdamW(self.p, self.g, self.m, self.v, self.step, masters=self.w, exp_avg_scales=self.ms,
                              exp_avg_sq_scales=self.vs, weight_decay=decay, lr_scale=rate)

    def new_grads(self):
        for t in self.g:
            t.copy_(self.rand(t.numel(), 1.0) * torch.exp(self.rand(t.numel(), self.spread)) * 1e-2)

    def tensors(self):
        return [t for ts in (self.p, self.w, self.m, self.v, self.ms, self.vs) if ts is not None for t in ts] + [self.step]

    def copy(self):
        return [t.clone() for t in self.tensors()]

    def same(self, old):
        return all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(self.tensors(), old))

    def want(self, lr, betas, eps, c=1.0):
        b1, b2 = betas
        t = int(self.step) + 1
        out = []
        for i, n in enumerate(self.sizes):
            g = self.g[i].double() * c
            p = (self.p if self.w is None else self.w)[i].double()
            if self.bits == 32:
                m, v = self.m[i].double(), self.v[i].double()
            else:
                spread = lambda s: s.double().repeat_interleave(256)[:n]  # noqa: E731
                m = self.m[i].double() * spread(self.ms[i])
                v = (self.v[i].double() * spread(self.vs[i])) ** 2
            size = b1 * m.abs() + (1 - b1) * g.abs()
            m = b1 * m + (1 - b1) * g
            v = b2 * v + (1 - b2) * g * g
            den = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
            rate = lr * self.rate[i] / (1 - b1 ** t)
            keep = 1 - lr * self.rate[i] * self.decay[i]
            up = rate * m / den
            p2 = p * keep - up
            # roundings (u each).  m: c, g c, 1 - b1, the product, the sum on g; b1, decoding, the product,
            # the sum on m.  v: twice c and g c, the square, 1 - b2, product, sum on g^2; b2, decoding twice, the square,
            # product, sum on v.  sqrt(v): half of v's and 2 of its own; times invRoot (2), plus eps (1): 9.
            # the step: rate, the quotient (2), the product and those 9, with m's own; p: keep, product, sum
            em = 6 * U * size + 2.0 ** -148
            ev = 9 * U * v + 2.0 ** -148
            ep = (4 * U) * (p * keep).abs() + 16 * U * up.abs() + abs(rate) / den * em
            out.append({"m": m, "v": v, "p": p2, "em": em, "ev": ev, "ep": ep})
        return out

    def check(self, want, t):
        assert int(self.step) == t
        for i, w in enumerate(want):
            if self.w is not None:
                close(self.w[i], w["p"], w["ep"], "master %d" % i)
                assert torch.equal(self.p[i], self.w[i].to(self.param)), "param %d is its copy rounded" % i
            else:
                close(self.p[i], w["p"], w["ep"] + (HALF[self.param] * w["p"].abs() + TINY[self.param] if self.param != F32 else 0), "param %d" % i)
            if self.bits == 32:
                close(self.m[i], w["m"], w["em"], "m %d" % i)
                close(self.v[i], w["v"], w["ev"], "v %d" % i)
                continue
            n = self.sizes[i]
            for code, scale, x, ex, floor in ((self.m[i], self.ms[i], w["m"], w["em"], False),
                                              (self.v[i], self.vs[i], w["v"].sqrt(), 7 * U * w["v"].sqrt(), True)):
                pad = torch.zeros(-(-n // 256) * 256 - n, dtype=torch.float64, device="cuda")
                runs = torch.cat([x, pad]).reshape(-1, 256)
                top = runs.abs().amax(1) / 448
                etop = torch.cat([ex, pad]).reshape(-1, 256).amax(1) / 448
                # the largest of values that are each off by ex, times 1 / 448 (2 roundings)
                close(scale, top, etop + 3 * U * top, "scale %d" % i)
                s = scale.double().repeat_interleave(256)[:n]
                value = code.double() * s
                # half a step: 2^-4 of the value, or 2^-10 of the scale under the smallest normal code; the
                # scale's own error and that of the quotient (4 roundings) move a value by as much
                bound = (2.0 ** -4 * x.abs()).maximum(2.0 ** -10 * s) * (1 + 1e-6) + ex + x.abs() * 6 * U + 450 * etop.repeat_interleave(256)[:n]
                if floor:   # a value above zero has at least the smallest code
                    bound = bound.maximum(torch.where((x > 0) & (x < 2.0 ** -9 * s), 2.0 ** -9 * s - x, 0.0) * (1 + 1e-6))
                    assert bool(((value > 0) | (x == 0)).all())
                close(value, x, bound, "codes %d" % i)
        for name, (buf, spans, old) in self.bufs.items():
            assert torch.equal(between(buf, spans), old), "%s: written beside the tensors" % name


SIZES = [1, 7, 8, 255, 256, 257, 0, 2047, 2048, 2049, 6151]
TYPES = [(F32, F32, False), (F32, BF16, False), (F32, F16, False), (BF16, BF16, True), (BF16, BF16, False), (BF16, F32, True),
         (BF16, F32, False), (F16, F16, True), (F16, F16, False), (F16, BF16, True), (F16, F32, False), (BF16, F16, True),
         (BF16, F16, False), (F16, BF16, False), (F16, F32, True)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,master", TYPES)
def test_adamw_types(param, grad, master, bits):
    k = Model(SIZES, param, grad, master, bits, decay=[0.1 * (i % 3) for i in range(len(SIZES))],
              rate=[1.0 + 0.5 * (i % 2) for i in range(len(SIZES))], odd=0)
    for t in range(1, 4):
        want = k.want(1e-2, (0.9, 0.99), 1e-8)
        k.plan.step(1e-2, betas=(0.9, 0.99), eps=1e-8)
        k.check(want, t)
        k.new_grads()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("odd", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("param,grad,master", [(F32, F32, False), (BF16, F16, True), (F16, BF16, False)])
def test_adamw_tensors_that_start_anywhere(param, grad, master, odd, bits):
    k = Model(SIZES, param, grad, master, bits, odd=odd)
    for t in range(1, 3):
        want = k.want(1e-2, (0.9, 0.999), 1e-8)
        k.plan.step(1e-2)
        k.check(want, t)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count,size", [(65, 3), (64, 2049), (5000, 1), (4097, 300)])
def test_adamw_many_tensors(count, size, bits):
    k = Model([size + i % 3 for i in range(count)], bits=bits, decay=[0.01 * (i % 7) for i in range(count)])
    flat = lambda ts: torch.cat([t.reshape(-1) for t in ts])  # noqa: E731
    want = k.want(1e-2, (0.9, 0.999), 1e-8)
    k.plan.step(1e-2)
    close(flat(k.p), flat([w["p"] for w in want]), flat([w["ep"] for w in want]), "params")
    assert int(k.step) == 1


@pytest.mark.parametrize("chunks", [31, 32, 33, 500, 2100])
def test_adamw_on_both_sides_of_one_launch(chunks):
    for bits in (32, 8):
        k = Model([2048 * chunks - 5], BF16, BF16, False, bits)
        for t in range(1, 4):
            want = k.want(1e-2, (0.9, 0.999), 1e-8)
            k.plan.step(1e-2)
            k.check(want, t)


def test_offsets_past_32_bits():
    """4.3 billion elements in one tensor: what lies behind the 2^32nd is stepped and summed like the rest."""
    n, tail = (1 << 32) + 5003, 5000
    grad = torch.zeros(n, dtype=BF16, device="cuda")
    param = torch.ones(n, dtype=BF16, device="cuda")
    m, v, ms, vs = ops.adamw_state(param, bits=8)
    grad[-tail:] = torch.randn(tail, generator=gen(1), device="cuda").to(BF16)
    grad[:3] = 2.0
    total = ops.SquareSum([grad])()
    want = float(grad[-tail:].double().square().sum()) + 12.0
    assert abs(float(total) - want) <= want * n * 2.0 ** -52
    small = Model([tail], BF16, BF16, False, 32, decay=0.0)
    small.p[0].copy_(param[-tail:])
    small.g[0].copy_(grad[-tail:])
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.AdamW([param], [grad], [m], [v], step, exp_avg_scales=[ms], exp_avg_sq_scales=[vs]).step(1e-2)
    small.plan.step(1e-2)
    assert torch.equal(param[-tail:], small.p[0]) and int(step) == 1
    assert bool((param[:3] < 1).all()) and bool((param[3:-tail] == 1).all())
    first = (n - tail) // 256   # the first run that the tail reaches
    got = ops.dequantize_state(m[first * 256:], ms[first:])[n - tail - first * 256:].double()
    exact = small.g[0].double() * 0.1
    # half a step of e4m3 (2^-4, or 2^-10 of the scale, itself the run's largest / 448) and its 6 roundings
    near = ms[first:].double().repeat_interleave(256)[n - tail - first * 256:][:tail]
    assert bool(((got - exact).abs() <= (2.0 ** -4 * exact.abs()).maximum(2.0 ** -10 * near) * (1 + 1e-5)).all())
    assert int((ms != 0).sum()) <= tail // 256 + 3


def test_adamw_large_tensor_and_step_count():
    k = Model([5_000_011], BF16, BF16, True, 32, t0=123_456)
    want = k.want(1e-3, (0.9, 0.999), 1e-8)
    k.plan.step(1e-3)
    k.check(want, 123_457)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_8bit_wide_range_within_a_run(bits):
    # gradients that differ by ten orders of magnitude within 256 neighbours, and exact zeros
    k = Model([4096], bits=bits, spread=6.0)
    for t in range(1, 4):
        k.g[0][::5] = 0
        want = k.want(1e-2, (0.9, 0.99), 1e-8)
        k.plan.step(1e-2, betas=(0.9, 0.99))
        k.check(want, t)
        k.new_grads()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_clip_scale_and_total(bits):
    k = Model([3000, 17], BF16, BF16, True, bits)
    sums = ops.SquareSum(k.g)
    for t, (scale, limit) in enumerate([(1.0, 1e-2), (0.125, 1e3), (0.125, 1e-3), (4.0, None)], 1):
        total = sums()
        norm = scale * math.sqrt(float(total))
        c = scale * (1.0 if limit is None else min(1.0, limit / (norm + 1e-6)))
        want = k.want(1e-2, (0.9, 0.999), 1e-8, c)
        k.plan.step(1e-2, grad_scale=scale, grad_square_sum=total, max_norm=limit)
        k.check(want, t)
        k.new_grads()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_adamw_leaves_everything_where_the_total_is_not_finite(bits, bad):
    k = Model([3000, 17], BF16, F16, True, bits)
    k.plan.step(1e-2)
    old = k.copy()
    k.g[0][2999] = bad
    total = ops.SquareSum(k.g)()
    k.plan.step(1e-2, grad_square_sum=total, max_norm=1.0)
    k.plan.step(1e-2, grad_square_sum=total)
    assert k.same(old)
    k.g[0][2999] = 1.0
    want = k.want(1e-2, (0.9, 0.999), 1e-8)
    k.plan.step(1e-2, grad_square_sum=ops.SquareSum(k.g)())
    k.check(want, 2)


def test_adamw_8bit_run_with_nan_and_its_neighbours():
    k = Model([1024], bits=8)
    k.plan.step(1e-2)
    k.g[0][300] = float("nan")
    k.g[0][600] = float("inf")
    before = k.p[0].clone()
    k.plan.step(1e-2)
    m = ops.dequantize_state(k.m[0], k.ms[0])
    v = ops.dequantize_state(k.v[0], k.vs[0], second=True)
    for x in (m, v):
        assert torch.isnan(x[256:768]).all() and torch.isfinite(x[:256]).all() and torch.isfinite(x[768:]).all()
    nan = torch.isnan(k.p[0])
    assert nan.nonzero().flatten().tolist() == [300, 600] and not torch.equal(k.p[0][:256], before[:256])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_zero_gradients_move_weights_by_decay_alone(bits):
    k = Model([777], bits=bits, decay=0.5)
    k.g[0].zero_()
    old = k.p[0].clone()
    k.plan.step(0.1)
    close(k.p[0], old.double() * (1 - 0.05), 3 * U * old.double().abs(), "p")
    assert all(float(t.float().abs().max()) == 0 for t in (k.m[0], k.v[0]))


def test_adamw_device_rate_and_graph():
    a, b = (Model([5000, 33], BF16, BF16, True, bits, seed=5) for bits in (32, 8))
    c, d = (Model([5000, 33], BF16, BF16, True, bits, seed=5) for bits in (32, 8))
    lr = torch.full((1,), 1e-2, device="cuda")
    total = torch.full((1,), 4.0, dtype=torch.float64, device="cuda")
    warm = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    old = a.copy() + b.copy()
    with torch.cuda.graph(graph, stream=warm):
        a.plan.step(lr, max_norm=0.5, grad_square_sum=total)
        b.plan.step(lr, max_norm=0.5, grad_square_sum=total)
    torch.cuda.synchronize()
    assert a.same(old[:len(a.tensors())]) and b.same(old[len(a.tensors()):])   # captured, not run
    for t in range(1, 6):
        lr.fill_(1e-2 / t)
        for x, y in ((a, c), (b, d)):
            for s, r in zip(x.g, y.g):
                s.copy_(torch.randn(s.numel(), generator=gen(t), device="cuda"))
                r.copy_(s)
        graph.replay()
        for y in (c, d):
            y.plan.step(float(lr), max_norm=0.5, grad_square_sum=total)
        torch.cuda.synchronize()
        assert a.same(c.copy()) and b.same(d.copy()) and int(a.step) == t


def test_adamw_set_grads_and_side_stream():
    a, b = Model([3000, 0, 5], seed=3), Model([3000, 0, 5], seed=3)
    other = [torch.randn(g.numel(), generator=gen(9), device="cuda") for g in a.g]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a.plan.step(1e-2)
        a.plan.set_grads(other)
        a.plan.step(1e-2)
    side.synchronize()
    b.plan.step(1e-2)
    for x, y in zip(b.g, other):
        x.copy_(y)
    b.plan.step(1e-2)
    assert a.same(b.copy())


def test_adamw_same_bits_again():
    a, b = (Model(SIZES, BF16, BF16, True, 8, seed=4) for _ in range(2))
    for _ in range(3):
        a.plan.step(1e-2)
        b.plan.step(1e-2)
    assert a.same(b.copy())


def test_adamw_refuses():
    k = Model([10, 20])
    p, g, m, v, s = k.p, k.g, k.m, k.v, k.step
    bad = [dict(grads=g[:1]), dict(grads=[g[0], g[0]]), dict(grads=[g[0], g[1].double()]), dict(grads=[g[0], g[1].bfloat16()]),
           dict(step=s.int()), dict(step=s.cpu()), dict(masters=[x.clone() for x in p]), dict(exp_avg_scales=[s.float()] * 2),
           dict(exp_avgs=[x.to(E4M3) for x in m]), dict(exp_avgs=[x.double() for x in m]), dict(weight_decay=[0.1]),
           dict(params=[p[1][:10], p[1]]), dict(grads=[p[0], g[1]]), dict(exp_avgs=[m[0], v[1]]),
           dict(params=[x.double() for x in p]), dict(lr_scale=[1.0] * 3)]
    for kw in bad:
        args = dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, step=s) | kw
        with pytest.raises((ValueError, TypeError, ops.NcclError)):
            ops.AdamW(**args)
    old = k.copy()
    total = torch.ones(1, dtype=torch.float64, device="cuda")
    for kw in [dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=-1.0), dict(eps=1e-40), dict(grad_scale=1e39),
               dict(eps=float("inf")), dict(grad_scale=0.0), dict(grad_scale=-1.0), dict(grad_scale=float("inf")),
               dict(max_norm=1.0), dict(max_norm=0.0, grad_square_sum=total), dict(max_norm=-1.0, grad_square_sum=total),
               dict(grad_square_sum=total.float()), dict(grad_square_sum=total.cpu()), dict(lr=s)]:
        with pytest.raises((ValueError, TypeError, ops.NcclError)):
            k.plan.step(**(dict(lr=1e-2) | kw))
    with pytest.raises(ValueError):
        k.plan.set_grads(g[:1])
    with pytest.raises(ValueError):
        k.plan.set_grads([g[1], g[0]])
    with pytest.raises(ops.NcclError):
        k.plan.set_grads([g[0], m[1]])
    torch.cuda.synchronize()
    assert k.same(old)
    k.plan.close()
    k.plan.close()
    with pytest.raises(ValueError):
        k.plan.step(1e-2)


# ---- balance loss --------------------------------------------------------------------------------

def scores64(x, score):
    x = x.double()
    if score == "sigmoid":
        z = torch.special.expit(x)
    else:
        top = x.amax(1, keepdim=True)
        z = torch.exp(x - torch.where(torch.isneginf(top), 0.0, top))
    s = z.sum(1, keepdim=True)
    return z, torch.where(s == 0, 0.0, z / s)


def rows_error(x, score):
    """Roundings of a probability, in u.  softmax, of a logit d below its row's largest: 1 d of the
    subtraction and 1.3 d of the product with log2(e) (its rounding and the constant's) in the exponential,
    whose own are 2; the same of the sum's terms, which weigh as p does, and sum p d <= 2 + ln 1024 = 9: 23;
    the sum's 15 additions, the reciprocal's 2 and the product's 1: 2.3 d + 43.  sigmoid: 1.3 |x| + 2 of
    the exponential, 1 of 1 + e, the reciprocal's 2, a product: 1.3 |x| + 6, twice with the sum's terms, its
    15 additions, the quotient and the product's 2: 2.6 |x| + 30."""
    x = x.double()
    fine = torch.where(torch.isfinite(x), x, 0.0)
    if score == "sigmoid":
        return 2.6 * fine.abs().amax(1, keepdim=True) + 30
    return 2.3 * (fine.amax(1, keepdim=True) - fine.amin(1, keepdim=True)) + 43


def router(tokens, experts, k, dtype, masked, seed=3, index=torch.int32, pad=0, scale=2.0):
    g = gen(seed)
    wide = (torch.randn(tokens, experts + pad, generator=g, device="cuda") * scale).to(dtype)
    logits = wide[:, :experts]
    ind = torch.argsort(torch.rand(tokens, experts, generator=g, device="cuda"), dim=1)[:, :k]
    if pad:
        room = torch.full((tokens, k + pad), -7, dtype=index, device="cuda")
        room[:, :k] = ind
        ind = room[:, :k]
    else:
        ind = ind.to(index).contiguous()
    valid = torch.rand(tokens, generator=g, device="cuda") < 0.7 if masked else None
    return logits, ind, valid


def check_stats(logits, ind, valid, score):
    t, e = logits.shape
    counts, probs = ops.balance_stats(logits, ind, valid=valid, score=score)
    here = torch.ones(t, dtype=torch.bool, device="cuda") if valid is None else valid.bool()
    chosen = ind[here].reshape(-1).long()
    chosen = chosen[(chosen >= 0) & (chosen < e)]
    assert torch.equal(counts[:e], torch.bincount(chosen, minlength=e)) and int(counts[e]) == int(here.sum())
    p = scores64(logits[here], score)[1]
    err = rows_error(logits[here], score) if t else 0
    # the sum's own: at most 64 additions in a lane, 16 in a workgroup, one rounding
    close(probs, p.sum(0), (p * (err + 81) * U).sum(0), "probs")
    again = ops.balance_stats(logits, ind, valid=valid, score=score)
    assert torch.equal(again[0], counts) and torch.equal(again[1], probs)
    return counts, probs


SHAPES = [(1, 1, 1), (1, 2, 1), (5, 7, 3), (64, 8, 2), (333, 9, 8), (1025, 16, 4), (700, 17, 2), (257, 60, 4), (4099, 64, 6),
          (130, 100, 3), (999, 128, 8), (65, 200, 5), (3001, 256, 8), (40, 511, 7), (100, 512, 2), (77, 513, 1), (50, 1000, 4),
          (33, 1024, 1024), (20011, 8, 2)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,experts,k", SHAPES)
def test_balance_stats_and_loss(tokens, experts, k, dtype, score):
    for masked, index, pad in ((False, torch.int32, 0), (True, torch.int64, 3)):
        logits, ind, valid = router(tokens, experts, k, dtype, masked, index=index, pad=pad)
        counts, probs = check_stats(logits, ind, valid, score)
        loss = ops.balance_loss(counts, probs, k, 0.25)
        n = int(counts[experts])
        want = 0.25 * experts / (k * n * n) * float((counts[:experts].double() * probs.double()).sum()) if n else 0.0
        assert abs(float(loss) - want) <= 1.01 * U * abs(want)


def check_backward(logits, counts, k, coef, up, valid, score, got, base=None):
    t, e = logits.shape
    n = int(counts[e])
    w = counts[:e].double() * (coef * e / (k * n * n) * up if n else 0.0)
    z, p = scores64(logits, score)
    mean = (p * w).sum(1, keepdim=True)
    d = p * (w - mean)
    size = (p * w.abs()).sum(1, keepdim=True)
    err = rows_error(logits, score)
    # p's roundings on d; w's two and the difference's; the sum's own 17 and those of its terms
    bound = p * U * (err * (w - mean).abs() + 4 * w.abs() + (err + 20) * size)
    if score == "sigmoid":
        d, bound = d * (1 - z), bound * (1 - z) + (d * (1 - z)).abs() * 10 * U
    if valid is not None:   # padded rows, whatever they hold: exact
        d, bound = (torch.where(valid.bool().reshape(-1, 1), x, 0.0) for x in (d, bound))
    if base is not None:
        bound, d = bound + U * (base.double() + d).abs(), base.double() + d
        if valid is not None:
            d = torch.where(valid.bool().reshape(-1, 1), d, base.double())
    dtype = logits.dtype
    close(got, d, bound + (HALF[dtype] * (d.abs() + bound) + TINY[dtype] if dtype != F32 else 2.0 ** -148), "gradient")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,experts,k", SHAPES)
def test_balance_backward(tokens, experts, k, dtype, score):
    for masked, pad in ((False, 0), (True, 5)):
        logits, ind, valid = router(tokens, experts, k, dtype, masked, pad=pad)
        counts, probs = ops.balance_stats(logits, ind, valid=valid, score=score)
        up = torch.tensor([256.0 * tokens], device="cuda")
        got = ops.balance_backward(logits, counts, k, 0.5, grad_output=up, valid=valid, score=score)
        check_backward(logits, counts, k, 0.5, float(up), valid, score, got)
        room = torch.randn(tokens, experts + pad, generator=gen(8), device="cuda").to(dtype)
        out, base = room[:, :experts], room.clone()
        ops.balance_backward(logits, counts, k, 0.5, grad_output=up, valid=valid, score=score, out=out, accumulate=True)
        check_backward(logits, counts, k, 0.5, float(up), valid, score, out, base[:, :experts])
        assert torch.equal(room[:, experts:], base[:, experts:])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_gradient_against_differences(score):
    logits, ind, valid = router(23, 11, 3, F32, True)
    counts, _ = ops.balance_stats(logits, ind, valid=valid, score=score)
    got = ops.balance_backward(logits, counts, 3, 1.0, valid=valid, score=score)
    n = int(counts[11])

    def loss(x):
        p = scores64(x, score)[1][valid]
        return float((counts[:11].double() * p.sum(0)).sum()) * 11 / (3 * n * n)
    h = 1e-4
    x = logits.double()
    for i, j in ((0, 0), (3, 5), (7, 10), (11, 2), (19, 9), (22, 1)):
        up, down = x.clone(), x.clone()
        up[i, j] += h
        down[i, j] -= h
        slope = (loss(up) - loss(down)) / (2 * h)
        # central differences leave h^2 / 6 of the third derivative, at most 6 w here, and 2^-52 of the loss over h;
        # the kernel's own: 200 roundings of terms up to w
        w = float(counts[:11].max()) * 11 / (3 * n * n)
        assert abs(float(got[i, j]) - slope) <= w * (h * h + 200 * U) + loss(x) * 2.0 ** -50 / h


def test_balance_loss_gradient_is_autograds():
    logits, ind, valid = router(50, 12, 3, F32, True)
    counts, _ = ops.balance_stats(logits, ind, valid=valid)
    got = ops.balance_backward(logits, counts, 3, 0.1, valid=valid)
    x = logits.double().cpu().requires_grad_(True)
    c, keep = counts.double().cpu(), valid.cpu()
    p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))[keep]
    (0.1 * 12 / (3 * c[12] ** 2) * (c[:12] * p.sum(0)).sum()).backward()
    w = float(c[:12].max() * 0.1 * 12 / (3 * c[12] ** 2))
    assert float((got.cpu().double() - x.grad).abs().max()) <= 200 * U * w


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_balance_masked_experts_rows_and_garbage(score, dtype):
    logits, ind, valid = router(200, 24, 4, dtype, True)
    valid[5], valid[6], valid[7], valid[8] = True, True, False, False
    logits[:, 3] = float("-inf")         # an expert that is off
    logits[5] = float("-inf")            # a row that leaves nothing
    logits[6, :23] = torch.finfo(dtype).min   # masked with the lowest value
    logits[7] = float("nan")             # padding holds anything
    logits[8] = float("inf")
    ind[7] = 1 << 30
    ind[9, 0], ind[9, 1], ind[10, 2] = -1, 24, ind[10, 1]   # dropped slots, one expert twice
    counts, probs = check_stats(logits, ind, valid, score)
    assert float(probs[3]) == 0 and torch.isfinite(probs).all()
    got = ops.balance_backward(logits, counts, 4, valid=valid, score=score, grad_output=torch.full((1,), 100.0, device="cuda"))
    assert torch.isfinite(got).all() and float(got[5].abs().max()) == 0 and float(got[:, 3].abs().max()) == 0
    assert float(got[7].abs().max()) == 0 and float(got[8].abs().max()) == 0
    rest = torch.ones(200, dtype=torch.bool, device="cuda")
    rest[6] = False   # (its lowest value would spoil the bound of the row's spread)
    check_backward(logits[rest], counts, 4, 1.0, 100.0, valid[rest], score, got[rest])


def test_balance_nan_in_a_valid_row_shows():
    logits, ind, _ = router(20, 8, 2, F32, False)
    logits[3, 2] = float("nan")
    counts, probs = ops.balance_stats(logits, ind)
    assert torch.isnan(probs).all() and int(counts[8]) == 20
    assert torch.isnan(ops.balance_loss(counts, probs, 2)).all()
    got = ops.balance_backward(logits, counts, 2)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[:3]).all() and torch.isfinite(got[4:]).all()


@pytest.mark.parametrize("tokens", [0, 3, 5000])
def test_balance_no_valid_tokens(tokens):
    logits, ind, _ = router(tokens, 32, 2, BF16, False)
    valid = torch.zeros(tokens, dtype=torch.uint8, device="cuda")
    counts, probs = ops.balance_stats(logits, ind, valid=valid)
    assert int(counts.abs().sum()) == 0 and float(probs.abs().sum()) == 0
    assert float(ops.balance_loss(counts, probs, 2)) == 0
    got = ops.balance_backward(logits, counts, 2, valid=valid)
    assert got.shape == logits.shape and float(got.float().abs().sum()) == 0


def test_balance_one_expert_takes_all():
    # 300000 slots on one counter
    logits, ind, _ = router(100_000, 40, 3, BF16, False)
    ind.fill_(17)
    counts, _ = check_stats(logits, ind, None, "softmax")
    assert int(counts[17]) == 300_000


def test_balance_many_rows_a_lane():
    # a lane adds up 300 rows: its sums of 64 rows go on in 64 bits (what the plain bound of 81 counts)
    logits, ind, valid = router(256 * 16 * 300, 500, 2, F16, False)
    check_stats(logits, ind, torch.ones(len(ind), dtype=torch.bool, device="cuda"), "softmax")


def test_plans_on_other_streams_keep_their_tables():
    # a plan that is dropped while another stream still has its calls to make
    x = torch.randn(1 << 22, device="cuda")
    want = ops.SquareSum([x])()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        plan = ops.SquareSum([x])
        with torch.cuda.stream(side):
            for _ in range(50):
                got = plan()
        del plan
        junk = [torch.full((64,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]
        side.synchronize()
        assert torch.equal(got, want)
        del junk


def test_balance_far_rows():
    # rows whose elements lie past 2^31 of the buffer
    rows, stride = 9, (1 << 28) + 8
    buf = torch.zeros(rows * stride, dtype=BF16, device="cuda")
    logits = buf.as_strided((rows, 64), (stride, 1))
    small, ind, _ = router(rows, 64, 4, BF16, False)
    logits.copy_(small)
    counts, probs = ops.balance_stats(logits, ind)
    want = ops.balance_stats(small, ind)
    assert torch.equal(counts, want[0]) and torch.equal(probs, want[1])
    got = ops.balance_backward(logits, counts, 4)
    assert torch.equal(got, ops.balance_backward(small, counts, 4))
    ops.balance_backward(logits, counts, 4, out=logits)   # in place, far too
    assert torch.equal(logits, got) and int((buf != 0).sum()) == int((got != 0).sum())


def test_balance_streams_and_graph():
    logits, ind, valid = router(3000, 64, 4, BF16, True)
    up = torch.full((1,), 1000.0, device="cuda")

    def pass_():
        counts, probs = ops.balance_stats(logits, ind, valid=valid)
        return counts, probs, ops.balance_loss(counts, probs, 4), ops.balance_backward(logits, counts, 4, 1.0, up, valid)
    want = pass_()
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(4):
        with torch.cuda.stream(sides[k % 2]):
            got.append(pass_())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pass_()
    for _ in range(4):
        logits.mul_(0.75)
        graph.replay()
        eager = pass_()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_balance_refuses():
    logits, ind, valid = router(20, 8, 2, F32, True)
    counts, probs = ops.balance_stats(logits, ind)
    with pytest.raises(TypeError):
        ops.balance_stats(logits.double(), ind)
    with pytest.raises(TypeError):
        ops.balance_stats(logits, ind.float())
    with pytest.raises(TypeError):
        ops.balance_stats(logits, ind[:10])
    with pytest.raises(ValueError):
        ops.balance_stats(logits.t(), ind[:8])
    with pytest.raises(ValueError):
        ops.balance_stats(logits, ind.cpu())
    with pytest.raises(ValueError):
        ops.balance_stats(logits, ind, valid=valid[:5])
    with pytest.raises(TypeError):
        ops.balance_stats(logits, ind, valid=valid.float())
    with pytest.raises(ValueError):
        ops.balance_stats(logits, ind, score="cosine")
    with pytest.raises(ValueError):
        ops.balance_stats(torch.zeros(4, 1025, device="cuda"), ind[:4])
    with pytest.raises(ops.NcclError):
        ops.balance_stats(logits, torch.zeros(20, 9, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.balance_loss(counts, probs, 9)
    with pytest.raises(ValueError):
        ops.balance_loss(counts[:8], probs, 2)
    with pytest.raises(ValueError):
        ops.balance_backward(logits, counts[:8], 2)
    with pytest.raises(ValueError):
        ops.balance_backward(logits, counts, 2, accumulate=True)
    with pytest.raises(ValueError):
        ops.balance_backward(logits, counts, 2, out=torch.zeros(20, 7, device="cuda"))
    with pytest.raises(ops.NcclError):
        ops.balance_backward(logits, counts, 2, out=logits, accumulate=True)
    with pytest.raises(ValueError):
        ops.balance_backward(logits, counts, 0)


def test_calls_from_another_current_device(monkeypatch):
    """The way round by the tensors' own device (taken once here, as if another were current)."""
    x = torch.randn(1000, generator=gen(1), device="cuda")
    logits, ind, valid = router(50, 12, 3, F32, True)
    a, b = Model([300], seed=2), Model([300], seed=2)
    plan = ops.SquareSum([x])
    total = plan()
    counts, probs = ops.balance_stats(logits, ind, valid=valid)
    loss, grad = ops.balance_loss(counts, probs, 3), ops.balance_backward(logits, counts, 3, valid=valid)
    b.plan.step(1e-2)
    once = []

    def elsewhere(device):
        once.append(device)
        return len(once) % 2 == 1

    def check(call, *want):
        once.clear()
        got = call()
        assert len(once) >= 1 and all(torch.equal(g, w) for g, w in zip(got, want))
    monkeypatch.setattr(ops, "_elsewhere", elsewhere)
    check(lambda: [plan()], total)
    check(lambda: ops.balance_stats(logits, ind, valid=valid), counts, probs)
    check(lambda: [ops.balance_loss(counts, probs, 3)], loss)
    check(lambda: [ops.balance_backward(logits, counts, 3, valid=valid)], grad)
    check(lambda: a.plan.step(1e-2) or [])
    assert a.same(b.copy())


# ---- a run of them, beside the collectives -----------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
def test_a_sharded_training_step(bits):
    """Two ranks on this GPU: the balance loss over both ranks' tokens and its gradient, then the gradients
    reduced, clipped, stepped and gathered, against one rank's step on the whole in 64 bits."""
    import msccl_amd as M
    comms = M.Comm.init_all([0, 0])
    try:
        run_sharded(comms, bits)
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def test_a_sharded_step_in_a_graph():
    """Captured once and replayed, with gradients that change, against the same steps one by one."""
    import msccl_amd as M
    n, block = 2, 6400

    def make(comms):
        params = [(torch.randn(n * block, generator=gen(1), device="cuda") * 0.1).to(BF16) for _ in range(n)]
        grads = [torch.zeros(n * block, dtype=BF16, device="cuda") for _ in range(n)]
        shards = [torch.zeros(block, dtype=BF16, device="cuda") for _ in range(n)]
        plans, sums, keep = [], [], []
        for r in range(n):
            p = params[r][r * block:(r + 1) * block]
            w, st, step = p.float(), ops.adamw_state(p, 8), torch.zeros(1, dtype=torch.int64, device="cuda")
            plans.append(ops.AdamW([p], [shards[r]], [st[0]], [st[1]], step, masters=[w], exp_avg_scales=[st[2]],
                                   exp_avg_sq_scales=[st[3]], weight_decay=0.1))
            sums.append(ops.SquareSum([shards[r]]))
            keep += [w, *st, step]
        return params, grads, shards, plans, sums, keep
    comms = M.Comm.init_all([0] * n)
    try:
        a, b = make(comms), make(comms)
        lr = torch.full((1,), 1e-2, device="cuda")
        ops.sharded_step(comms, a[1], a[2], a[0], a[3], a[4], lr=1e-2, max_norm=1.0)   # gradients of zero
        ops.sharded_step(comms, b[1], b[2], b[0], b[3], b[4], lr=1e-2, max_norm=1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            totals = ops.sharded_step(comms, a[1], a[2], a[0], a[3], a[4], lr=[lr] * n, max_norm=1.0)
        for t in range(1, 5):
            lr.fill_(1e-2 / t)
            for r in range(n):
                a[1][r].copy_(torch.randn(n * block, generator=gen(10 * t + r), device="cuda"))
                b[1][r].copy_(a[1][r])
            graph.replay()
            eager = ops.sharded_step(comms, b[1], b[2], b[0], b[3], b[4], lr=[lr] * n, max_norm=1.0)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(totals, eager))
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[0] + a[5], b[0] + b[5]))
            assert int(a[5][-1]) == t + 1
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def run_sharded(comms, bits):
    # the balance loss over both ranks
    data = [router(301, 24, 3, BF16, True, seed=r) for r in range(2)]
    stats = [ops.balance_stats(x, i, valid=v) for x, i, v in data]
    local = [(c.clone(), p.clone()) for c, p in stats]
    ops.balance_all_reduce(comms, [s[0] for s in stats], [s[1] for s in stats])
    for c, p in stats:
        assert torch.equal(c, local[0][0] + local[1][0]) and torch.equal(p, local[0][1] + local[1][1])
    losses = [ops.balance_loss(c, p, 3, 0.01) for c, p in stats]
    assert torch.equal(losses[0], losses[1])
    for (x, _, v), (c, p) in zip(data, stats):
        got = ops.balance_backward(x, c, 3, 0.01, grad_output=torch.full((1,), 1e4, device="cuda"), valid=v)
        check_backward(x, c, 3, 0.01, 1e4, v, "softmax", got)
    # the sharded step: a block of each rank holds tensors of odd sizes
    sizes, block = [1000, 3, 517, 2049], 4352
    spans, at = [], 0
    for n in sizes:
        spans.append((at, n))
        at += -(-n // 256) * 256
    start = (torch.randn(2 * block, generator=gen(1), device="cuda") * 0.1).to(BF16)
    params = [start.clone() for _ in range(2)]
    shards = [torch.zeros(block, dtype=BF16, device="cuda") for _ in range(2)]
    plans, sums, states = [], [], []
    for r in range(2):
        mine = params[r][r * block:(r + 1) * block]
        cut = lambda t: [t[a:a + n] for a, n in spans]  # noqa: E731
        p, g = cut(mine), cut(shards[r])
        st = [ops.adamw_state(x, bits) for x in p]
        w = [x.float() for x in p]
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        plans.append(ops.AdamW(p, g, [s[0] for s in st], [s[1] for s in st], step, masters=w,
                               exp_avg_scales=[s[2] for s in st] if bits == 8 else None,
                               exp_avg_sq_scales=[s[3] for s in st] if bits == 8 else None, weight_decay=0.1))
        sums.append(ops.SquareSum(g))
        states.append((w, st, step))
    for t in range(1, 4):
        grads = [(torch.randn(2 * block, generator=gen(10 * t + r), device="cuda")).to(BF16) for r in range(2)]
        before = [[w.clone() for w in s[0]] for s in states]
        old = [[(s[0].clone(), s[1].clone()) for s in st[1]] for st in states]
        oldscale = [[(s[2].clone(), s[3].clone()) for s in st[1]] for st in states] if bits == 8 else None
        totals = ops.sharded_step(comms, grads, shards, params, plans, sums, lr=1e-2, betas=(0.9, 0.99), max_norm=1.0)
        # ReduceScatter adds two bfloat16 values and rounds once
        whole = (grads[0].float() + grads[1].float()).to(BF16)
        total = sum(float(whole[r * block + a:r * block + a + n].double().square().sum()) for r in range(2) for a, n in spans)
        assert all(abs(float(x) - total) <= total * 1e-12 for x in totals)
        assert torch.equal(params[0], params[1])
        c = 0.5 * min(1.0, 1.0 / (0.5 * math.sqrt(total) + 1e-6))
        for r in range(2):
            w, st, step = states[r]
            assert int(step) == t
            for i, (a, n) in enumerate(spans):
                g = whole[r * block + a:r * block + a + n].double() * c
                m, v = (x.double() for x in old[r][i])
                if bits == 8:
                    ms, vs = (s.double().repeat_interleave(256)[:n] for s in oldscale[r][i])
                    m, v = m * ms, (v * vs) ** 2
                size = 0.9 * m.abs() + 0.1 * g.abs()
                m, v = 0.9 * m + 0.1 * g, 0.99 * v + 0.01 * g * g
                den = v.sqrt() / math.sqrt(1 - 0.99 ** t) + 1e-8
                rate = 1e-2 / (1 - 0.9 ** t)
                p = before[r][i].double() * (1 - 1e-3)
                up = rate * m / den
                close(w[i], p - up, 4 * U * p.abs() + 16 * U * up.abs() + rate / den * 6 * U * size, "weights")
                assert torch.equal(params[0][r * block + a:r * block + a + n], w[i].to(BF16))
    # one rank's bad gradient leaves every rank as it was
    bad = [g.clone() for g in grads]
    bad[1][5] = float("nan")
    kept, weights = params[0].clone(), [w.clone() for s in states for w in s[0]]
    ops.sharded_step(comms, bad, shards, params, plans, sums, lr=1e-2, max_norm=1.0)
    assert torch.equal(params[0], kept) and torch.equal(params[1], kept)
    assert all(torch.equal(a, b) for a, b in zip(weights, [w for s in states for w in s[0]]))
    assert all(int(s[2]) == 3 for s in states)
    with pytest.raises(ValueError):
        ops.sharded_step(comms, bad, shards, params, plans, sums[:1], lr=1e-2)
    with pytest.raises(ValueError):
        ops.sharded_step(comms, [g[:-1] for g in bad], shards, params, plans, sums, lr=1e-2)
    with pytest.raises(ValueError):
        ops.sharded_step(comms, bad, [s.clone() for s in shards], params, plans, sums, lr=1e-2)
    with pytest.raises(ValueError):
        ops.sharded_step(comms, bad, shards, [p.clone() for p in params], plans, sums, lr=1e-2)
    with pytest.raises(ValueError):
        ops.sharded_step(comms, bad, shards, params, plans[::-1], sums, lr=1e-2)
