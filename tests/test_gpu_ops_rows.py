"""Balance statistics and gradients of rows whose logits are large, far below zero or masked with a finite
value, against the definitions in 64 bits.

u = 2^-24 is half a step of a 32-bit value.  Bounds count roundings, element by element: a logit's own
distance from its row's largest says how many its exponential has."""
import pytest
import torch

from msccl_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # of the output's type (32 bits: counted in the bound)
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}
EXPERTS = [3, 8, 24, 100, 700]   # one lane a row (part and whole), four, sixteen, sixty-four with two vectors


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def definition(x, score):
    """(p, 1 - sigmoid, roundings of p): p from logarithms, so that no size of logit leaves 64 bits."""
    x = x.double()
    a = x if score == "softmax" else torch.where(x < -40, x, torch.nn.functional.logsigmoid(x))
    top = a.amax(1, keepdim=True)
    z = torch.exp(a - torch.where(torch.isneginf(top), 0.0, top))
    s = z.sum(1, keepdim=True)
    p = torch.where(s == 0, 0.0, z / s)
    # softmax of a logit d below the largest: the subtraction 1 d, the product with log2(e) 1.3 d, the
    # exponential's own 2; the same of the sum's terms, which weigh as p does (sum p d <= 2 + ln 1024 = 9): 23;
    # the sum's 15 additions, the reciprocal 2, the product 1
    # (differences past 150 belong to a p of zero)
    d = (x.amax(1, keepdim=True) - x).clamp(max=150.0).nan_to_num(150.0, 150.0, 0.0)
    err = 2.3 * d + 43
    if score == "sigmoid":
        # near zero instead: the exponential's argument 1.3 |x|, its own 2, the sum, the reciprocal and the
        # product 4; the sum's terms the same, weighing as p does; 15 additions, quotient and product 2.
        # (a sum of 1024 scores below e^-26 is below 2^-25: from there on the differences count again)
        far = x.abs().clamp(max=150.0)
        err = torch.where(x.amax(1, keepdim=True) > -26, 1.3 * far + (p * 1.3 * far).sum(1, keepdim=True) + 30, err)
    return p, torch.special.expit(-x), err


def close(got, want, bound, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    off = (got - want).abs() - bound
    assert off.max() <= 0, (what, int(off.argmax()), float(off.max()), float(want.flatten()[off.argmax()]))


def check_rows(x, score, up=1.0):
    """Each row's statistics by themselves, all rows', and the gradient."""
    t, e = x.shape
    p, slope, err = definition(x, score)
    index = torch.zeros(t, 1, dtype=torch.int32, device="cuda")
    # (a probability below 2^-100 may be zero: its score beside the row's sum leaves 32 bits)
    one = p * (err + 2) * U + 2.0 ** -100
    for r in range(t) if e == 24 else ():
        valid = torch.zeros(t, dtype=torch.bool, device="cuda")
        valid[r] = True
        close(ops.balance_stats(x, index, valid=valid, score=score)[1], p[r], one[r], "row %d" % r)
    # the sums over rows: in 32 bits at most 80 roundings
    close(ops.balance_stats(x, index, score=score)[1], p.sum(0), (one + p * 80 * U).sum(0), "all rows")
    counts = torch.randint(0, 1000, (e + 1,), generator=gen(2), device="cuda")
    counts[e] = 500
    k = min(2, e)
    w = counts[:e].double() * (0.5 * e / (k * 500.0 ** 2)) * up
    got = ops.balance_backward(x, counts, k, 0.5, grad_output=torch.full((1,), up, device="cuda"), score=score)
    w = w - 500.0 * k / e * (0.5 * e / (k * 500.0 ** 2)) * up   # the same for every expert: no part of the gradient
    mean = (p * w).sum(1, keepdim=True)
    d = p * (w - mean)
    size = (p * w.abs()).sum(1, keepdim=True)
    bound = p * U * (err * (w - mean).abs() + 4 * w.abs() + (err + 20) * size) + 2.0 ** -100 * (w.abs() + size)
    if score == "sigmoid":   # 1 - sigmoid and its product: 10 roundings, and those of its exponential
        d, bound = d * slope, bound * slope + (d * slope).abs() * (10 + 1.3 * x.double().abs().clamp(max=150.0)) * U
    close(got, d, bound + HALF[x.dtype] * (d.abs() + bound) + TINY[x.dtype], "gradient")


def rows_at(values, e, dtype, seed=1):
    """For each value a row of it alone, one with it once among ordinary logits, one where every second
    logit has it, and ordinary rows between them."""
    rows = []
    g = gen(seed)
    for v in values:
        plain = torch.randn(4, e, generator=g, device="cuda", dtype=torch.float64)
        plain[0] = v
        plain[1, e // 2] = v
        plain[2, ::2] = v
        rows.append(plain)
    top = float(torch.finfo(dtype).max)
    return torch.cat(rows).clamp(-top, top).to(dtype)


LARGE = [1e6, 2.0 ** 20, 1e8, 1e9, 2.0 ** 31, 5e9, 1e10, 1e12, 1e15, 1e20, 1e30, 3.4e38]


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_softmax_of_large_finite_logits(dtype, experts):
    values = LARGE + [-v for v in LARGE]
    check_rows(rows_at(values, experts, dtype), "softmax")
    for v in values:   # (the rows of a wave may take one another's way)
        check_rows(rows_at([v], experts, dtype), "softmax")


def test_softmax_rows_masked_throughout_weigh_alike():
    for low in (-1e9, -1e10, -1e30, torch.finfo(F32).min):
        x = torch.full((64, 8), low, device="cuda")
        counts, probs = ops.balance_stats(x, torch.zeros(64, 2, dtype=torch.int64, device="cuda"))
        assert probs.tolist() == [8.0] * 8, low


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("up", [1e-30, 1e-6, 1.0, 1e14, 1e25])
def test_sigmoid_gradient_where_all_scores_are_small(experts, up):
    """The mean of the weights over a row is of the weights' size, however small the scores are: it neither
    loses its digits in 32 bits nor passes their range."""
    x = -73.0 - 12.0 * torch.rand(64, experts, generator=gen(4), device="cuda")
    counts = torch.randint(1, 100_000, (experts + 1,), generator=gen(5), device="cuda")
    counts[experts] = 1_000_000
    k = min(2, experts)
    got = ops.balance_backward(x, counts, k, 0.01, grad_output=torch.full((1,), up, device="cuda"), score="sigmoid")
    p = definition(x, "sigmoid")[0]
    scale = 0.01 * experts / (k * 1e12) * up
    w = (counts[:experts].double() - 1e6 * k / experts) * scale
    mean = (p * w).sum(1, keepdim=True)
    d = p * (w - mean)
    # a score: its exponential's argument 1.3 |x|, and 8; a probability that of the sum's terms too, 15
    # additions, the quotient 2; the weights 3; the mean's terms as many again, and 17 additions
    err = 2.6 * x.double().abs() + 33
    bound = U * p * ((err + 10) * (w - mean).abs() + (p * w.abs()).sum(1, keepdim=True) * (err + 20)) + 2.0 ** -140
    close(got, d, bound, "gradient")


LOW = [-15.0, -17.0, -17.5, -18.0, -25.0, -60.0, -70.0, -85.0, -87.0, -88.0, -95.0, -103.0, -150.0, -1e3, -60000.0, -1e10, -1e30, -3.4e38]


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sigmoid_rows_far_below_zero(dtype, experts):
    """Their scores leave 32 bits, their probabilities do not."""
    g = gen(6)
    rows = [rows_at(LOW, experts, dtype)]
    for v in LOW:   # a few units apart from each other, as scores of one row are
        rows.append((v - 6.0 * torch.rand(3, experts, generator=g, device="cuda", dtype=torch.float64)).clamp(min=float(torch.finfo(dtype).min)).to(dtype))
    check_rows(torch.cat(rows), "sigmoid")
    for r in rows[1:]:
        check_rows(r, "sigmoid")


def test_sigmoid_rows_between_infinities():
    """A row of -inf alone has nothing; one score among them has everything; +inf counts as one does."""
    inf = float("inf")
    x = torch.tensor([[-inf] * 4, [-inf, -200.0, -inf, -inf], [-90.0, -inf, -90.0, -inf], [inf, -300.0, -inf, inf]], device="cuda")
    index = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    for r, want in enumerate([[0, 0, 0, 0], [0, 1, 0, 0], [0.5, 0, 0.5, 0], [0.5, 0, 0, 0.5]]):
        assert ops.balance_stats(x[r:r + 1], index[r:r + 1], score="sigmoid")[1].tolist() == want
    got = ops.balance_backward(x, torch.tensor([5, 1, 1, 1, 4], device="cuda"), 1, score="sigmoid")
    assert bool(torch.isfinite(got).all()) and float(got[:2].abs().max()) == 0 and float(got[3].abs().max()) == 0
    # p (w - mean) of weights 20 / 16 and 1 / 4 on halves
    assert got[2].tolist() == [0.25, 0, -0.25, 0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts", [(1000, 3), (40_000, 7), (5000, 60), (131_072, 100), (999_999, 100), (100_000, 200), (65_536, 700)])
def test_equal_rows_add_up(tokens, experts, score):
    """A router whose weights are zero: every row the same, so that the roundings of a sum do not average out."""
    x = torch.zeros(tokens, experts, dtype=BF16, device="cuda")
    counts, probs = ops.balance_stats(x, torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), score=score)
    want = tokens / experts
    # one over the row's sum (exact here) is within 2 roundings, its product with the score 1; the sums are in
    # 64 bits and rounded once
    assert int(counts[experts]) == tokens and float((probs.double() - want).abs().max()) <= 4 * U * want * (1 + 1e-6)

