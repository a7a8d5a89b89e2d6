"""A layer of experts around its products, against plain implementations in 64 bits: which experts a row goes to and with which weights, rows
ordered by expert, their weighted sums; gradients against the formulas and against differences.

Bounds. Choices, orders and copies: equal. Weights (fp32): an exponential of a rounded difference (2^-24 of up to 64), a sum, a quotient and
a product, 2^-18 in all at most. Their gradients subtract a mean of k terms of which each is off as much: 2^-17 of the largest term, and a
rounding of the result. Weighted sums of k terms in fp32: k 2^-23 of the terms' magnitudes, and a rounding: 2^-8 (bf16) or 2^-11 (f16) of the
result at most. Dots over D elements: (D + 8) 2^-24 of the sum of the terms' magnitudes."""
import pytest
import torch

import apt_b200
from apt_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
INF = float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------- router
def _route64(logits, k, score, bias, groups, top_groups, best, renormalize, scale):
    """Row by row, from the definition, in Python numbers (doubles)."""
    experts, weights = [], []
    n = logits.shape[1]
    table = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    for row, s in zip(logits.double().tolist(), table.tolist()):
        c = [z if bias is None else v + float(b) for z, v, b in zip(row, s, [0.0] * n if bias is None else bias)]
        there = [e for e in range(n) if row[e] != -INF and c[e] != -INF]
        if groups > 1:
            per, values = n // groups, []
            for g in range(groups):
                mine = sorted((s[e] if bias is None and best == 2 else c[e] for e in there if e // per == g), reverse=True)
                values.append(sum(mine[:best]) if mine else -INF)
            first = sorted(range(groups), key=lambda g: (-values[g], g))[:top_groups]
            there = [e for e in there if e // per in first]
        chosen = sorted(there, key=lambda e: (-c[e], e))[:k]
        total = sum(s[e] for e in chosen)
        experts.append(chosen + [-1] * (k - len(chosen)))
        weights.append([scale * s[e] / (total if renormalize else 1.0) for e in chosen] + [0.0] * (k - len(chosen)))
    return torch.tensor(experts, device="cuda").view(-1, k), torch.tensor(weights, device="cuda", dtype=torch.float64).view(-1, k)


def _route_grad64(logits, experts, grad, score, renormalize, scale):
    leaf = logits.detach().double().requires_grad_()
    z = torch.where(leaf.isneginf().all(1, keepdim=True), 0.0, leaf)
    s = torch.softmax(z, 1) if score == "softmax" else torch.sigmoid(z)
    real = experts >= 0
    picked = torch.where(real, s.gather(1, experts.clamp(min=0)), 0.0)
    w = scale * (picked / picked.sum(1, keepdim=True).clamp(min=1e-300) if renormalize else picked)
    return torch.autograd.grad(w, leaf, torch.where(real, grad.double(), 0.0))[0]


def _check_route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, best=1, renormalize=True, scale=1.0):
    args = (k, score, bias, groups, top_groups, best, renormalize, scale)
    experts, weights = apt_b200.route_experts(logits, *args)
    want_e, want_w = _route64(logits, *args)
    assert torch.equal(experts, want_e)
    assert weights.dtype == torch.float32 and float(((weights - want_w).abs() - 2.0 ** -18 * want_w.abs()).max()) <= 1e-37
    leaf = logits.clone().requires_grad_()
    e2, w2 = apt_b200.RouteExperts.apply(leaf, *args)
    assert torch.equal(e2, experts) and torch.equal(w2, weights) and not e2.requires_grad
    grad = torch.randn(weights.shape, device="cuda", generator=_gen(5))
    got = torch.autograd.grad(w2, leaf, grad)[0]
    want = _route_grad64(logits, experts, grad, score, renormalize, scale)
    assert got.dtype == logits.dtype
    # the largest term of a row's mean: the largest |scale w g|, times 4 for the two factors behind it
    term = 4 * (want_w * grad.double()).abs().amax(1, keepdim=True)
    # numbers below the type's smallest normal one are a step of its denormals off
    tiny = torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps
    assert bool(((got.double() - want).abs() <= 2.0 ** -17 * term + HALF[logits.dtype] * want.abs() + tiny).all())
    assert torch.equal(got, apt_b200.route_experts_backward(leaf.detach(), experts, grad, score, renormalize, scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (1, 64, 6), (5, 2, 2), (300, 8, 2), (77, 7, 7), (129, 47, 5), (64, 64, 64), (33, 65, 3), (40, 256, 8),
                                            (9, 300, 16), (7, 1000, 12), (5, 1024, 64)])
def test_routes(rows, experts, k, score, dtype):
    logits = (torch.randn((rows, experts), device="cuda", generator=_gen(rows + experts)) * 2).to(dtype)
    bias = torch.randn(experts, device="cuda", generator=_gen(3)) * 0.1
    _check_route(logits, k, score)
    _check_route(logits, k, score, bias, renormalize=False, scale=2.5)
    _check_route(logits, k, score, bias)
    _check_route(logits, k, score, renormalize=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(4, 2, 1, 1), (8, 8, 3, 3), (24, 3, 2, 4), (60, 5, 2, 6), (64, 32, 7, 8), (100, 4, 3, 20), (256, 8, 4, 8),
                                                         (1023, 3, 2, 10), (1023, 31, 9, 9), (1020, 17, 5, 16)])
def test_routes_by_groups(experts, groups, top_groups, k, best, dtype):
    logits = (torch.randn((45, experts), device="cuda", generator=_gen(experts)) * 1.5).to(dtype)
    bias = torch.randn(experts, device="cuda", generator=_gen(4)) * 0.05
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            _check_route(logits, k, score, b, groups, top_groups, best)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_routes_of_masked_experts_and_rows(score, dtype):
    logits = torch.randn((64, 24), device="cuda", generator=_gen(1)).to(dtype)
    logits[torch.rand(logits.shape, device="cuda", generator=_gen(2)) < 0.7] = -INF
    logits[::5] = -INF                                  # nothing is left
    logits[1] = torch.finfo(dtype).min                  # all as low as can be, and yet there
    logits[2] = -INF
    logits[2, 17] = torch.finfo(dtype).min
    bias = torch.randn(24, device="cuda", generator=_gen(3)) * 0.1
    bias[3] = -INF
    for b in (None, bias):
        _check_route(logits, 4, score, b, renormalize=False)
        _check_route(logits, 4, score, b, 6, 2, 2, renormalize=False)
    experts, weights = apt_b200.route_experts(logits, 4, score)
    assert torch.equal(experts, _route64(logits, 4, score, None, 1, 1, 1, False, 1.0)[0])
    # scores that are all nothing in 32 bits still have shares
    some = (experts >= 0).any(1)
    assert torch.allclose(weights.sum(1)[some], torch.ones((), device="cuda"), atol=2e-6) and not weights[~some].any()
    grad = apt_b200.route_experts_backward(logits, experts, torch.ones_like(weights), score)
    assert torch.isfinite(grad).all() and not grad[::5].any()


def test_equal_scores_go_by_their_index():
    logits = torch.zeros((3, 40), device="cuda")
    logits[1, ::3] = -0.0                               # the same number
    logits[2, 20:] = 1.0
    for b in (None, torch.zeros(40, device="cuda")):
        for score in ("softmax", "sigmoid"):
            experts, weights = apt_b200.route_experts(logits, 4, score, b)
            assert experts.tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [20, 21, 22, 23]]
            assert apt_b200.route_experts(logits, 4, score, b, 8, 2, 2)[0].tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [20, 21, 22, 23]]


def test_scores_that_are_one_in_32_bits():
    """Neighbours by 1e-9: 32 bits do not tell them apart, 64 do."""
    logits = torch.randn((2000, 64), device="cuda", generator=_gen(8)).clamp_(-3, 3)
    table = torch.sigmoid(logits.double())
    # every expert's score and bias come to nearly the same
    bias = (1.0 - table[0]).float()
    logits = logits[0].repeat(2000, 1)
    logits += torch.randn(logits.shape, device="cuda", generator=_gen(9)) * 1e-7
    args = (8, "sigmoid", bias, 1, 1, 1, True, 1.0)
    assert torch.equal(apt_b200.route_experts(logits, *args)[0], _route64(logits, *args)[0])
    args = (8, "sigmoid", bias, 8, 3, 2, True, 1.0)
    assert torch.equal(apt_b200.route_experts(logits, *args)[0], _route64(logits, *args)[0])


@pytest.mark.parametrize("experts,groups,top_groups,k", [(64, 1, 1, 8), (64, 1, 1, 33), (130, 1, 1, 16), (130, 1, 1, 64), (256, 1, 1, 8), (256, 1, 1, 33), (256, 8, 4, 8),
                                                         (512, 1, 1, 47), (1000, 1, 1, 64), (1024, 1, 1, 63), (1024, 8, 2, 64), (1020, 17, 5, 31)])
def test_many_equal_scores(experts, groups, top_groups, k):
    """Rows of very few values and biases: more equal ones at the last place than there is room for, and neighbours by less than 32 bits tell behind them."""
    few = torch.randint(0, 3, (40, experts), device="cuda", generator=_gen(experts)).float()
    few[:4] = 0.0
    few[4, :] = -1.0
    few[5, experts // 2:] = -INF
    round_ = torch.randn((40, experts), device="cuda", generator=_gen(k)).bfloat16()
    near = few + torch.randint(0, 2, few.shape, device="cuda", generator=_gen(7)) * 2.0 ** -22
    zeros, two = torch.zeros(experts, device="cuda"), torch.randint(0, 2, (experts,), device="cuda", generator=_gen(8)) * 0.5
    for logits in (few, round_, near):
        for best in (1, 2):
            if groups == 1 and best == 2:
                continue
            for score, bias in (("softmax", None), ("softmax", zeros), ("sigmoid", zeros), ("sigmoid", two)):
                args = (k, score, bias, groups, top_groups, best, True, 1.0)
                got, weights = apt_b200.route_experts(logits, *args)
                want, want_weights = _route64(logits, *args)
                assert torch.equal(got, want)
                assert float(((weights - want_weights).abs() - 2.0 ** -18 * want_weights.abs()).max()) <= 1e-37


def _choice64(logits, k, score, bias, groups=1, top_groups=1, best=1):
    """_route64's choice for a bias, many rows at once."""
    s = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    c = torch.where(logits == -INF, -INF, s + bias.double())
    if groups > 1:
        values = c.view(len(c), groups, -1).sort(dim=2, descending=True).values[:, :, :best]
        values = torch.where(values[:, :, -1] == -INF, values[:, :, 0], values.sum(2))
        stay = torch.zeros_like(values, dtype=torch.bool).scatter_(1, values.sort(dim=1, descending=True, stable=True).indices[:, :top_groups], True)
        c = torch.where(stay.repeat_interleave(c.shape[1] // groups, 1), c, -INF)
    order = c.sort(dim=1, descending=True, stable=True)
    return torch.where(order.values == -INF, -1, order.indices)[:, :k]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,k", [(6, 1), (16, 2), (64, 3), (256, 8)])
def test_near_ones_that_are_not_among_the_picks(experts, k, score):
    """The last pick and the next are one logit and bias; others, of another logit and bias, come to the same 32 bits, and in the exact scores some are above."""
    gen = _gen(experts)
    base = torch.rand((1, experts), device="cuda", generator=gen) * 2 - 1
    table = torch.softmax(base.double(), 1) if score == "softmax" else torch.sigmoid(base.double())
    bias = (1.0 - table[0]).float()
    logits = base.repeat(20_000, 1)
    # half of the experts are the same, the others neighbours by a unit or two
    logits[:, ::2], bias[::2] = logits[0, 0].clone(), bias[0].clone()
    step = torch.randint(-3, 4, logits.shape, device="cuda", generator=gen) * 2.0 ** -24
    step[:, ::2] = 0.0
    logits += step
    assert torch.equal(apt_b200.route_experts(logits, k, score, bias)[0], _choice64(logits, k, score, bias))


def test_groups_by_their_best_that_are_one_in_32_bits():
    """The best of two groups are one number in 32 bits, logistics next to 1, and not in the exact scores."""
    zeros = torch.zeros(4, device="cuda")
    for dtype in DTYPES:
        logits = torch.tensor([[20.0, -5.0, 25.0, -5.0], [25.0, 1.0, 20.0, 2.0], [-5.0, 21.0, 22.0, 21.0], [22.0, 22.0, 22.0, 22.0]], device="cuda").to(dtype)
        assert apt_b200.route_experts(logits, 1, "sigmoid", zeros, 2, 1)[0].tolist() == [[2], [0], [2], [0]]
        assert apt_b200.route_experts(logits, 2, "sigmoid", zeros, 2, 1)[0].tolist() == [[2, 3], [0, 1], [2, 3], [0, 1]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(4, 2, 1, 1), (16, 8, 3, 1), (64, 8, 3, 4), (60, 5, 2, 1), (256, 8, 4, 8), (1023, 31, 9, 9), (1020, 17, 5, 1)])
def test_groups_by_their_best_are_those_of_the_exact_scores(experts, groups, top_groups, k, score):
    rows = 40_000 if experts < 1000 else 8000
    gen = _gen(experts + k)
    # logistics next to 1 in many of the groups
    wide = (torch.randn((rows, experts), device="cuda", generator=gen) * 6).clamp_(-30, 30)
    # neighbours by a unit of their last place
    close = torch.randn((1, experts), device="cuda", generator=gen).clamp_(-2, 2)
    table = torch.softmax(close.double(), 1) if score == "softmax" else torch.sigmoid(close.double())
    level = (table.max() - table[0]).float()
    close = close + torch.randint(-4, 5, (rows, experts), device="cuda", generator=gen) * 2.0 ** -23
    few = torch.randint(0, 3, (rows, experts), device="cuda", generator=gen).float() + torch.randint(0, 2, (rows, experts), device="cuda", generator=gen) * 2.0 ** -22
    zeros, constant = torch.zeros(experts, device="cuda"), torch.full((experts,), 0.75, device="cuda")
    for logits, bias in ((wide, zeros), (wide.bfloat16(), zeros), (wide.half(), constant), (close, level), (few, zeros), (few, constant)):
        got = apt_b200.route_experts(logits, k, score, bias, groups, top_groups, 1)[0]
        assert torch.equal(got, _choice64(logits, k, score, bias, groups, top_groups, 1))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(16, 8, 3, 1), (16, 8, 3, 4), (8, 4, 2, 2), (96, 32, 5, 3)])
def test_groups_whose_two_best_take_each_other_away(experts, groups, top_groups, k, score):
    """Biases of 64 and more, and minus as much: each sum with one is rounded to steps of 2^-17, the two best together are as little as two scores."""
    gen = _gen(experts + k)
    per = experts // groups
    own = 64.0 + 2.0 * (torch.arange(experts, device="cuda") // per)
    bias = torch.where(torch.arange(experts, device="cuda") % per == 0, own, -own)
    logits = torch.randn((1, per), device="cuda", generator=gen).repeat(20_000, groups)
    logits += torch.randn(logits.shape, device="cuda", generator=gen) * 2e-5
    got = apt_b200.route_experts(logits, k, score, bias, groups, top_groups, 2)[0]
    assert torch.equal(got, _choice64(logits, k, score, bias, groups, top_groups, 2))


def test_wild_logits_stay_in_their_rows():
    logits = torch.randn((64, 32), device="cuda", generator=_gen(1))
    bias = torch.zeros(32, device="cuda")
    clean = apt_b200.route_experts(logits, 4, "softmax", bias)
    wild = logits.clone()
    wild[::2, 5] = float("nan")
    wild[1::4, 7] = INF
    for b in (None, bias):
        experts, weights = apt_b200.route_experts(wild, 4, "softmax", b)
        assert bool(((experts >= 0) & (experts < 32)).all()) and torch.isnan(weights[::2]).all()
        assert torch.equal(experts[3::4], clean[0][3::4]) and torch.equal(weights[3::4], clean[1][3::4])
    grad = apt_b200.route_experts_backward(wild, clean[0], torch.ones_like(clean[1]), "softmax", False)
    assert torch.isfinite(grad[3::4]).all() and torch.isnan(grad[::2]).all()


def test_route_gradient_against_differences():
    logits = torch.randn((6, 12), device="cuda", generator=_gen(3))
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            experts, _ = apt_b200.route_experts(logits, 3, score, None, 1, 1, 1, renormalize, 2.0)
            grad = torch.randn((6, 3), device="cuda", generator=_gen(4))
            got = apt_b200.route_experts_backward(logits, experts, grad, score, renormalize, 2.0)
            step = 2.0 ** -7

            def value(z):
                s = torch.softmax(z.double(), 1) if score == "softmax" else torch.sigmoid(z.double())
                p = s.gather(1, experts)
                return (2.0 * (p / p.sum(1, keepdim=True) if renormalize else p) * grad).sum(1)

            for e in range(12):
                d = torch.zeros_like(logits)
                d[:, e] = step
                slope = (value(logits.double() + d.double()) - value(logits.double() - d.double())) / (2 * step)
                # a third derivative below 4 |g| k leaves step^2 / 6 of it
                assert float((got[:, e].double() - slope).abs().max()) < 4 * 3 * 3.5 * step ** 2 / 6 + 1e-5


def test_an_expert_named_twice_has_both_gradients():
    logits = torch.randn((4, 9), device="cuda", generator=_gen(1))
    experts = torch.tensor([[3, 3, 1]] * 4, device="cuda")
    grad = torch.randn((4, 3), device="cuda", generator=_gen(2))
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            got = apt_b200.route_experts_backward(logits, experts, grad, score, renormalize)
            want = _route_grad64(logits, experts, grad, score, renormalize, 1.0)
            assert float((got - want).abs().max()) < 2.0 ** -17 * 8 * float(grad.abs().max())


# -------------------------------------------------------------------------------------------------- rows to their experts
def _places64(experts, num_experts):
    flat = experts.reshape(-1).tolist()
    order = sorted(range(len(flat)), key=lambda p: (flat[p] if flat[p] >= 0 else num_experts, p))
    place = [0] * len(flat)
    for at, p in enumerate(order):
        place[p] = at if flat[p] >= 0 else -1 - at
    counts = [0] * (num_experts + 1)
    for e in flat:
        if e >= 0:
            counts[e + 1] += 1
    return order, torch.tensor(place, device="cuda").view(experts.shape), torch.tensor(counts, device="cuda").cumsum(0)


def _check_rows(x, experts, num_experts):
    rows, offsets, place = apt_b200.expert_rows(x, experts, num_experts)
    order, want_place, ends = _places64(experts, num_experts)
    k = experts[0].numel() if experts.dim() == 2 else 1
    at = torch.tensor(order, device="cuda", dtype=torch.int64)
    real = (experts.reshape(-1)[at] >= 0).unsqueeze(1)
    assert torch.equal(offsets, ends) and torch.equal(place, want_place)
    assert torch.equal(rows, torch.where(real, x[at // k], torch.zeros((), device="cuda", dtype=x.dtype)))
    leaf = x.clone().requires_grad_()
    got = apt_b200.ExpertRows.apply(leaf, experts, num_experts)
    assert all(torch.equal(a, b) for a, b in zip(got, (rows, offsets, place)))
    grad = torch.randn(rows.shape, device="cuda", generator=_gen(2)).to(x.dtype)
    gx = torch.autograd.grad(got[0], leaf, grad)[0]
    parts = torch.where((place >= 0).reshape(-1, 1), grad.double()[place.clamp(min=0).reshape(-1)], 0.0).view(x.shape[0], k, -1)
    want = parts.sum(1)
    assert bool(((gx.double() - want).abs() <= k * 2.0 ** -23 * parts.abs().sum(1) + HALF[x.dtype] * want.abs() + 1e-7 * HALF[x.dtype]).all())
    assert torch.equal(gx, apt_b200.expert_rows_backward(grad, place))
    ops.check_status()


def _experts(rows, k, num_experts, seed, none=0.1):
    e = torch.randint(0, num_experts, (rows, k), device="cuda", generator=_gen(seed))
    e = (e * e) // max(1, num_experts)                   # low ones are the likelier
    e[torch.rand(e.shape, device="cuda", generator=_gen(seed + 1)) < none] = -1
    return e


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,num_experts,dim", [(1, 1, 1, 1), (1, 6, 64, 256), (3, 2, 2, 7), (31, 3, 5, 8), (129, 8, 512, 33), (512, 2, 16, 100), (513, 2, 16, 4),
                                                    (1024, 1, 3, 64), (2500, 3, 47, 119), (1500, 7, 4096, 16), (3000, 5, 700, 258), (2048, 2, 1024, 6), (4097, 1, 1024, 6), (1, 1, 1025, 5),
                                                    (2, 2, 4096, 3)])
def test_rows_by_expert(rows, k, num_experts, dim, dtype):
    x = torch.randn((rows, dim), device="cuda", generator=_gen(dim)).to(dtype)
    _check_rows(x, _experts(rows, k, num_experts, rows), num_experts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_one_expert_of_none_and_of_views(dtype):
    x = torch.randn((1700, 24), device="cuda", generator=_gen(1)).to(dtype)
    for e in (torch.zeros((1700, 2), device="cuda", dtype=torch.int64), torch.full((1700, 2), -1, device="cuda"), torch.full((1700, 2), 8, device="cuda"),
              torch.arange(1700, device="cuda") % 9, torch.arange(3400, device="cuda").view(2, 1700).t() % 9):
        _check_rows(x, e, 9)
    wide = torch.randn((1700, 60), device="cuda", generator=_gen(2)).to(dtype)
    _check_rows(wide[:, 3:34], _experts(1700, 2, 9, 5), 9)
    flat = torch.randn(1700 * 24 + 1, device="cuda", generator=_gen(2)).to(dtype)
    _check_rows(flat[1:].view(1700, 24), _experts(1700, 2, 9, 5), 9)


def test_experts_that_are_none_are_reported():
    x = torch.randn((600, 8), device="cuda", generator=_gen(1))
    for bad in (5, -2, 2 ** 40):
        for rows in (600, 3):
            e = _experts(rows, 3, 5, 1)
            e[rows - 1, 1] = bad
            rows_, offsets, place = apt_b200.expert_rows(x[:rows], e, 5)
            with pytest.raises(RuntimeError, match="id outside"):
                ops.check_status()
            e[rows - 1, 1] = -1
            assert all(torch.equal(a, b) for a, b in zip((rows_, offsets, place), apt_b200.expert_rows(x[:rows], e, 5)))
    ops.check_status()


# -------------------------------------------------------------------------------------------------------- and their sum
def _check_sum(y, weights, place):
    k = place.shape[1]
    real = (place >= 0).unsqueeze(2)
    leaves = [y.clone().requires_grad_(), weights.clone().requires_grad_()]
    out = apt_b200.ExpertSum.apply(*leaves, place)
    assert torch.equal(out, apt_b200.expert_sum(y, weights, place))
    parts = torch.where(real, y.double()[place.clamp(min=0)], 0.0)
    terms = parts * torch.where(real, weights.double().unsqueeze(2), 0.0)
    want = terms.sum(1)
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert out.dtype == y.dtype and bool(((out.double() - want).abs() <= k * 2.0 ** -23 * terms.abs().sum(1) + HALF[y.dtype] * want.abs() + tiny).all())
    grad = torch.randn(out.shape, device="cuda", generator=_gen(9)).to(y.dtype)
    gy, gw = torch.autograd.grad(out, leaves, grad)
    want_y = torch.zeros_like(y, dtype=torch.float64)
    want_y[torch.where(place >= 0, place, -1 - place).reshape(-1)] = (torch.where(real, weights.double().unsqueeze(2), 0.0) * grad.double().unsqueeze(1)).reshape(y.shape)
    assert bool(((gy.double() - want_y).abs() <= 2 * HALF[y.dtype] * want_y.abs() + tiny).all())
    products = parts * grad.double().unsqueeze(1)
    assert gw.dtype == torch.float32
    assert bool(((gw.double() - products.sum(2)).abs() <= (y.shape[1] + 8) * 2.0 ** -24 * products.abs().sum(2)).all())
    # either alone
    a, b = apt_b200.expert_sum_backward(y, weights, place, grad, True, False), apt_b200.expert_sum_backward(y, weights, place, grad, False, True)
    assert torch.equal(a[0], gy) and a[1] is None and b[0] is None and torch.equal(b[1], gw)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,dim", [(1, 1, 1), (1, 6, 256), (3, 2, 7), (61, 6, 119), (130, 3, 33), (129, 8, 64), (1000, 2, 100), (2000, 1, 256), (300, 5, 1024), (40, 4, 2050)])
def test_sums_over_experts(rows, k, dim, dtype):
    experts = _experts(rows, k, 11, rows + dim)
    place = apt_b200.expert_rows(torch.zeros((rows, 1), device="cuda"), experts, 11)[2]
    y = torch.randn((rows * k, dim), device="cuda", generator=_gen(dim)).to(dtype)
    _check_sum(y, torch.rand((rows, k), device="cuda", generator=_gen(1)) - 0.3, place)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,dim", [(1, 8, 8192), (1, 3, 5001), (2, 2, 300), (7, 2, 4100), (70, 5, 2500), (150, 1, 3000), (590, 3, 1000), (1200, 2, 600)])
def test_few_wide_rows(rows, k, dim, dtype):
    """Rows that several warps share."""
    x = torch.randn((rows, dim), device="cuda", generator=_gen(dim)).to(dtype)
    experts = _experts(rows, k, 16, 4)
    _check_rows(x, experts, 16)
    y, _, place = apt_b200.expert_rows(x, experts, 16)
    _check_sum(y, torch.randn((rows, k), device="cuda", generator=_gen(6)), place)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_expert_count_for_nothing_whatever_they_hold(dtype):
    experts = _experts(200, 3, 6, 1, none=0.4)
    experts[:7] = -1
    place = apt_b200.expert_rows(torch.zeros((200, 1), device="cuda"), experts, 6)[2]
    y = torch.randn((600, 40), device="cuda", generator=_gen(2)).to(dtype)
    weights = torch.rand((200, 3), device="cuda", generator=_gen(3))
    clean = apt_b200.expert_sum(y, weights, place)
    wild, lost = y.clone(), weights.clone()
    wild[-1 - place[place < 0]] = float("nan")
    lost[place < 0] = INF
    assert torch.equal(apt_b200.expert_sum(wild, lost, place), clean) and not clean[:7].any()
    grad = torch.randn((200, 40), device="cuda", generator=_gen(4)).to(dtype)
    for a, b in zip(apt_b200.expert_sum_backward(wild, lost, place, grad), apt_b200.expert_sum_backward(y, weights, place, grad)):
        assert torch.equal(a, b)


def test_places_beyond_the_rows_are_reported():
    y, w = torch.randn((12, 8), device="cuda", generator=_gen(2)), torch.ones((6, 2), device="cuda")
    place = torch.arange(12, device="cuda").view(6, 2)
    for bad in (12, -14, 2 ** 40, -2 ** 40):
        p = place.clone()
        p[2, 1] = bad
        got = apt_b200.expert_sum(y, w, p)
        with pytest.raises(RuntimeError, match="id outside"):
            ops.check_status()
        assert torch.equal(got[2], y[4])
        apt_b200.expert_sum_backward(y, w, p, torch.ones((6, 8), device="cuda"))
        with pytest.raises(RuntimeError, match="id outside"):
            ops.check_status()
    ops.check_status()


# ---------------------------------------------------------------------------------------------------------- all together
def _layer(x, router, weight, k, num_experts):
    experts, weights = apt_b200.RouteExperts.apply(x @ router, k)
    rows, offsets, place = apt_b200.ExpertRows.apply(x, experts, num_experts)
    return apt_b200.ExpertSum.apply(apt_b200.GroupedLinear.apply(rows, weight, offsets), weights, place)


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 4e-6), (torch.bfloat16, 2.0 ** -7)])
def test_a_layer_of_experts(dtype, bound):
    """Against every row times all experts' weights, masked. fp32: some ten roundings and sums of at most 300 terms; bf16: three roundings of
    2^-8 at most one behind the other."""
    x = torch.randn((300, 48), device="cuda", generator=_gen(1)).to(dtype).requires_grad_()
    router = (torch.randn((48, 6), device="cuda", generator=_gen(2)) * 0.2).to(dtype).requires_grad_()
    weight = (torch.randn((6, 32, 48), device="cuda", generator=_gen(3)) * 0.15).to(dtype).requires_grad_()
    out = _layer(x, router, weight, 2, 6)
    grad = torch.randn(out.shape, device="cuda", generator=_gen(4)).to(dtype)
    got = torch.autograd.grad(out, [x, router, weight], grad)
    wide = [t.detach().double().requires_grad_() for t in (x, router, weight)]
    logits = wide[0] @ wide[1]
    # the choice is that of the logits as they were rounded
    chosen = (x @ router).detach().topk(2, 1).indices
    p = torch.softmax(logits, 1).gather(1, chosen)
    p = p / p.sum(1, keepdim=True)
    every = torch.einsum("rd,eod->reo", wide[0], wide[2])
    want = (every.gather(1, chosen.unsqueeze(2).expand(-1, -1, 32)) * p.unsqueeze(2)).sum(1)
    for a, b in zip((out,) + got, (want,) + torch.autograd.grad(want, wide, grad.double())):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < bound
    ops.check_status()


def _step(x, router, weight, out_weight, out_bias, labels, k, padded=None):
    logits = x @ router
    if padded is not None:
        logits = logits.masked_fill(padded.unsqueeze(1), -INF)
    experts, weights = apt_b200.RouteExperts.apply(logits, k)
    rows, offsets, place = apt_b200.ExpertRows.apply(x, experts, weight.shape[0])
    h = apt_b200.ExpertSum.apply(apt_b200.GroupedLinear.apply(rows, weight, offsets), weights, place)
    return apt_b200.LinearCrossEntropy.apply(h, out_weight, labels, out_bias)


def _step_leaves(rows, dim, hidden, num_experts, classes, dtype, seed=1):
    gen = _gen(seed)
    shapes = [(rows, dim), (dim, num_experts), (num_experts, hidden, dim), (classes, hidden), (classes,)]
    scales = [1.0, 0.2, 0.15, 0.3, 0.5]
    return [(torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype).requires_grad_() for shape, scale in zip(shapes, scales)]


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-4), (torch.bfloat16, 2.0 ** -5)])
def test_a_layer_of_experts_and_its_loss(dtype, bound):
    """A padded batch through all of them, against every row times all experts' weights. fp32: logits of the loss of some 18 (their terms'
    magnitudes and eight more) are (32 2^-23 + 2^-19) of that off, 1e-4, and the slopes with them. bf16: the layer's half steps move the
    logits by 2^-7, and six roundings of 2^-8 at most follow one another."""
    leaves = _step_leaves(320, 48, 32, 6, 500, dtype)
    labels = torch.randint(0, 500, (320,), device="cuda", generator=_gen(9))
    padded = torch.arange(320, device="cuda") >= 300
    labels[padded] = -100
    with torch.no_grad():
        leaves[0][padded] = 0.0
    loss = _step(*leaves, labels, 2, padded)
    got = torch.autograd.grad(loss, leaves)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    x, router, weight, out_weight, out_bias = wide
    chosen = (leaves[0] @ leaves[1]).detach().topk(2, 1).indices
    p = torch.softmax(x @ router, 1).gather(1, chosen)
    p = p / p.sum(1, keepdim=True)
    every = torch.einsum("rd,eod->reo", x, weight)
    h = (every.gather(1, chosen.unsqueeze(2).expand(-1, -1, 32)) * p.unsqueeze(2)).sum(1)
    want = torch.nn.functional.cross_entropy((h @ out_weight.t() + out_bias)[:300], labels[:300])
    assert abs(loss.item() - want.item()) < bound * want.item()
    for a, b in zip(got, torch.autograd.grad(want, wide)):
        assert bool(torch.isfinite(a).all()) and float((a.double() - b).norm() / b.norm()) < bound
    assert not got[0][300:].any()
    ops.check_status()


def test_calls_at_once():
    """Steps of two sizes on two streams, none waiting for another's: what each gives alone."""
    steps, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed, rows, experts, classes in ((1, 4000, 16, 3001), (2, 2500, 24, 5000)):
        leaves = _step_leaves(rows, 64, 64, experts, classes, torch.bfloat16, seed)
        steps.append((leaves, torch.randint(0, classes, (rows,), device="cuda", generator=_gen(seed))))

    def run(n):
        loss = _step(*steps[n][0], steps[n][1], 3)
        return [loss.detach()] + list(torch.autograd.grad(loss, steps[n][0]))

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(run(n))
    torch.cuda.synchronize()
    for n in (0, 1):
        for one in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[n]))
    ops.check_status()


def test_more_than_31_bits_of_elements():
    rows, dim, k, n = 1_100_000, 1024, 2, 500
    logits = torch.empty((2 * rows, dim), device="cuda", dtype=torch.bfloat16).normal_(generator=_gen(1))
    assert logits.numel() > 2 ** 31
    experts, weights = apt_b200.route_experts(logits, k)
    tail = apt_b200.route_experts(logits[-n:].clone(), k)
    assert torch.equal(experts[-n:], tail[0]) and torch.equal(weights[-n:], tail[1])
    grad = torch.randn(weights.shape, device="cuda", generator=_gen(2))
    for renormalize in (True, False):
        whole = apt_b200.route_experts_backward(logits, experts, grad, "softmax", renormalize)[-n:].clone()
        assert torch.equal(whole, apt_b200.route_experts_backward(logits[-n:].clone(), tail[0], grad[-n:].clone(), "softmax", renormalize))
    x, experts, weights = logits[:rows].clone(), experts[:rows] % 4, weights[:rows].contiguous()
    del logits, grad
    y, offsets, place = apt_b200.expert_rows(x, experts, 4)
    assert y.numel() > 2 ** 31 and int(place.max()) == rows * k - 1 and int(offsets[-1]) == rows * k
    last = (place == rows * k - 1).nonzero()[0, 0]
    some = torch.cat([torch.arange(rows - n, rows, device="cuda"), last.view(1)])
    assert torch.equal(y[place[some]], x[some].unsqueeze(1).expand(-1, k, -1))
    out = apt_b200.expert_sum(y, weights, place)
    want = (x[some].double().unsqueeze(1) * weights[some].double().unsqueeze(2)).sum(1)
    assert bool(((out[some].double() - want).abs() <= (HALF[x.dtype] + 2.0 ** -22) * want.abs() + 1e-37).all())
    grad_y, grad_weights = apt_b200.expert_sum_backward(y, weights, place, out)
    want = weights[some].double().unsqueeze(2) * out[some].double().unsqueeze(1)
    assert bool(((grad_y[place[some]].double() - want).abs() <= (HALF[x.dtype] + 2.0 ** -22) * want.abs() + 1e-37).all())
    # 1024 terms in fp32: at most 2^-14 of their magnitudes
    terms = out[some].double().unsqueeze(1) * y[place[some]].double()
    assert bool(((grad_weights[some].double() - terms.sum(2)).abs() <= 2.0 ** -14 * terms.abs().sum(2)).all())
    ops.check_status()


def test_another_stream_and_a_captured_graph():
    x = torch.randn((700, 64), device="cuda", generator=_gen(1)).requires_grad_()
    router = (torch.randn((64, 8), device="cuda", generator=_gen(2)) * 0.2).requires_grad_()
    weight = (torch.randn((8, 40, 64), device="cuda", generator=_gen(3)) * 0.1).requires_grad_()
    grad = torch.randn((700, 40), device="cuda", generator=_gen(4))

    def step():
        out = _layer(x, router, weight, 3, 8)
        return (out,) + torch.autograd.grad(out, [x, router, weight], grad)

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    with torch.no_grad():
        x.copy_(x.flip(0).clone())
    graph.replay()
    again = [t.detach().clone() for t in captured]
    assert all(torch.equal(a, b.detach()) for a, b in zip(again, step()))
    assert not torch.equal(again[0], want[0])
    ops.check_status()


def test_no_rows():
    logits = torch.empty((0, 8), device="cuda").requires_grad_()
    experts, weights = apt_b200.RouteExperts.apply(logits, 2)
    assert experts.shape == weights.shape == (0, 2) and torch.autograd.grad(weights, logits, torch.empty((0, 2), device="cuda"))[0].shape == (0, 8)
    x = torch.empty((0, 16), device="cuda").requires_grad_()
    rows, offsets, place = apt_b200.ExpertRows.apply(x, experts, 8)
    assert rows.shape == (0, 16) and place.shape == (0, 2) and not offsets.any() and offsets.shape == (9,)
    out = apt_b200.ExpertSum.apply(rows, weights, place)
    assert out.shape == (0, 16) and torch.autograd.grad(out, x, torch.empty((0, 16), device="cuda"))[0].shape == (0, 16)


def test_second_derivatives_raise():
    logits = torch.randn((5, 8), device="cuda", generator=_gen(1)).requires_grad_()
    _, w = apt_b200.RouteExperts.apply(logits, 2)
    g = torch.autograd.grad(w.square().sum(), logits, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(g.sum(), logits)
    y = torch.randn((10, 4), device="cuda", generator=_gen(1)).requires_grad_()
    out = apt_b200.ExpertSum.apply(y, torch.ones((5, 2), device="cuda"), torch.arange(10, device="cuda").view(5, 2))
    g = torch.autograd.grad(out.square().sum(), y, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(g.sum(), y)


def test_refusals():
    z, x = torch.zeros((4, 8), device="cuda"), torch.zeros((4, 16), device="cuda")
    e = torch.zeros((4, 2), device="cuda", dtype=torch.int64)
    w, y = torch.zeros((4, 2), device="cuda"), torch.zeros((8, 16), device="cuda")
    for call, text in [
            (lambda: apt_b200.route_experts(z, 9), "9 of 8 experts"), (lambda: apt_b200.route_experts(z, 0), "at least 1"),
            (lambda: apt_b200.route_experts(z, 2, "tanh"), "unknown score"), (lambda: apt_b200.route_experts(z, 2, num_groups=3), "3 groups"),
            (lambda: apt_b200.route_experts(z, 5, num_groups=4, top_groups=2), "2 of 4 groups"), (lambda: apt_b200.route_experts(z, 2, num_groups=4, top_groups=5), "5 of 4"),
            (lambda: apt_b200.route_experts(z, 2, num_groups=4, top_groups=2, group_best=3), "not 3"),
            (lambda: apt_b200.route_experts(z.double(), 2), "float64"), (lambda: apt_b200.route_experts(z[0], 2), "rows, experts"),
            (lambda: apt_b200.route_experts(z, 2, bias=torch.zeros(7, device="cuda")), "one value an expert"),
            (lambda: apt_b200.route_experts(z, 2, bias=torch.zeros(8, device="cuda").half()), "torch.float32"),
            (lambda: apt_b200.route_experts(torch.zeros((2, 1025), device="cuda"), 2), "1025 experts"),
            (lambda: apt_b200.route_experts_backward(z, e[:3], w[:3]), "rows, k"), (lambda: apt_b200.route_experts_backward(z, e, w[:, :1]), "like experts"),
            (lambda: apt_b200.expert_rows(x, e[:3], 8), "rows, k"), (lambda: apt_b200.expert_rows(x, e.int(), 8), "int64"), (lambda: apt_b200.expert_rows(x, e, 0), "at least 1"),
            (lambda: apt_b200.expert_rows(x, e, 5000), "5000 experts"), (lambda: apt_b200.expert_rows(x.double(), e, 8), "float64"),
            (lambda: apt_b200.expert_rows(x, e[:, :0], 8), "one expert a row"),
            (lambda: apt_b200.expert_sum(y[:7], w, e), "8 places"), (lambda: apt_b200.expert_sum(y, w[:3], e), "like place"),
            (lambda: apt_b200.expert_sum(y, w.half(), e), "torch.float32"), (lambda: apt_b200.expert_sum_backward(y, w, e, x.half()), "y's dtype"),
            (lambda: apt_b200.expert_rows(x, e.cpu(), 8), "CUDA tensor"), (lambda: apt_b200.route_experts(z.cpu(), 2), "CUDA tensor")]:
        with pytest.raises((RuntimeError, _lib.AptError), match=text):
            call()
