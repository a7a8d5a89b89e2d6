"""linear_cross_entropy against a plain implementation in 64 bits; its gradients against the formula's and against differences.

Bounds. A logit is a sum of K terms in fp32, at most K 2^-23 of its terms' magnitudes off (2^-21 more of them in pieces of fewer bits for
fp32; tensor cores cut sums off), and a loss is as much off as its logits are, with ten roundings of numbers of its logits' size:
loss <= (K 2^-23 + 2^-19) (max |x| . |w| + 8). Slopes: rounded to the type (half a step, HALF), of exponentials that are off by what the logits
are: with E = that and HALF, gradients are E times the sum of the magnitudes of their terms, p and the label's one, and a rounding of the
result. What cutting sums over rows or classes
off takes, in parts of 8192 terms (fp32: 1024): 3e-5 of the magnitudes.
"""
import pytest
import torch

import apt_b200
from apt_b200 import _lib, ops
from apt_b200._lib import check

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
IGNORE = -100


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(rows, dim, classes, dtype, bias=True, seed=1, scale=2.0, ignored=0.1):
    gen = _gen(seed + rows + 3 * dim + 7 * classes)
    x = torch.randn((rows, dim), device="cuda", generator=gen).to(dtype)
    w = (torch.randn((classes, dim), device="cuda", generator=gen) * scale * dim ** -0.5).to(dtype)
    b = (torch.randn(classes, device="cuda", generator=gen) * 0.5).to(dtype) if bias else None
    labels = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    labels[torch.rand(rows, device="cuda", generator=gen) < ignored] = IGNORE
    return x, w, b, labels


def _plain(x, w, b, labels, ignore=IGNORE):
    """(losses, slopes, rows that count) in 64 bits."""
    z = x.double() @ w.double().t() + (0 if b is None else b.double())
    counted = labels != ignore
    at = torch.where(counted, labels, 0).unsqueeze(1)
    lse = torch.logsumexp(z, 1)
    losses = torch.where(counted, lse - z.gather(1, at).squeeze(1), 0.0)
    slopes = torch.exp(z - lse.unsqueeze(1))
    magnitudes = slopes.clone()
    slopes.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    magnitudes.scatter_add_(1, at, torch.ones_like(at, dtype=torch.float64))
    return losses, torch.where(counted.unsqueeze(1), slopes, 0.0), torch.where(counted.unsqueeze(1), magnitudes, 0.0), counted


def _check(x, w, b, labels, reduction, ignore=IGNORE):
    rows, dim = x.shape
    dtype = x.dtype
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b) if t is not None]
    loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2] if b is not None else None, reduction, ignore)
    assert torch.equal(loss, apt_b200.linear_cross_entropy(x, w, labels, b, reduction, ignore)) and loss.dtype == torch.float32
    losses, slopes, magnitudes, counted = _plain(x, w, b, labels, ignore)
    count = max(1, int(counted.sum()))
    size = float((x.double().abs() @ w.double().abs().t()).max()) + (0 if b is None else float(b.double().abs().max()))
    off = (dim * 2.0 ** -23 + 2.0 ** -19) * (size + 8)
    want = losses if reduction == "none" else losses.sum() / (count if reduction == "mean" else 1)
    times = count if reduction == "sum" else 1
    assert bool(((loss.double() - want).abs() <= off * times + 2.0 ** -23 * want.abs()).all())
    grad = torch.rand(loss.shape, device="cuda", generator=_gen(3)) + 0.5
    got = torch.autograd.grad(loss, leaves, grad)
    g = (grad.double() / (count if reduction == "mean" else 1)).expand(rows).unsqueeze(1)
    slopes, magnitudes = slopes * g, magnitudes * g
    near = off + HALF[dtype] + 3e-5
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    pairs = [(got[0], slopes @ w.double(), magnitudes @ w.double().abs()), (got[1], slopes.t() @ x.double(), magnitudes.t() @ x.double().abs())]
    if b is not None:
        pairs.append((got[2], slopes.sum(0), magnitudes.sum(0)))
    for a, want, terms in pairs:
        assert a.dtype == dtype and bool(((a.double() - want).abs() <= near * terms + HALF[dtype] * want.abs() + tiny).all())
        # and in the 2-norm, where roundings that go either way take one another away: a result's own and those of its terms
        norm = float(want.norm())
        if norm:
            assert float((a.double() - want).norm()) <= (1.5 * HALF[dtype] + 1e-5 + off) * norm + tiny * want.numel() ** 0.5, (float((a.double() - want).norm()) / norm)
    if reduction != "none":
        assert not got[0][~counted].any()
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes", [(1, 1, 1), (1, 16, 2), (1, 64, 5000), (2, 7, 47), (15, 8, 16), (17, 100, 257), (100, 33, 1000), (128, 64, 256), (129, 72, 300),
                                              (300, 256, 47), (513, 128, 2983), (40, 1100, 700), (1000, 17, 130), (257, 520, 513)])
def test_loss_and_gradients(rows, dim, classes, dtype):
    x, w, b, labels = _inputs(rows, dim, classes, dtype)
    for reduction in ("mean", "sum", "none"):
        _check(x, w, b, labels, reduction)
    _check(x, w, None, labels, "mean")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes", [(3000, 256, 20_000), (20_000, 64, 700), (700, 1024, 9000), (9000, 512, 1500), (4, 128, 60_001), (2000, 72, 30_011), (9000, 300, 30_000)])
def test_larger(rows, dim, classes, dtype):
    x, w, b, labels = _inputs(rows, dim, classes, dtype)
    _check(x, w, b, labels, "mean")
    _check(x, w, None, labels, "none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_classes_in_several_pieces(dtype):
    """More slopes than are there at a time: 512 MB are 8192 x 32768 of 16 bits."""
    rows, classes = (8192, 40_000) if dtype != torch.float32 else (8192, 20_000)
    _check(*_inputs(rows, 40, classes, dtype), "mean")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_do_not_count(dtype):
    x, w, b, labels = _inputs(300, 64, 90, dtype)
    labels[:] = IGNORE
    for reduction in ("mean", "sum", "none"):
        _check(x, w, b, labels, reduction)
        assert not apt_b200.linear_cross_entropy(x, w, labels, b, reduction).any()
    labels[7] = 89
    for reduction in ("mean", "sum", "none"):
        _check(x, w, b, labels, reduction)
    # a class that is not asked for
    labels = torch.randint(0, 4, (300,), device="cuda", generator=_gen(1))
    _check(x, w, b, labels, "mean", ignore=2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    x, w, b, labels = _inputs(200, 96, 150, dtype)
    wide = torch.cat([x, x], 1)
    args = (labels, b, "none")
    want = apt_b200.linear_cross_entropy(x, w, *args)
    assert torch.equal(apt_b200.linear_cross_entropy(wide[:, 96:], w, *args), want)
    assert torch.equal(apt_b200.linear_cross_entropy(x.t().contiguous().t(), w, *args), want)
    flat = torch.cat([w.reshape(-1)[:1], w.reshape(-1)])
    assert torch.equal(apt_b200.linear_cross_entropy(x, flat[1:].view(150, 96), *args), want)
    assert torch.equal(apt_b200.linear_cross_entropy(x, w, torch.stack([labels, labels], 1)[:, 0], torch.stack([b, b], 1)[:, 0], "none"), want)


def test_a_row_that_is_all_but_sure():
    """Losses of 1e-6 have digits of their own: they are not the difference of two numbers of the logits' size."""
    x = torch.eye(4, device="cuda") * 30.0
    w = torch.zeros((6, 4), device="cuda")
    labels = torch.arange(4, device="cuda")
    for k in range(4):
        w[k, k] = 1.0
    # one other class 12 + k below the label's
    w[5] = torch.tensor([(30.0 - 12.0 - k) / 30.0 for k in range(4)], device="cuda")
    z = x.double() @ w.double().t()
    want = torch.log1p((torch.exp(z - z.gather(1, labels.unsqueeze(1))).sum(1) - 1))
    got = apt_b200.linear_cross_entropy(x, w, labels, None, "none")
    # the exponent is a multiply-add of numbers up to 43: 2^-24 of them; the sum is 1 + 6e-6 in steps of 2^-23, half a step of which remains
    assert float((got.double() - want).abs().max()) < 2 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_classes(dtype):
    """A bias of -inf, or of the type's lowest value, takes a class out."""
    x, w, b, labels = _inputs(150, 48, 400, dtype, ignored=0.0)
    labels %= 100
    out = torch.arange(400, device="cuda") >= 100
    want = apt_b200.linear_cross_entropy(x, w[:100], labels, b[:100], "none")
    for v in (-float("inf"), torch.finfo(dtype).min):
        masked = torch.where(out, torch.tensor(v, device="cuda", dtype=dtype), b)
        leaves = [t.clone().requires_grad_() for t in (x, w, masked)]
        loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2], "none")
        assert torch.allclose(loss, want, rtol=1e-5, atol=1e-5)
        gx, gw, gb = torch.autograd.grad(loss.sum(), leaves)
        assert torch.isfinite(gx).all() and not gw[100:].any() and not gb[100:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_wild_values_stay_in_their_rows(dtype):
    x, w, b, labels = _inputs(200, 64, 300, dtype, ignored=0.0)
    clean = apt_b200.linear_cross_entropy(x, w, labels, b, "none")
    wild = x.clone()
    wild[3] = float("nan")
    wild[77, 5] = float("inf")
    leaf = wild.clone().requires_grad_()
    got = apt_b200.LinearCrossEntropy.apply(leaf, w, labels, b, "none")
    fine = torch.ones(200, dtype=torch.bool, device="cuda")
    fine[3] = fine[77] = False
    assert torch.equal(got[fine], clean[fine]) and not torch.isfinite(got[~fine]).any()
    gx = torch.autograd.grad(got, leaf, torch.ones_like(got))[0]
    plain = x.clone().requires_grad_()
    want = torch.autograd.grad(apt_b200.LinearCrossEntropy.apply(plain, w, labels, b, "none"), plain, torch.ones_like(got))[0]
    assert torch.equal(gx[fine], want[fine]) and torch.isnan(gx[3]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes", [(200, 64, 300), (333, 100, 47), (100, 40, 24_000)])
def test_rows_that_do_not_count_may_hold_anything(rows, dim, classes, dtype):
    x, w, b, labels = _inputs(rows, dim, classes, dtype)
    out = labels == IGNORE
    clean = torch.where(out.unsqueeze(1), 0.0, x.float()).to(dtype)

    def step(x, reduction):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2], reduction)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, torch.ones_like(loss))

    for reduction in ("mean", "none"):
        want = step(clean, reduction)
        assert int(out.sum()) > 3 and all(torch.isfinite(t).all() for t in want)
        for v in (float("nan"), float("inf"), -float("inf")):
            wild = x.clone()
            wild[out, 3:] = v
            assert all(torch.equal(a, b) for a, b in zip(step(wild, reduction), want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes", [(200, 64, 300), (90, 33, 9000)])
def test_gradients_that_are_no_numbers_stay_in_their_rows(rows, dim, classes, dtype):
    """A row's own gradient that is infinite, or none: the other rows' dx is what it is without."""
    x, w, b, labels = _inputs(rows, dim, classes, dtype)
    labels[5], labels[9] = 3, IGNORE
    saved = apt_b200.linear_cross_entropy(x, w, labels, b, "none", return_saved=True)[1]
    fine = torch.arange(rows, device="cuda") != 5
    for size in (2.0 ** 10, 2.0 ** -12):
        grad = torch.full((rows,), size, device="cuda")
        want = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none")[0]
        assert torch.isfinite(want).all()
        for bad in (float("inf"), -float("inf"), float("nan")):
            grad[5], grad[9] = bad, bad
            got = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none")[0]
            assert torch.equal(got[fine], want[fine]) and not torch.isfinite(got[5]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes", [(200, 64, 300), (300, 128, 9000), (1, 40, 77)])
def test_rows_that_do_not_count_have_no_gradient_whatever_the_loss_has(rows, dim, classes, dtype):
    x, w, b, labels = _inputs(rows, dim, classes, dtype, ignored=0.3)
    labels[0] = IGNORE
    for none_counts in (False, True):
        if none_counts:
            labels = torch.full_like(labels, IGNORE)
        for reduction in ("mean", "sum", "none"):
            saved = apt_b200.linear_cross_entropy(x, w, labels, b, reduction, return_saved=True)[1]
            for bad in (float("inf"), -float("inf"), float("nan")):
                grad = torch.full((rows,) if reduction == "none" else (), bad, device="cuda")
                gx, gw, gb = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, reduction)
                counted = labels != IGNORE
                assert not gx[~counted].any() and not (gx[~counted] != gx[~counted]).any()
                if counted.any():
                    assert not torch.isfinite(gx[counted]).all(1).any() and not torch.isfinite(gw).any() and not torch.isfinite(gb).any()
                else:
                    assert all(torch.equal(t, torch.zeros_like(t)) for t in (gw, gb))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,classes,bias", [(300, 64, 50_000, True), (200, 32, 6000, False), (257, 33, 8000, True), (20_000, 64, 700, True),
                                                   (8192, 40, 40_000, False)])
def test_row_gradients_over_seven_decades(rows, dim, classes, bias, dtype):
    """dx of every row is right next to its own gradient. In f16 what a row adds to dW has steps of 2^-24 of 2^-14 of the largest gradient."""
    x, w, b, labels = _inputs(rows, dim, classes, dtype, bias=bias, scale=0.5)
    w += 1.0      # what probabilities lose as a whole shows in dx then
    grad = 1e3 * 10.0 ** (-7.0 * torch.arange(rows, device="cuda") / rows)
    grad[::3] *= -1.0
    grad[7] = 0.0
    _, slopes, magnitudes, counted = _plain(x, w, b, labels)
    size = float((x.double().abs() @ w.double().abs().t()).max()) + (float(b.double().abs().max()) if bias else 0.0)
    near, half = (dim * 2.0 ** -23 + 2.0 ** -19) * (size + 8) + HALF[dtype] + 3e-5, HALF[dtype]
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    saved = apt_b200.linear_cross_entropy(x, w, labels, b, "none", return_saved=True)[1]
    g = grad.double().unsqueeze(1)
    slopes, magnitudes = slopes * g, magnitudes * g.abs()
    step = 2.0 ** -39 * 1e3 if dtype == torch.float16 else 0.0
    wants = [(slopes @ w.double(), magnitudes @ w.double().abs(), 0.0), (slopes.t() @ x.double(), magnitudes.t() @ x.double().abs(), step * float(x.double().abs().sum(0).max()))]
    if bias:
        wants.append((slopes.sum(0), magnitudes.sum(0), step * rows))
    every = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none")
    for i, (want, terms, least) in enumerate(wants):
        alone = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none", i == 0, i == 1, i == 2)[i]
        for got in (every[i], alone):
            assert bool(((got.double() - want).abs() <= near * terms + half * want.abs() + tiny + least).all())
        assert i == 2 or torch.equal(every[i], alone)
    assert not every[0][~counted].any() and not every[0][7].any()
    fine = torch.arange(rows, device="cuda") != 11
    grad[~counted], grad[11] = float("nan"), float("inf")
    assert torch.equal(apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none", True, False, False)[0][fine], every[0][fine])
    ops.check_status()



@pytest.mark.parametrize("rows,dim,classes", [(300, 64, 5000), (20_000, 64, 700)])
def test_a_captured_backward_takes_row_gradients_of_any_range(rows, dim, classes):
    """f16: whether slopes are made once or twice goes by the gradients that are there at the replay."""
    x, w, b, labels = _inputs(rows, dim, classes, torch.float16)
    saved = apt_b200.linear_cross_entropy(x, w, labels, b, "none", return_saved=True)[1]
    near = torch.rand(rows, device="cuda", generator=_gen(1)) + 0.5
    far = near * 10.0 ** (-6.0 * torch.arange(rows, device="cuda") / rows)
    grad = near.clone()

    def call():
        return apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b, "none")

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    torch.cuda.current_stream().wait_stream(side)
    seen = []
    for now in (far, near, far):
        grad.copy_(now)
        graph.replay()
        seen.append([t.clone() for t in captured])
        assert all(torch.equal(a, b) for a, b in zip(seen[-1], call()))
    assert all(torch.equal(a, b) for a, b in zip(seen[0], seen[2])) and not torch.equal(seen[0][0], seen[1][0])
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("polls", [0, 1, 6, 50])
@pytest.mark.parametrize("rows,dim,classes", [(300, 128, 700), (3000, 64, 1500), (700, 1024, 25_000)])
def test_the_kernels_end_when_a_wait_runs_out(rows, dim, classes, dtype, polls):
    x, w, b, labels = _inputs(rows, dim, classes, dtype)
    saved = apt_b200.linear_cross_entropy(x, w, labels, b, return_saved=True)[1]
    grad = torch.ones((), device="cuda")

    def call():
        return (apt_b200.linear_cross_entropy(x, w, labels, b),) + apt_b200.linear_cross_entropy_backward(x, w, labels, saved, grad, b)

    want = call()
    ops.check_status()
    check(_lib.lib.apt_set_tunable(b"bulk_wait_polls", polls))
    try:
        got = call()
        torch.cuda.synchronize()
    finally:
        check(_lib.lib.apt_set_tunable(b"bulk_wait_polls", 1 << 20))
    flagged = False
    try:
        ops.check_status()
    except RuntimeError as e:
        assert "did not reach shared memory" in str(e)
        flagged = True
    assert flagged or (polls > 0 and all(torch.equal(a, b) for a, b in zip(got, want)))
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
    ops.check_status()


def test_small_gradients_of_f16_are_numbers():
    """A mean over many rows makes slopes of 1e-9, below f16's smallest number: they are held times the common factor."""
    x, w, b, labels = _inputs(4096, 32, 3000, torch.float16, scale=0.5, ignored=0.0)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss = apt_b200.LinearCrossEntropy.apply(*leaves, labels, None, "mean")
    scale = torch.tensor(2.0 ** 20, device="cuda")
    got = torch.autograd.grad(loss, leaves, scale)
    _, slopes, _, _ = _plain(x, w, None, labels)
    for a, want in zip(got, (slopes @ w.double(), slopes.t() @ x.double())):
        want = want * 2.0 ** 20 / 4096
        assert float((a.double() - want).norm() / want.norm()) < 2 * 2.0 ** -11


def test_gradient_against_differences():
    x, w, b, labels = _inputs(9, 12, 31, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2], "mean")
    grads = torch.autograd.grad(loss, leaves)
    for i, leaf in enumerate((x, w, b)):
        for seed in range(4):
            d = torch.randn(leaf.shape, device="cuda", generator=_gen(seed), dtype=torch.float64)
            d /= d.norm()
            args = [t.double() for t in (x, w, b)]

            def value(step):
                moved = list(args)
                moved[i] = moved[i] + step * d
                losses, _, _, counted = _plain(*moved, labels)
                return float(losses.sum() / counted.sum())

            slope = (value(1e-4) - value(-1e-4)) / 2e-4
            # the third derivative of a mean of losses along a unit direction is below 2 (max |x|, |w| row norms, 6)^3
            assert abs(float((grads[i].double() * d).sum()) - slope) < 2 * 6 ** 3 * 1e-8 / 6 + 2e-5


def test_labels_that_are_none_are_reported():
    x, w, b, labels = _inputs(70, 16, 20, torch.float32, ignored=0.0)
    for bad in (20, -1, 2 ** 40, -2 ** 40):
        marked = labels.clone()
        marked[33] = bad
        got, saved = apt_b200.linear_cross_entropy(x, w, marked, b, "none", return_saved=True)
        with pytest.raises(RuntimeError, match="id outside"):
            ops.check_status()
        gx = apt_b200.linear_cross_entropy_backward(x, w, marked, saved, torch.ones_like(got), b, "none")[0]
        assert got[33] == 0 and not gx[33].any() and gx[32].any()
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_each_gradient_alone(dtype):
    x, w, b, labels = _inputs(260, 40, 600, dtype)
    loss, saved = apt_b200.linear_cross_entropy(x, w, labels, b, return_saved=True)
    g = torch.tensor(1.5, device="cuda")
    every = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, g, b)
    for k in range(3):
        wants = [k == 0, k == 1, k == 2]
        alone = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, g, b, "mean", *wants)
        assert [t is not None for t in alone] == wants
        if k < 2:
            assert torch.equal(alone[k], every[k])
        else:      # another order of sums in fp32
            assert float((alone[2].double() - every[2].double()).abs().max()) <= 2 * HALF[dtype] * float(every[2].double().abs().max()) + 1e-6
    assert apt_b200.linear_cross_entropy_backward(x, w, labels, saved, g, b, "mean", False, False, False) == (None, None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_again_and_again(dtype):
    x, w, b, labels = _inputs(5000, 96, 3000, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def step():
        loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2])
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)

    first = step()
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


@pytest.mark.parametrize("rows,dim,classes,dtype", [(8_500_000, 24, 250, torch.bfloat16)] + [(200_000, 16, 50_000, dtype) for dtype in DTYPES])
def test_more_than_31_bits_of_slopes(rows, dim, classes, dtype):
    """Rows of which the first and the last ones count: what these are alone. Slopes at once, and in many pieces, with statistics in several."""
    n = 400
    x, w, b, _ = _inputs(rows, dim, classes, dtype)
    some = torch.cat([torch.arange(n, device="cuda"), torch.arange(rows - n, rows, device="cuda")])
    labels = torch.full((rows,), IGNORE, device="cuda")
    labels[some] = torch.randint(0, classes, (2 * n,), device="cuda", generator=_gen(5))
    loss, saved = apt_b200.linear_cross_entropy(x, w, labels, b, "sum", return_saved=True)
    losses, slopes, magnitudes, _ = _plain(x[some], w, b, labels[some])
    off = (dim * 2.0 ** -23 + 2.0 ** -19) * (float((x[some].double().abs() @ w.double().abs().t()).max()) + float(b.double().abs().max()) + 8)
    assert abs(float(loss) - float(losses.sum())) <= off * 2 * n + 2.0 ** -23 * float(losses.sum())
    gx, gw, gb = apt_b200.linear_cross_entropy_backward(x, w, labels, saved, torch.ones((), device="cuda"), b, "sum")
    near, half, tiny = off + HALF[dtype] + 3e-5, HALF[dtype], torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for got, want, terms in ((gx[some], slopes @ w.double(), magnitudes @ w.double().abs()), (gw, slopes.t() @ x[some].double(), magnitudes.t() @ x[some].double().abs()),
                             (gb, slopes.sum(0), magnitudes.sum(0))):
        assert bool(((got.double() - want).abs() <= near * terms + half * want.abs() + tiny).all())
    gx[some] = 0
    assert not gx.any()
    ops.check_status()


def test_another_stream_and_a_captured_graph():
    x, w, b, labels = _inputs(600, 64, 900, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def step():
        loss = apt_b200.LinearCrossEntropy.apply(leaves[0], leaves[1], labels, leaves[2])
        return (loss,) + torch.autograd.grad(loss, leaves)

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
        leaves[0].copy_(leaves[0].flip(0).clone())
        labels.copy_(labels.roll(5))
    graph.replay()
    again = [t.detach().clone() for t in captured]
    assert all(torch.equal(a, b.detach()) for a, b in zip(again, step()))
    assert not torch.equal(again[0], want[0])
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    w, b = torch.randn((9, 16), device="cuda").to(dtype).requires_grad_(), torch.zeros(9, device="cuda", dtype=dtype).requires_grad_()
    x, labels = torch.empty((0, 16), device="cuda", dtype=dtype).requires_grad_(), torch.empty(0, device="cuda", dtype=torch.int64)
    for reduction in ("mean", "sum", "none"):
        loss = apt_b200.LinearCrossEntropy.apply(x, w, labels, b, reduction)
        assert not loss.any() and loss.shape == ((0,) if reduction == "none" else ())
        gx, gw, gb = torch.autograd.grad(loss, [x, w, b], torch.ones_like(loss))
        assert gx.shape == (0, 16) and not gw.any() and not gb.any()


def test_second_derivatives_raise():
    x, w, _, labels = _inputs(9, 12, 31, torch.float32)
    leaf = x.clone().requires_grad_()
    g = torch.autograd.grad(apt_b200.LinearCrossEntropy.apply(leaf, w, labels), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(g.sum(), leaf)


def test_refusals():
    x, w, b, labels = _inputs(9, 12, 31, torch.float32)
    for call, text in [
            (lambda: apt_b200.linear_cross_entropy(x, w, labels, b, "all"), "unknown reduction"), (lambda: apt_b200.linear_cross_entropy(x, w[:, :11], labels), "classes, dim"),
            (lambda: apt_b200.linear_cross_entropy(x, w.half(), labels), "mixed dtypes"), (lambda: apt_b200.linear_cross_entropy(x.double(), w.double(), labels), "float64"),
            (lambda: apt_b200.linear_cross_entropy(x, w, labels.int()), "int64"), (lambda: apt_b200.linear_cross_entropy(x, w, labels[:8]), "labels must be"),
            (lambda: apt_b200.linear_cross_entropy(x, w, labels, b[:30]), "bias must be"), (lambda: apt_b200.linear_cross_entropy(x, w, labels, b.half()), "mixed dtypes"),
            (lambda: apt_b200.linear_cross_entropy(x, w.cpu(), labels), "CUDA tensor"), (lambda: apt_b200.linear_cross_entropy(x, w[:0], labels), "0 classes"),
            (lambda: apt_b200.linear_cross_entropy(torch.zeros((2, 8200), device="cuda"), torch.zeros((3, 8200), device="cuda"), labels[:2]), "rows of 8200"),
            (lambda: apt_b200.linear_cross_entropy_backward(x, w, labels, torch.zeros(5, device="cuda"), torch.zeros((), device="cuda")), "saved"),
            (lambda: apt_b200.linear_cross_entropy_backward(x, w, labels, torch.zeros(20, device="cuda"), torch.zeros(9, device="cuda")), "like the loss")]:
        with pytest.raises((RuntimeError, _lib.AptError), match=text):
            call()
