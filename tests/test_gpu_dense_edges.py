"""The operators of a layer's dense half where they end: waits that run out, sizes at the ends of what a call takes, numbers that a mean error
would hide."""
import numpy as np
import pytest
import torch

import apt_b200
from apt_b200 import ops
from apt_b200._lib import check, lib

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ends(*sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), device="cuda")


# ------------------------------------------------------------------------------------------------- grouped products
def _given_up(call, polls):
    """The call's results with so few polls a wait, and whether one of them ran out."""
    check(lib.apt_set_tunable(b"bulk_wait_polls", polls))
    try:
        got = call()
        torch.cuda.synchronize()
    finally:
        check(lib.apt_set_tunable(b"bulk_wait_polls", 1 << 20))
    try:
        ops.check_status()
    except RuntimeError as e:
        assert "did not reach shared memory" in str(e)
        return got, True
    return got, False


def _right_or_flagged(call, polls):
    want = call()
    ops.check_status()
    got, flagged = _given_up(call, polls)
    assert flagged or all(torch.equal(a, b) for a, b in zip(got, want))
    assert flagged or polls > 0
    for a, b in zip(call(), want):
        assert torch.equal(a, b)
    ops.check_status()


# weights that stay in shared memory, tiles in pairs, two blocks a stage, few rows a group
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,dim,out_dim", [([60000, 1], 128, 256), ([40000, 40000], 1024, 264), ([300, 0, 5], 256, 40), ([3] * 64, 1024, 512)])
@pytest.mark.parametrize("polls", [0, 1, 6, 50])
def test_products_of_rows_end_when_a_wait_runs_out(sizes, dim, out_dim, dtype, polls):
    gen = _gen(1)
    make = lambda *shape: torch.randn(shape, device="cuda", generator=gen).to(dtype)
    offsets, rows = _ends(*sizes), sum(sizes)
    x, weight, bias, grad = make(rows, dim), make(len(sizes), out_dim, dim), make(len(sizes), out_dim), make(rows, out_dim)
    _right_or_flagged(lambda: (apt_b200.grouped_linear(x, weight, offsets, bias),
                               apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_weight=False, want_bias=False)[0]), polls)


# sums within a run and across runs, groups without rows, an end within a stage
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,dim,out_dim", [([60000, 1], 128, 256), ([4000, 0, 777], 264, 136), ([3] * 64, 256, 512), ([17], 16, 8)])
@pytest.mark.parametrize("polls", [0, 1, 6, 50])
def test_weight_gradients_end_when_a_wait_runs_out(sizes, dim, out_dim, dtype, polls):
    """The partial sums that a run did not make are not there; which of them belong together the join knows all the same."""
    gen = _gen(2)
    make = lambda *shape: torch.randn(shape, device="cuda", generator=gen).to(dtype)
    offsets, rows = _ends(*sizes), sum(sizes)
    x, weight, grad = make(rows, dim), make(len(sizes), out_dim, dim), make(rows, out_dim)
    _right_or_flagged(lambda: apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_x=False)[1:], polls)


def test_infinite_results_take_no_longer():
    """Rows that are infinite all over, long contractions: right, and without a wait that runs out."""
    gen = _gen(3)
    rows, dim, n = 2000, 4096, 512
    offsets = _ends(1500, 300, 200)
    x, weight = torch.randn((rows, dim), device="cuda", generator=gen), torch.randn((3, n, dim), device="cuda", generator=gen)
    grad = torch.randn((rows, n), device="cuda", generator=gen)
    calm = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    wild = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    def both(events):
        for k in range(2):
            events[0].record()
            got = (apt_b200.grouped_linear(x, weight, offsets),) + apt_b200.grouped_linear_backward(x, weight, offsets, grad)
            events[1].record()
        torch.cuda.synchronize()
        return got

    both(calm)
    x[:, 17] = float("inf")
    grad[:, 5] = float("-inf")
    out, gx, gw, gb = both(wild)
    ops.check_status()
    for g, (b, e) in enumerate(((0, 1500), (1500, 1800), (1800, 2000))):
        assert torch.equal(out[b:e], torch.copysign(torch.full((e - b, n), float("inf"), device="cuda"), weight[g, :, 17].expand(e - b, n)))
        assert torch.equal(gx[b:e], torch.copysign(torch.full((e - b, dim), float("inf"), device="cuda"), -weight[g, 5].expand(e - b, dim)))
        # infinite terms of either sign in one sum, but where an infinite factor meets the other
        nan = torch.zeros((n, dim), dtype=torch.bool, device="cuda")
        nan[:, 17] = nan[5] = True
        nan[5, 17] = False
        assert torch.equal(torch.isnan(gw[g]), nan) and float(gw[g, 5, 17]) == float("-inf") == float(gb[g, 5])
    assert wild[0].elapsed_time(wild[1]) < 4 * calm[0].elapsed_time(calm[1])


@pytest.mark.parametrize("bits", [0x7FC00000, 0x7F800001, -1, 0xFF800001 - 2 ** 32])
def test_a_nan_is_one_whatever_its_bits(bits):
    gen = _gen(4)
    x, weight = torch.randn((200, 64), device="cuda", generator=gen), torch.randn((1, 48, 64), device="cuda", generator=gen)
    x[77].view(torch.int32)[9] = bits
    weight[0, 30].view(torch.int32)[3] = bits
    offsets = _ends(200)
    out = apt_b200.grouped_linear(x, weight, offsets)
    nan = torch.zeros((200, 48), dtype=torch.bool, device="cuda")
    nan[77], nan[:, 30] = True, True
    assert torch.equal(torch.isnan(out), nan) and torch.isfinite(out[~nan]).all()
    grad = torch.randn((200, 48), device="cuda", generator=gen)
    gx, gw, _ = apt_b200.grouped_linear_backward(x, weight, offsets, grad)
    assert torch.isnan(gx[:, 3]).all() and torch.isfinite(gx[:, :3]).all() and torch.isnan(gw[0, :, 9]).all() and torch.isfinite(gw[0, :, :9]).all()
    ops.check_status()


def _one_sign(*shape, seed, dtype=torch.float32, scale=1.0):
    """Numbers of 0.5 to 1.5, and columns of factors of 1 to 2, so that roundings of their sums are of either sign."""
    gen = _gen(seed)
    return ((torch.rand(shape, device="cuda", generator=gen) + 0.5) * (torch.rand(shape[-1], device="cuda", generator=gen) + 1.0) * scale).to(dtype)


# A part of a sum has at most 64 steps of 16 terms, each of which loses less than a unit of 2^-23 of it; eight parts are rounded as they are added up,
# and operands taken apart lose 2^-22: 74 units, whatever the number of terms. In one sum 8192 terms lose 216 units.
@pytest.mark.parametrize("dim,n", [(1024, 130), (1040, 64), (2049, 47), (8192, 200), (8190, 130)])
def test_long_contractions_of_one_sign(dim, n):
    offsets = _ends(200, 0, 101)
    for rows_of, out_dim in ((dim, n), (n, dim)):
        x, weight = _one_sign(310, rows_of, seed=6), _one_sign(3, out_dim, rows_of, seed=7)
        bias, grad = _one_sign(3, out_dim, seed=8), _one_sign(310, out_dim, seed=9)
        out = apt_b200.grouped_linear(x, weight, offsets, bias)
        gx = apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_weight=False, want_bias=False)[0]
        for g, (b, e) in enumerate(((0, 200), (200, 200), (200, 301))):
            for got, want in ((out, x[b:e].double() @ weight[g].double().T + bias[g].double()), (gx, grad[b:e].double() @ weight[g].double())):
                assert ((got[b:e].double() - want).abs() <= 74 * 2.0 ** -23 * want).all()
        assert not out[301:].any() and not gx[301:].any()
    ops.check_status()


# Parts of 8192 rows (fp32: 1024) have 512 (64) steps, and are added up one by one with errors of either sign, m of them: sqrt(m) / 2 units at three
# deviations. The mean over what is looked at has the roundings of the results, uniform in half a unit of theirs, as noise besides, at five deviations.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,dim,n", [([262144], 512, 264), ([131072], 1100, 1000), ([70000, 3, 60007], 130, 70)])
def test_weight_gradients_of_long_groups_of_one_sign(sizes, dim, n, dtype):
    rows = sum(sizes)
    x, grad = _one_sign(rows, dim, seed=10, dtype=dtype, scale=1 / 64), _one_sign(rows, n, seed=11, dtype=dtype, scale=1 / 64)
    weight = torch.zeros((len(sizes), n, dim), device="cuda", dtype=dtype)
    _, gw, gb = apt_b200.grouped_linear_backward(x, weight, _ends(*sizes), grad, want_x=False)
    ops.check_status()
    steps, unit = (64, 0.0) if dtype == torch.float32 else (512, UNIT[dtype])
    end = 0
    for g, size in enumerate(sizes):
        b, end = end, end + size
        for columns in (slice(0, 40), slice(n - 40, n)):
            want = grad[b:end, columns].double().T @ x[b:end].double()
            off = (gw[g, columns].double() - want) / want
            parts = size / (16 * steps) + 1
            loss = (steps + 3 * parts ** 0.5 / 2 + 4) * 2.0 ** -23
            assert float(off.abs().max()) <= loss + unit
            assert abs(float(off.mean())) <= loss + 5 * unit / (3 * off.numel()) ** 0.5
        want = grad[b:end].double().sum(0)
        assert (((gb[g].double() - want) / want).abs() <= 2e-6 + unit).all()


def test_weight_gradients_of_very_many_tiles():
    """4096 tiles of 16500 rows: as many runs as there are blocks, and no more."""
    rows, dim = 16500, 8192
    x, grad = torch.randn((rows, dim), device="cuda", generator=_gen(12)), torch.randn((rows, dim), device="cuda", generator=_gen(13))
    weight = torch.zeros((2, dim, dim), device="cuda")
    gw = apt_b200.grouped_linear_backward(x, weight, _ends(16000, 500), grad, want_x=False)[1]
    ops.check_status()
    for g, (b, e) in enumerate(((0, 16000), (16000, 16500))):
        for some in (slice(0, 64), slice(4000, 4064), slice(8128, 8192)):
            want = grad[b:e, some].double().T @ x[b:e].double()
            size = grad[b:e, some].double().abs().T @ x[b:e].double().abs()
            assert ((gw[g, some].double() - want).abs() <= 80 * 2.0 ** -23 * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,out_dim", [([1, 0, 300, 5000, 31], 70), ([0], 1), ([33] * 200, 32), ([20000], 257)])
def test_the_gradient_of_the_bias_alone(sizes, out_dim, dtype):
    """Sums of a column: 256 rows' side by side, 8 of them and then 32 partial ones added up, in all 20000 / 256 + 40 roundings of either sign."""
    rows, offsets = sum(sizes) + 9, _ends(*sizes)
    grad = torch.randn((rows, out_dim), device="cuda", generator=_gen(5)).to(dtype)
    grad[sum(sizes):] = float("nan")      # of no group
    x, weight = torch.randn((rows, 8), device="cuda").to(dtype), torch.randn((len(sizes), out_dim, 8), device="cuda").to(dtype)
    gx, gw, gb = apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_x=False, want_weight=False)
    assert gx is None and gw is None
    ends = offsets.tolist()
    for g, (b, e) in enumerate(zip(ends, ends[1:])):
        want, size = grad[b:e].double().sum(0), grad[b:e].double().abs().sum(0)
        assert ((gb[g].double() - want).abs() <= 32 * 2.0 ** -24 * size + UNIT[dtype] * want.abs()).all()
    bias = torch.zeros((len(sizes), out_dim), device="cuda", dtype=dtype, requires_grad=True)
    out = apt_b200.GroupedLinear.apply(x, weight, offsets, bias)
    assert torch.equal(torch.autograd.grad(out, bias, grad)[0], gb)
    # with the weight's, whose kernel makes it beside: another order
    _, _, beside = apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_x=False)
    for g, (b, e) in enumerate(zip(ends, ends[1:])):
        size = grad[b:e].double().abs().sum(0)
        assert ((gb[g].double() - beside[g].double()).abs() <= 64 * 2.0 ** -24 * size + 2 * UNIT[dtype] * gb[g].double().abs()).all()
    ops.check_status()


# ------------------------------------------------------------------------------------------------------ group norm
def test_statistics_of_segments_without_rows_are_zeros():
    for rows in (0, 7):
        filled = torch.full((4, 3, 2), 7.0, device="cuda")
        del filled      # what the statistics are written to held something else before
        offsets = torch.tensor([0, 0, rows, rows, rows], device="cuda")
        _, stats = apt_b200.group_norm_act(torch.randn((rows, 12), device="cuda"), 3, offsets=offsets, return_stats=True)
        assert stats.shape == (4, 3, 2) and not stats[[0, 2, 3]].any() and bool(stats[1].all()) == (rows > 0)
    ops.check_status()


def test_blocks_without_rows_are_segments():
    x = torch.zeros((5, 0, 12), device="cuda")
    weight = torch.ones(12, device="cuda")
    y, stats = apt_b200.group_norm_act(x, 3, weight, return_stats=True)
    assert y.shape == x.shape and stats.shape == (5, 3, 2) and not stats.any()
    gx, gw, _ = apt_b200.group_norm_act_backward(x, x, stats, 3, weight)
    assert gx.shape == x.shape and not gw.any()
    for empty in (torch.zeros((0, 4, 12), device="cuda"), torch.zeros((0, 12), device="cuda")):
        assert apt_b200.group_norm_act(empty, 3, return_stats=True)[1].shape == (0, 3, 2)


# tiles of segments, many segments (joined eight a block), groups that a block walks over
@pytest.mark.parametrize("dim,segments", [(64, 2), (64, 1500), (4106, 2)])
def test_the_backward_looks_at_the_ends_too(dim, segments):
    x = torch.randn((2000, dim), device="cuda", generator=_gen(14))
    good = torch.arange(segments + 1, device="cuda")
    good[-1] = 2000
    _, stats = apt_b200.group_norm_act(x, 2, offsets=good, return_stats=True)
    ops.check_status()
    for place, end in ((0, 1), (1, 1999), (-1, 2001), (1, -5)):
        bad = good.clone()
        bad[place] = end
        if segments == 1500 or not (bad.diff() >= 0).all() or place != 1:
            apt_b200.group_norm_act_backward(x, x, stats, 2, offsets=bad)
            with pytest.raises(RuntimeError, match="row groups"):
                ops.check_status()
    apt_b200.group_norm_act_backward(x, x, stats, 2, offsets=good)
    ops.check_status()


def test_ends_of_calls_without_rows_are_looked_at():
    x, weight = torch.zeros((0, 16), device="cuda"), torch.ones((2, 4, 16), device="cuda")
    grad, stats = torch.zeros((0, 4), device="cuda"), torch.zeros((2, 2, 2), device="cuda")
    for ends in ([0, 0, 0], [0, 0, 5], [1, 1, 1], [0, 3, 0]):
        offsets = torch.tensor(ends, device="cuda")
        for call in (lambda: apt_b200.grouped_linear(x, weight, offsets), lambda: apt_b200.grouped_linear_backward(x, weight, offsets, grad),
                     lambda: apt_b200.group_norm_act(x, 2, offsets=offsets), lambda: apt_b200.group_norm_act_backward(x, x, stats, 2, offsets=offsets)):
            call()
            if any(ends):
                with pytest.raises(RuntimeError, match="row groups"):
                    ops.check_status()
            ops.check_status()


def _statistics(x, groups, ends):
    """Mean and 1 / deviation of each segment that has rows, in 64 bits."""
    v = [x[b:e].double().view(e - b, groups, -1) for b, e in zip(ends, ends[1:])]
    return torch.stack([t.mean((0, 2)) for t in v]), torch.stack([1 / torch.sqrt(t.var((0, 2), unbiased=False) + 1e-5) for t in v])


# 301 with a deviation of 0.3. A mean is a sum rounded eight times as it is joined: 16 units. The variance's terms are 0.3^2, off by 2^-22 of themselves
# each way and by the square of the mean's error, (3e-4)^2: 2e-5 of it. A sum whose losses are lost had the mean off by 0.27 in 20000 rows of 2053.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,groups,sizes", [(2053, 1, [19000, 1000]), (70001, 1, [1, 2]), (4106, 2, [1, 3000])])
def test_groups_that_a_block_walks_over_far_from_zero(dim, groups, sizes, dtype):
    x = (torch.randn((sum(sizes), dim), device="cuda", generator=_gen(15)) * 0.3 + 301.0).to(dtype)
    ends = _ends(*sizes)
    _, stats = apt_b200.group_norm_act(x, groups, offsets=ends, return_stats=True)
    mean, rstd = _statistics(x, groups, ends.tolist())
    assert ((stats[..., 0].double() - mean).abs() <= 16 * 2.0 ** -24 * 302).all()
    assert ((stats[..., 1].double() / rstd - 1).abs() <= 2e-5).all()


def test_a_gradient_without_a_slope_over_a_long_segment():
    """dxh is 0.9 everywhere, so dx is zero but for roundings of its three terms: 2^-22 of 0.9 and of |xh|'s share of the second mean, itself zero but for
    the mean of xh (2e-5) and roundings."""
    rows, dim = 40000, 2053
    x = torch.randn((rows, dim), device="cuda", generator=_gen(16))
    ends = _ends(rows)
    _, stats = apt_b200.group_norm_act(x, 1, offsets=ends, return_stats=True)
    grad = apt_b200.group_norm_act_backward(x, torch.full_like(x, 0.9), stats, 1, offsets=ends)[0]
    assert float(grad.abs().max()) <= 0.9 * (2.0 ** -22 + 7 * 2e-5)


def _time(call):
    """The shorter of two calls behind a first one, in milliseconds."""
    call()
    times = []
    for _ in range(2):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


# groups of which not one is a whole number of 16-byte slices, in rows that are, of more than a block's columns
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,groups", [(4104, 8), (4112, 16), (4120, 2), (2056, 8), (2570, 10)])
def test_segments_of_groups_of_odd_widths(dim, groups, dtype):
    sizes = [12000, 1, 0, 8000]
    ends, rows = _ends(*sizes), sum(sizes)
    x = (torch.randn((rows, dim), device="cuda", generator=_gen(17)) * 0.3 + 301.0).to(dtype)
    call = lambda t, o: apt_b200.group_norm_act(t, groups, offsets=o, act="silu", return_stats=True)
    _, stats = call(x, ends)
    mean, rstd = _statistics(x, groups, [0, 12000, 12001, 20001])
    some = [0, 1, 3]
    assert ((stats[some, :, 0].double() - mean).abs() <= 16 * 2.0 ** -24 * 302).all()
    assert ((stats[some, :, 1].double() / rstd - 1).abs() <= 2e-5).all() and not stats[2].any()
    # single elements take six times as long as whole slices, one block for a long segment's group thirty times and more
    even = torch.randn((rows, 2048), device="cuda", generator=_gen(18)).to(dtype)
    assert _time(lambda: call(x, ends)) < 12 * (dim / 2048) * _time(lambda: apt_b200.group_norm_act(even, 8, offsets=ends, act="silu"))


# more than 65535 times what a block has of them: of rows by themselves 8 groups, and 256 where a group is one channel; of segments 64 in the join
@pytest.mark.parametrize("dim,groups,sizes", [(17 * 600_000, 600_000, None), (16_777_215, 16_777_215, None), (5_000_000, 5_000_000, [2])])
def test_very_many_groups(dim, groups, sizes):
    x = torch.randn((2, dim), device="cuda", generator=_gen(19))
    ends = None if sizes is None else _ends(*sizes)
    out, stats = apt_b200.group_norm_act(x, groups, offsets=ends, return_stats=True)
    grad, _, _ = apt_b200.group_norm_act_backward(x, x, stats, groups, offsets=ends)
    ops.check_status()
    for part in (slice(0, 17 * 64), slice(dim - 17 * 64 if dim % 17 == 0 else dim - 64, dim)):
        v = x[:, part].double()
        v = v.view(2, -1, dim // groups) if sizes is None else v.t().reshape(1, -1, 2)
        mean, var = v.mean(2, keepdim=True), v.var(2, unbiased=False, keepdim=True)
        rstd = 1 / torch.sqrt(var + 1e-5)
        xh = (v - mean) * rstd
        dx = rstd * (v - mean - xh * (v * xh).mean(2, keepdim=True))
        back = lambda t: t.reshape(2, -1) if sizes is None else t.view(-1, 2).t()
        # ten roundings of numbers of at most |x| rstd, which the gradient multiplies by rstd: 316 each at most
        assert ((out[:, part].double() - back(xh)).abs() <= 2e-6 * back(v.abs() * rstd + rstd * mean.abs()) + 1e-7).all()
        assert ((grad[:, part].double() - back(dx)).abs() <= 2e-5 * back(rstd * (v.abs() + mean.abs()) * (1 + xh * xh)) + 1e-7).all()


# Without a slope of its own (gamma 0) z is beta. q's exponent z^2 / 2 is a product of three numbers, rounded each: 1.5 z^2 units of 2^-24; the exponential, the
# reciprocal, the polynomial (6; of 16 bits 20) and the products: 24 (38) units. Below -13 the exponential is smaller than a normal number, and f16 ends at
# 2^-24, bf16's normal numbers at 2^-126.
@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_where_it_is_small(dtype):
    z = torch.linspace(-13.0, 13.0, 4096, device="cuda")
    x, gamma = torch.randn((1, 4096), device="cuda", generator=_gen(20)).to(dtype), torch.zeros(4096, device="cuda")
    out, stats = apt_b200.group_norm_act(x, 1, gamma, z, act="gelu", return_stats=True)
    slope = apt_b200.group_norm_act_backward(x, torch.ones_like(x), stats, 1, gamma, z, act="gelu")[2]
    wide = z.double()
    below = 0.5 * torch.erfc(-wide / 2 ** 0.5)
    density = torch.exp(-wide * wide / 2) / (2 * np.pi) ** 0.5
    share = (1.5 * wide * wide + (24 if dtype == torch.float32 else 38)) * 2.0 ** -24
    least = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
    assert ((out[0].double() - wide * below).abs() <= (share + UNIT[dtype] * (1 + share)) * (wide * below).abs() + least).all()
    assert ((slope.double() - (below + wide * density)).abs() <= share * (below + wide.abs() * density)).all()
    low, high = (apt_b200.group_norm_act(x, 1, gamma, torch.full_like(z, end), act="gelu") for end in (-40.0, 40.0))
    assert not low.any() and (high == 40.0).all()


# ------------------------------------------------------------------------------------------------------ derivatives
def test_second_derivatives_are_right_or_refused():
    x = torch.randn((6, 8), device="cuda", generator=_gen(21), requires_grad=True)
    weight = torch.randn((2, 4, 8), device="cuda", generator=_gen(22), requires_grad=True)
    y = apt_b200.Dropout.apply(x, 0.5, 1)
    g = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)[0]
    keep = 2.0 * (apt_b200.dropout(torch.ones_like(x), 0.5, 1) > 0)
    assert torch.equal(g, 3 * (x * keep) ** 2 * keep)
    assert torch.allclose(torch.autograd.grad(g.sum(), x)[0], 6 * x * keep ** 3, rtol=1e-6)
    for name, y in (("grouped_linear", apt_b200.GroupedLinear.apply(x, weight, _ends(2, 4))),
                    ("group_norm_act", apt_b200.GroupNormAct.apply(x, 2, None, None, None, 1e-5, "silu"))):
        plain = torch.autograd.grad((y * y).sum(), x, retain_graph=True)[0]
        g = torch.autograd.grad((y * y).sum(), x, create_graph=True)[0]
        assert torch.equal(g, plain) and not plain.requires_grad
        with pytest.raises(RuntimeError, match=f"{name} has no second derivatives"):
            torch.autograd.grad((g * g).sum() + (x * x).sum(), x)
