"""The dense half of a layer against plain implementations in 64 bits: dropout, group norm with an activation, grouped products; their
gradients against the formulas and against differences.

Bounds. Dropout: equal, one product and one rounding. Products: a sum of n terms in fp32, in whatever order, is off by at most
n 2^-23 of the sum of the terms' magnitudes where each step may cut instead of round, and operands held in pieces of fewer bits add 2^-21
of it; a rounding to 16 bits adds 2^-8 (bf16) or 2^-11 (f16) of the result. Norms, in the 2-norm: some ten roundings an element and
sums whose terms a thread adds up a few hundred of, 4e-6 in all, times 1 + |mean| / deviation of a group where the mean is far from zero,
times 4 for gradients, which subtract two means; roundings to 16 bits as above."""
import numpy as np
import pytest
import torch

import apt_b200
from apt_b200 import ops
from oracle import oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _offsets(sizes, tail=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), device="cuda"), int(sum(sizes)) + tail


# --------------------------------------------------------------------------------------------------------- dropout
def _words(n, key, call_id, first=0):
    """The generator's words by the CPU oracle's Philox, from element `first` (of a whole quad) on."""
    quads = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(first // 4)
    low, high = (quads & np.uint64(0xFFFFFFFF)).astype(np.uint32), (quads >> np.uint64(32)).astype(np.uint32)
    w = orc.philox4x32_10(low, high, np.full_like(low, call_id & 0xFFFFFFFF), np.full_like(low, 0x64726F70),
                          np.uint32(key & 0xFFFFFFFF), np.uint32(key >> 32 & 0xFFFFFFFF))
    return np.stack(w, axis=-1).reshape(-1)[:n].astype(np.uint64)


def _dropped(x, p, key, call_id):
    if p >= 1.0:
        return torch.zeros_like(x)
    keep = torch.from_numpy(_words(x.numel(), key, call_id) >= np.uint64(int(p * 2 ** 32))).view(x.shape).to(x.device)
    return torch.where(keep, x.float() * np.float32(1.0 / (1.0 - p)), torch.zeros((), device=x.device)).to(x.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7, 1), (8,), (1, 47), (33, 119), (1024, 256), (5, 3, 31)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0 - 2.0 ** -32, 1.0])
def test_dropout_against_the_oracle(shape, dtype, p):
    x = torch.randn(shape, device="cuda", generator=_gen(len(shape))).to(dtype)
    key, call = 2 ** 63 + 12345, 7
    got = apt_b200.dropout(x, p, key, call)
    assert torch.equal(got, _dropped(x, p, key, call))
    leaf = x.clone().requires_grad_()
    y = apt_b200.Dropout.apply(leaf, p, key, call)
    g = torch.randn(shape, device="cuda", generator=_gen(2)).to(dtype)
    assert torch.equal(y, got)
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], _dropped(g, p, key, call))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_of_views_and_masked_places(dtype):
    base = torch.randn(2000, device="cuda", generator=_gen(1)).to(dtype)
    for x in (base[1:1998], base[3:], base.view(40, 50).t(), base.view(40, 50)[:, 7:19], base[:5].expand(9, 5)):
        assert torch.equal(apt_b200.dropout(x, 0.3, 5, 1), _dropped(x, 0.3, 5, 1))
    wild = torch.full((4096,), float("nan"), device="cuda", dtype=dtype)
    wild[::2] = float("inf")
    got = apt_b200.dropout(wild, 0.5, 9)
    gone = torch.from_numpy(_words(4096, 9, 0) < 2 ** 31).cuda()
    assert torch.equal(got == 0, gone) and not torch.isfinite(got[~gone]).any()
    assert apt_b200.dropout(base[:0], 0.5, 1).shape == (0,)


def test_dropout_streams_differ_and_keep_their_share():
    x = torch.ones(1 << 20, device="cuda")
    a, b, c = apt_b200.dropout(x, 0.25, 1, 0), apt_b200.dropout(x, 0.25, 1, 1), apt_b200.dropout(x, 0.25, 2, 0)
    for u, v in ((a, b), (a, c)):
        # both kept: 0.75^2 of 2^20 elements, five deviations of a binomial either way
        assert abs(float(((u > 0) & (v > 0)).double().mean()) - 0.5625) < 5 * (0.5625 * 0.4375 / 2 ** 20) ** 0.5
    assert abs(float((a > 0).double().mean()) - 0.75) < 5 * (0.75 * 0.25 / 2 ** 20) ** 0.5


# ------------------------------------------------------------------------------------------------------ group norm
ACTS = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}


def _norm64(x, groups, weight, bias, offsets, eps, act, p, key, call):
    """The definition through PyTorch's autograd in 64 bits."""
    rows = x.reshape(-1, x.shape[-1])
    if offsets is not None:
        ends = offsets.tolist()
    else:
        per = rows.shape[0] // x.shape[0] if x.shape[0] else 0
        ends = [k * per for k in range(x.shape[0] + 1)]
    parts = []
    if offsets is None and per == 1:
        v = rows.reshape(rows.shape[0], groups, -1)
        var, mean = torch.var_mean(v, dim=2, unbiased=False, keepdim=True)
        parts = [((v - mean) / torch.sqrt(var + eps)).reshape(rows.shape)]
    else:
        for b, e in zip(ends, ends[1:]):
            if e > b:
                v = rows[b:e].reshape(e - b, groups, -1)
                var, mean = torch.var_mean(v, dim=(0, 2), unbiased=False, keepdim=True)
                parts.append(((v - mean) / torch.sqrt(var + eps)).reshape(e - b, -1))
    n = torch.cat(parts) if parts else rows[:0]
    z = n if weight is None else n * weight
    y = ACTS[act](z if bias is None else z + bias)
    if p > 0.0:
        keep = torch.from_numpy(_words(x.numel(), key, call) >= np.uint64(int(p * 2 ** 32))).cuda().view(rows.shape)[: y.shape[0]]
        y = y * keep / (1.0 - p)
    y = torch.cat([y, torch.zeros_like(rows[y.shape[0]:])])
    return y.reshape(x.shape)


def _close(got, want, bound):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    scale = float(want.norm())
    off = float((got - want).norm())
    assert off <= bound * scale + 1e-12 * want.numel() ** 0.5, (off / max(scale, 1e-300), bound)


def _check_norm(x, groups, offsets=None, act="none", p=0.0, params="f32", eps=1e-5, seed=0, shift=0.0):
    dim, dtype = x.shape[-1], x.dtype
    gen = _gen(seed + 77)
    weight = bias = None
    if params is not None:
        t = torch.float32 if params == "f32" else dtype
        weight = (torch.randn(dim, device="cuda", generator=gen) * 0.2 + 1).to(t)
        bias = (torch.randn(dim, device="cuda", generator=gen) * 0.2).to(t)
    grad = torch.randn(x.shape, device="cuda", generator=gen).to(dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (x, weight, bias) if t is not None]
    args = leaves if params is not None else [leaves[0], None, None]
    out = apt_b200.GroupNormAct.apply(args[0], groups, args[1], args[2], offsets, eps, act, p, 11, 3)
    grads = torch.autograd.grad(out, leaves, grad)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    wargs = wide if params is not None else [wide[0], None, None]
    want = _norm64(wargs[0], groups, wargs[1], wargs[2], offsets, eps, act, p, 11, 3)
    wgrads = torch.autograd.grad(want, wide, grad.double()) if want.requires_grad else [torch.zeros_like(t) for t in wide]
    base = 4e-6 * (1.0 + shift)
    _close(out, want, base + UNIT[dtype])
    _close(grads[0], wgrads[0], 4 * base + UNIT[dtype])
    for a, b in zip(grads[1:], wgrads[1:]):
        _close(a, b, 4 * base + UNIT[a.dtype])
    plain, stats = apt_b200.group_norm_act(x, groups, weight, bias, offsets, eps, act, p, 11, 3, return_stats=True)
    assert torch.equal(plain, out)
    again = apt_b200.group_norm_act_backward(x, grad, stats, groups, weight, bias, offsets, eps, act, p, 11, 3)
    for a, b in zip(again, grads):
        assert torch.equal(a, b)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,groups", [(1, 8, 1), (1, 32, 8), (3, 100, 4), (931, 100, 4), (257, 256, 8), (64, 47, 1), (40, 119, 7), (300, 37, 1),
                                             (5, 1024, 1), (17, 1024, 32), (2, 5000, 1), (2, 20000, 2), (130, 64, 64), (1000, 16, 2), (6, 2304, 3)])
@pytest.mark.parametrize("act,p,params", [("none", 0.0, None), ("silu", 0.5, "f32"), ("gelu", 0.1, "own")])
def test_norm_of_rows(rows, dim, groups, dtype, act, p, params):
    x = (torch.randn((rows, dim), device="cuda", generator=_gen(rows + dim)) * 1.5 + 0.3).to(dtype)
    _check_norm(x, groups, act=act, p=p, params=params)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,tail", [([5], 0), ([1], 0), ([0, 1, 0, 2, 300, 0], 0), ([1000, 3, 3000], 0), ([7] * 60, 5), ([0, 0], 9), ([64, 128, 1, 63], 1),
                                        ([9000], 0), ([1] * 40 + [700], 3)])
@pytest.mark.parametrize("dim,groups", [(64, 64), (256, 32), (100, 4), (47, 1), (24, 8), (1024, 2)])
def test_norm_of_ragged_segments(sizes, tail, dim, groups, dtype):
    offsets, rows = _offsets(sizes, tail)
    x = (torch.randn((rows, dim), device="cuda", generator=_gen(rows + dim)) * 0.7 - 0.2).to(dtype)
    if dim // groups == 1 and rows < 10:      # statistics over one or two numbers: all there is to compare are roundings of a zero
        x = x.float().mul(4).to(dtype)
    _check_norm(x, groups, offsets, act="silu" if dim % 8 else "gelu", p=0.25 if groups > 8 else 0.0, params="f32" if groups != 4 else "own")


# groups wider than a block's columns: cut into parts of whole slices, or (2053 is a prime) walked over by a block
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,tail", [([90, 0, 1, 400], 7), ([3] * 70, 0)])
@pytest.mark.parametrize("dim,groups", [(8192, 1), (6000, 2), (2053, 1), (4106, 1), (2068, 1)])
def test_norm_of_wide_groups(sizes, tail, dim, groups, dtype):
    offsets, rows = _offsets(sizes, tail)
    x = (torch.randn((rows, dim), device="cuda", generator=_gen(rows + dim)) * 0.7 - 0.2).to(dtype)
    _check_norm(x, groups, offsets, act="gelu", p=0.1)
    if dim == 8192:
        _check_norm(x[: rows // 6 * 6].view(-1, 3, dim), groups, act="none", p=0.0)


# rows whose groups are slices of 8 bytes, rows of 1433
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,groups", [(100, 1), (36, 3), (42, 3), (138, 1), (316, 1), (1433, 1), (2060, 1)])
def test_norm_of_rows_of_narrow_slices(dim, groups, dtype):
    x = (torch.randn((301, dim), device="cuda", generator=_gen(dim)) * 1.5 + 0.3).to(dtype)
    _check_norm(x, groups, act="silu", p=0.5)
    offsets, _ = _offsets([200, 1, 0, 70], 30)
    _check_norm(x, groups, offsets, act="gelu", p=0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", [((2, 5, 7, 32), 4), ((1, 3000, 16), 16), ((3, 1, 48), 6), ((40, 9, 64), 1), ((2, 2, 2, 2, 10), 5)])
def test_norm_channels_last(shape, groups, dtype):
    x = torch.randn(shape, device="cuda", generator=_gen(3)).to(dtype)
    _check_norm(x, groups, act="silu", p=0.1)


@pytest.mark.parametrize("rows,offsets", [(500, None), (500, [0, 100, 500])])
def test_norm_far_from_zero(rows, offsets):
    x = torch.randn((rows, 64), device="cuda", generator=_gen(4)) + 300.0
    _check_norm(x, 2, None if offsets is None else torch.tensor(offsets, device="cuda"), act="silu", shift=300.0)


def test_norm_relu_and_its_kinks():
    x = torch.randn((333, 64), device="cuda", generator=_gen(5))
    weight, bias = torch.full((64,), 2.0, device="cuda"), torch.full((64,), 0.25, device="cuda")
    leaf = x.clone().requires_grad_()
    out = apt_b200.GroupNormAct.apply(leaf, 4, weight, bias, None, 1e-5, "relu")
    z = _norm64(x.double(), 4, weight.double(), bias.double(), None, 1e-5, "none", 0.0, 0, 0)
    _close(out, torch.relu(z), 4e-6)
    # behind the kink: zeros, and rows of zeros have gradients of zero
    assert (out[z < -1e-4] == 0).all()
    low = torch.full((64,), -50.0, device="cuda")
    out = apt_b200.GroupNormAct.apply(leaf, 4, weight, low, None, 1e-5, "relu")
    assert not out.any() and not torch.autograd.grad(out, leaf, torch.ones_like(out))[0].any()
    x[7, 3] = float("nan")
    got = apt_b200.group_norm_act(x, 4, act="relu")
    assert torch.isnan(got[7, :16]).all() and torch.isfinite(got[7, 16:]).all() and torch.isfinite(got[8]).all()


def test_norm_wild_values_stay_in_their_segment():
    offsets = torch.tensor([0, 40, 41, 100], device="cuda")
    x = torch.randn((110, 32), device="cuda", generator=_gen(6))
    x[40] = float("inf")
    x[105] = float("nan")      # of no segment
    leaf = x.clone().requires_grad_()
    out = apt_b200.GroupNormAct.apply(leaf, 4, None, None, offsets)
    assert torch.isnan(out[40]).all() and torch.isfinite(out[:40]).all() and torch.isfinite(out[41:]).all() and not out[100:].any()
    g = torch.autograd.grad(out, leaf, torch.ones_like(out))[0]
    assert torch.isfinite(g[:40]).all() and torch.isfinite(g[41:]).all() and not g[100:].any()


def test_norm_gradient_against_differences():
    gen = _gen(8)
    x, weight, bias = torch.randn((6, 12), device="cuda", generator=gen), torch.rand(12, device="cuda", generator=gen) + 0.5, torch.randn(12, device="cuda", generator=gen)
    offsets = torch.tensor([0, 4, 6], device="cuda")
    direction = torch.randn(x.shape, device="cuda", generator=gen)
    grad = torch.randn(x.shape, device="cuda", generator=gen)
    leaf = x.clone().requires_grad_()
    f = lambda t: apt_b200.GroupNormAct.apply(t, 3, weight, bias, offsets, 1e-5, "gelu", 0.25, 5, 6)
    got = float((torch.autograd.grad(f(leaf), leaf, grad)[0].double() * direction.double()).sum())
    # central differences with steps of 2^-6: third derivatives of order one leave about h^2 / 6 = 4e-5, roundings 2^-24 / h = 4e-6, of terms whose
    # magnitudes sum up to about 70: 5e-3
    h = 2.0 ** -6
    want = float(((f(x + h * direction).double() - f(x - h * direction).double()) * grad.double()).sum()) / (2 * h)
    assert abs(got - want) < 5e-3 * max(1.0, abs(want))


# ------------------------------------------------------------------------------------------------- grouped products
def _linear64(x, weight, offsets, bias, grad):
    x, weight, grad = x.double(), weight.double(), grad.double()
    ends = offsets.tolist()
    out, gx = torch.zeros((x.shape[0], weight.shape[1]), dtype=torch.float64, device="cuda"), torch.zeros_like(x)
    gw, gb = torch.zeros_like(weight), torch.zeros(weight.shape[:2], dtype=torch.float64, device="cuda")
    for g, (b, e) in enumerate(zip(ends, ends[1:])):
        out[b:e] = x[b:e] @ weight[g].T + (0 if bias is None else bias[g].double())
        gx[b:e], gw[g], gb[g] = grad[b:e] @ weight[g], grad[b:e].T @ x[b:e], grad[b:e].sum(0)
    return out, gx, gw, gb


def _close_sums(got, want, terms, magnitude, dtype):
    """Element by element: `terms` added up, the magnitudes of which sum up to `magnitude`."""
    got, want = got.detach().double(), want.detach().double()
    assert torch.isfinite(got).all()
    bound = (terms * 2.0 ** -23 + 2.0 ** -21) * magnitude + UNIT[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    off = (got - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


def _check_linear(sizes, dim, out_dim, dtype, tail=0, with_bias=True, seed=0, scale=1.0):
    gen = _gen(seed + 1000 * dim + out_dim)
    offsets, rows = _offsets(sizes, tail)
    make = lambda *shape: (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)
    x, weight, grad = make(rows, dim), make(len(sizes), out_dim, dim), make(rows, out_dim)
    bias = make(len(sizes), out_dim) if with_bias else None
    want = _linear64(x, weight, offsets, bias, grad)
    sizes_of = _linear64(x.abs(), weight.abs(), offsets, None if bias is None else bias.abs(), grad.abs())
    longest = max(list(sizes) + [1])
    terms = [dim + 1, out_dim, longest, longest]
    leaves = [t.requires_grad_() for t in (x, weight) + ((bias,) if with_bias else ())]
    out = apt_b200.GroupedLinear.apply(x, weight, offsets, bias)
    got = (out,) + torch.autograd.grad(out, leaves, grad)
    for a, b, n, m in zip(got, want, terms, sizes_of):
        _close_sums(a, b, n, m, dtype)
    with torch.no_grad():
        assert torch.equal(apt_b200.grouped_linear(x, weight, offsets, bias), out)
        again = apt_b200.grouped_linear_backward(x, weight, offsets, grad)
        for a, b in zip(again, got[1:]):
            assert torch.equal(a, b)      # sums in an order of their own, the same every time
        only = apt_b200.grouped_linear_backward(x, weight, offsets, grad, want_x=False, want_bias=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1], again[1])
    ops.check_status()


SIZES = [([1], 0), ([0], 3), ([5, 0, 1], 0), ([128], 0), ([129, 127, 0, 1], 2), ([300, 1, 1000], 0), ([1] * 70, 0), ([0] * 9 + [17], 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,tail", SIZES)
@pytest.mark.parametrize("dim,out_dim", [(128, 256), (64, 64), (100, 47), (1, 1), (8, 300), (257, 24), (36, 40)])
def test_linear(sizes, tail, dim, out_dim, dtype):
    _check_linear(sizes, dim, out_dim, dtype, tail, with_bias=dim != 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,dim,out_dim", [([3000, 5000], 256, 256), ([700] * 3, 1024, 520), ([20000], 16, 8), ([1, 4000, 2, 33], 136, 72), ([64] * 64, 72, 1000),
                                               ([2, 1, 0, 3], 2048, 1032), ([6131], 96, 172)])
def test_linear_larger(sizes, dim, out_dim, dtype):
    _check_linear(sizes, dim, out_dim, dtype, scale=0.25)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_many_groups(dtype):
    rng = np.random.default_rng(3)
    _check_linear([int(n) for n in rng.integers(0, 4, 1500)], 32, 24, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_views(dtype):
    gen = _gen(12)
    offsets = torch.tensor([0, 60, 90], device="cuda")
    wide = torch.randn((100, 200), device="cuda", generator=gen).to(dtype)
    flat = torch.randn(2 * 48 * 64 + 8, device="cuda", generator=gen).to(dtype)
    for x in (wide[:90, 3:67], wide.t()[:90, :64], wide[5:95, 64:128], wide[:1, :64].expand(90, 64)):
        for weight in (flat[1:1 + 2 * 48 * 64].view(2, 48, 64), flat[:2 * 48 * 64].view(2, 64, 48).transpose(1, 2)):
            grad = torch.ones((1, 1), device="cuda", dtype=dtype).expand(90, 48)
            want = _linear64(x, weight, offsets, None, grad)
            got = (apt_b200.grouped_linear(x, weight, offsets),) + apt_b200.grouped_linear_backward(x, weight, offsets, grad)
            size = _linear64(x.abs(), weight.abs(), offsets, None, grad)
            for a, b, n, m in zip(got, want, (64, 48, 60, 60), size):
                _close_sums(a, b, n, m, dtype)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_wild_values_stay_in_their_rows_and_groups(dtype):
    gen = _gen(13)
    offsets = torch.tensor([0, 50, 101, 130], device="cuda")
    x = torch.randn((150, 72), device="cuda", generator=gen).to(dtype)
    weight = torch.randn((3, 40, 72), device="cuda", generator=gen).to(dtype)
    grad = torch.randn((150, 40), device="cuda", generator=gen).to(dtype)
    x[20, 5], x[77], x[140:] = float("inf"), float("nan"), float("nan")
    grad[90, 3], grad[145] = float("-inf"), float("inf")
    out = apt_b200.grouped_linear(x, weight, offsets)
    gx, gw, gb = apt_b200.grouped_linear_backward(x, weight, offsets, grad)
    ops.check_status()
    fine = torch.ones(150, dtype=torch.bool, device="cuda")
    fine[20] = fine[77] = False
    assert torch.isfinite(out[fine]).all() and torch.isnan(out[77]).all() and not out[130:].any()
    # an infinite product in a sum of finite ones is infinite, of the sign of its factors
    assert torch.equal(out[20].float(), torch.copysign(torch.full((40,), float("inf"), device="cuda"), weight[0, :, 5].float()))
    fine[:] = True
    fine[90] = False
    assert torch.isfinite(gx[fine]).all() and not gx[130:].any()
    assert torch.equal(gx[90].float(), torch.copysign(torch.full((72,), float("inf"), device="cuda"), -weight[1, 3].float()))
    assert torch.isfinite(gw[2]).all() and torch.isfinite(gb[0]).all() and torch.isfinite(gb[2]).all()
    assert torch.isfinite(gw[0][:, [k for k in range(72) if k != 5]]).all()
    assert torch.equal(gw[0][:, 5].float(), torch.copysign(torch.full((40,), float("inf"), device="cuda"), grad[20].float()))
    assert torch.isnan(gw[1]).all() and float(gb[1, 3]) == float("-inf")


def test_linear_values_of_any_size():
    """fp32 operands keep their 24 bits and their range: rows of very large and very small numbers beside one another."""
    gen = _gen(14)
    offsets = torch.tensor([0, 200], device="cuda")
    scale = torch.logspace(-15, 15, 200, device="cuda").view(200, 1)
    x = torch.randn((200, 96), device="cuda", generator=gen) * scale
    weight = torch.randn((1, 64, 96), device="cuda", generator=gen)
    want = x.double() @ weight[0].double().T
    size = x.double().abs() @ weight[0].double().abs().T
    _close_sums(apt_b200.grouped_linear(x, weight, offsets), want, 96, size, torch.float32)
    # sums that leave the range are infinite, not NaN
    big = torch.full((3, 96), 3e38, device="cuda")
    got = apt_b200.grouped_linear(big, torch.ones((1, 64, 96), device="cuda"), torch.tensor([0, 3], device="cuda"))
    assert torch.equal(got, torch.full_like(got, float("inf")))
    ops.check_status()


def test_linear_gradient_against_differences():
    gen = _gen(15)
    offsets = torch.tensor([0, 3, 3, 9], device="cuda")
    x, weight, bias = (torch.randn(s, device="cuda", generator=gen) for s in ((9, 20), (3, 11, 20), (3, 11)))
    grad = torch.randn((9, 11), device="cuda", generator=gen)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    f = lambda *a: (apt_b200.GroupedLinear.apply(a[0], a[1], offsets, a[2]).double() * grad.double()).sum()
    got = torch.autograd.grad(f(*leaves), leaves)
    for k in range(3):
        step = [torch.zeros_like(t) for t in leaves]
        step[k] = torch.randn(leaves[k].shape, device="cuda", generator=gen)
        # a linear map in each of them: differences over steps of one are off by roundings only, 1e-6 of a thousand products
        want = float(f(*[a + s for a, s in zip(leaves, step)]) - f(*[a - s for a, s in zip(leaves, step)])) / 2
        assert abs(float((got[k].double() * step[k].double()).sum()) - want) < 2e-3


# --------------------------------------------------------------------------------------- streams, graphs, refusals
def test_another_stream_and_a_captured_graph():
    gen = _gen(16)
    sizes = [100, 0, 411, 90]
    offsets, rows = _offsets(sizes)
    x, weight = torch.randn((rows, 64), device="cuda", generator=gen).bfloat16(), torch.randn((4, 64, 64), device="cuda", generator=gen).bfloat16()

    def layer():
        h = apt_b200.grouped_linear(x, weight, offsets)
        y = apt_b200.group_norm_act(h, 4, offsets=offsets, act="silu", p=0.5, key=3, call_id=1)
        return y, apt_b200.dropout(y, 0.5, 3, 2), *apt_b200.grouped_linear_backward(x, weight, offsets, y)

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer()
    # other ends of the groups and other rows, as a replayed mini-batch has them
    other = torch.tensor([0, 1, 300, 300, 580], device="cuda")
    offsets.copy_(other)
    x.copy_(torch.randn((rows, 64), device="cuda", generator=gen))
    graph.replay()
    for a, b in zip(held, layer()):
        assert torch.equal(a, b)
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_again_and_again(dtype):
    """The same bits every time, from the first call on and with the cache full of something else: nothing is read before it is there."""
    gen = _gen(17)
    offsets, rows = _offsets([7000, 0, 9000, 4001])
    make = lambda *shape: torch.randn(shape, device="cuda", generator=gen).to(dtype)
    x, weight, bias, grad = make(rows, 328), make(4, 88, 328), make(4, 88), make(rows, 88)
    other = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for k in range(60):
        if k % 2:
            other.fill_(k)
        got = (apt_b200.grouped_linear(x, weight, offsets, bias),) + apt_b200.grouped_linear_backward(x, weight, offsets, grad)
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b), k
    ops.check_status()


def test_a_thread_that_has_not_used_the_gpu():
    """The autograd engine's threads, or a caller's: nothing has bound them to the device's context yet."""
    import threading

    x, weight, offsets = torch.randn((64, 32), device="cuda"), torch.randn((1, 32, 32), device="cuda"), torch.tensor([0, 64], device="cuda")
    want = apt_b200.grouped_linear(x, weight, offsets)
    got = []

    def call():
        try:
            got.append(apt_b200.grouped_linear(x, weight, offsets))
        except RuntimeError as e:
            got.append(e)

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert torch.is_tensor(got[0]), got[0]
    assert torch.equal(got[0], want)


@pytest.mark.parametrize("ends", [[1, 5, 20], [0, 9, 5], [0, 5, 21], [-1, 5, 20], [0, -5, 2 ** 60]])
def test_bad_offsets_are_reported(ends):
    offsets = torch.tensor(ends, device="cuda")
    x, weight = torch.randn((20, 16), device="cuda"), torch.randn((2, 16, 16), device="cuda")
    for call in (lambda: apt_b200.grouped_linear(x, weight, offsets), lambda: apt_b200.grouped_linear_backward(x, weight, offsets, x),
                 lambda: apt_b200.group_norm_act(x, 2, offsets=offsets)):
        call()
        with pytest.raises(RuntimeError, match="row groups"):
            ops.check_status()
    ops.check_status()


def test_refusals():
    x, weight = torch.randn((8, 16), device="cuda"), torch.randn((2, 4, 16), device="cuda")
    offsets = torch.tensor([0, 3, 8], device="cuda")
    refused = [
        (lambda: apt_b200.dropout(x.cpu(), 0.5, 1), "CUDA tensor"), (lambda: apt_b200.dropout(x.double(), 0.5, 1), "unsupported dtype"),
        (lambda: apt_b200.dropout(x, -0.1, 1), "probability"), (lambda: apt_b200.dropout(x, 1.5, 1), "probability"),
        (lambda: apt_b200.dropout(x, float("nan"), 1), "probability"),
        (lambda: apt_b200.grouped_linear(x.cpu(), weight, offsets), "CUDA tensor"), (lambda: apt_b200.grouped_linear(x, weight, offsets.int()), "int64"),
        (lambda: apt_b200.grouped_linear(x, weight, offsets[:2]), "groups \\+ 1"), (lambda: apt_b200.grouped_linear(x.half(), weight, offsets), "mixed dtypes"),
        (lambda: apt_b200.grouped_linear(x[:, :8], weight, offsets), "dim"), (lambda: apt_b200.grouped_linear(x.double(), weight.double(), offsets), "unsupported"),
        (lambda: apt_b200.grouped_linear(x, weight, offsets, torch.zeros((4, 2), device="cuda")), "bias"),
        (lambda: apt_b200.grouped_linear(x, weight, offsets, torch.zeros((2, 4), device="cuda").half()), "mixed dtypes"),
        (lambda: apt_b200.grouped_linear(x, weight[:0], offsets[:1]), "groups"),
        (lambda: apt_b200.grouped_linear_backward(x, weight, offsets, x), "grad_out"),
        (lambda: apt_b200.group_norm_act(x, 3), "whole number"), (lambda: apt_b200.group_norm_act(x, 0), "whole number"),
        (lambda: apt_b200.group_norm_act(x[0], 2), "dimension"), (lambda: apt_b200.group_norm_act(x, 2, act="tanh"), "activation"),
        (lambda: apt_b200.group_norm_act(x, 2, weight=x[0, :8]), "one value a channel"), (lambda: apt_b200.group_norm_act(x, 2, p=2.0), "probability"),
        (lambda: apt_b200.group_norm_act(x, 2, eps=-1.0), "eps"), (lambda: apt_b200.group_norm_act(x, 2, weight=x[0].half()), "beside"),
        (lambda: apt_b200.group_norm_act(x.view(2, 4, 16), 2, offsets=offsets), "two dimensions"),
        (lambda: apt_b200.group_norm_act_backward(x, x, torch.zeros((8, 4, 2), device="cuda"), 2), "stats"),
        (lambda: apt_b200.group_norm_act_backward(x, x[:4], torch.zeros((8, 2, 2), device="cuda"), 2), "like x"),
    ]
    for call, text in refused:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    offsets = torch.zeros(3, dtype=torch.int64, device="cuda")
    x, weight = torch.zeros((0, 16), device="cuda", dtype=dtype), torch.ones((2, 4, 16), device="cuda", dtype=dtype)
    assert apt_b200.grouped_linear(x, weight, offsets).shape == (0, 4)
    gx, gw, gb = apt_b200.grouped_linear_backward(x, weight, offsets, x.new_zeros((0, 4)))
    assert gx.shape == (0, 16) and not gw.any() and not gb.any()
    y, stats = apt_b200.group_norm_act(x, 2, x.new_ones(16), x.new_ones(16), offsets, return_stats=True)
    assert y.shape == (0, 16)
    gx, gw, gb = apt_b200.group_norm_act_backward(x, x, stats, 2, x.new_ones(16), x.new_ones(16), offsets)
    assert gx.shape == (0, 16) and not gw.any() and not gb.any()
    ops.check_status()


def test_more_than_31_bits_of_elements():
    rows, dim, n = 8_400_000, 256, 1000
    x = torch.randn((rows, dim), device="cuda", generator=_gen(5), dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    tail = x[-n:].clone()
    ends = torch.tensor([0, 10, rows - n, rows], device="cuda")
    one = torch.tensor([0, n], device="cuda")
    # rows by themselves: what they are alone
    y = apt_b200.group_norm_act(x, 4, act="silu")
    assert torch.equal(y[-n:], apt_b200.group_norm_act(tail, 4, act="silu"))
    # the last segment, alone in other tiles: roundings of its statistics
    y, stats = apt_b200.group_norm_act(x, 4, None, None, ends, 1e-5, "silu", return_stats=True)
    alone, alone_stats = apt_b200.group_norm_act(tail, 4, None, None, one, 1e-5, "silu", return_stats=True)
    _close(y[-n:], alone, UNIT[x.dtype])
    _close(stats[2], alone_stats[0], 1e-5)
    grad = apt_b200.group_norm_act_backward(x, y, stats, 4, None, None, ends, 1e-5, "silu")[0]
    _close(grad[-n:], apt_b200.group_norm_act_backward(tail, y[-n:].clone(), alone_stats, 4, None, None, one, 1e-5, "silu")[0], UNIT[x.dtype])
    del y, grad
    # dropout: words by the element's number
    first = rows * dim - 4096
    keep = torch.from_numpy(_words(4096, 7, 2, first) >= 2 ** 31).cuda()
    out = apt_b200.dropout(x, 0.5, 7, 2)
    assert torch.equal(out.view(-1)[first:], torch.where(keep, x.view(-1)[first:] * 2, 0.0))
    del out
    weight = (torch.randn((3, dim, dim), device="cuda", generator=_gen(6)) / 16).bfloat16()
    out = apt_b200.grouped_linear(x, weight, ends)
    _close(out[-n:], tail.double() @ weight[2].double().T, 4e-6 + UNIT[x.dtype])
    _close(out[10:1010], x[10:1010].double() @ weight[1].double().T, 4e-6 + UNIT[x.dtype])
    grad_x, grad_weight, _ = apt_b200.grouped_linear_backward(x, weight, ends, out)
    _close(grad_x[-n:], out[-n:].double() @ weight[2].double(), 4e-6 + UNIT[x.dtype])
    _close(grad_weight[2], out[-n:].double().T @ tail.double(), 4e-6 + UNIT[x.dtype])
    ops.check_status()
