"""The dense half of a layer, as cases that can be timed: products of rows with the weights of their type (or expert), group
norm with an activation, and dropout.

A case names its kind:

  linear   grouped_linear: rows in ragged groups, each group with weights and a bias of its own
  norm     group_norm_act: statistics over each row, or over the rows of each ragged group (a node type, a graph of a batch)
  dropout  dropout, whose mask follows from a key, the number of the call and the place of the element

`train` cases are a forward and the gradients of all inputs for a given gradient of the output, the others a forward alone.
With `own` false the operators are computed in elementary torch operations, in 32 bits and rounded once at the end.

The activations of the cases are smooth ones: behind a kink two computations of one gradient may differ by all of it where an
input is a rounding away from the kink.
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5
_M0, _M1, _W0, _W1, _DROP = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0x64726F70


def listed():
    return [
        # hidden rows of one batch of 1024 seeds: launches and host work count
        dict(name="drop_seeds_f32", kind="dropout", rows=1024, dim=256, dtype="f32", p=0.5, train=True),
        # rows that are no whole vectors, an odd number of elements: no layer in between, forward alone
        dict(name="drop_odd_f16", kind="dropout", rows=30_011, dim=119, dtype="f16", p=0.1, train=False),
        # the input layer of the papers-shaped block, hidden size 256
        dict(name="drop_papers_bf16", kind="dropout", rows=151_552, dim=256, dtype="bf16", p=0.5, train=True),
        # inference for the short last batch of an epoch, rows of 100 features
        dict(name="norm_seeds_f32", kind="norm", rows=931, dim=100, groups=4, segments=0, dtype="f32", act="silu", p=0.0, train=False),
        # every row by itself over the destinations of the papers-shaped block, with the dropout behind it
        dict(name="norm_rows_f32", kind="norm", rows=67_584, dim=256, groups=8, segments=0, dtype="f32", act="silu", p=0.5, train=True),
        # statistics a node type: eight long ragged segments
        dict(name="norm_types_bf16", kind="norm", rows=151_552, dim=256, groups=32, segments=8, dtype="bf16", act="silu", p=0.5, train=True),
        # a batch of small graphs, statistics a graph and channel
        dict(name="norm_graphs_f16", kind="norm", rows=55_001, dim=64, groups=64, segments=2048, dtype="f16", act="gelu", p=0.0, train=True),
        # single nodes (or tokens) answered one by one: about a row for each of 64 experts, and experts without any
        dict(name="linear_tokens_bf16", kind="linear", rows=61, dim=1024, out=1024, groups=64, dtype="bf16", train=False),
        # the last layer of a batch of 1024 seeds: 47 classes, five types
        dict(name="linear_classes_f32", kind="linear", rows=1024, dim=256, out=47, groups=5, dtype="f32", train=True),
        # the outermost layer of the papers-shaped block: 128 features in, 256 out
        dict(name="linear_papers_f32", kind="linear", rows=67_584, dim=128, out=256, groups=8, dtype="f32", train=True),
        # the layer behind it, over all sources, with sixteen types
        dict(name="linear_papers_bf16", kind="linear", rows=151_552, dim=256, out=256, groups=16, dtype="bf16", train=True),
        # rows of the feature stress test, inference
        dict(name="linear_stress_f16", kind="linear", rows=495_616, dim=1024, out=256, groups=4, dtype="f16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "norm", "dropout"])
    dtype, train = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.6
    if kind == "linear":
        dim, out, groups = _log(rng, 16, 1024), _log(rng, 8, 1024), _log(rng, 1, 64)
        if rng.random() < 0.5:
            dim, out = max(16, dim // 16 * 16), max(16, out // 16 * 16)
        most = min(495_616, int(4e10 / (dim * out) / (3 if train else 1)), (1 << 29) // _BYTES[dtype] // max(dim, out))
        return dict(kind=kind, rows=_log(rng, 8, most), dim=dim, out=out, groups=groups, dtype=dtype, train=train)
    dim = _log(rng, 16, 1024)
    if rng.random() < 0.5:
        dim = max(16, dim // 16 * 16)
    rows = _log(rng, 100, min(495_616, (1 << 28) // _BYTES[dtype] // dim))
    if kind == "dropout":
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, p=rng.choice([0.1, 0.25, 0.5, 0.8]), train=train)
    segments = rng.choice([0, _log(rng, 1, 2048)])
    groups = rng.choice([g for g in (1, 2, 4, 8, 16, 32, dim) if dim % g == 0 and (segments or dim // g >= 8)])
    return dict(kind=kind, rows=rows, dim=dim, groups=groups, segments=min(segments, rows // 4), dtype=dtype,
                act=rng.choice(["none", "silu", "gelu"]), p=rng.choice([0.0, 0.0, 0.1, 0.5]), train=train)


# ---------------------------------------------------------------------------------------------------------- inputs
def _sizes(rows, groups, seed):
    """Rows of each group: some groups several times as long as others, now and then one without any."""
    share = np.random.RandomState(seed % (1 << 31)).lognormal(0.0, 0.8, groups)
    if groups > 4:
        share[seed % groups] = 0.0
    ends = np.round(np.cumsum(share) / share.sum() * rows).astype(np.int64)
    return [int(n) for n in np.diff(np.concatenate([[0], ends]))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = _TORCH[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dtype, leaf=train):
        t = torch.randn(shape, device="cuda", generator=gen).mul_(scale).add_(mean).to(dtype)
        return t.requires_grad_() if leaf else t

    s = dict(case=case, key=1 + seed * 7919, call_id=seed % 1000)
    rows, dim = case["rows"], case["dim"]
    s["x"] = normal(rows, dim, mean=0.25 if case["kind"] == "norm" else 0.0)
    width = dim
    if case["kind"] == "linear":
        width = case["out"]
        s["sizes"] = _sizes(rows, case["groups"], seed)
        s["weight"] = normal(case["groups"], width, dim, scale=dim ** -0.5)
        s["bias"] = normal(case["groups"], width, scale=0.1)
    if case["kind"] == "norm":
        s["sizes"] = _sizes(rows, case["segments"], seed) if case["segments"] else None
        # the parameters of a norm are kept in 32 bits beside 16-bit activations
        s["weight"] = normal(dim, scale=0.1, mean=1.0, dtype=torch.float32)
        s["bias"] = normal(dim, scale=0.1, dtype=torch.float32)
    if s.get("sizes") is not None:
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(s["sizes"])]), device="cuda")
    if train:
        s["grad"] = normal(rows, width, leaf=False)
    return s


# ------------------------------------------------------------------------------------------------- plain operators
def _mulhilo(a, b):
    """High and low word of the product of two 32-bit numbers held in 64 bits (the low 64 bits of a product do not depend on signs)."""
    p = a * b
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _keep(n, p, key, call_id, device):
    """Which of n elements stay: Philox4x32-10 of (number of the element's quad, call, tag), a word an element."""
    q = torch.arange((n + 3) // 4, device=device)
    c = [q & 0xFFFFFFFF, q >> 32, torch.full_like(q, call_id), torch.full_like(q, _DROP)]
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for r in range(10):
        h0, l0 = _mulhilo(c[0], _M0)
        h1, l1 = _mulhilo(c[2], _M1)
        c = [h1 ^ c[1] ^ ((k0 + r * _W0) & 0xFFFFFFFF), l1, h0 ^ c[3] ^ ((k1 + r * _W1) & 0xFFFFFFFF), l0]
    return torch.stack(c, 1).view(-1)[:n] >= int(p * 2.0 ** 32)


def _drop(t, keep, p):
    return torch.where(keep.view(t.shape), t * (1.0 / (1.0 - p)), torch.zeros((), device=t.device))


def _act(z, act):
    """act(z) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    keep = _keep(x.numel(), case["p"], s["key"], s["call_id"], x.device)
    out = {"out": _drop(x.float(), keep, case["p"]).to(x.dtype)}
    if case["train"]:
        keep = _keep(x.numel(), case["p"], s["key"], s["call_id"], x.device)
        out["grad_x"] = _drop(s["grad"].float(), keep, case["p"]).to(x.dtype)
    return out


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    rows, dim, groups = case["rows"], case["dim"], case["groups"]
    x, gamma, beta = s["x"].float().view(rows, groups, -1), s["weight"].view(groups, -1), s["bias"].view(groups, -1)
    if s["sizes"] is None:
        mean_of = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    else:
        offsets = s["offsets"]
        segment = torch.searchsorted(offsets, torch.arange(rows, device=x.device), right=True) - 1
        count = ((offsets[1:] - offsets[:-1]).clamp(min=1) * (dim // groups)).float().view(-1, 1)

        def mean_of(t):
            sums = torch.zeros((case["segments"], groups), device=t.device).index_add_(0, segment, t.sum(-1))
            return (sums / count)[segment].unsqueeze(-1)
    xh = x - mean_of(x)
    rstd = torch.rsqrt(mean_of(xh * xh) + _EPS)
    xh = xh * rstd
    y, slope = _act(xh * gamma + beta, case["act"])
    keep = _keep(x.numel(), case["p"], s["key"], s["call_id"], x.device) if case["p"] else None
    out = {"out": (y if keep is None else _drop(y, keep, case["p"])).view(rows, dim).to(dtype)}
    if case["train"]:
        dz = s["grad"].float().view_as(x)
        dz = (dz if keep is None else _drop(dz, keep, case["p"])) * slope
        dxh = dz * gamma
        dx = rstd * (dxh - mean_of(dxh) - xh * mean_of(dxh * xh))
        out.update(grad_x=dx.view(rows, dim).to(dtype), grad_weight=(dz * xh).view(rows, dim).sum(0), grad_bias=dz.view(rows, dim).sum(0))
    return out


def _plain_linear(s):
    x, weight, bias = s["x"].float(), s["weight"].float(), s["bias"].float()
    dtype, parts = s["x"].dtype, x.split(s["sizes"])
    out = {"out": torch.cat([a @ w.t() + b for a, w, b in zip(parts, weight, bias)]).to(dtype)}
    if s["case"]["train"]:
        grads = s["grad"].float().split(s["sizes"])
        out["grad_x"] = torch.cat([g @ w for g, w in zip(grads, weight)]).to(dtype)
        out["grad_weight"] = torch.stack([g.t() @ a for g, a in zip(grads, parts)]).to(dtype)
        out["grad_bias"] = torch.stack([g.sum(0) for g in grads]).to(dtype)
    return out


# --------------------------------------------------------------------------------------- the framework's operators
def _own_run(s):
    import apt_b200

    case, x = s["case"], s["x"]
    if case["kind"] == "dropout":
        args, op, fn = (x, case["p"], s["key"], s["call_id"]), apt_b200.dropout, apt_b200.Dropout
        leaves = {"grad_x": x}
    elif case["kind"] == "norm":
        args = (x, case["groups"], s["weight"], s["bias"], s.get("offsets"), _EPS, case["act"], case["p"], s["key"], s["call_id"])
        op, fn = apt_b200.group_norm_act, apt_b200.GroupNormAct
        leaves = {"grad_x": x, "grad_weight": s["weight"], "grad_bias": s["bias"]}
    else:
        args, op, fn = (x, s["weight"], s["offsets"], s["bias"]), apt_b200.grouped_linear, apt_b200.GroupedLinear
        leaves = {"grad_x": x, "grad_weight": s["weight"], "grad_bias": s["bias"]}
    if not case["train"]:
        return {"out": op(*args)}
    out = fn.apply(*args)
    return {"out": out, **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), s["grad"])))}


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return {"dropout": _plain_dropout, "norm": _plain_norm, "linear": _plain_linear}[state["case"]["kind"]](state)


def work(case):
    size, rows, dim, train = _BYTES[case["dtype"]], case["rows"], case["dim"], case["train"]
    if case["kind"] == "linear":
        width, groups = case["out"], case["groups"]
        # groups without a row need none of their weights: counted for as many groups as can have one
        used = min(groups, rows)
        params = used * width * (dim + 1) * size
        grads = groups * width * (dim + 1) * size if train else 0
        return {"bytes": rows * (dim + width) * size * (2 if train else 1) + params + grads,
                "flops": 2.0 * rows * dim * width * (3 if train else 1)}
    n = rows * dim
    passes = 4 if train else 2
    if case["kind"] == "dropout":
        return {"bytes": n * size * passes, "flops": n * 1.0 * (2 if train else 1)}
    return {"bytes": n * size * passes + dim * 4 * passes, "flops": n * (25.0 if train else 10.0)}


# --------------------------------------------------------------------------------------------- results in 64 bits
def _exact_words(n, key, call_id):
    """The generator's words in numpy, products of 32-bit numbers in unsigned 64 bits."""
    u = np.uint64
    quad = np.arange(-(-n // 4), dtype=u)
    low, half = u(0xFFFFFFFF), u(32)
    x0, x1, x2, x3 = quad & low, quad >> half, np.full_like(quad, call_id), np.full_like(quad, _DROP)
    a, b = key & 0xFFFFFFFF, key >> 32 & 0xFFFFFFFF
    for _ in range(10):
        first, second = x0 * u(_M0), x2 * u(_M1)
        x0, x1, x2, x3 = (second >> half) ^ x1 ^ u(a), second & low, (first >> half) ^ x3 ^ u(b), first & low
        a, b = (a + _W0) & 0xFFFFFFFF, (b + _W1) & 0xFFFFFFFF
    return np.stack([x0, x1, x2, x3], axis=1).reshape(-1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    x, train = s["x"].detach().double(), case["train"]
    rows, dim = x.shape
    grad = s["grad"].double() if train else None
    factor = None
    if case.get("p"):
        kept = _exact_words(rows * dim, s["key"], s["call_id"]) >= np.uint64(math.floor(case["p"] * 4294967296.0))
        factor = torch.from_numpy(kept.reshape(rows, dim)).cuda().double() / (1.0 - case["p"])
    if case["kind"] == "dropout":
        return {"out": x * factor, **({"grad_x": grad * factor} if train else {})}
    weight, bias = s["weight"].detach().double(), s["bias"].detach().double()
    if case["kind"] == "linear":
        out = torch.empty((rows, case["out"]), dtype=torch.float64, device="cuda")
        gx, gw, gb = torch.empty_like(x), torch.zeros_like(weight), torch.zeros_like(bias)
        at = 0
        for g, n in enumerate(s["sizes"]):
            here = slice(at, at + n)
            out[here] = torch.addmm(bias[g], x[here], weight[g].T)
            if train and n:
                gx[here] = torch.mm(grad[here], weight[g])
                gw[g] = torch.mm(grad[here].T, x[here])
                gb[g] = grad[here].sum(dim=0)
            at += n
        return {"out": out, "grad_x": gx, "grad_weight": gw, "grad_bias": gb} if train else {"out": out}
    leaves = [t.requires_grad_(train) for t in (x, weight, bias)]
    per = dim // case["groups"]
    if s["sizes"] is None:
        view = leaves[0].view(rows, case["groups"], per)
        var, mean = torch.var_mean(view, dim=2, unbiased=False, keepdim=True)
        normed = ((view - mean) / torch.sqrt(var + _EPS)).view(rows, dim)
    else:
        at, done = 0, []
        for n in s["sizes"]:
            if n:
                view = leaves[0][at:at + n].view(n, case["groups"], per)
                var, mean = torch.var_mean(view, dim=(0, 2), unbiased=False, keepdim=True)
                done.append(((view - mean) / torch.sqrt(var + _EPS)).view(n, dim))
            at += n
        normed = torch.cat(done)
    z = normed * leaves[1] + leaves[2]
    out = {"none": lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["act"]](z)
    if factor is not None:
        out = out * factor
    if not train:
        return {"out": out}
    return {"out": out.detach(), **dict(zip(("grad_x", "grad_weight", "grad_bias"), torch.autograd.grad(out, leaves, grad)))}
