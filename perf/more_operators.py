"""A layer of experts around its products, and the loss behind the last layer, as cases that can be timed.

A case names its kind:

  route    route_experts: a row's logits over the experts -> the k that it goes to, and their weights
  rows     expert_rows: a copy of every row for each of its experts, ordered by expert, and where the experts' groups end
  sum      expert_sum: the experts' results of a row, weighted and added up
  loss     linear_cross_entropy: rows times the classes' weights -> softmax cross entropy against labels, logits never kept

`train` cases are a forward and the gradients of all inputs for a given gradient of the output, the others a forward alone.
With `own` false the operators are computed in elementary torch operations, in 32 bits and rounded once at the end; which experts a
row goes to is decided on 64-bit scores, so that neighbouring scores have one order.
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_INF = float("inf")
_IGNORE = -100


def listed():
    return [
        # one node (or token) answered by itself: launches and host work are the time
        dict(name="route_one_f32", kind="route", rows=1, experts=64, k=6, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=True,
             scale=1.0, dtype="f32", train=False),
        # the hidden rows of one batch of 1024 seeds, eight experts
        dict(name="route_seeds_f32", kind="route", rows=1024, experts=8, k=2, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=True,
             scale=1.0, dtype="f32", train=True),
        # many experts in groups that are chosen first, with a bias that balances their load: destinations of the papers-shaped block
        dict(name="route_groups_f32", kind="route", rows=67_584, experts=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, best=2, renorm=True,
             scale=2.5, dtype="f32", train=True),
        # all sources of the papers-shaped block, weights that do not add up to one
        dict(name="route_papers_bf16", kind="route", rows=151_552, experts=64, k=6, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=False,
             scale=1.0, dtype="bf16", train=True),
        # the short last batch of an epoch, rows of 100 features, inference
        dict(name="rows_seeds_f32", kind="rows", rows=931, k=2, experts=8, dim=100, dtype="f32", train=False),
        # the layer behind the input of the papers-shaped block
        dict(name="rows_papers_bf16", kind="rows", rows=151_552, k=2, experts=16, dim=256, dtype="bf16", train=True),
        # single nodes answered together, rows that are no whole vectors
        dict(name="sum_tokens_f16", kind="sum", rows=61, k=6, experts=64, dim=119, dtype="f16", train=False),
        # the same layer's results on their way back
        dict(name="sum_papers_bf16", kind="sum", rows=151_552, k=2, experts=16, dim=256, dtype="bf16", train=True),
        # the last layer of a batch of 1024 seeds: 47 classes
        dict(name="loss_classes_f32", kind="loss", rows=1024, dim=256, classes=47, bias=True, reduction="mean", dtype="f32", train=True),
        # losses of single rows that are weighted afterwards, the short last batch of an epoch, a large odd number of classes
        dict(name="loss_odd_f16", kind="loss", rows=931, dim=100, classes=50_021, bias=False, reduction="none", dtype="f16", train=True),
        # thousands of classes over a large batch
        dict(name="loss_many_bf16", kind="loss", rows=67_584, dim=256, classes=2_983, bias=True, reduction="mean", dtype="bf16", train=True),
        # which of 131072 nodes (or words) comes next
        dict(name="loss_nodes_bf16", kind="loss", rows=8_192, dim=256, classes=131_072, bias=False, reduction="mean", dtype="bf16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "rows", "sum", "loss", "loss"])
    dtype, train = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.6
    if kind == "loss":
        dim, classes = _log(rng, 16, 1024), _log(rng, 8, 131_072)
        if rng.random() < 0.5:
            dim = max(16, dim // 16 * 16)
        # work of the largest listed case; in 32 bits a product is six of 16
        most = min(67_584, (1 << 30) // classes, int(2.7e11 / (dim * classes)) // (6 if dtype == "f32" else 1))
        return dict(kind=kind, rows=_log(rng, 16, max(17, most)), dim=dim, classes=classes, bias=rng.random() < 0.5,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]), dtype=dtype, train=train)
    if kind == "route":
        groups = rng.choice([1, 1, 1, 2, 4, 8])
        per = max(2, _log(rng, 4, 512) // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(16, per * top_groups))
        rows = _log(rng, 1, min(151_552, (1 << 24) // (per * groups)))
        return dict(kind=kind, rows=rows, experts=per * groups, k=k, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    top_groups=top_groups, best=rng.choice([1, 2]), renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]), dtype=dtype, train=train)
    dim, k = _log(rng, 16, 1024), rng.randint(1, 8)
    if rng.random() < 0.5:
        dim = max(16, dim // 16 * 16)
    rows = _log(rng, 1, min(151_552, (1 << 28) // _BYTES[dtype] // (dim * k)))
    return dict(kind=kind, rows=rows, k=k, experts=_log(rng, 2, 512), dim=dim, dtype=dtype, train=train)


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train, kind, rows = _TORCH[case["dtype"]], case["train"], case["kind"], case["rows"]

    def normal(*shape, scale=1.0, dtype=dtype, leaf=train):
        t = torch.randn(shape, device="cuda", generator=gen).mul_(scale).to(dtype)
        return t.requires_grad_() if leaf else t

    s = dict(case=case)
    if kind == "loss":
        s["x"] = normal(rows, case["dim"])
        # logits that favour some classes, as behind some training
        s["weight"] = normal(case["classes"], case["dim"], scale=2.0 * case["dim"] ** -0.5)
        s["bias"] = normal(case["classes"], scale=0.5) if case["bias"] else None
        # small classes are the likelier ones; a row in about sixteen has no label
        u = torch.rand(rows, device="cuda", generator=gen)
        s["labels"] = (u * u * case["classes"]).long().clamp_(max=case["classes"] - 1)
        s["labels"][torch.rand(rows, device="cuda", generator=gen) < 1 / 16] = _IGNORE
        if train:
            s["grad"] = torch.rand(rows if case["reduction"] == "none" else (), device="cuda", generator=gen) + 0.5
        return s
    if kind == "route":
        experts = case["experts"]
        logits = normal(rows, experts, scale=1.5, leaf=False)
        # the rows behind the last real one of a padded batch go nowhere
        logits[rows - rows // 64:] = -_INF
        s["logits"] = logits.requires_grad_() if train else logits
        s["bias"] = normal(experts, scale=0.05, dtype=torch.float32, leaf=False) if case["bias"] else None
        if train:
            s["grad"] = normal(rows, case["k"], dtype=torch.float32, leaf=False)
        return s
    # experts as a router leaves them: some of them much liked, rows behind the last real one without any
    k, experts, dim = case["k"], case["experts"], case["dim"]
    liked = torch.randn(experts, device="cuda", generator=gen) * 0.7
    if k <= experts:
        noise = torch.rand((rows, experts), device="cuda", generator=gen).clamp_(1e-7, 1 - 1e-7)
        chosen = (liked - torch.log(-torch.log(noise))).topk(k, dim=1).indices
    else:
        chosen = torch.randint(0, experts, (rows, k), device="cuda", generator=gen)
    chosen[rows - rows // 64:] = -1
    s["experts"] = chosen
    if kind == "rows":
        s["x"] = normal(rows, dim)
        if train:
            s["grad"] = normal(rows * k, dim, leaf=False)
        return s
    s["place"] = _places(chosen, experts)[0]
    s["y"] = normal(rows * k, dim)
    w = torch.rand((rows, k), device="cuda", generator=gen) / k
    s["weights"] = w.requires_grad_() if train else w
    if train:
        s["grad"] = normal(rows, dim, leaf=False)
    return s


# ------------------------------------------------------------------------------------------------- plain operators
def _places(chosen, experts):
    """Where each (row, expert) goes when they are ordered by expert, which is at each place, and the experts' ends. Without an
    expert: behind all others, the place's complement."""
    flat = chosen.reshape(-1)
    order = torch.sort(torch.where(flat < 0, experts, flat), stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel(), device=flat.device)
    counts = torch.zeros(experts, dtype=torch.int64, device=flat.device)
    counts.index_add_(0, flat.clamp(min=0), (flat >= 0).long())
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return torch.where(flat < 0, -1 - place, place).view(chosen.shape), order, offsets


def _choose(case, logits, bias):
    """The experts that the rows go to: by 64-bit scores."""
    rows, experts, groups = case["rows"], case["experts"], case["groups"]
    z = logits.detach().double()
    none = z == -_INF
    if case["score"] == "softmax":
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - torch.where(top == -_INF, 0.0, top))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-z))
    if bias is not None:
        score = score + bias.double()
    # without a bias experts are ranked as their logits are
    choice = torch.where(none, -_INF, score if bias is not None else z)
    if groups > 1:
        per = torch.where(none, -_INF, score if bias is not None or case["best"] == 2 else z).view(rows, groups, -1)
        best = per.sort(dim=2, descending=True).values
        if case["best"] == 2:
            # a second expert counts where there is one
            value = best[..., 0] + torch.where(best[..., 1] == -_INF, 0.0, best[..., 1])
        else:
            value = best[..., 0]
        first = value.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((rows, groups), dtype=torch.bool, device=z.device).scatter_(1, first, True)
        choice = torch.where(kept.repeat_interleave(experts // groups, 1), choice, -_INF)
    value, chosen = choice.sort(dim=1, descending=True, stable=True)
    value, chosen = value[:, :case["k"]], chosen[:, :case["k"]]
    return torch.where(value == -_INF, -1, chosen)


def _plain_route(s):
    case, logits = s["case"], s["logits"]
    chosen = _choose(case, logits, s["bias"])
    z, real, at = logits.float(), chosen >= 0, chosen.clamp(min=0)
    if case["score"] == "softmax":
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - torch.where(top == -_INF, 0.0, top))
        score = e / e.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        score = 1 / (1 + torch.exp(-z))
    picked = torch.where(real, score.gather(1, at), 0.0)
    scale = case["scale"]
    total = picked.sum(1, keepdim=True).clamp(min=1e-30) if case["renorm"] else torch.ones_like(picked[:, :1])
    weights = picked / total * scale
    out = {"experts": chosen, "weights": weights}
    if case["train"]:
        g = torch.where(real, s["grad"], 0.0) * scale
        if case["renorm"]:
            g = (g - (g * picked).sum(1, keepdim=True) / total) / total
        ds = torch.zeros_like(z).scatter_add_(1, at, torch.where(real, g, 0.0))
        dz = score * (ds - (ds * score).sum(1, keepdim=True)) if case["score"] == "softmax" else ds * score * (1 - score)
        out["grad_logits"] = dz.to(logits.dtype)
    return out


def _plain_rows(s):
    case, x = s["case"], s["x"]
    place, order, offsets = _places(s["experts"], case["experts"])
    real = (s["experts"].reshape(-1)[order] >= 0).unsqueeze(1)
    out = {"rows": torch.where(real, x[order // case["k"]], 0.0), "offsets": offsets, "place": place}
    if case["train"]:
        back = s["grad"].float()[place.clamp(min=0).reshape(-1)] * (place.reshape(-1, 1) >= 0)
        out["grad_x"] = back.view(case["rows"], case["k"], -1).sum(1).to(x.dtype)
    return out


def _plain_sum(s):
    case, y, place = s["case"], s["y"], s["place"]
    real = place >= 0
    w = torch.where(real, s["weights"], 0.0)
    parts = y.float()[place.clamp(min=0).reshape(-1)].view(case["rows"], case["k"], -1)
    out = {"out": (parts * w.unsqueeze(2)).sum(1).to(y.dtype)}
    if case["train"]:
        g = s["grad"].float().unsqueeze(1)
        out["grad_y"] = torch.zeros_like(y).index_copy_(0, torch.where(real, place, -1 - place).reshape(-1), (g * w.unsqueeze(2)).view_as(y).to(y.dtype))
        out["grad_weights"] = torch.where(real, (parts * g).sum(2), 0.0)
    return out


def _plain_loss(s):
    case, labels = s["case"], s["labels"]
    x, weight = s["x"].float(), s["weight"].float()
    z = x @ weight.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    counted, at = labels != _IGNORE, labels.clamp(min=0).unsqueeze(1)
    top = z.amax(1, keepdim=True)
    picked = z.gather(1, at)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    losses = torch.where(counted, (torch.log(total) + top - picked).squeeze(1), 0.0)
    count = counted.sum().clamp(min=1)
    out = {"loss": losses if case["reduction"] == "none" else losses.sum() if case["reduction"] == "sum" else losses.sum() / count}
    if case["train"]:
        g = torch.where(counted, s["grad"] / count if case["reduction"] == "mean" else s["grad"], 0.0).unsqueeze(1)
        dz = e.mul_(g / total)
        dz.scatter_add_(1, at, -g)
        out["grad_x"] = (dz @ weight).to(s["x"].dtype)
        out["grad_weight"] = (dz.t() @ x).to(s["x"].dtype)
        if s["bias"] is not None:
            out["grad_bias"] = dz.sum(0).to(s["x"].dtype)
    return out


# --------------------------------------------------------------------------------------- the framework's operators
def _own_run(s):
    import apt_b200

    case = s["case"]
    kind, train = case["kind"], case["train"]
    if kind == "route":
        args = (s["logits"], case["k"], case["score"], s["bias"], case["groups"], case["top_groups"], case["best"], case["renorm"], case["scale"])
        experts, weights = (apt_b200.RouteExperts.apply if train else apt_b200.route_experts)(*args)
        out = {"experts": experts, "weights": weights}
        return {**out, "grad_logits": torch.autograd.grad(weights, s["logits"], s["grad"])[0]} if train else out
    if kind == "rows":
        rows, offsets, place = (apt_b200.ExpertRows.apply if train else apt_b200.expert_rows)(s["x"], s["experts"], case["experts"])
        out = {"rows": rows, "offsets": offsets, "place": place}
        return {**out, "grad_x": torch.autograd.grad(rows, s["x"], s["grad"])[0]} if train else out
    if kind == "sum":
        out = (apt_b200.ExpertSum.apply if train else apt_b200.expert_sum)(s["y"], s["weights"], s["place"])
        leaves = {"grad_y": s["y"], "grad_weights": s["weights"]}
        name = "out"
    else:
        op = apt_b200.LinearCrossEntropy.apply if train else apt_b200.linear_cross_entropy
        out = op(s["x"], s["weight"], s["labels"], s["bias"], case["reduction"], _IGNORE)
        leaves = {"grad_x": s["x"], "grad_weight": s["weight"], **({"grad_bias": s["bias"]} if s["bias"] is not None else {})}
        name = "loss"
    return {name: out, **(dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), s["grad"]))) if train else {})}


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return {"route": _plain_route, "rows": _plain_rows, "sum": _plain_sum, "loss": _plain_loss}[state["case"]["kind"]](state)


def work(case):
    size, rows, train = _BYTES[case["dtype"]], case["rows"], case["train"]
    if case["kind"] == "loss":
        dim, classes = case["dim"], case["classes"]
        params = classes * (dim + (1 if case["bias"] else 0)) * size
        return {"bytes": rows * dim * size * (2 if train else 1) + params * (2 if train else 1) + rows * 8,
                "flops": 2.0 * rows * dim * classes * (3 if train else 1)}
    k = case["k"]
    if case["kind"] == "route":
        logits = rows * case["experts"]
        return {"bytes": logits * size * (2 if train else 1) + rows * k * (16 if train else 12), "flops": logits * (4.0 + 2.0 * k) * (2 if train else 1)}
    row = case["dim"] * size
    if case["kind"] == "rows":
        return {"bytes": rows * row * (k + 1) * (2 if train else 1) + rows * k * 16 + (case["experts"] + 1) * 8, "flops": rows * k * case["dim"] * (1.0 if train else 0.0)}
    # y read once and its gradient written once; the gradient of the weights needs y beside what the forward read it for
    return {"bytes": rows * row * (k + 1) + rows * k * 12 + (rows * row * (k + 1) + rows * k * 4 if train else 0), "flops": rows * k * case["dim"] * (5.0 if train else 2.0)}


# --------------------------------------------------------------------------------------------- results in 64 bits
def _exact_route(case, s):
    """Row by row of a sorted list of pairs in numpy for the choice, autograd in 64 bits for the weights and the gradient."""
    rows, experts, k = case["rows"], case["experts"], case["k"]
    z = s["logits"].detach().double().cpu().numpy()
    bias = None if s["bias"] is None else s["bias"].double().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        if case["score"] == "softmax":
            shifted = np.exp(z - np.where(np.isfinite(z.max(1)), z.max(1), 0.0)[:, None])
            score = shifted / np.maximum(shifted.sum(1, keepdims=True), 1e-300)
        else:
            score = 1.0 / (1.0 + np.exp(-z))
    barred = np.isneginf(z)
    rank = z.copy() if bias is None else score + bias
    rank[barred] = -np.inf
    if case["groups"] > 1:
        value = rank if bias is not None or case["best"] == 1 else np.where(barred, -np.inf, score)
        value = np.sort(value.reshape(rows, case["groups"], -1), axis=2)[:, :, ::-1]
        group = value[:, :, 0] + (np.where(np.isneginf(value[:, :, 1]), 0.0, value[:, :, 1]) if case["best"] == 2 else 0.0)
        order = np.argsort(-group, axis=1, kind="stable")[:, case["top_groups"]:]
        out = np.zeros((rows, case["groups"]), dtype=bool)
        np.put_along_axis(out, order, True, axis=1)
        rank[np.repeat(out, experts // case["groups"], axis=1)] = -np.inf
    chosen = np.argsort(-rank, axis=1, kind="stable")[:, :k]
    chosen[np.isneginf(np.take_along_axis(rank, chosen, axis=1))] = -1
    chosen = torch.from_numpy(chosen).cuda()
    real = chosen >= 0
    # rows that go nowhere have weights and gradients of zero: any finite logits will do for them
    leaf = torch.where(real[:, :1], s["logits"].detach().double(), 0.0).requires_grad_()
    score = torch.softmax(leaf, 1) if case["score"] == "softmax" else torch.sigmoid(leaf)
    picked = score.gather(1, chosen.clamp(min=0)) * real
    weights = case["scale"] * (picked / picked.sum(1, keepdim=True).clamp(min=1e-300) if case["renorm"] else picked)
    out = {"experts": chosen, "weights": weights.detach()}
    if case["train"]:
        out["grad_logits"] = torch.autograd.grad(weights, leaf, s["grad"].double())[0]
    return out


def _exact_rows(case, s):
    flat = s["experts"].reshape(-1).cpu().numpy()
    known = np.flatnonzero(flat >= 0)
    order = np.concatenate([known[np.argsort(flat[known], kind="stable")], np.flatnonzero(flat < 0)])
    place = np.empty_like(order)
    place[order] = np.arange(len(order))
    offsets = np.searchsorted(flat[order[:len(known)]], np.arange(case["experts"] + 1))
    x, n = s["x"].detach().double(), len(known)
    rows = torch.zeros((len(flat), case["dim"]), dtype=torch.float64, device="cuda")
    rows[:n] = x[torch.from_numpy(order[:n] // case["k"]).cuda()]
    out = {"rows": rows, "offsets": torch.from_numpy(offsets.astype(np.int64)).cuda(),
           "place": torch.from_numpy(np.where(flat < 0, -1 - place, place)).view(case["rows"], case["k"]).cuda()}
    if case["train"]:
        out["grad_x"] = torch.zeros_like(x).index_add_(0, torch.from_numpy(order[:n] // case["k"]).cuda(), s["grad"].double()[:n])
    return out


def _exact_sum(case, s):
    y, w = s["y"].detach().double().requires_grad_(), s["weights"].detach().double().requires_grad_()
    row, slot = torch.nonzero(s["place"] >= 0, as_tuple=True)
    at = s["place"][row, slot]
    out = torch.zeros((case["rows"], case["dim"]), dtype=torch.float64, device="cuda").index_add(0, row, w[row, slot].unsqueeze(1) * y[at])
    if not case["train"]:
        return {"out": out.detach()}
    gy, gw = torch.autograd.grad(out, [y, w], s["grad"].double())
    return {"out": out.detach(), "grad_y": gy, "grad_weights": gw}


def _exact_loss(case, s):
    x, weight = s["x"].detach().double(), s["weight"].detach().double()
    bias = torch.zeros(case["classes"], dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].detach().double()
    counted = s["labels"] != _IGNORE
    share = 1.0 / max(1, int(counted.sum())) if case["reduction"] == "mean" else 1.0
    losses = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    gx, gw, gb = torch.zeros_like(x), torch.zeros_like(weight), torch.zeros_like(bias)
    step = max(1, (1 << 28) // case["classes"])
    for a in range(0, case["rows"], step):
        here = torch.nonzero(counted[a:a + step]).squeeze(1) + a
        if not len(here):
            continue
        label = s["labels"][here]
        p = torch.log_softmax(torch.addmm(bias, x[here], weight.T), dim=1)
        mine = torch.arange(len(here), device="cuda")
        losses[here] = -p[mine, label]
        if case["train"]:
            p.exp_()
            p[mine, label] -= 1.0
            p *= share * (s["grad"].double()[here].unsqueeze(1) if case["reduction"] == "none" else s["grad"].double())
            gx[here] = torch.mm(p, weight)
            gw.addmm_(p.T, x[here])
            gb += p.sum(dim=0)
    out = {"loss": losses if case["reduction"] == "none" else losses.sum() * share}
    if case["train"]:
        out.update(grad_x=gx, grad_weight=gw, **({"grad_bias": gb} if case["bias"] else {}))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "rows": _exact_rows, "sum": _exact_sum, "loss": _exact_loss}[case["kind"]](case, s)
