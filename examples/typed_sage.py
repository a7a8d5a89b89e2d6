"""A GraphSAGE model with weights of its own for every node type, trained on sampled mini-batches of one GPU.

    python examples/typed_sage.py [--nodes 20000] [--steps 30] [--dtype bf16]

A mini-batch is sampled and its feature rows gathered by the data path; a layer then is

    neighbour means -> rows grouped by the type of their node -> grouped_linear -> group_norm_act (statistics of each row,
    silu, dropout) -> rows back in their places

How many nodes of a type a mini-batch has only the device knows, and nothing here asks: the groups' ends go from one kernel to the
next. The graph, the types, the features and the labels (which follow from type and features, so that there is something to learn) are
synthetic.
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import apt_b200  # noqa: E402
from apt_b200 import ops  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def install(num_nodes, degree, dim, types, classes, dtype, seed):
    """A random graph with self loops and a feature table, in the process-wide state; the nodes' types and labels."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    neighbours = torch.randint(0, num_nodes, (num_nodes, degree), device="cuda", generator=gen)
    neighbours[:, 0] = torch.arange(num_nodes, device="cuda")
    indptr = torch.arange(num_nodes + 1, device="cuda") * degree
    none = torch.empty(0, dtype=torch.int64)
    ops.mix_cache_graphs(0, none, none, none, indptr, neighbours.reshape(-1))
    ops.register_min_vids(torch.tensor([0, num_nodes]))
    node_type = torch.randint(0, types, (num_nodes,), device="cuda", generator=gen)
    feats = torch.randn((num_nodes, dim), device="cuda", generator=gen)
    planes = torch.randn((types, classes, dim), device="cuda", generator=gen)
    labels = torch.einsum("nd,ncd->nc", feats, planes[node_type]).argmax(1)
    cached = torch.arange(num_nodes)
    feats = feats.to(dtype)
    ops.cache_feats_shared(num_nodes, feats[:1].cpu().pin_memory(), feats, cached, cached[:1], 0)
    return node_type, labels


class NeighbourMean(torch.autograd.Function):
    """Means over a block's edges; the gradient is the sum over the same block with its two sides swapped."""

    @staticmethod
    def forward(ctx, x, block):
        ends = [torch.tensor([0, n], device=x.device) for n in (block.coo_row.numel(), block.num_src, block.num_dst)]
        ctx.block, ctx.ends = block, ends
        return ops.spmm_copy_u_sum(block.coo_row, block.coo_col, x, *ends).div_(block.fanout)

    @staticmethod
    def backward(ctx, grad):
        edges, src, dst = ctx.ends
        grad = (grad / ctx.block.fanout).contiguous()
        return ops.spmm_copy_u_sum(ctx.block.coo_col, ctx.block.coo_row, grad, edges, dst, src), None


class RowOrder(torch.autograd.Function):
    """Rows in another order, `order` a permutation; the gradient's rows go back."""

    @staticmethod
    def forward(ctx, x, order, back):
        ctx.order, ctx.back = order, back
        return ops.rows_scatter(x, order, x.shape[0]) if back else ops.rows_gather(x, order)

    @staticmethod
    def backward(ctx, grad):
        grad = grad.contiguous()
        return (ops.rows_gather(grad, ctx.order) if ctx.back else ops.rows_scatter(grad, ctx.order, grad.shape[0])), None, None


class TypedLayer(torch.nn.Module):
    def __init__(self, dim, out, types, norm_groups, drop, key, layer, dtype):
        super().__init__()
        self.weight = torch.nn.Parameter((torch.randn(types, out, 2 * dim, device="cuda") * (2 * dim) ** -0.5).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(types, out, device="cuda", dtype=dtype))
        self.last = norm_groups == 0
        if not self.last:
            self.gamma = torch.nn.Parameter(torch.ones(out, device="cuda"))
            self.beta = torch.nn.Parameter(torch.zeros(out, device="cuda"))
        self.types, self.norm_groups, self.drop, self.key, self.layer = types, norm_groups, drop, key, layer

    def forward(self, x, block, node_type, step):
        dst = torch.cat([x[:block.num_dst], NeighbourMean.apply(x, block)], 1)
        types, order = node_type[block.src_ids[:block.num_dst]].sort(stable=True)
        ends = torch.searchsorted(types, torch.arange(self.types + 1, device=types.device))
        h = apt_b200.GroupedLinear.apply(RowOrder.apply(dst, order, False), self.weight, ends, self.bias)
        h = RowOrder.apply(h, order, True)
        if self.last:
            return h
        # a stream of its own for every layer and step
        p = self.drop if self.training else 0.0
        return apt_b200.GroupNormAct.apply(h, self.norm_groups, self.gamma, self.beta, None, 1e-5, "silu", p, self.key, 64 * step + self.layer)


class TypedSAGE(torch.nn.Module):
    def __init__(self, dim, hidden, classes, types, layers, dtype, drop=0.1, key=2025):
        super().__init__()
        sizes = [dim] + [hidden] * (layers - 1) + [classes]
        self.layers = torch.nn.ModuleList(
            TypedLayer(a, b, types, 4 if k + 1 < layers else 0, drop, key, k, dtype) for k, (a, b) in enumerate(zip(sizes, sizes[1:])))

    def forward(self, x, blocks, node_type, step):
        for layer, block in zip(self.layers, blocks):
            x = layer(x, block, node_type, step)
        return x


def train(num_nodes=20000, degree=12, dim=64, hidden=128, classes=7, types=5, fanouts=(8, 5), batch=512, steps=30, dtype="bf16", seed=1, log=print):
    """Losses of the steps."""
    torch.manual_seed(seed)
    node_type, labels = install(num_nodes, degree, dim, types, classes, DTYPES[dtype], seed)
    model = TypedSAGE(dim, hidden, classes, types, len(fanouts), DTYPES[dtype])
    optimizer = torch.optim.Adam(model.parameters(), lr=5e-3, eps=1e-5)
    ops.set_sampling(key=seed, call_id=0)
    sampler = apt_b200.DPNeighborSampler(0, list(fanouts))
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    losses = []
    for step in range(steps):
        seeds = torch.randperm(num_nodes, device="cuda", generator=gen)[:batch]
        input_nodes, _, blocks = sampler.sample(None, seeds)
        logits = model(ops.load_subtensor(input_nodes), blocks, node_type, step)
        loss = torch.nn.functional.cross_entropy(logits.float(), labels[seeds])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if log and step % 10 == 0:
            log(f"step {step:4d}  loss {losses[-1]:.4f}  {input_nodes.numel()} input nodes")
    ops.check_status()
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--nodes", type=int, default=20000)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    args = parser.parse_args()
    found = train(num_nodes=args.nodes, steps=args.steps, dtype=args.dtype)
    print(f"loss of the first and the last five steps: {sum(found[:5]) / 5:.4f}  {sum(found[-5:]) / 5:.4f}")
