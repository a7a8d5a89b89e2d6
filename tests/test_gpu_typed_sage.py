"""examples/typed_sage.py: a layer against the same in plain PyTorch in 64 bits, gradients included, and a training run that learns."""
import os
import sys

import pytest
import torch

import apt_b200
from apt_b200 import ops

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(autouse=True)
def _state_as_before():
    """The graph and the feature table that a test installs go with it: other tests' samplers look rows up in whatever is installed."""
    state = ops.STATE
    before = state.feat, state.graph
    state.feat, state.graph = ops.FeatStorage(), ops.GraphStorage()
    yield
    state.feat, state.graph = before
    state.generation += 1


def test_a_layer_and_its_gradients():
    import typed_sage

    torch.manual_seed(0)
    node_type, _ = typed_sage.install(3000, 6, 32, 4, 3, torch.float32, 5)
    ops.set_sampling(key=9, call_id=0)
    _, _, (block,) = apt_b200.DPNeighborSampler(0, [5]).sample(None, torch.arange(300, device="cuda") * 7)
    layer = typed_sage.TypedLayer(32, 24, 4, 3, 0.0, 1, 0, torch.float32)
    x = torch.randn((block.num_src, 32), device="cuda", requires_grad=True)
    grad = torch.randn((block.num_dst, 24), device="cuda")
    leaves = [x] + list(layer.parameters())
    out = layer(x, block, node_type, 0)
    got = (out,) + torch.autograd.grad(out, leaves, grad)

    wide = [t.detach().double().requires_grad_() for t in leaves]
    names = dict(zip([n for n, _ in layer.named_parameters()], wide[1:]))
    mean = torch.zeros((block.num_dst, 32), dtype=torch.float64, device="cuda").index_add(0, block.coo_col, wide[0][block.coo_row]) / block.fanout
    both = torch.cat([wide[0][:block.num_dst], mean], 1)
    kind = node_type[block.src_ids[:block.num_dst]]
    h = torch.einsum("rk,rnk->rn", both, names["weight"][kind]) + names["bias"][kind]
    v = h.view(-1, 3, 8)
    var, centre = torch.var_mean(v, dim=2, unbiased=False, keepdim=True)
    z = ((v - centre) / torch.sqrt(var + 1e-5)).view_as(h) * names["gamma"] + names["beta"]
    want = torch.nn.functional.silu(z)
    want = (want,) + torch.autograd.grad(want, wide, grad.double())
    # sums of at most 300 terms in fp32 and some twenty roundings one after another, of which the norm's gradient subtracts two means: 2e-5
    for a, b in zip(got, want):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 2e-5
    ops.check_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_training_learns(dtype):
    import typed_sage

    losses = typed_sage.train(num_nodes=4000, steps=60, batch=256, dtype=dtype, log=None)
    # seven classes: log 7 = 1.95 knows nothing
    assert sum(losses[:3]) / 3 > 1.6 and sum(losses[-5:]) / 5 < 1.3, losses
