"""Which captures gated_matmul refuses next to living eager graphs: on the graphs alone, and on a GPU."""
from __future__ import annotations

import pytest
import torch

from helion_b200 import gated


class Node:
    """Stands for the backward node of an eager forward pass over ``tensors``."""

    def __init__(self, *tensors):
        self.next_functions = tuple((torch.autograd.graph.get_gradient_edge(t).node, 0) for t in tensors if t.requires_grad) + ((None, 0),)


def test_leaves_are_found_below_what_is_computed_from_them():
    a, b, c = (torch.ones(2, requires_grad=True) for _ in range(3))
    living = Node(a * 2, b)
    gated._eager_nodes.add(living)
    for inputs in ((a,), (b,), (a * 3,), (c, (b + c).exp()), (c * 2, a[:1].sum().reshape(1) + c)):
        with pytest.raises(RuntimeError, match="still alive"):
            gated._refuse_capture(*inputs)
    gated._refuse_capture(c, c * 2, torch.ones(2))
    gated._refuse_capture((a * 2).detach().requires_grad_(), b.detach())
    del living
    gated._refuse_capture(a, b, a * b)


@pytest.mark.gpu
def test_an_input_computed_from_a_leaf_of_a_living_graph(built_library):
    import helion_b200 as hb

    g = torch.Generator(device="cuda").manual_seed(1)
    x0 = torch.randn(140, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    w = [torch.randn(64, 48, generator=g, device="cuda").bfloat16() for _ in range(2)]
    dh = torch.randn(140, 48, generator=g, device="cuda").bfloat16()
    eager = hb.gated_matmul(x0 * 2, *w)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            hb.gated_matmul(x0 * 2, *w)
    (want,) = torch.autograd.grad(eager, x0, dh)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(hb.gated_matmul(x0 * 2, *w), x0, dh)
    graph.replay()
    assert torch.equal(got, want)
