"""Captured backwards of logits and weights that are made from leaves: where an eager graph of the leaves is alive, its default stream cannot join
the capture, which would end the process."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls(device):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    g = torch.Generator(device=device).manual_seed(3)
    index = torch.randint(0, 20, (300, 2), generator=g, device=device)
    leaf = lambda *s: torch.randn(*s, generator=g, device=device, requires_grad=True)
    return [(leaf(300, 20), lambda x: balance_loss(x * 2, 3)[0]),
            (leaf(300, 2), lambda x: neighbour_balance(x.softmax(-1), index, 20)[0]),
            (leaf(300, 20), lambda x: neighbour_balance(torch.gather(x, 1, index).softmax(-1), index, 20)[2].square().sum())]


def test_leaves_behind_the_logits(device):
    for leaf, call in _calls(device):
        alive = call(leaf)
        want, = torch.autograd.grad(alive, leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match='eager graph'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(leaf), leaf)
        torch.cuda.synchronize()
        assert torch.equal(torch.autograd.grad(alive, leaf)[0], want)  # the eager graph is whole
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(leaf), leaf)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(torch.autograd.grad(call(leaf), leaf)[0], want)


def test_eager_graphs_of_other_leaves_are_no_matter(device):
    """And so are those behind what the gradient is asked for: a detached tensor of the same memory is a leaf of its own."""
    for leaf, call in _calls(device):
        other = leaf.detach().clone().requires_grad_(True)
        alive = call(other) + call(leaf)
        want, = torch.autograd.grad(alive, leaf, retain_graph=True)
        fresh = leaf.detach().requires_grad_(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(fresh), fresh)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        del alive
