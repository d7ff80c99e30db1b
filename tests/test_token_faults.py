"""Faults found in the token-model operators, one test each: what a call answered wrongly, and what it answers."""
import math

import pytest
import torch

import beyond_deep_ensembles_amd as bde
from tests.test_token_ops import F32, BF16, U, backend, gen, teacher  # noqa: F401  (backend: the fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["nodes", "python"])
def test_forward_and_backward_captured_into_two_graphs(path, monkeypatch):
    """The backward's graph computes the gradient itself at every replay: the forward's graph may not run in between, the caller
    may have changed the last result in place, and the upstream value may have been another one."""
    if path == "python":
        import beyond_deep_ensembles_amd.bbb_layers as L
        monkeypatch.setattr(L, "_native_nodes", lambda ops: None)
    dev = "cuda:0"
    z, values, indices, rest = (t.to(dev) for t in teacher(20, 2000, 8, F32, 0))

    def eager(logits, factor):
        y = logits.clone().requires_grad_()
        (g,) = torch.autograd.grad(bde.distillation_loss(y, values, indices, rest), y, torch.tensor(factor, device=dev))
        return g
    want = {f: eager(z, f) for f in (1.0, 0.5)}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = z.clone().requires_grad_()                 # (a leaf of this stream's)
        up = torch.ones((), device=dev)
        forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(forward, stream=s):
            loss = bde.distillation_loss(x, values, indices, rest)
        with torch.cuda.graph(backward, stream=s):
            (g,) = torch.autograd.grad(loss, x, up)
    torch.cuda.current_stream().wait_stream(s)

    def run(graph):
        graph.replay()
        torch.cuda.synchronize()
    run(forward)
    run(backward)
    assert torch.equal(g, want[1.0])
    up.fill_(0.5)
    run(backward)
    assert torch.equal(g, want[0.5])
    up.fill_(1.0)
    run(backward)
    assert torch.equal(g, want[1.0]), "what an upstream value of 0.5 left"
    g.mul_(3.0)
    run(backward)
    assert torch.equal(g, want[1.0]), "what the caller made of the last gradient"
    with torch.no_grad():
        x.add_(torch.randn(x.shape, generator=gen(1)).to(dev))
    run(forward)
    run(backward)
    assert torch.equal(g, eager(x.detach(), 1.0))


@pytest.mark.gpu
def test_two_steps_captured_into_graphs_of_their_own():
    """Each graph holds a forward and its backward: both still take the gradient the forward pass finished, and neither takes the
    other's."""
    dev = "cuda:0"
    sides = [[t.to(dev) for t in teacher(12, 3000, 5, BF16, seed)] for seed in (1, 2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        leaves = [side[0].clone().requires_grad_() for side in sides]
        s.synchronize()
        for x, side in zip(leaves, sides):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                loss = bde.distillation_loss(x, *side[1:])
                (g,) = torch.autograd.grad(loss, x)
            graphs.append(graph)
            outs.append((loss, g))
            del loss, g
    torch.cuda.current_stream().wait_stream(s)
    for order in ((0, 1), (1, 0), (1, 1), (0, 0)):
        for i in order:
            graphs[i].replay()
            torch.cuda.synchronize()
            y = sides[i][0].clone().requires_grad_()
            want = bde.distillation_loss(y, *sides[i][1:])
            (gy,) = torch.autograd.grad(want, y)
            assert torch.equal(outs[i][0], want) and torch.equal(outs[i][1], gy)
            outs[i][1].zero_()
