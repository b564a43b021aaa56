"""Backward passes of the operators in a graph, and calls on streams at the same time."""

import pytest
import torch

from purin_b200 import (clip_gradients, combine_from_experts, dispatch_to_experts, gradient_norm,
                        linear_cross_entropy, route_to_experts, token_embedding)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,slots", [(200, 2), (9001, 3)])  # one-launch sorts, and many blocks
def test_backward_passes_in_a_graph(tokens, slots, dtype):
    g = torch.Generator(device=DEV).manual_seed(tokens)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)

    vocab, dim, experts = 700, 72, 9
    table, head = normal(vocab, dim).requires_grad_(), normal(vocab, dim, scale=0.3).requires_grad_()
    weights = torch.rand(tokens, slots, generator=g, device=DEV).requires_grad_()
    ids = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    targets = torch.randint(-100, vocab, (tokens,), generator=g, device=DEV)
    chosen = torch.randint(-1, experts, (tokens, slots), generator=g, device=DEV)

    def step():
        x = token_embedding(table, ids, scale=0.5)
        routing = route_to_experts(chosen, experts)
        y = x + combine_from_experts(torch.tanh(dispatch_to_experts(x, routing)), weights, routing)
        loss = linear_cross_entropy(y, head, targets)
        grads = list(torch.autograd.grad(loss, (table, weights, head)))
        return [loss.detach(), clip_gradients(grads, 0.01), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        g.manual_seed(seed)
        ids.copy_(torch.randint(-1, vocab, (tokens,), generator=g, device=DEV))
        targets.copy_(torch.randint(-50, vocab, (tokens,), generator=g, device=DEV))
        chosen.copy_(torch.randint(-2, experts + 1, (tokens, slots), generator=g, device=DEV))
        graph.replay()
        got = [t.clone() for t in captured]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("slots", [64, 2500, 20000])  # a block's sort, a cluster's, many blocks'
def test_sorts_and_clips_on_two_streams(slots):
    g = torch.Generator(device=DEV).manual_seed(slots)
    inputs = []
    for _ in range(2):
        chosen = torch.randint(-1, 3000, (slots, 1), generator=g, device=DEV)
        grads = [torch.randn(n, generator=g, device=DEV) for n in (5, 3001, 70 * slots)]
        table = torch.randn(3000, 24, generator=g, device=DEV, requires_grad=True)
        inputs.append((chosen, grads, table))

    def run(chosen, grads, table):
        routing = route_to_experts(chosen, 3000)
        outs = [torch.empty_like(t) for t in grads]
        norm = clip_gradients(grads, 1.0, out=outs)
        grad, = torch.autograd.grad(token_embedding(table, chosen[:, 0]).sum(), table)
        return [*routing, norm, gradient_norm(grads), *outs, grad]

    want = [run(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for results in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(results, want[k]))
