"""Calls that the operators have to refuse, or answer in full, rather than lose a derivative."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from purin_b200 import (clip_gradients, combine_from_experts, dispatch_to_experts, gradient_norm,
                        linear_cross_entropy, route_to_experts, token_embedding)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operators():
    """(name, function of one tensor, that tensor) of everything that is differentiable."""
    g = torch.Generator(device=DEV).manual_seed(4)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    ids = torch.tensor([3, 0, 3, 5], device=DEV)
    routing = route_to_experts(torch.tensor([[0, 2], [1, 0], [2, -1], [0, 1]], device=DEV), 3)
    x, rows, weights, head = normal(4, 8), normal(8, 8), normal(4, 2), normal(6, 8)
    return [
        ("embedding", lambda t: token_embedding(t, ids), head),
        ("dispatch", lambda t: dispatch_to_experts(t, routing), x),
        ("combine rows", lambda t: combine_from_experts(t, weights, routing), rows),
        ("combine weights", lambda t: combine_from_experts(rows, t, routing), weights),
        ("loss hidden", lambda t: linear_cross_entropy(t, head, ids), x),
        ("loss weight", lambda t: linear_cross_entropy(x, t, ids), head),
    ]


@pytest.mark.parametrize("index", range(6))
@pytest.mark.parametrize("needs", [False, True])
def test_forward_mode_tangents_are_not_lost(index, needs):
    name, run, t = operators()[index]
    t = t.clone().requires_grad_(needs)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            run(fwd.make_dual(t, torch.ones_like(t)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            run(fwd.make_dual(t, torch.ones_like(t)))
        run(t)  # no tangent: as ever


@pytest.mark.parametrize("index", range(6))
def test_forward_mode_tangents_of_a_cotangent_are_not_lost(index):
    name, run, t = operators()[index]
    t = t.clone().requires_grad_()
    out = run(t)
    with fwd.dual_level():
        cotangent = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, t, cotangent)


def test_forward_mode_tangents_of_gradients_are_not_lost():
    t = torch.ones(40, 6, device=DEV)
    with fwd.dual_level():
        for of in (lambda d: d, lambda d: d[:, ::2]):
            dual = of(fwd.make_dual(t, torch.ones_like(t)))
            for run in (lambda: gradient_norm([dual]), lambda: clip_gradients([dual], 1.0)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    run()
        dual = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            clip_gradients([t.clone()], 1.0, out=[dual])
    assert bool((t == 1).all())
