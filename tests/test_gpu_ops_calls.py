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


def test_norm_of_tensors_with_a_graph_raises_when_differentiated():
    x = torch.arange(6.0, device=DEV).view(2, 3).requires_grad_()
    y = x * x
    want = float(y.detach().double().square().sum().sqrt())
    for of in (lambda t: t, lambda t: t[:, ::2]):
        norm = gradient_norm([of(y), torch.zeros(3, device=DEV)])
        with pytest.raises(RuntimeError, match="gradient_norm is not differentiable"):
            norm.backward()
    assert abs(gradient_norm(y).item() - want) <= 1e-6 * want
    with torch.no_grad():
        assert not gradient_norm(y).requires_grad
    assert not gradient_norm(y.detach()).requires_grad


@pytest.mark.parametrize("index", range(6))
@pytest.mark.parametrize("tracer", ["make_fx", "make_fx before dispatch", "jit"])
def test_operators_are_not_traced_as_empty_memory(index, tracer):
    from torch.fx.experimental.proxy_tensor import make_fx

    _, run, t = operators()[index]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        if tracer == "jit":
            torch.jit.trace(run, t, check_trace=False)
        else:
            make_fx(run, pre_dispatch="before" in tracer)(t)
    run(t)


def test_gradients_and_routes_are_not_traced_as_empty_memory():
    from torch.fx.experimental.proxy_tensor import make_fx

    t = torch.ones(9, device=DEV)
    for run in (lambda v: gradient_norm([v]), lambda v: clip_gradients([v], 1.0),
                lambda v: route_to_experts((v > 0).int().view(9, 1), 2)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(run)(t)
    assert bool((t == 1).all())


def test_other_dispatch_modes_see_the_operators_run():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Passing(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for _, run, t in operators():
        with Passing():
            got = run(t)
        assert torch.equal(got, run(t))


def test_clipping_does_not_write_what_it_refuses():
    """Tensors of inference mode are not written outside it."""
    with torch.inference_mode():
        t = torch.full((1000,), 2.0, device=DEV)
    with pytest.raises(RuntimeError, match="nference"):
        clip_gradients([t], 1.0)
    assert bool((t == 2).all())
    with torch.inference_mode():
        clip_gradients([t], 1.0)
    assert abs(float(t.double().norm()) - 1.0) < 1e-5


def test_clipping_by_an_infinite_norm():
    """As documented: finite values become zero, infinite ones NaN; a NaN norm makes all NaN."""
    for bad, others in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        t = torch.ones(5000, device=DEV)
        t[777] = bad
        norm = clip_gradients([t], 1.0)
        assert not bool(torch.isfinite(norm)) and bool(torch.isnan(t[777]))
        t[777] = others
        assert torch.equal(t.nan_to_num(7.0), torch.full_like(t, others).nan_to_num(7.0))
    big = [torch.full((100,), 3e38, device=DEV) for _ in range(2)]  # beyond float32, not float64
    norm = clip_gradients(big, 1.0)
    assert bool(torch.isinf(norm))
    assert all(abs(float(b.double().square().sum()) - 0.5) < 1e-5 for b in big)


def test_scale_that_needs_a_gradient_is_refused():
    table, ids = torch.ones(4, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    scale = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(TypeError, match="number"):
        token_embedding(table, ids, scale=scale)
    with torch.no_grad():
        assert bool((token_embedding(table, ids, scale=scale) == 2).all())
    assert bool((token_embedding(table, ids, scale=scale.detach()) == 2).all())


@pytest.mark.parametrize("dim", [5, 72, 130, 1031])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_outside_the_rows_are_neither_read_nor_written(dtype, dim):
    """A routing made by hand: such slots are dropped, and the memory around keeps its values."""
    tokens, slots, far = 6, 3, 2 ** 31 - 1
    routing = route_to_experts(torch.arange(18, device=DEV).view(6, 3) % 5, 5)
    position = routing.position.clone()
    bad = torch.zeros(6, 3, dtype=torch.bool, device=DEV)
    for at, value in (((0, 0), 18), ((1, 2), far), ((2, 1), -1), ((5, 2), -far - 1), ((4, 0), 19)):
        position[at] = value
        bad[at] = True
    offsets = routing.offsets.clone()
    offsets[-1] = 1000  # more rows than there are
    made = routing._replace(position=position, offsets=offsets)
    g = torch.Generator(device=DEV).manual_seed(dim)
    x = torch.randn(tokens, dim, generator=g, device=DEV).to(dtype).requires_grad_()
    rows = torch.randn(18, dim, generator=g, device=DEV).to(dtype).requires_grad_()
    weights = torch.rand(tokens, slots, generator=g, device=DEV).requires_grad_()
    kept = ~bad
    at = torch.where(kept, position, 0).long()
    sent = dispatch_to_experts(x, made)
    assert torch.equal(sent[position[kept].long()], x[kept.nonzero()[:, 0]])
    picked = torch.where(kept[:, :, None], rows.detach().double()[at], 0.0)
    out = combine_from_experts(rows, weights, made)
    want = (picked * weights.detach().double()[:, :, None]).sum(1)
    limit = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -20
    assert (out.double() - want).abs().max() <= limit * (1 + want.abs().max())
    grad = torch.randn(tokens, dim, generator=g, device=DEV).to(dtype)
    drows, dweights = torch.autograd.grad(out, (rows, weights), grad)
    want = (picked * grad.double()[:, None, :]).sum(2)
    assert (dweights.double() - want).abs().max() <= 2.0 ** -16 * (1 + want.abs().max())
    assert bool((dweights[bad] == 0).all())
    want = (grad.double()[:, None, :] * weights.detach().double()[:, :, None])[kept]
    assert (drows.double()[position[kept].long()] - want).abs().max() <= limit * (1 + want.abs().max())
    back = torch.randn(18, dim, generator=g, device=DEV).to(dtype)
    dx, = torch.autograd.grad(sent, x, back)
    want = torch.where(kept[:, :, None], back.double()[at], 0.0).sum(1)
    assert (dx.double() - want).abs().max() <= limit * (1 + want.abs().max())


def test_routings_that_are_not_whole_are_refused():
    routing = route_to_experts(torch.arange(18, device=DEV).view(6, 3) % 5, 5)
    x, rows, weights = torch.ones(6, 8, device=DEV), torch.ones(18, 8, device=DEV), torch.ones(6, 3, device=DEV)
    cases = [(ValueError, dict(position=routing.position[:, :1])), (ValueError, dict(position=routing.position[:2])),
             (ValueError, dict(offsets=routing.offsets.cpu())), (ValueError, dict(offsets=routing.offsets[::2])),
             (ValueError, dict(position=routing.position.cpu())), (TypeError, dict(position=routing.position.long()))]
    for error, change in cases:
        made = routing._replace(**change)
        tokens, slots = made.position.shape
        with pytest.raises(error):
            dispatch_to_experts(x[:tokens], made)
        with pytest.raises(error):
            combine_from_experts(rows[:tokens * slots], weights[:tokens, :slots], made)


def test_recording_leaves_captured_calls_out():
    """A captured call has no time of its own; asking for it is not the next call's error."""
    from purin_b200 import _native_ops

    x, ids = torch.ones(5, 4, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    token_embedding(x, ids)
    torch.cuda.synchronize()
    _native_ops.recorded_launches()
    _native_ops.record_launches(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = token_embedding(x, ids)
    gradient_norm(x)
    _native_ops.record_launches(False)
    assert [name for name, ms in _native_ops.recorded_launches() if ms > 0] == ["purin_gradients"]
    graph.replay()
    assert torch.equal(captured, token_embedding(x, ids))
