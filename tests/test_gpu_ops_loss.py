"""The linear cross entropy over several pieces of the vocabulary, and its float32 accuracy."""

import ctypes
import math

import pytest
import torch

import loss_parts
import ops_helpers as plain
from purin_b200 import linear_cross_entropy
from test_ops_interface import entry, structure

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def release():
    yield
    torch.cuda.empty_cache()


def inputs(tokens, vocab, dim, dtype, ignored=0.05):
    g = torch.Generator(device=DEV).manual_seed(tokens + vocab)
    hidden = torch.randn(tokens, dim, generator=g, device=DEV).to(dtype)
    weight = (torch.randn(vocab, dim, generator=g, device=DEV) * (3 / math.sqrt(dim))).to(dtype)
    targets = (torch.rand(tokens, generator=g, device=DEV) * vocab).long()
    targets[torch.rand(tokens, generator=g, device=DEV) < ignored] = -100
    return hidden, weight, targets, g


def workspace(tokens, vocab, dim, dtype, backward):
    loss = structure("PurinLossArgs")(dtype=2 if dtype == torch.bfloat16 else 1, tokens=tokens, vocab=vocab,
                                      dim=dim, hidden=4096, hidden_stride=dim, weight=4096, weight_stride=dim)
    size = ctypes.c_size_t()
    assert entry("purin_loss_workspace_size")(ctypes.byref(loss), backward, ctypes.byref(size)) == 0
    return size.value


def in_rows(hidden, weight, targets, cotangent, step=500):
    """Losses and gradients for a cotangent per token, in 64 bits, some rows at a time."""
    w = weight.double()
    losses = torch.zeros(len(targets), dtype=torch.float64, device=DEV)
    dh = torch.zeros(hidden.shape, dtype=torch.float64, device=DEV)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    for at in range(0, len(targets), step):
        h, y = hidden[at:at + step].double(), targets[at:at + step]
        real = y >= 0
        y = torch.where(real, y, 0)[:, None]
        z = h @ w.t()
        lse = torch.logsumexp(z, 1, keepdim=True)
        losses[at:at + step] = torch.where(real, (lse - z.gather(1, y))[:, 0], 0.0)
        if cotangent is None:
            continue
        dz = z.sub_(lse).exp_().scatter_add_(1, y, torch.full(y.shape, -1.0, dtype=torch.float64, device=DEV))
        dz *= torch.where(real, cotangent[at:at + step].double(), 0.0)[:, None]
        dh[at:at + step] = dz @ w
        dw += dz.t() @ h
    return losses, dh, dw


# bfloat16: dz is rounded before its products, and so is the gradient, each by 2^-9 at most.
LIMIT = {torch.bfloat16: 2.0 ** -8, torch.float32: loss_parts.GRADIENT_LIMIT}


def assert_rows(got, exact, limit, step):
    """Norm-wise over every ``step`` rows, so that a part left out shows wherever it is."""
    for at in range(0, len(exact), step):
        assert loss_parts.relative(got[at:at + step], exact[at:at + step]) <= limit, at


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_over_pieces_of_the_vocabulary(dtype, reduction):
    """More columns of dz than one piece holds, the last piece shorter; two groups of rows."""
    tokens, vocab, dim = 5000, 60001, 24
    parts = 1 if dtype == torch.bfloat16 else 3
    whole = 2 * parts * tokens * vocab
    assert workspace(tokens, vocab, dim, dtype, 1) < whole / 2  # three pieces, or seven
    hidden, weight, targets, g = inputs(tokens, vocab, dim, dtype)
    count = int((targets >= 0).sum())
    assert count > 4096
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets, reduction=reduction)
    if reduction == "mean":
        cotangent, given = torch.full((tokens,), 1.0 / count, dtype=torch.float64, device=DEV), None
    else:
        cotangent = given = torch.randn(tokens, generator=g, device=DEV)
    got = torch.autograd.grad(loss, (h, w), given)
    losses, dh, dw = in_rows(hidden.detach(), weight.detach(), targets, cotangent)
    if reduction == "mean":
        losses = losses.sum() / count
    assert loss_parts.relative(loss.detach(), losses) <= loss_parts.LOSS_LIMIT
    assert_rows(got[0], dh, LIMIT[dtype], 500)
    assert_rows(got[1], dw, LIMIT[dtype], 1000)
    assert bool((got[0][targets < 0] == 0).all())
    again = torch.autograd.grad(linear_cross_entropy(h, w, targets, reduction=reduction), (h, w), given)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 1_100_003), (torch.float32, 560_003)])
def test_loss_with_several_tiles_to_a_partial_result(dtype, vocab):
    """Beyond some 8e9 logits a partial result covers several tiles of columns."""
    tokens, dim = 8192, 8
    one_tile = 8 * tokens * (vocab // 256 + 1) * (1 if dtype == torch.bfloat16 else 2)
    packed = (0 if dtype == torch.bfloat16 else 6 * vocab * dim) + 64 * tokens
    assert workspace(tokens, vocab, dim, dtype, 0) < packed + 0.6 * one_tile
    hidden, weight, targets, _ = inputs(tokens, vocab, dim, dtype)
    targets[0], targets[1], targets[2] = vocab - 1, 255, 256
    each = linear_cross_entropy(hidden, weight, targets, reduction="none")
    losses, _, _ = in_rows(hidden, weight, targets, None, step=256)
    assert loss_parts.relative(each, losses) <= loss_parts.LOSS_LIMIT
    # No row alone is off: a tile left out would change its loss by some 256 / vocab.
    assert bool(((each.double() - losses).abs() <= 2.0 ** -16 * (1 + losses.abs())).all())


@pytest.mark.parametrize("tokens,vocab,dim", [(100, 1000, 515), (300, 1000, 515), (257, 5000, 264), (700, 9000, 72),
                                              (129, 4099, 1031)])
def test_float32_loss_accuracy(tokens, vocab, dim):
    hidden, weight, targets, _ = inputs(tokens, vocab, dim, torch.float32, ignored=0.2)
    want = plain.cross_entropy(hidden, weight, targets, -100)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    each = linear_cross_entropy(h, w, targets, reduction="none")
    assert loss_parts.relative(each.detach(), want["loss"]) <= loss_parts.LOSS_LIMIT
    dh, dw = torch.autograd.grad(each.sum() / want["count"], (h, w))
    mean = torch.autograd.grad(linear_cross_entropy(h, w, targets), (h, w))
    for got in ((dh, dw), mean):
        assert loss_parts.relative(got[0], want["dh"]) <= loss_parts.GRADIENT_LIMIT
        assert loss_parts.relative(got[1], want["dw"]) <= loss_parts.GRADIENT_LIMIT


@pytest.mark.parametrize("side", ["hidden", "weight"])
@pytest.mark.parametrize("repeat", [1, 2])
def test_float32_logits_of_third_parts(side, repeat):
    """repeat: rows for a single CTA, and for a pair."""
    hidden, weight, targets, exact = loss_parts.third_part_decides(DEV, side)
    rows = 1 if repeat == 1 else 129
    loss = linear_cross_entropy(hidden.repeat(rows, 1), weight, targets.repeat(rows), reduction="none")
    assert (loss.double() - exact.repeat(rows)).abs().max().item() <= 0.5
