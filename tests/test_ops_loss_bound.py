"""The limits of the float32 loss's accuracy tell three bfloat16 parts from two (no GPU needed)."""

import ctypes
import math

import pytest
import torch

import loss_parts
import ops_helpers as plain
from test_ops_interface import entry, structure


@pytest.mark.parametrize("tokens,vocab,dim", [(300, 1000, 515), (129, 1500, 72)])
def test_limits_pass_three_parts_and_fail_fewer(tokens, vocab, dim):
    g = torch.Generator().manual_seed(tokens)
    hidden = torch.randn(tokens, dim, generator=g)
    weight = torch.randn(vocab, dim, generator=g) * (3 / math.sqrt(dim))
    targets = torch.randint(0, vocab, (tokens,), generator=g)
    targets[::5] = -100
    want = plain.cross_entropy(hidden, weight, targets, -100)
    for parts in (3, 2, 1):
        got = loss_parts.cross_entropy(hidden, weight, targets, parts)
        limits = (loss_parts.LOSS_LIMIT, loss_parts.GRADIENT_LIMIT, loss_parts.GRADIENT_LIMIT)
        for value, exact, limit in zip(got, (want["loss"], want["dh"], want["dw"]), limits):
            assert (loss_parts.relative(value, exact) <= limit) == (parts == 3)


@pytest.mark.parametrize("side", ["hidden", "weight"])
def test_third_part_decides(side):
    hidden, weight, targets, exact = loss_parts.third_part_decides("cpu", side)
    want = plain.cross_entropy(hidden, weight, targets, -100)["loss"]
    assert (want - exact).abs().max() <= 1e-12
    for parts in (3, 2):
        loss = loss_parts.cross_entropy(hidden, weight, targets, parts)[0]
        assert ((loss.double() - exact).abs().max() <= 0.5) == (parts == 3)


@pytest.mark.parametrize("tokens", [1000, 40000, 131072, 300000])
@pytest.mark.parametrize("code,parts", [(2, 1), (1, 3)])
def test_backward_workspace_is_bounded(tokens, code, parts):
    """The piece of dz takes 256 MB at most, or 1024 columns where those are more."""
    vocab, dim = 500_000, 64
    args = structure("PurinLossArgs")(dtype=code, tokens=tokens, vocab=vocab, dim=dim, hidden=4096,
                                      hidden_stride=dim, weight=4096, weight_stride=dim)
    size = ctypes.c_size_t()
    assert entry("purin_loss_workspace_size")(ctypes.byref(args), 1, ctypes.byref(size)) == 0
    piece = max(256 << 20, 1024 * 2 * parts * tokens)
    packed = 2 * parts * dim * (tokens + (vocab if parts == 3 else 0))
    splits = 148 // max(1, -(-tokens // 128)) + 1  # sums of dh: one for each part of K
    assert size.value <= piece + packed + splits * tokens * dim * 4 + 20 * tokens + 4096
