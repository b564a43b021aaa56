"""Accuracy of the float32 loss: limits, and a CPU emulation with fewer bits that must fail them.

The operator takes a float32 value as three bfloat16 parts and six products of parts.  Errors
are compared norm-wise, rms(got - exact) / rms(exact):

* a logit's terms lose at most 2^-22 of |a||b| to the products left out, about 2^-25 in the
  mean, and each addition of the tensor cores truncates by at most 2^-23 of the running sum: some
  1e-7 of the logits' rms.  The loss adds a few roundings of its own size: LOSS_LIMIT is ten times that.
* the softmax gradient takes the logits' absolute error (they are of order 3) as a relative one,
  and that of its exponential, 2^-22: some 3e-7, and GRADIENT_LIMIT is six times that.

Two parts of a value keep 16 or 17 bits of it: 1.7e-6 in the loss and 7e-6 in the gradients.
"""

import math

import torch

LOSS_LIMIT = 2.0 ** -20
GRADIENT_LIMIT = 2.0 ** -19
LOG2E = 1.4426950408889634


def rms(x):
    return x.double().square().mean().sqrt().item()


def relative(got, exact):
    return rms(got.double() - exact) / rms(exact)


def _parts(x, count):
    """bfloat16 parts of float32 values; of three the first is cut off, as the operator does."""
    if count == 1:
        return [x.bfloat16().double()]
    first = (x.view(torch.int32) & ~0xffff).view(torch.float32)
    second = (x - first).bfloat16().float()
    third = (x - first - second).bfloat16()
    return [first.double(), second.double(), third.double()][:count]


def _truncated(x):
    y = x.float()
    too_far = y.double().abs() > x.abs()
    return torch.where(too_far, torch.nextafter(y, torch.zeros_like(y)), y).double()


def product(a, b, count):
    """``a @ b.T`` of float32 matrices by products of ``count`` parts of their values."""
    order = [(i, j) for i, j in ((0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)) if max(i, j) < count]
    pa, pb = _parts(a.contiguous(), count), _parts(b.contiguous(), count)
    out = torch.zeros(a.shape[0], b.shape[0])
    for k in range(0, a.shape[1], 64):
        block = torch.zeros(out.shape, dtype=torch.float64)
        for i, j in order:
            for at in range(k, min(k + 64, a.shape[1]), 16):
                end = min(at + 16, a.shape[1])
                block = _truncated(block + pa[i][:, at:end] @ pb[j][:, at:end].t())
        out += block.float()
    return out


def cross_entropy(hidden, weight, targets, count):
    """Losses and gradients of their mean as the operator makes them, from ``count`` parts."""
    z = product(hidden, weight, count)
    real = (targets >= 0) & (targets < weight.shape[0])
    y = torch.where(real, targets, 0)[:, None]
    top = z.max(1, keepdim=True).values * LOG2E
    e = torch.exp2((z.double() * LOG2E - top.double()).float())
    total = e.sum(1, keepdim=True)
    at_target = z.gather(1, y).double() * LOG2E
    loss = ((top.double() - at_target).float() + torch.log2(total)) * math.log(2.0)
    dz = (e / total).scatter_add(1, y, torch.full(y.shape, -1.0))
    dz = torch.where(real[:, None], dz, 0.0)
    n = max(int(real.sum()), 1)
    return (torch.where(real, loss[:, 0], 0.0), product(dz, weight.t(), count) / n,
            product(dz.t(), hidden.t(), count) / n)


def third_part_decides(device, side):
    """hidden, weight, targets, exact losses: logits k / 8 that are a difference of values which
    agree in their first two parts.  The two coordinates lie in different blocks of K, so their sums
    are added in registers.  ``side``: whether hidden or weight holds the values."""
    k = torch.arange(0, 128, dtype=torch.float64, device=device)
    wide = torch.zeros(128, 72, dtype=torch.float32, device=device)
    wide[:, 0] = (1 + 2.0 ** -8 + k * 2.0 ** -23).float()
    wide[:, 64] = 1 + 2.0 ** -8
    other = torch.zeros(2, 72, dtype=torch.float32, device=device)
    other[0, 0], other[0, 64] = 2.0 ** 20, -(2.0 ** 20)
    if side == "hidden":  # logits (k / 8, 0), target 1
        targets = torch.ones(128, dtype=torch.long, device=device)
        return wide, other, targets, torch.nn.functional.softplus(k / 8)
    # Two tokens, 128 words with the logits k / 8 and (second token) 0; targets: word 0.
    z = torch.stack([k / 8, torch.zeros_like(k)])
    return other, wide, torch.zeros(2, dtype=torch.long, device=device), torch.logsumexp(z, 1) - z[:, 0]
