"""Routings that are not whole are refused on the host (no GPU needed)."""

import pytest
import torch

from purin_b200 import ExpertRouting, routing


def whole(tokens=4, slots=2, experts=3):
    n = tokens * slots
    return ExpertRouting(torch.zeros(experts + 1, dtype=torch.int32),
                         torch.arange(n, dtype=torch.int32).view(tokens, slots), torch.arange(n, dtype=torch.int32))


@pytest.fixture(autouse=True)
def any_device(monkeypatch):
    """The checks behind that of the device."""
    monkeypatch.setattr(routing._ops, "require_cuda", lambda what, *tensors: None)


def test_a_whole_routing_passes():
    routing._check_routing("dispatch", torch.zeros(4, 8), whole())
    routing._check_routing("dispatch", torch.zeros(4, 8), whole()._replace(source=None))
    routing._check_routing("dispatch", torch.zeros(0, 8), whole(tokens=0))


@pytest.mark.parametrize("error,change", [
    (ValueError, lambda r: r._replace(position=r.position[:, :1])),      # a view with another stride
    (ValueError, lambda r: r._replace(position=r.position[:2])),         # positions of rows that are not there
    (ValueError, lambda r: r._replace(position=r.position.t())),
    (ValueError, lambda r: r._replace(position=r.position.reshape(-1))),
    (ValueError, lambda r: r._replace(offsets=r.offsets[:, None])),
    (ValueError, lambda r: r._replace(offsets=r.offsets[:1])),
    (ValueError, lambda r: r._replace(offsets=r.offsets[::2])),
    (TypeError, lambda r: r._replace(position=r.position.long())),
    (TypeError, lambda r: r._replace(offsets=r.offsets.float())),
])
def test_parts_and_views_are_refused(error, change):
    with pytest.raises(error, match="routing"):
        routing._check_routing("dispatch", torch.zeros(4, 8), change(whole()))


def test_a_view_read_as_contiguous_names_rows_behind_the_output():
    """Why they are refused: the values at the view's address, one after another."""
    position = whole().position
    view = position[:, :1]
    read = view.as_strided((4,), (1,))  # what a kernel that knows no strides reads
    assert read.tolist() != view[:, 0].tolist()
    assert int(view.max()) >= view.numel()  # rows of dispatch's output
