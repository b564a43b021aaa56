"""Routings that are not whole are refused on the host (no GPU needed)."""

import pytest
import torch

from purin_b200 import ExpertRouting, routing


def whole(tokens=4, slots=2, experts=3):
    n = tokens * slots
    return ExpertRouting(torch.zeros(experts + 1, dtype=torch.int32),
                         torch.arange(n, dtype=torch.int32).view(tokens, slots), torch.arange(n, dtype=torch.int32))


@pytest.fixture(autouse=True, scope="module")
def built():
    from purin_b200.csrc.build import build

    build()


def test_a_whole_routing_passes_up_to_the_device():
    for made, tokens in ((whole(), 4), (whole()._replace(source=None), 4), (whole(tokens=0), 0)):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            routing._check_routing("dispatch", torch.zeros(tokens, 8), made)


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
