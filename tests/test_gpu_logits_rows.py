"""Controls from rows of one alignment into rows of another (the input is copied, then edited where it went)."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_logits import DEV, Case, assert_controlled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [4100, 9001])
@pytest.mark.parametrize("src,dst", [  # (padding of a row, floats before the first)
    ((4, 0), (4, 1)), ((4, 0), (3, 0)), ((3, 1), (4, 0)), ((1, 3), (2, 2)), ((0, 1), (0, 0)), ((7, 0), (3, 1)),
])
def test_rows_of_two_alignments(V: int, src: tuple[int, int], dst: tuple[int, int]) -> None:
    from microserve_b200 import _lib

    c = Case(4, 3, V, seed=V + 10 * src[0] + dst[0], gamma=3, first=1)
    want, mag = c.want()
    rows = c.B * c.R

    def place(pad: int, shift: int) -> tuple[torch.Tensor, torch.Tensor]:
        buf = torch.full((rows * (V + pad) + 8,), 7.0, device=DEV)
        return buf, buf[shift : shift + rows * (V + pad)].view(rows, V + pad)[:, :V]

    bufs, x = place(*src)
    bufd, y = place(*dst)
    x.copy_(torch.from_numpy(c.x))
    assert c.run(x, out=y) is y
    assert_controlled(y.cpu().numpy(), want, mag)
    assert torch.equal(y, c.run(x.contiguous()))  # the bits of the other kernel
    assert torch.equal(x.cpu(), torch.from_numpy(c.x))  # the input is only read
    for buf, view in ((bufs, x), (bufd, y)):
        view.fill_(7.0)
        assert (buf == 7.0).all()
    assert _lib.device_error() == 0


def test_a_single_row_of_any_stride() -> None:
    """A column of logits, transposed, is one row whose stride is 1."""
    c = Case(1, 1, 4100, seed=3)
    want, mag = c.want()
    x = torch.from_numpy(c.x).to(DEV).reshape(4100, 1).t()
    assert x.shape == (1, 4100) and x.stride(0) == 1
    assert_controlled(c.run(x).cpu().numpy(), want, mag)
    assert c.run(x, out=x) is x
    assert_controlled(x.cpu().numpy(), want, mag)
