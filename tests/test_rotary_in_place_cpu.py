"""What rotary refuses in place; the check comes before any launch, so no device is needed."""

import pytest
import torch

from saelens_b200.ops import _build

pytestmark = pytest.mark.skipif(_build._so_path() is None, reason="the extension is not built")
F = torch.ones(32, dtype=torch.float64)


def in_place(q, k=None):
    _build.load().rotary(q, k, F, None, 0, False, 1.0, True)


@pytest.mark.parametrize("size,stride", [((1, 2, 3, 64), (0, 200, 32, 1)), ((1, 2, 3, 64), (0, 64, 64, 1)), ((2, 1, 3, 64), (1, 0, 64, 1)),
                                         ((1, 2, 2, 64), (0, 127, 64, 1)), ((2, 2, 2, 64), (256, 128, 0, 1)), ((1, 1, 1, 64), (0, 0, 0, 2))])
def test_values_that_are_there_twice(size, stride):
    """Windows over one buffer: threads that turn neighbouring heads would write the same values."""
    t = torch.zeros(2000).as_strided(size, stride)
    with pytest.raises(ValueError, match="no value twice"):
        in_place(t)
    with pytest.raises(ValueError, match="no value twice"):
        in_place(torch.zeros(*size), t)


def test_views_that_hold_each_value_once():
    qkv = torch.zeros(2, 5, 8 * 64 + 24)
    heads = qkv[..., 8 : 8 + 4 * 64].view(2, 5, 4, 64)
    whole = torch.zeros(4, 3, 5, 80)
    for t in (heads, heads[:, ::2], heads.transpose(0, 1), heads.transpose(1, 2), whole[..., 7:71], whole.permute(2, 0, 1, 3)[..., :64], heads[:1],
              heads[:, :1, 3:], torch.zeros(2, 5, 4, 2, 64)[..., 1, :], torch.zeros(1, 2, 3, 64).as_strided((1, 2, 3, 64), (0, 192, 64, 1))):
        with pytest.raises(RuntimeError, match="must be CUDA"):  # past the check, at the launch
            in_place(t)
