"""Sizes that the entries' 32-bit arguments cannot hold are refused: the binding would cut them off, and a part of the rows would be computed."""
import pytest
import torch

from dun_amd import act8
from dun_amd.layer_norm import layer_norm, layer_norm_forward
from tests.test_row_buffers_cpu import entries  # noqa: F401  (nothing may be launched: any call of an entry is counted)


def one_element(*shape, dtype=torch.float32):
    return torch.zeros(1, dtype=dtype).expand(*shape)


@pytest.mark.parametrize("cols", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 8])
def test_rows_that_are_too_long(entries, cols):  # noqa: F811
    x = one_element(1, cols, dtype=torch.float16)
    for call in (lambda: layer_norm(x), lambda: layer_norm_forward(x), lambda: act8.pack(x), lambda: layer_norm(one_element(cols))):
        with pytest.raises(RuntimeError, match="elements a row"):
            call()
    small = torch.zeros(1, 8)
    entries.hold(small)
    p = act8.pack(small)
    with pytest.raises(RuntimeError, match="elements a row"):
        act8.weight_grad(x, p)
    assert entries.calls == ["pack"]


@pytest.mark.parametrize("x,w", [((2 ** 31, 3), (5, 3)), ((2 ** 32 + 4, 3), (5, 3)), ((2 ** 16, 2 ** 16, 3), (5, 3)), ((4, 2 ** 32 + 4), (5, 2 ** 32 + 4)),
                                 ((4, 3), (2 ** 32 + 5, 3))])
def test_products_that_are_too_large(entries, x, w):  # noqa: F811
    with pytest.raises(RuntimeError, match="linear: .*2\\^31"):
        act8.linear(one_element(*x), one_element(*w))
    assert not entries.calls
