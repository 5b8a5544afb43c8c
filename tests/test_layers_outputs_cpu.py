"""Which maps a group norm may write: any whose elements lie apart, in any order of the axes."""
import ctypes as C
import itertools

import pytest

from tests.test_layers_cpu import _norm


def _strides(order):
    """Strides of a dense 2 x 4 x 5 x 12 map whose axes lie in `order`, the innermost first."""
    extents, step, out = {"image": 2, "row": 4, "texel": 5}, 12, {}
    for axis in order:
        out[axis + "_stride"] = step
        step *= extents[axis]
    return out


@pytest.mark.parametrize("order", list(itertools.permutations(("image", "row", "texel"))), ids="-".join)
def test_written_maps_may_have_any_order(native, order):
    """Not an argument error: on a machine without a GPU the call gets as far as its launch."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses here are no memory")
    from neural_textures_b200 import _native as N
    for entry, name in ((native.nt_group_norm_forward, "y"), (native.nt_group_norm_backward, "dx")):
        fits = {f"{name}__{k}": v for k, v in _strides(order).items()}
        assert entry(C.byref(_norm(**fits)), None) != 1, N.last_error()
        for axis in order:  # one element less and that axis steps into what lies inside it
            less = dict(fits)
            less[f"{name}__{axis}_stride"] -= 1
            assert entry(C.byref(_norm(**less)), None) == 1
            assert "overlap" in N.last_error()
