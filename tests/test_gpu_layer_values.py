"""Values of the texel layers where they can go wrong: copies, far arguments, long sums, small gradients."""
import copy
import io

import numpy as np
import pytest
import torch

from tests import layer_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def f64(t):
    return t.detach().double().cpu().numpy()


def test_a_copied_layer_keeps_its_weights(cuda):
    import neural_textures_b200 as nt
    layer = nt.TexelLayer(48, 24, groups=6, seed=5)
    x = torch.randn((9, 13, 48), device="cuda").half()
    want = layer.forward(x)
    f = io.BytesIO()
    torch.save(layer, f)
    f.seek(0)
    copies = [copy.deepcopy(layer), torch.load(f, weights_only=False)]
    layer.weight.mul_(-2)
    layer.pack()
    torch.full((1 << 20,), 0xff, dtype=torch.uint8, device="cuda")  # over what the original's weights left
    for other in copies:
        assert torch.equal(other.forward(x), want)
    assert not torch.equal(layer.forward(x), want)
