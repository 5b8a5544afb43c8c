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


@pytest.mark.parametrize("block,k", [(16, (1 << 28) + (1 << 20) + 40), (32, (1 << 29) + (1 << 21) + 72)])
def test_product_of_rows_whose_scales_pass_32_bits(cuda, block, k):
    """Rows that are zero but for 300 places, the last ones behind 2^31 bytes of scale tiles.  Zeros add nothing, so
    the sum rounds 300 times at most."""
    import neural_textures_b200 as nt
    g = torch.Generator().manual_seed(block)
    at = torch.cat((torch.randint(0, k, (280,), generator=g), k - 1 - torch.arange(0, 2000, 100))).unique().cuda()
    value = torch.exp2(torch.randint(-3, 4, (2, at.numel()), generator=g).float()).cuda()
    x = torch.zeros((1, k), dtype=torch.float16, device="cuda")
    packed, values = [], []
    for v in value:
        x[0, at] = v.half()
        packed.append(nt.mx4_quantize(x, block=block))
        back = nt.mx4_dequantize(packed[-1], torch.float16)
        values.append(f64(back[0, at]))
        assert int(torch.count_nonzero(back)) == at.numel()
        del back
    got = float(nt.mx4_product(*packed, dtype=torch.float32))
    want, size = float(values[0] @ values[1]), float(np.abs(values[0]) @ np.abs(values[1]))
    far = (at >= k - 2001).cpu().numpy()
    assert float(values[0][far] @ values[1][far]) > 1e-2 * size, "the far places count"
    assert abs(got - want) <= 308 * U * size


def test_encoder_gradients_of_many_samples(cuda, monkeypatch):
    """The gradients of 262,144 samples that are off by about 0.01 are 10^-8 each, below fp16's smallest step: the
    encoder's come out as those of 2^18 times larger ones, divided by 2^18, bit for bit."""
    import neural_textures_b200 as nt
    from neural_textures_b200 import encoder
    from tests.model_utils import make_texture
    tex = make_texture((512, 512), ((512, 512), (256, 256)), 8, 8, lattice=(512, 512), seed=3)
    g = torch.Generator(device="cuda").manual_seed(8)
    d = 1e-8 * torch.randn((512, 512, 8), generator=g, device="cuda")
    features = torch.randn((512, 512, 32), generator=g, device="cuda").half()
    monkeypatch.setattr(encoder, "InvokeTraining", lambda p, *a, stream=None: tex.ggrads[0].copy_(d))
    enc = nt.LatentEncoder(tex, grid=0, features=32)
    first, second = copy.deepcopy(enc.layers)
    enc.train_step(features)
    second.forward(first.forward(features, keep=True), keep=True)
    first.backward(second.backward(d * 2.0 ** 18))
    for layer, want in zip(enc.layers, (first, second)):
        for got, large in zip(layer.grads, want.grads):
            assert float(large.abs().max()) > 0
            assert torch.equal(got, large * 2.0 ** -18)


def test_layer_gradients_with_factors(cuda):
    """A gain is that of the result alone, a scale is taken out of the parameters' gradients: bit for bit."""
    import neural_textures_b200 as nt
    layer = nt.TexelLayer(48, 24, groups=6, seed=5)
    x, d = torch.randn((9, 13, 48), device="cuda").half(), torch.randn((9, 13, 24), device="cuda")
    layer.forward(x, keep=True)
    dx = layer.backward(d)
    grads = layer.grads
    tiny = layer.backward(d * 2.0 ** -30, gain=2.0 ** 30)
    assert torch.equal(tiny, dx) and all(torch.equal(a, b * 2.0 ** -30) for a, b in zip(layer.grads, grads))
    large = layer.backward(d * 2.0 ** 10, scale=2.0 ** 10, gain=2.0 ** -10)
    assert torch.equal(large, dx) and all(torch.equal(a, b) for a, b in zip(layer.grads, grads))
    for factors in ((0.0, 1.0), (1.0, -2.0), (float("nan"), 1.0), (1.0, float("inf"))):
        with pytest.raises(ValueError, match="positive"):
            layer.backward(d, *factors)
