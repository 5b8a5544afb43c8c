"""The texel-layer operators together: TexelLayer against its formula in 64 bits, a LatentEncoder that
learns a texture's latents through the texture's training pass, latents stored in 4 bits."""
import numpy as np
import pytest
import torch

from tests import layer_oracle as O
from tests.model_utils import make_texture

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().double().cpu().numpy()


def test_texel_layer_forward_and_backward(cuda):
    """Operands are the layer's own 4-bit tensors read back, so only fp32 sums and the fp16 results differ:
    K / 16 + 8 units of the sum of magnitudes, then one rounding to fp16 (2^-11)."""
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(3)
    layer = nt.TexelLayer(48, 24, groups=6, seed=5)
    x = torch.randn((9, 13, 48), generator=g, device="cuda").half()
    d = torch.randn((9, 13, 24), generator=g, device="cuda") * 1e-6  # the size of a training pass's gradients
    out = layer.forward(x, keep=True)
    dx = layer.backward(d)
    y, mean, rstd = nt.group_norm(x, 6, layer.gamma, layer.beta, activation="silu")
    u = 2.0 ** -24

    def product(a, b, block, bias, dtype):
        A, B = (f64(nt.mx4_dequantize(nt.mx4_quantize(t, block=block), torch.float32)) for t in (a, b))
        return A @ B.T + bias, (A.shape[1] / 16 + 8) * u * (np.abs(A) @ np.abs(B).T + np.abs(bias))

    rows = y.view(-1, 48)
    want, tol = product(rows, layer.weight, 16, f64(layer.bias), torch.float16)
    got = f64(out).reshape(-1, 24)
    assert (np.abs(got - want) <= tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
    flat = d.view(-1, 24)
    want, tol = product(flat.t(), rows.t(), 32, 0.0, torch.float32)
    assert (np.abs(f64(layer.grads[0]) - want) <= tol + u * np.abs(want)).all()
    assert np.allclose(f64(layer.grads[1]), f64(flat).sum(axis=0), rtol=1e-5, atol=1e-9)
    dy = nt.mx4_product(nt.mx4_quantize(flat), nt.mx4_quantize(layer.weight.t()), dtype=torch.float16)
    again = nt.group_norm_backward(dy.view(x.shape), x, mean, rstd, 6, layer.gamma, layer.beta, activation="silu")
    for a, b in zip((dx, layer.grads[2], layer.grads[3]), again):
        assert torch.equal(a, b)
    assert float(dx.float().abs().max()) > 0, "gradients of 1e-6 survive the 4-bit products"


def test_latent_encoder_learns(cuda):
    """A grid texel covers a 2 x 2 block of the target, whose 32 values are its features.  The loss of
    the last 20 of 150 steps is at most half that of the first 20."""
    import neural_textures_b200 as nt
    tex = make_texture((64, 64), ((32, 32), (16, 16)), 8, 8, lattice=(32, 32), seed=7)
    features = tex.target.view(32, 2, 32, 2, 8).permute(0, 2, 1, 3, 4).reshape(32, 32, 32).contiguous()
    enc = nt.LatentEncoder(tex, grid=0, features=32)
    losses = []
    for _ in range(150):
        tex.loss_accum.zero_()
        enc.train_step(features)
        losses.append(tex.loss_accum.item())
    assert np.isfinite(losses).all()
    assert np.mean(losses[-20:]) <= 0.5 * np.mean(losses[:20]), (losses[:20], losses[-20:])
    grid = enc.encode(features)
    assert torch.isfinite(grid).all() and torch.equal(grid, tex.grids[0])
    with pytest.raises(ValueError, match="grid"):
        enc.encode(features[:16])


@pytest.mark.parametrize("block", [16, 32])
def test_latents_in_4_bits(cuda, block):
    """Grids of 8 and 12 channels, with and without mips, come back as the 64-bit restatement's values."""
    import neural_textures_b200 as nt
    for channels, mips in ((8, (1, 1)), (12, (3, 1))):
        tex = nt.NeuralTexture(64, 48, grid_sizes=((32, 24), (16, 12)), latent_channels=channels, num_mips=mips)
        tex.init(seed=2)
        before = [tex._mx4_rows(g).clone() for g in range(2)]
        packed = tex.export_mx4(block=block)
        for c in tex.grid_chains:
            c.zero_()
        tex.from_mx4(packed)
        for g in range(2):
            _, _, values = O.mx4_quantize(f64(before[g]), block)
            assert np.array_equal(f64(tex._mx4_rows(g)), values.astype(np.float16).astype(np.float64))
