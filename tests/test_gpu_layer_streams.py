"""The texel layers and the encoder on streams other than the default one."""
import pytest
import torch

from tests.model_utils import make_texture, rel_l2

pytestmark = pytest.mark.gpu


def _encoder(seed):
    import neural_textures_b200 as nt
    tex = make_texture((64, 64), ((32, 32), (16, 16)), 8, 8, lattice=(32, 32), seed=seed)
    features = tex.target.view(32, 2, 32, 2, 8).permute(0, 2, 1, 3, 4).reshape(32, 32, 32).contiguous()
    return nt.LatentEncoder(tex, grid=0, features=32), features


def test_encoder_step_on_a_side_stream(cuda):
    """The same step on the default stream and, behind 20 ms of other work, on another.  The passes add in no fixed
    order, so gradients differ by fp32 rounding, and by one 4-bit step (1/4 of a value at most) where that
    moves a value across a tie: one value in 10^4 does, 1/4 sqrt(10^-4) of the norm."""
    plain, features = _encoder(7)
    plain.train_step(features)
    torch.cuda.synchronize()
    enc, features = _encoder(7)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
        enc.train_step(features)
    side.synchronize()
    assert torch.equal(enc.tex.grids[0], plain.tex.grids[0])
    for a, b in zip(enc.layers, plain.layers):
        for g, h in zip(a.grads, b.grads):
            assert float(h.abs().max()) > 0
            assert rel_l2(g.cpu().numpy(), h.cpu().numpy()) <= 2.5e-3
    assert not any(g.any() for g in enc.tex.ggrads)
