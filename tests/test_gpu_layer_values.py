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


# arguments of an activation, far ones among them
FAR = [-3e38, -1e20, -1e4, -200.0, -104.0, -100.0, -88.5, -87.0, -60.0, -50.0, -43.5, -43.0, -42.5, -30.0, -12.0, -5.0, -1.0,
       -1e-3, -1e-30, 0.0, 1e-30, 1e-3, 1.0, 5.0, 30.0, 60.0, 88.5, 200.0, 1e4, 1e20, 3e38]
FLT_MIN = 2.0 ** -126


def _far(act):
    """(z, activation(z), its slope, both as fp32 holds them, their tolerances).  silu's exponential is rounded relative to its argument,
    8 + |z| units; results below FLT_MIN may be 0.  gelu's integral of the normal distribution is good to 1.5e-7."""
    z = np.array(FAR, np.float32).astype(np.float64)
    with np.errstate(over="ignore"):
        value, slope = (v.astype(np.float32).astype(np.float64) for v in (O.activate(z, act), O.slope(z, act)))
    if act == "silu":
        s = np.exp(-np.logaddexp(0, -z))
        units = 2 * U * (8 + np.minimum(np.abs(z), 104))
        return z, value, slope, units * np.abs(value) + 104 * FLT_MIN, units * s * (2 + np.minimum(np.abs(z), 104)) + 104 * FLT_MIN
    bell = np.abs(z) * np.exp(-np.minimum(z * z, 2000) / 2)
    tail = np.where(z < -16, 0.0, 1.5e-7)
    return z, value, slope, tail * np.minimum(np.abs(z), 16) + 8 * U * np.abs(value), tail + 32 * U * (bell + 1) * (z > -16)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_of_far_arguments(cuda, act):
    """A map of zeros is normalised to zeros, so that z is beta and the gradient of beta the slope; zero codes leave
    a product its bias."""
    import neural_textures_b200 as nt
    z, value, slope, value_tol, slope_tol = _far(act)
    c = z.size
    beta = torch.tensor(z, dtype=torch.float32, device="cuda")
    x = torch.zeros((1, 1, 1, c), device="cuda")
    y, mean, rstd = nt.group_norm(x, 1, None, beta, activation=act)
    assert (np.abs(f64(y).ravel() - value) <= value_tol).all(), f64(y).ravel() - value
    _, _, dbeta = nt.group_norm_backward(torch.ones_like(x), x, mean, rstd, 1, None, beta, activation=act)
    assert (np.abs(f64(dbeta) - slope) <= slope_tol).all(), f64(dbeta) - slope
    for m, k in ((1, 64), (1, 4096), (200, 64)):
        a, b = nt.mx4_quantize(torch.zeros((m, k), device="cuda")), nt.mx4_quantize(torch.zeros((c, k), device="cuda"))
        d = f64(nt.mx4_product(a, b, bias=beta, activation=act, dtype=torch.float32))
        assert (np.abs(d - value) <= value_tol).all(), (m, k, d[0] - value)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_activations_of_infinities(cuda, act):
    """+inf stays; -inf is 0 under relu and, as 0 x inf, NaN under silu and gelu; a NaN is one."""
    import neural_textures_b200 as nt
    inf = float("inf")
    bias = torch.tensor([inf, -inf, float("nan"), 1.0], device="cuda")
    q = nt.mx4_quantize(torch.zeros((4, 64), device="cuda"))
    for m in (1, 200):
        d = nt.mx4_product(nt.mx4_quantize(torch.zeros((m, 64), device="cuda")), q, bias=bias, activation=act, dtype=torch.float32)
        assert (d[:, 0] == inf).all() and torch.isnan(d[:, 2]).all() and torch.isfinite(d[:, 3]).all()
        low = d[:, 1]
        assert {"none": (low == -inf).all(), "relu": (low == 0).all()}.get(act, torch.isnan(low).all())


def test_encoder_step_optimises_the_other_grid(cuda):
    """Beside a plain texture that starts from the encoded latents: its step moves the other grid by as much.  The two
    passes add in no fixed order, and a first step of Adam has a gradient's sign, so one value in 100 may differ."""
    import neural_textures_b200 as nt
    from tests.model_utils import make_texture
    make = lambda: make_texture((64, 64), ((32, 32), (16, 16)), 8, 8, lattice=(32, 32), seed=7)
    tex, plain = make(), make()
    features = tex.target.view(32, 2, 32, 2, 8).permute(0, 2, 1, 3, 4).reshape(32, 32, 32).contiguous()
    enc = nt.LatentEncoder(tex, grid=0, features=32)
    before = tex.grids[1].clone()
    plain.grids[0].copy_(enc.encode(features))
    enc.train_step(features)
    assert torch.equal(tex.grids[0], plain.grids[0])
    plain.train_step()
    assert float((plain.grids[1] != before).float().mean()) > 0.9
    assert float((plain.grids[1] == tex.grids[1]).float().mean()) >= 0.99
    assert not any(g.any() for g in tex.ggrads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("offset", [20.0, 1000.0])
def test_group_norm_statistics_behind_a_black_border(cuda, offset, dtype):
    """Every thread's first texels are 0 and the 8,000 after them `offset` deviations away: the variance must not
    be a difference of sums about that 0. Rounding errors of n values add like sqrt(n) = 91 units; sums about a
    pivot within the values so far are at most 4 times the centred ones: 364 of the 512 units of SUM. The mean is one
    fp32 number of the offset's size."""
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(5)
    image = offset + torch.randn((512, 512, 64), generator=g, device="cuda")
    image[0] = 0
    image = image.to(dtype)
    x = image.expand(150, 512, 512, 64)  # as many images as leave one block to each
    y, mean, rstd = nt.group_norm(x, 64)
    v = image.double().view(-1, 64)
    want = v.mean(dim=0)
    var = (v - want).square().mean(dim=0)
    wrstd = (var + 1e-5).rsqrt()
    assert torch.equal(mean[0].expand_as(mean), mean) and torch.equal(rstd[0].expand_as(rstd), rstd)
    assert float((mean[0].double() - want).abs().max()) <= 16 * U * offset
    assert float((rstd[0].double() / wrstd - 1).abs().max()) <= 512 * U, float((rstd[0].double() / wrstd - 1).abs().max())
    z = (image.double() - want) * wrstd
    tol = 512 * U * (1 + z.abs()) + 16 * U * offset * wrstd.max()
    tol = tol + O.HALF_ULP[dtype] * (z.abs() + tol)
    assert bool(((y[149].double() - z).abs() <= tol).all())


@pytest.mark.parametrize("act", ["none", "silu"])
def test_group_norm_gradient_sums_of_equal_terms(cuda, act):
    """A gradient of 0.1 everywhere, 11,000 texels a thread: adding equal terms one by one rounds one way.  The bound
    is SUM of the magnitudes, 512 units, as for short sums."""
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(6)
    image = torch.randn((512, 512, 64), generator=g, device="cuda")
    x = image.expand(150, 512, 512, 64)
    dy = torch.full((64,), 0.1, device="cuda").expand(150, 512, 512, 64)
    mean, rstd = torch.zeros((150, 8), device="cuda"), torch.ones((150, 8), device="cuda")
    _, dgamma, dbeta = nt.group_norm_backward(dy, x, mean, rstd, 8, activation=act)
    h = image.double().view(-1, 64)
    s = torch.sigmoid(h)
    slope = s * (1 + h * (1 - s)) if act == "silu" else torch.ones_like(h)
    e = 150 * float(np.float32(0.1)) * slope
    for got, terms in ((dbeta, e), (dgamma, e * h)):
        err, size = (got.double() - terms.sum(dim=0)).abs(), terms.abs().sum(dim=0)
        assert bool((err <= 512 * U * size).all()), float((err / size).max()) / U


def test_group_norm_into_a_transposed_map(cuda):
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((2, 9, 13, 24), generator=g, device="cuda").half()
    want, mean, rstd = nt.group_norm(x, 3, activation="relu")
    wdx, _, _ = nt.group_norm_backward(x, x, mean, rstd, 3, activation="silu")
    for axes in ((0, 2, 1, 3), (1, 2, 0, 3), (2, 1, 0, 3)):
        back = [axes.index(i) for i in range(4)]
        y, dx = (torch.empty([x.shape[a] for a in axes], dtype=x.dtype, device="cuda").permute(back) for _ in range(2))
        nt.group_norm(x, 3, activation="relu", out=y)
        nt.group_norm_backward(x, x, mean, rstd, 3, activation="silu", out=dx)
        assert float((y.float() - want.float()).abs().max()) <= 2.0 ** -10 * float(want.abs().max())
        assert float((dx.float() - wdx.float()).abs().max()) <= 2.0 ** -10 * float(wdx.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("period", [1, 3, 256, 512])
def test_group_norm_of_values_whose_squares_overflow(cuda, dtype, period):
    """+-10^20 in turn: the variance is past fp32, so rstd is 0 (and y beta) or a NaN, never that of a small variance."""
    import neural_textures_b200 as nt
    sign = 1 - 2.0 * ((torch.arange(64 * 64, device="cuda") // period) % 2)
    x = (1e20 * sign)[:, None].repeat(1, 8).view(1, 64, 64, 8).to(dtype)
    for images in (1, 150):
        y, mean, rstd = nt.group_norm(x.expand(images, 64, 64, 8), 2)
        assert not (rstd > 0).any(), rstd
        assert not (y.abs() > 0).any()
