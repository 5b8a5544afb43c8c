"""Group normalisation and 4-bit microscaled matrices against their 64-bit definitions
(tests/layer_oracle.py), on the device.

Tolerances.  u = 2^-24 is fp32's rounding unit.  The kernels add in fp32 in chains of at most a
few hundred terms before joining partial sums pairwise, and evaluate exp / erf to a few units:
SUM = 512 u of the sum of the magnitudes bounds either.  A result is then rounded once to its type.
Products: every E2M1 x E2M1 product and scale product is exact in fp32; at least 16 of them are
added per fp32 rounding, so K / 16 + 8 units of the sum of magnitudes bound the sum.
4-bit codes, scales and read-back are exact: no tolerance.
"""
import numpy as np
import pytest
import torch

from tests import layer_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SUM = 512 * U
ALL = [torch.float16, torch.bfloat16, torch.float32]


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, tol, what):
    err = np.abs(f64(got) - want)
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err / tol):.3g} x the tolerance"


def rounded(dtype, want, tol):
    return tol + O.HALF_ULP[dtype] * (np.abs(want) + tol) + O.TINY[dtype]


def norm_case(shape, dtype, seed, pad=0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, h, w, c = shape
    wide = torch.randn((n, h, w, c + pad), generator=g, device="cuda") * 1.5 + offset
    wide += torch.randn(c + pad, generator=g, device="cuda")
    x = wide.to(dtype)[..., :c]
    gamma = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    beta = 0.3 * torch.randn(c, generator=g, device="cuda")
    dy = torch.randn((n, h, w, c), generator=g, device="cuda").to(dtype)
    return x, gamma, beta, dy


# images, height, width, channels, groups, pad
NORM_SIZES = [
    (1, 1, 1, 1, 1, 0),        # one value: variance 0
    (1, 1, 1, 24, 3, 0),       # one texel
    (2, 1, 3, 8, 8, 0),        # a channel a group
    (1, 16, 16, 64, 8, 0),
    (3, 5, 7, 12, 3, 4),       # a slice of wider texels
    (2, 9, 11, 10, 5, 1),      # nothing aligned
    (5, 33, 17, 96, 12, 0),
    (1, 61, 67, 7, 1, 0),      # odd channels
    (40, 3, 5, 16, 4, 0),
    (300, 2, 2, 8, 2, 0),      # more images than thread blocks run at once
    (1, 200, 150, 32, 4, 0),
    (2, 2, 3, 4100, 4, 0),     # more channels than threads
    (1, 3, 2, 8192, 8192, 0),
    (1, 512, 509, 16, 2, 0),
    # more texels than a block keeps in shared memory
    (160, 64, 40, 32, 4, 0),
    (150, 200, 100, 3, 1, 0),   # single channels
    (150, 33, 31, 20, 10, 4),   # vectors across groups, unaligned
    (150, 4, 3, 8192, 16, 0),   # several turns along a texel
    (1, 1000, 1100, 24, 3, 0),  # the whole grid
]


@pytest.mark.parametrize("dtype", ALL, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_group_norm_forward_and_backward(cuda, size, dtype):
    import neural_textures_b200 as nt
    n, h, w, c, groups, pad = size
    act = ["none", "relu", "silu", "gelu"][(n + h + w + c) % 4]
    x, gamma, beta, dy = norm_case((n, h, w, c), dtype, 7, pad)
    eps = 1e-3
    y, mean, rstd = nt.group_norm(x, groups, gamma, beta, activation=act, eps=eps)
    dx, dgamma, dbeta = nt.group_norm_backward(dy, x, mean, rstd, groups, gamma, beta, activation=act)
    torch.cuda.synchronize()
    ga, be = f64(gamma), f64(beta)
    wy, z, hat, wmean, wrstd = O.group_norm(f64(x), groups, ga, be, act, eps)
    size_x = np.abs(f64(x)).max()
    close(mean, wmean, SUM * size_x, "mean")
    close(rstd, wrstd, SUM * wrstd * (1 + size_x * wrstd), "rstd")
    # an error of the statistics moves h by at most SUM (1 + |h|) (1 + size_x rstd)
    moved = SUM * (1 + np.abs(ga)) * (1 + np.abs(hat)) * (1 + size_x * O._spread(wrstd, c)) + SUM * np.abs(z)
    close(y, wy, rounded(dtype, wy, 1.2 * moved), "y")
    # the backward pass from the statistics that it was given
    wdx, wdg, wdb, sx, sg, sb = O.group_norm_backward(f64(dy), f64(x), f64(mean), f64(rstd), groups, ga, be, act)
    if act == "relu":  # z at rounding distance of 0 may take either slope: compare where no such z is
        hat32 = (f64(x) - O._spread(f64(mean), c)) * O._spread(f64(rstd), c)
        if (np.abs(ga * hat32 + be) < 16 * U * (np.abs(ga * hat32) + np.abs(be)) + 1e-30).any():
            return
    lipschitz = 1.2 * (1 + np.abs(ga).max() + np.abs(be).max())
    close(dx, wdx, rounded(dtype, wdx, SUM * lipschitz * sx + 1e-30), "dx")
    close(dgamma, wdg, SUM * lipschitz * sg + 1e-30, "dgamma")
    close(dbeta, wdb, SUM * lipschitz * sb + 1e-30, "dbeta")


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_group_norm_gradient_against_differences(cuda, act):
    """Central differences of the forward kernel's output: step s = 2^-7 leaves s^2 / 6 of the third
    derivative (order 1 for these activations and unit inputs) and u / s of rounding: 1e-3 of the
    norms of the two directions bounds their sum."""
    import neural_textures_b200 as nt
    x, gamma, beta, w = norm_case((2, 6, 7, 12), torch.float32, 11)
    groups, s = 3, 2.0 ** -7
    loss = lambda x, ga, be: float((nt.group_norm(x, groups, ga, be, activation=act)[0].double() * w.double()).sum())
    y, mean, rstd = nt.group_norm(x, groups, gamma, beta, activation=act)
    grads = nt.group_norm_backward(w, x, mean, rstd, groups, gamma, beta, activation=act)
    for k, (value, grad) in enumerate(zip((x, gamma, beta), grads)):
        d = torch.randn(value.shape, generator=torch.Generator().manual_seed(k)).cuda()
        at = lambda t: [value + t * d if j == k else v for j, v in enumerate((x, gamma, beta))]
        numeric = (loss(*at(s)) - loss(*at(-s))) / (2 * s)
        exact = float((grad.double() * d.double()).sum())
        assert abs(numeric - exact) <= 1e-3 * float(w.double().norm()) * float(d.double().norm()), (k, numeric, exact)


def test_group_norm_large_common_offset(cuda):
    """Values 4096 + unit noise: the variance loses no digits to the offset.  x itself is exact in
    fp32 to 2^-12, so the oracle sees the same values; the tolerance is that of unit inputs."""
    import neural_textures_b200 as nt
    x, gamma, beta, _ = norm_case((2, 64, 65, 16), torch.float32, 3, offset=4096.0)
    y, mean, rstd = nt.group_norm(x, 4, gamma, beta)
    wy, z, hat, wmean, wrstd = O.group_norm(f64(x), 4, f64(gamma), f64(beta), "none", 1e-5)
    close(mean, wmean, 16 * U * 4096, "mean")
    close(rstd, wrstd, 2 * SUM * wrstd, "rstd")
    # mean is one fp32 number near 4096: half a unit of it, 2^-12, over the deviation
    close(y, wy, 2 * SUM * (1 + np.abs(z)) + (2.0 ** -11) * np.abs(f64(gamma)) * O._spread(wrstd, 16), "y")


def test_group_norm_keeps_infinities_in_their_group(cuda):
    import neural_textures_b200 as nt
    x, gamma, beta, dy = norm_case((2, 6, 5, 12), torch.float16, 5)
    clean, *_ = nt.group_norm(x, 3, gamma, beta, activation="silu")
    x = x.clone()
    x[0, 2, 3, 5] = float("inf")   # image 0, group 1
    x[1, 0, 0, 11] = float("nan")  # image 1, group 2
    y, mean, rstd = nt.group_norm(x, 3, gamma, beta, activation="relu")
    dx, dgamma, dbeta = nt.group_norm_backward(dy, x, mean, rstd, 3, gamma, beta, activation="none")
    torch.cuda.synchronize()
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, ..., 4:8] = True
    bad[1, ..., 8:12] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    assert torch.isfinite(dgamma[:4]).all() and torch.isnan(dgamma[4:]).all()
    assert torch.isfinite(dbeta).all()  # no activation: dbeta is a sum of dy alone
    assert torch.isfinite(clean).all()


def test_group_norm_strides_in_place_and_broadcast(cuda):
    import neural_textures_b200 as nt
    x, gamma, beta, dy = norm_case((3, 10, 9, 16), torch.float16, 9)
    want, mean, rstd = nt.group_norm(x, 4, gamma, beta, activation="silu")
    wdx, wdg, wdb = nt.group_norm_backward(dy, x, mean, rstd, 4, gamma, beta, activation="silu")
    # a window of a larger map, written into a window of another
    big = torch.zeros((3, 20, 30, 24), dtype=torch.float16, device="cuda")
    view = big[:, 4:14, 7:16, 8:24]
    view.copy_(x)
    out = torch.full((3, 12, 11, 16), 7.0, dtype=torch.float16, device="cuda")
    y, m2, _ = nt.group_norm(view, 4, gamma, beta, activation="silu", out=out[:, 1:11, 1:10])
    assert torch.equal(out[:, 1:11, 1:10], y)
    tol = 4 * float(np.abs(f64(want)).max()) * 2.0 ** -11
    assert float((y.float() - want.float()).abs().max()) <= tol  # another split of the sums
    border = out.clone()
    border[:, 1:11, 1:10] = 7.0
    assert (border == 7.0).all(), "nothing outside the view is written"
    # a transposed image (rows and texels swapped) holds the same groups
    yt, *_ = nt.group_norm(x.transpose(1, 2), 4, gamma, beta, activation="silu")
    assert float((yt.transpose(1, 2).float() - want.float()).abs().max()) <= tol
    # in place
    inplace = x.clone()
    nt.group_norm(inplace, 4, gamma, beta, activation="silu", out=inplace)
    assert torch.equal(inplace, want)
    for target in (dy.clone(), x.clone()):
        args = (target, x) if torch.equal(target, dy) else (dy, target)
        got, dg, db = nt.group_norm_backward(*args, mean, rstd, 4, gamma, beta, activation="silu", out=target)
        assert torch.equal(got, wdx) and torch.equal(dg, wdg) and torch.equal(db, wdb)
    # one image repeated by a zero stride: dy broadcast over texels
    flat = torch.randn((1, 1, 1, 16), device="cuda").half()
    got = nt.group_norm_backward(flat.expand(3, 10, 9, 16), x, mean, rstd, 4, gamma, beta, activation="silu")
    full = nt.group_norm_backward(flat.expand(3, 10, 9, 16).contiguous(), x, mean, rstd, 4, gamma, beta, activation="silu")
    assert all(float((a.float() - b.float()).abs().max()) <= 1e-3 * float(b.float().abs().max()) for a, b in zip(got, full))
    # [H][W][C], no parameters
    y3, *_ = nt.group_norm(x[1], 4)
    y4, *_ = nt.group_norm(x[1:2], 4, torch.ones(16, device="cuda"), torch.zeros(16, device="cuda"))
    assert torch.equal(y3, y4[0])


def test_group_norm_no_images(cuda):
    import neural_textures_b200 as nt
    x = torch.empty((0, 4, 4, 8), device="cuda")
    y, mean, rstd = nt.group_norm(x, 2)
    assert y.shape == x.shape and mean.shape == (0, 2)
    dx, dgamma, dbeta = nt.group_norm_backward(x, x, mean, rstd, 2)
    assert dx.shape == x.shape and not dgamma.any() and not dbeta.any()


def test_group_norm_repeats_bit_for_bit(cuda):
    """No result depends on the order in which thread blocks run."""
    import neural_textures_b200 as nt
    x, gamma, beta, dy = norm_case((1, 700, 600, 32), torch.float16, 21)
    first = None
    for _ in range(3):
        y, mean, rstd = nt.group_norm(x, 4, gamma, beta, activation="gelu")
        got = (y, mean, rstd, *nt.group_norm_backward(dy, x, mean, rstd, 4, gamma, beta, activation="gelu"))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


# ---- 4-bit microscaled matrices --------------------------------------------------------------------

def matrix(rows, cols, dtype, seed):
    """Rows of different sizes, with zeros, ties, subnormals, saturating and special values among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(3 * torch.randn((rows, 1), generator=g))
    flat = x.view(-1)
    some = torch.randperm(flat.numel(), generator=g)[: max(1, flat.numel() // 6)]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -2.5, -0.0, 0.0, 1e-7, -6.5])
    flat[some] = ties[torch.randint(0, len(ties), some.shape, generator=g)] * torch.exp2(torch.randint(-3, 4, some.shape, generator=g).float())
    return x.to(dtype).cuda()


def check_quantized(nt, x, block):
    q = nt.mx4_quantize(x, block=block)
    codes, byte, values = O.mx4_quantize(f64(x), block)
    data, scales = O.mx4_pack(codes, byte, block)
    torch.cuda.synchronize()
    assert np.array_equal(q.scales.cpu().numpy(), scales), "scales"
    finite = np.isfinite(values)
    got = q.data.cpu().numpy()
    unpacked = np.stack((got & 15, got >> 4), axis=2).reshape(got.shape[0], -1)
    assert np.array_equal(unpacked[:, :x.shape[1]][finite], codes[finite]), "codes"
    assert not unpacked[:, x.shape[1]:].any(), "padding"
    for dtype in ALL:
        back = nt.mx4_dequantize(q, dtype)
        want = torch.from_numpy(values.astype(np.float32)).to(dtype)  # exact in fp32, rounded once
        assert torch.equal(torch.nan_to_num(back.cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0)), dtype
    return q


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", ALL, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 31), (129, 33), (200, 260), (31, 127), (5, 16), (640, 1000)])
def test_mx4_quantize_is_exact(cuda, rows, cols, dtype, block):
    import neural_textures_b200 as nt
    x = matrix(rows, cols, dtype, rows * 131 + cols)
    check_quantized(nt, x, block)
    # the same matrix read along its columns, and out of a wider one
    q = nt.mx4_quantize(x, block=block)
    for view in (x.t().contiguous().t(), torch.cat((x, x), dim=1)[:, :cols], x.repeat_interleave(2, dim=1)[:, ::2]):
        again = nt.mx4_quantize(view, block=block)
        assert torch.equal(again.data, q.data) and torch.equal(again.scales, q.scales)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", ALL, ids=["f16", "bf16", "f32"])
def test_mx4_special_values(cuda, dtype, block):
    import neural_textures_b200 as nt
    top = torch.finfo(dtype).max
    small = torch.finfo(dtype).smallest_normal
    x = matrix(16, 256, dtype, 77)
    x[0, 3] = float("nan")
    x[1, 40] = float("inf")
    x[2, 100] = -float("inf")
    x[3, :64] = 0.0
    x[4, :64] = -0.0
    x[5, 7] = top
    x[6, 130] = -top
    x[7] = small * torch.arange(-128, 128, device="cuda").to(dtype) / 16
    x[8] = top
    x[9] = 2.0 ** -9 * torch.linspace(-6.5, 6.5, 256, device="cuda").to(dtype)  # around E4M3's smallest scale
    check_quantized(nt, x, block)


def test_mx4_fp32_neighbours_of_ties(cuda):
    """fp32 values one step beside t * scale, and on it, for every E4M3 scale: the quotient alone,
    rounded to fp32, cannot tell them apart."""
    import neural_textures_b200 as nt
    s = torch.tensor(O.E4M3[1:127], dtype=torch.float32)[:, None]
    t = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5], dtype=torch.float32)[None, :]
    tie = s * t
    x = torch.cat((tie, torch.nextafter(tie, torch.tensor(1e9)), torch.nextafter(tie, torch.tensor(0.0)), 6 * s), dim=1)
    assert x.shape[1] == 16
    check_quantized(nt, x.cuda(), 16)


@pytest.mark.parametrize("dtype", ALL, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k,block", [
    (4000, 2500, 160, 16),   # tiles of 256 columns, several to a block
    (4000, 2501, 96, 32),    # rows of d that no tensor map takes
    (40000, 64, 64, 32),     # epilogue warps in turns, several tiles to a block
    (40001, 50, 30, 16), (20000, 24, 130, 32), (5000, 128, 300, 16)])
def test_mx4_product_of_many_tiles(cuda, m, n, k, block, dtype):
    """Against 64-bit products on the device; the tolerance of test_mx4_product."""
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(m + n)
    qa = nt.mx4_quantize(torch.randn((m, k), generator=g, device="cuda"), block=block)
    qb = nt.mx4_quantize(torch.randn((n, k), generator=g, device="cuda"), block=block)
    bias = torch.randn(n, generator=g, device="cuda")
    d = nt.mx4_product(qa, qb, bias=bias, activation="relu", alpha=0.5, dtype=dtype)
    a, b = nt.mx4_dequantize(qa, torch.float32).double(), nt.mx4_dequantize(qb, torch.float32).double()
    want = torch.relu(0.5 * (a @ b.t()) + bias.double())
    size = 0.5 * (a.abs() @ b.abs().t()) + bias.double().abs()
    tol = (k / 16 + 8) * U * size
    tol = tol + O.HALF_ULP[dtype] * (want + tol) + O.TINY[dtype]
    assert bool(((d.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 5, 16), (1, 300, 4096), (7, 129, 100), (33, 64, 64), (128, 128, 256), (130, 257, 1111), (1000, 24, 48),
    (64, 512, 2048), (300, 1000, 513), (4, 2048, 8192), (513, 384, 640)])
def test_mx4_product(cuda, m, n, k, block):
    import neural_textures_b200 as nt
    dtype, act = ALL[(m + n) % 3], ["none", "relu", "silu", "gelu"][(m + k) % 4]
    alpha = 0.75 / k ** 0.5
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n)
    qa = nt.mx4_quantize(torch.randn((m, k), generator=g, device="cuda") * torch.exp2(torch.randn((m, 1), generator=g, device="cuda")), block=block)
    qb = nt.mx4_quantize(torch.randn((n, k), generator=g, device="cuda").half(), block=block)
    bias = torch.randn(n, generator=g, device="cuda") if (m + n + k) % 5 else None
    d = nt.mx4_product(qa, qb, bias=bias, activation=act, alpha=alpha, dtype=dtype)
    a, b = f64(nt.mx4_dequantize(qa, torch.float32)), f64(nt.mx4_dequantize(qb, torch.float32))
    wide = np.zeros(n) if bias is None else f64(bias)
    z = alpha * (a @ b.T) + wide
    want = O.activate(z, act)
    tol = (k / 16 + 8) * U * (alpha * (np.abs(a) @ np.abs(b).T) + np.abs(wide) + np.abs(z))
    close(d, want, rounded(dtype, want, 1.2 * tol), "product")


def test_mx4_product_into_a_wider_matrix_and_rows(cuda):
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn((70, 96), generator=g, device="cuda"), torch.randn((50, 96), generator=g, device="cuda")
    a, b = nt.mx4_quantize(x), nt.mx4_quantize(w)
    want = nt.mx4_product(a, b, dtype=torch.float16)
    out = torch.full((70, 64), 9.0, device="cuda", dtype=torch.float16)
    nt.mx4_product(a, b, out=out[:, 7:57])
    assert torch.equal(out[:, 7:57], want) and (out[:, :7] == 9).all() and (out[:, 57:] == 9).all()
    # the first rows of a larger buffer, codes with a wider pitch
    data = torch.full((80, 80), 0xff, dtype=torch.uint8, device="cuda")
    data[:70, :48] = a.data
    again = nt.mx4_product(nt.Mx4Tensor(data[:, :48], a.scales, 70, 96, 32), b, dtype=torch.float16)
    assert torch.equal(again, want)
    assert nt.mx4_product(nt.Mx4Tensor.empty(0, 96), b).shape == (0, 50)
    assert nt.mx4_product(a, nt.Mx4Tensor.empty(0, 96)).shape == (70, 0)


@pytest.mark.parametrize("block", [16, 32])
def test_mx4_product_keeps_nan_in_its_rows(cuda, block):
    import neural_textures_b200 as nt
    g = torch.Generator(device="cuda").manual_seed(6)
    x, w = torch.randn((200, 192), generator=g, device="cuda"), torch.randn((150, 192), generator=g, device="cuda")
    x[133, 70] = float("nan")
    w[17, 0] = float("inf")
    d = nt.mx4_product(nt.mx4_quantize(x, block=block), nt.mx4_quantize(w, block=block), activation="relu", dtype=torch.float32)
    bad = torch.zeros_like(d, dtype=torch.bool)
    bad[133] = True
    bad[:, 17] = True
    assert torch.isnan(d[bad]).all() and torch.isfinite(d[~bad]).all()


def test_layers_on_another_stream(cuda):
    """Tensors made on one stream, used on another, by torch's current stream and by argument."""
    import neural_textures_b200 as nt
    x, gamma, beta, dy = norm_case((2, 40, 40, 32), torch.float16, 2)
    want, *_ = nt.group_norm(x, 4, gamma, beta, activation="silu")
    wq = nt.mx4_quantize(x.view(-1, 32))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, *_ = nt.group_norm(x, 4, gamma, beta, activation="silu")
    y2, *_ = nt.group_norm(x, 4, gamma, beta, activation="silu", stream=s)
    y3, *_ = nt.group_norm(x, 4, gamma, beta, activation="silu", stream=s.cuda_stream)
    q = nt.mx4_quantize(x.view(-1, 32), stream=s)
    s.synchronize()
    assert torch.equal(y1, want) and torch.equal(y2, want) and torch.equal(y3, want) and torch.equal(q.data, wq.data)


def test_layers_in_a_graph(cuda):
    """Captured once, replayed on new inputs."""
    import neural_textures_b200 as nt
    x, gamma, beta, dy = norm_case((1, 64, 64, 32), torch.float16, 2)
    w = nt.mx4_quantize(torch.randn((48, 32), device="cuda"))

    def layer():
        y, mean, rstd = nt.group_norm(x, 4, gamma, beta, activation="silu")
        grads = nt.group_norm_backward(dy, x, mean, rstd, 4, gamma, beta, activation="silu")
        return (nt.mx4_product(nt.mx4_quantize(y.view(-1, 32)), w), *grads)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for seed in (31, 32):
        x.copy_(norm_case((1, 64, 64, 32), torch.float16, seed)[0])
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, layer()))


def test_offsets_past_32_bits(cuda):
    """Rows and images 2^31 elements apart: reading, writing, and a product's rows 2^25 apart."""
    import neural_textures_b200 as nt
    far = 1 << 31
    pool = torch.empty(far + (1 << 26), dtype=torch.float16, device="cuda")
    x = torch.as_strided(pool, (2, 200), (far, 1))
    values = matrix(2, 200, torch.float16, 5)
    x.copy_(values)
    q, want = nt.mx4_quantize(x), nt.mx4_quantize(values.contiguous())
    assert torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)
    nt.mx4_dequantize(want, out=torch.as_strided(pool, (2, 200), (far, 1), 512))
    assert torch.equal(torch.as_strided(pool, (2, 200), (far, 1), 512), nt.mx4_dequantize(want))
    small, gamma, beta, _ = norm_case((2, 5, 6, 16), torch.float16, 4)
    apart = torch.as_strided(pool, (2, 5, 6, 16), (far, 96, 16, 1), 4096)
    apart.copy_(small)
    y, *_ = nt.group_norm(apart, 4, gamma, beta, activation="silu")
    w, *_ = nt.group_norm(small, 4, gamma, beta, activation="silu")
    assert float((y.float() - w.float()).abs().max()) <= 2.0 ** -10 * float(w.float().abs().max())
    out = torch.as_strided(pool, (2, 5, 6, 16), (far, 96, 16, 1), 8192)
    nt.group_norm(small, 4, gamma, beta, activation="silu", out=out)
    assert torch.equal(out, w)
    a, b = nt.mx4_quantize(torch.randn((65, 128), device="cuda")), nt.mx4_quantize(torch.randn((96, 128), device="cuda"))
    rows = torch.as_strided(pool, (65, 96), (1 << 25, 1), 1 << 14)
    nt.mx4_product(a, b, out=rows)
    assert torch.equal(rows, nt.mx4_product(a, b))
