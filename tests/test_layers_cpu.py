"""Texel-layer operators on the host: the parameter blocks match the C structs, sizes, and every
refusal (all before any CUDA call); the 64-bit restatements agree with torch's own gradient."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import layer_oracle as O


def test_parameter_blocks_match(native):
    from neural_textures_b200 import _native as N, layers
    assert C.sizeof(N.NtGroupNorm) == layers._GROUP_NORM.size
    import neural_textures_b200 as nt
    q = nt.Mx4Tensor.empty(5, 70, 16, device="cpu")
    m = N.NtMx4Matrix.from_buffer_copy(q._packed)
    assert (m.data, m.scales, m.pitch, m.rows, m.cols, m.block) == (q.data.data_ptr(), q.scales.data_ptr(), 48, 5, 70, 16)
    packed = layers._GROUP_NORM.pack(*range(1, 8), 0.5, *range(8, 32))
    p = N.NtGroupNorm.from_buffer_copy(packed)
    assert (p.images, p.activation, p.epsilon, p.x.data, p.x.texel_stride, p.gamma, p.rstd) == (1, 7, 0.5, 8, 11, 12, 15)
    assert (p.y.data, p.dy.data, p.dx.texel_stride, p.dgamma, p.workspace, p.workspace_bytes) == (16, 20, 27, 28, 30, 31)


def _norm(**change):
    from neural_textures_b200 import _native as N
    p = N.NtGroupNorm(images=2, height=4, width=5, channels=12, groups=3, dtype=N.NT_DTYPE_F16, activation=N.NT_ACT_SILU,
                      epsilon=1e-5)
    for f in (p.x, p.y, p.dy, p.dx):
        f.data, f.image_stride, f.row_stride, f.texel_stride = 0x10000, 240, 60, 12
    p.gamma = p.beta = p.mean = p.rstd = p.dgamma = p.dbeta = p.workspace = 0x10000
    p.workspace_bytes = 1 << 30
    for name, value in change.items():
        at, names = p, name.split("__")
        for part in names[:-1]:
            at = getattr(at, part)
        setattr(at, names[-1], value)
    return p


@pytest.mark.parametrize("change,needle", [
    (dict(images=-1), "images"), (dict(height=0), "image size"), (dict(width=-3), "image size"),
    (dict(height=1 << 16, width=1 << 15), "image size"), (dict(channels=0), "channels"), (dict(channels=8193, groups=1), "channels"),
    (dict(groups=5), "multiple of groups"), (dict(groups=0), "multiple of groups"), (dict(dtype=2), "dtype"),
    (dict(activation=4), "activation"), (dict(activation=-1), "activation"), (dict(epsilon=0.0), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"), (dict(x__data=None), "x must be"), (dict(x__data=0x10001), "x must be"),
    (dict(x__row_stride=-1), "x: strides"), (dict(gamma=0x10002), "gamma"), (dict(workspace=0x10008), "workspace"),
])
def test_group_norm_refuses(native, change, needle):
    from neural_textures_b200 import _native as N
    for entry in (native.nt_group_norm_forward, native.nt_group_norm_backward):
        assert entry(C.byref(_norm(**change)), None) == 1
        assert needle in N.last_error(), N.last_error()


@pytest.mark.parametrize("backward,change,needle", [
    (False, dict(y__data=None), "y must be"), (False, dict(y__texel_stride=11), "y: texels overlap"),
    (False, dict(y__row_stride=59), "y: rows overlap"), (False, dict(y__image_stride=0), "y: images overlap"),
    (True, dict(dy__data=None), "dy must be"), (True, dict(dx__image_stride=239), "dx: images overlap"),
    (True, dict(mean=None), "mean and rstd"), (True, dict(rstd=None), "mean and rstd"),
    (True, dict(workspace_bytes=8), "workspace"), (True, dict(workspace=None), "workspace"),
])
def test_group_norm_refuses_outputs(native, backward, change, needle):
    from neural_textures_b200 import _native as N
    entry = native.nt_group_norm_backward if backward else native.nt_group_norm_forward
    assert entry(C.byref(_norm(**change)), None) == 1
    assert needle in N.last_error(), N.last_error()
    assert entry(None, None) == 1


def test_group_norm_of_no_images_needs_nothing(native):
    p = _norm(images=0, workspace=None, workspace_bytes=0, x__data=None, y__data=None)
    assert native.nt_group_norm_workspace_bytes(C.byref(p), 0) == 0
    assert native.nt_group_norm_workspace_bytes(C.byref(p), 1) == 0
    assert native.nt_group_norm_forward(C.byref(p), None) == 0
    assert native.nt_group_norm_workspace_bytes(None, 0) == 0
    assert native.nt_group_norm_workspace_bytes(C.byref(_norm(groups=5)), 0) == 0


def test_mx4_sizes(native):
    assert [native.nt_mx4_pitch(c) for c in (-1, 0, 1, 31, 32, 33, 64)] == [0, 0, 16, 16, 16, 32, 32]
    assert native.nt_mx4_scales_bytes(128, 64, 16) == 512 and native.nt_mx4_scales_bytes(128, 128, 32) == 512
    assert native.nt_mx4_scales_bytes(129, 65, 16) == 2048 and native.nt_mx4_scales_bytes(1, 129, 32) == 1024
    assert native.nt_mx4_scales_bytes(0, 64, 16) == 0 and native.nt_mx4_scales_bytes(4, 0, 16) == 0
    assert native.nt_mx4_scales_bytes(4, 64, 8) == 0
    assert native.nt_mx4_scales_bytes(1 << 30, 1 << 20, 16) == (1 << 30) * (1 << 20) // 16  # past 32 bits


def _matrix(**change):
    from neural_textures_b200 import _native as N
    m = N.NtMx4Matrix(data=0x10000, scales=0x10000, pitch=64, rows=8, cols=100, block=32)
    for name, value in change.items():
        setattr(m, name, value)
    return m


@pytest.mark.parametrize("change,needle", [
    (dict(block=8), "block"), (dict(rows=-1), "matrix size"), (dict(cols=0), "matrix size"), (dict(pitch=48), "pitch"),
    (dict(pitch=72), "pitch"), (dict(data=None), "data and scales"), (dict(scales=0x10004), "data and scales"),
    (dict(data=0x10008), "data and scales"),
])
def test_mx4_refuses_matrices(native, change, needle):
    from neural_textures_b200 import _native as N
    bad, good = _matrix(**change), _matrix()
    calls = [lambda: native.nt_mx4_quantize(0x10000, 0, 100, 1, C.byref(bad), None),
             lambda: native.nt_mx4_dequantize(C.byref(bad), 0x10000, 0, 100, None),
             lambda: native.nt_mx4_product(C.byref(bad), C.byref(good), None, 0, 1.0, 0x10000, 0, 100, None),
             lambda: native.nt_mx4_product(C.byref(good), C.byref(bad), None, 0, 1.0, 0x10000, 0, 100, None)]
    for call in calls:
        assert call() == 1
        assert needle in N.last_error(), N.last_error()


def test_mx4_refuses_arguments(native):
    from neural_textures_b200 import _native as N
    m, product = C.byref(_matrix()), native.nt_mx4_product
    for status, needle in [
        (lambda: native.nt_mx4_quantize(None, 0, 100, 1, m, None), "src"),
        (lambda: native.nt_mx4_quantize(0x10001, 0, 100, 1, m, None), "src"),
        (lambda: native.nt_mx4_quantize(0x10000, 2, 100, 1, m, None), "dtype"),
        (lambda: native.nt_mx4_quantize(0x10000, 0, -1, 1, m, None), "strides"),
        (lambda: native.nt_mx4_quantize(0x10000, 0, 100, 1, None, None), "dst is null"),
        (lambda: native.nt_mx4_dequantize(m, None, 0, 100, None), "dst"),
        (lambda: native.nt_mx4_dequantize(m, 0x10000, 3, 100, None), "dtype"),
        (lambda: native.nt_mx4_dequantize(m, 0x10000, 0, 99, None), "row_stride"),
        (lambda: product(m, C.byref(_matrix(cols=99)), None, 0, 1.0, 0x10000, 0, 8, None), "same cols"),
        (lambda: product(m, C.byref(_matrix(block=16)), None, 0, 1.0, 0x10000, 0, 8, None), "block"),
        (lambda: product(m, m, None, 9, 1.0, 0x10000, 0, 8, None), "activation"),
        (lambda: product(m, m, None, 0, 1.0, 0x10000, 5, 8, None), "dtype"),
        (lambda: product(m, m, None, 0, 1.0, 0x10000, 0, 7, None), "row_stride"),
        (lambda: product(m, m, None, 0, 1.0, None, 0, 8, None), "d must be"),
        (lambda: product(m, m, 0x10002, 0, 1.0, 0x10000, 0, 8, None), "bias"),
    ]:
        assert status() == 1
        assert needle in N.last_error(), N.last_error()
    empty = C.byref(_matrix(rows=0, data=None, scales=None))
    assert native.nt_mx4_quantize(None, 0, 100, 1, empty, None) == 0
    assert native.nt_mx4_dequantize(empty, None, 0, 100, None) == 0
    assert product(empty, m, None, 0, 1.0, None, 0, 8, None) == 0


def test_python_refusals(native):
    import neural_textures_b200 as nt
    x = torch.zeros((2, 4, 4, 8), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        nt.group_norm(x, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        nt.mx4_quantize(x.view(-1, 8))
    with pytest.raises(TypeError, match="x must be"):
        nt.group_norm(x.int(), 2)
    with pytest.raises(TypeError, match="x must be"):
        nt.mx4_quantize(x.view(-1, 8).double())
    with pytest.raises(ValueError, match=r"\[N\]\[H\]\[W\]\[C\]"):
        nt.group_norm(x.view(-1, 8), 2)
    with pytest.raises(ValueError, match="activation"):
        nt.group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="gamma"):
        nt.group_norm(x, 2, gamma=torch.zeros(8, dtype=torch.float16))
    with pytest.raises(ValueError, match="beta"):
        nt.group_norm(x, 2, beta=torch.zeros(7))
    with pytest.raises(ValueError, match="channels must be contiguous"):
        nt.group_norm(x.transpose(1, 3), 1)
    with pytest.raises(ValueError, match="out must be"):
        nt.group_norm(x, 2, out=torch.zeros((2, 4, 4, 9), dtype=torch.float16))
    with pytest.raises(ValueError, match="dy must be"):
        nt.group_norm_backward(x[:1], x, torch.zeros(2, 2), torch.zeros(2, 2), 2)
    with pytest.raises(ValueError, match="mean must be"):
        nt.group_norm_backward(x, x, torch.zeros(2, 3), torch.zeros(2, 2), 2)
    with pytest.raises(ValueError, match="matrix"):
        nt.mx4_quantize(x)
    with pytest.raises(ValueError, match="blocks of 8"):
        nt.mx4_quantize(x.view(-1, 8), block=8)
    with pytest.raises(ValueError, match="data must be"):
        nt.Mx4Tensor(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 4, 33)
    with pytest.raises(ValueError, match="scales must be"):
        nt.Mx4Tensor(torch.zeros((129, 16), dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 129, 32)
    q = nt.Mx4Tensor.empty(4, 64, device="cpu")
    with pytest.raises(ValueError, match="out must be"):
        nt.mx4_dequantize(q, torch.float16, out=torch.zeros((4, 63), dtype=torch.float16))
    with pytest.raises(TypeError, match="dtype must be"):
        nt.mx4_dequantize(q, torch.float64)
    with pytest.raises(ValueError, match="bias"):
        nt.mx4_product(q, q, bias=torch.zeros(5))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_oracle_against_torch(act):
    """The restatement's forward and gradient against torch.group_norm's in 64 bits."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn((2, 5, 6, 12), generator=g, dtype=torch.float64, requires_grad=True)
    gamma = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    beta = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(x.shape, generator=g, dtype=torch.float64)
    z = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 3, gamma, beta, 1e-3).permute(0, 2, 3, 1)
    y = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](z)
    y.backward(dy)
    n = lambda t: t.detach().numpy()
    wy, _, _, mean, rstd = O.group_norm(n(x), 3, n(gamma), n(beta), act, 1e-3)
    dx, dg, db, *_ = O.group_norm_backward(n(dy), n(x), mean, rstd, 3, n(gamma), n(beta), act)
    for got, want in ((wy, y), (dx, x.grad), (dg, gamma.grad), (db, beta.grad)):
        assert np.allclose(got, n(want), rtol=1e-10, atol=1e-11)


def test_oracle_mx4_values():
    """Rounding and packing on a hand-made row: ties to even, saturation, the place of codes and scales."""
    x = np.zeros((130, 40))
    x[129, :9] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.3]
    codes, byte, values = O.mx4_quantize(x, 32)
    assert byte[129].tolist() == [127, 0]  # floor(log2 7.9) - 2 = 0
    assert codes[129, :9].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 9]
    assert values[129, :9].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -0.5]
    data, scales = O.mx4_pack(codes, byte, 32)
    assert data.shape == (130, 32) and data[129, 0] == 0x20 and data[129, 4] == 9
    assert scales.size == 2 * 1 * 512 and scales[512 + 16 * 1] == 127
    assert O.nearest(O.E4M3[:127], np.array([449.0, 0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0])).tolist() == [126, 0, 0, 2, 88]
