"""Texel-layer operators: channels-last group normalisation with an activation (forward and
backward), 4-bit microscaled matrices (quantise, read back, product), and TexelLayer, which runs
them as one layer of a network over a feature map.

Every call queues its kernels on `stream` (a torch.cuda.Stream or a raw handle; None: torch's
current stream of the tensors' device) and returns without waiting.  Results are new tensors unless
`out` is given, from the memory pool of that stream; a caller that passes `stream` orders it behind what made the
inputs, and keeps them until it is done.  Invalid arguments raise: TypeError / ValueError for what only the tensors
show (device, dtype, shape), NtError for what the library rejects.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import operator
import os
import struct

from . import _native as N
from . import build as _build
from ._native import check, load

ACTIVATIONS = {"none": N.NT_ACT_NONE, "relu": N.NT_ACT_RELU, "silu": N.NT_ACT_SILU, "gelu": N.NT_ACT_GELU}

_torch = None
_fast = None  # lib/nt_torch.so: the usual calls, at a third of the host time; None from it: not a usual call
_DTYPES = {}


def _lazy_torch():
    """torch, imported at the first call as everywhere in this package, and the shortcut module."""
    global _torch, _fast
    if _torch is None:
        import torch
        load()
        path = _build.TORCH_LIB
        if not os.path.exists(path):
            raise OSError(f"{path} is missing: build it with `python -m neural_textures_b200.build`")
        spec = importlib.util.spec_from_file_location("nt_torch", path)
        _fast = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_fast)
        _DTYPES.update({torch.float16: N.NT_DTYPE_F16, torch.bfloat16: N.NT_DTYPE_BF16, torch.float32: N.NT_DTYPE_F32})
        _torch = torch
    return _torch


def _dtype(t, name: str) -> int:
    d = _DTYPES.get(t.dtype if hasattr(t, "dtype") else t)
    if d is None:
        raise TypeError(f"{name} must be float16, bfloat16 or float32, not {getattr(t, 'dtype', t)}")
    return d


def _activation(name: str) -> int:
    a = ACTIVATIONS.get(name)
    if a is None:
        raise ValueError(f"unknown activation {name!r} (one of {', '.join(ACTIVATIONS)})")
    return a


def _vector(t, n: int, device, name: str) -> int:
    """Data pointer of an optional contiguous fp32 vector of n elements, 0 for None."""
    if t is None:
        return 0
    if t.dtype is not _torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} elements")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr()


_shapes = {}


def _new(shape, dtype, device):
    """torch.empty(shape) on a device with its index, at less than half its host time: empty_like of a one-element
    tensor expanded to the shape, kept per shape."""
    key = (shape, dtype, device)
    t = _shapes.get(key)
    if t is None:
        if len(_shapes) > 4096:
            _shapes.clear()
        t = _shapes[key] = _torch.empty(1, dtype=dtype, device=device).expand(shape)
    return _torch.empty_like(t)


def _launch(device, fn, *args):
    """fn(*args, torch's current stream) on `device`."""
    torch = _torch
    if device.type != "cuda":
        raise ValueError(f"a CUDA tensor is needed, not one on {device}")
    index = device.index
    handle = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, handle)
    else:
        with torch.cuda.device(index):
            status = fn(*args, handle)
    if status:
        check(status)


def _on(stream, device, fn, *args, out=None):
    """fn(*args, out=out) with `stream` as torch's current one.  Results and workspace come from its pool then:
    memory of the caller's current stream may have been freed with work pending there, which nothing orders before
    `stream`.  New results are recorded on the caller's stream, so that it may use them too."""
    torch = _torch
    if device.type != "cuda":
        raise ValueError(f"a CUDA tensor is needed, not one on {device}")
    if getattr(stream, "device", device) != device:
        raise ValueError(f"the stream is on {stream.device}, not on {device}")
    current = torch.cuda.current_stream(device)
    if not isinstance(stream, torch.cuda.Stream):
        handle = stream if isinstance(stream, int) else int(stream.cuda_stream)
        stream = current if handle == current.cuda_stream else torch.cuda.ExternalStream(handle, device=device)
    with torch.cuda.stream(stream):
        result = fn(*args, out=out)
    if stream != current:
        parts = (result.data, result.scales) if isinstance(result, Mx4Tensor) else result if isinstance(result, tuple) else (result,)
        for t in parts if out is None else parts[1:] if isinstance(result, tuple) else ():
            t.record_stream(current)
    return result


# ---------------------------------------------------------------------------------------
# group normalisation

_GROUP_NORM = struct.Struct("@7if" + "P3q" + "4P" + "P3q" * 3 + "3Pq")
_workspaces = {}


def _map(t, shape, dtype, device, name: str):
    """(pointer, strides) of a channels-last map [N][H][W][C] or [H][W][C]."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} of {dtype} on {device}, not {tuple(t.shape)} of {t.dtype} on {t.device}")
    return _strides(t, name)


def _strides(t, name: str):
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the channels must be contiguous (stride 1, not {s[-1]})")
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), 0, s[0], s[1])


def _norm_sizes(x, groups: int):
    shape = x.shape
    if len(shape) == 4:
        return (*shape, int(groups))
    if len(shape) != 3:
        raise ValueError(f"x must be [N][H][W][C] or [H][W][C], not {tuple(shape)}")
    return (1, *shape, int(groups))


def _norm_workspace(L, sizes, dtype: int, device, backward: int):
    """(tensor or None, pointer, bytes) of the call's workspace."""
    key = (sizes, dtype, backward, device)
    need = _workspaces.get(key)
    if need is None:
        if len(_workspaces) > 4096:
            _workspaces.clear()
        p = N.NtGroupNorm(*sizes, dtype, 0, 1.0)
        if device.type == "cuda":
            with _torch.cuda.device(device):
                need = _workspaces[key] = int(L.nt_group_norm_workspace_bytes(C.byref(p), backward))
        else:
            need = 0
    if not need:
        return None, 0, 0
    ws = _new((need,), _torch.uint8, device)
    return ws, ws.data_ptr(), need


def group_norm(x, groups: int, gamma=None, beta=None, activation: str = "none", eps: float = 1e-5, out=None, stream=None):
    """activation(gamma (x - mean) rstd + beta) of a channels-last feature map [N][H][W][C] (or one
    image [H][W][C]) over `groups` groups of consecutive channels; float16, bfloat16 or float32,
    any strides over images, rows and texels.  gamma and beta are float32 [C] or None.  Returns
    (y, mean, rstd) with float32 statistics [N][groups], which group_norm_backward takes.  `out`
    receives y and may be x."""
    torch = _torch or _lazy_torch()
    if stream is not None:
        return _on(stream, x.device, group_norm, x, groups, gamma, beta, activation, eps, out=out)
    if out is None:
        made = _fast.group_norm(x, groups, gamma, beta, ACTIVATIONS.get(activation), eps)
        if made is not None:
            return made
    sizes, kind, device = _norm_sizes(x, groups), x.dtype, x.device
    n, h, w, c, g = sizes
    dtype, act, L = _dtype(x, "x"), _activation(activation), load()
    xp, x0, x1, x2 = _strides(x, "x")
    ga, be = _vector(gamma, c, device, "gamma"), _vector(beta, c, device, "beta")
    if out is not None:
        y = out
        yp, y0, y1, y2 = _map(y, x.shape, kind, device, "out")
    else:
        y = torch.empty_like(x) if x.is_contiguous() else _new(x.shape, kind, device)
        yp, y0, y1, y2 = _strides(y, "y")
    mean, rstd = _new((n, max(g, 0)), torch.float32, device), _new((n, max(g, 0)), torch.float32, device)
    ws, wp, size = _norm_workspace(L, sizes, dtype, device, 0)
    _launch(device, L.nt_group_norm_forward,
            _GROUP_NORM.pack(n, h, w, c, g, dtype, act, eps, xp, x0, x1, x2, ga, be, mean.data_ptr(), rstd.data_ptr(),
                             yp, y0, y1, y2, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, wp, size))
    return y, mean, rstd


def group_norm_backward(dy, x, mean, rstd, groups: int, gamma=None, beta=None, activation: str = "none", out=None, stream=None):
    """Gradients of group_norm at its input x, with the statistics that it returned: (dx, dgamma,
    dbeta).  dx has x's type; dgamma and dbeta are float32 [C], summed over images and texels.
    `out` receives dx and may be dy or x."""
    torch = _torch or _lazy_torch()
    if stream is not None:
        return _on(stream, x.device, group_norm_backward, dy, x, mean, rstd, groups, gamma, beta, activation, out=out)
    if out is None:
        made = _fast.group_norm_backward(dy, x, mean, rstd, groups, gamma, beta, ACTIVATIONS.get(activation))
        if made is not None:
            return made
    sizes, kind, device = _norm_sizes(x, groups), x.dtype, x.device
    n, h, w, c, g = sizes
    dtype, act, L = _dtype(x, "x"), _activation(activation), load()
    xp, x0, x1, x2 = _strides(x, "x")
    gp, g0, g1, g2 = _map(dy, x.shape, kind, device, "dy")
    ga, be = _vector(gamma, c, device, "gamma"), _vector(beta, c, device, "beta")
    mp, rp = _vector(mean, n * g, device, "mean"), _vector(rstd, n * g, device, "rstd")
    if out is not None:
        dx = out
        dp, d0, d1, d2 = _map(dx, x.shape, kind, device, "out")
    else:
        dx = torch.empty_like(x) if x.is_contiguous() else _new(x.shape, kind, device)
        dp, d0, d1, d2 = _strides(dx, "dx")
    dgamma, dbeta = _new((c,), torch.float32, device), _new((c,), torch.float32, device)
    ws, wp, size = _norm_workspace(L, sizes, dtype, device, 1)
    _launch(device, L.nt_group_norm_backward,
            _GROUP_NORM.pack(n, h, w, c, g, dtype, act, 1.0, xp, x0, x1, x2, ga, be, mp, rp, 0, 0, 0, 0, gp, g0, g1, g2,
                             dp, d0, d1, d2, dgamma.data_ptr(), dbeta.data_ptr(), wp, size))
    return dx, dgamma, dbeta


# ---------------------------------------------------------------------------------------
# 4-bit microscaled matrices

def _matrix(q):
    """The NtMx4Matrix of q's tensors as they are now, packed as bytes."""
    torch = _torch or _lazy_torch()
    data, scales, rows, cols, block = q._data, q._scales, q._rows, q._cols, q._block
    q._packed = _fast.mx4_pack(data, scales, rows, cols, block)
    if q._packed is not None:
        return q._packed
    # not a matrix: say why
    if block not in (16, 32):
        raise ValueError(f"block must be 16 or 32, not {block}")
    if not 0 <= rows <= 0x7fffff00 or not 1 <= cols <= 0x7fffff00:
        raise ValueError(f"{rows} x {cols} is not a matrix size")
    pitch, size = -(-cols // 32) * 16, -(-rows // 128) * -(-cols // (4 * block)) * 512
    if data.dtype is not torch.uint8 or data.dim() != 2 or data.shape[0] < rows or data.shape[1] < pitch or rows and data.stride(1) != 1:
        raise ValueError(f"data must be uint8 [{rows}][{pitch}] or larger, the codes of a row contiguous")
    if scales.dtype is not torch.uint8 or not scales.is_contiguous() or scales.numel() < size:
        raise ValueError(f"scales must be contiguous uint8 of {size} bytes")
    if scales.device != data.device:
        raise ValueError(f"scales is on {scales.device}, not on {data.device}")
    raise TypeError("data and scales must be torch tensors, rows, cols and block integers")


class Mx4Tensor:
    """A rows x cols matrix in 4-bit microscaled form (NtMx4Matrix): `data`, the uint8 codes
    [rows][pitch], two to a byte, and `scales`, a byte per block of `block` columns (32: powers of
    two, 16: E4M3) in tiles of 128 rows x 4 blocks.  Padding must be zero, as mx4_quantize leaves it.  The fields
    are read-only; copies, pickles and torch.save carry the tensors."""
    __slots__ = ("_data", "_scales", "_rows", "_cols", "_block", "_packed")  # _packed: the NtMx4Matrix of a call
    data, scales, rows, cols, block = (property(operator.attrgetter(f)) for f in __slots__[:5])

    def __init__(self, data, scales, rows: int, cols: int, block: int = 32):
        self._data, self._scales, self._rows, self._cols, self._block = data, scales, rows, cols, block
        _matrix(self)

    def __reduce__(self):  # copies and loaded matrices name the memory of their own tensors
        return Mx4Tensor, (self._data, self._scales, self._rows, self._cols, self._block)

    @classmethod
    def empty(cls, rows: int, cols: int, block: int = 32, device="cuda"):
        torch = _torch or _lazy_torch()
        if block not in (16, 32) or rows < 0 or cols < 1:
            raise ValueError(f"{rows} x {cols} in blocks of {block} is not a 4-bit matrix")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        pitch = -(-cols // 32) * 16
        return cls(_new((rows, pitch), torch.uint8, device),
                   _new((-(-rows // 128) * -(-cols // (4 * block)) * 512,), torch.uint8, device), rows, cols, block)

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel() + self.scales.numel()

    def __repr__(self):
        return f"Mx4Tensor({self.rows} x {self.cols}, block {self.block}, {self.device})"


def mx4_quantize(x, block: int = 32, out: Mx4Tensor | None = None, stream=None) -> Mx4Tensor:
    """The float16, bfloat16 or float32 matrix x (2-D, any strides: x.t() is read in place) in 4-bit
    microscaled form, blocks along its columns (nt_mx4_quantize)."""
    _torch or _lazy_torch()
    if stream is not None:
        return _on(stream, x.device, mx4_quantize, x, block, out=out)
    if out is None:
        made = _fast.mx4_quantize(x, block)
        if made is not None:
            out = Mx4Tensor.__new__(Mx4Tensor)
            (out._rows, out._cols), out._block = x.shape, block
            out._data, out._scales, out._packed = made
            return out
    dtype = _dtype(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, not {tuple(x.shape)}")
    if out is None:
        out = Mx4Tensor.empty(x.shape[0], x.shape[1], block, x.device)
    elif out.shape != tuple(x.shape) or out.block != block or out.device != x.device:
        raise ValueError(f"out must be {tuple(x.shape)} in blocks of {block} on {x.device}")
    rs, cs = x.stride()
    _launch(x.device, load().nt_mx4_quantize, x.data_ptr(), dtype, rs, cs, _matrix(out))
    return out


def _output(out, rows: int, cols: int, dtype, device):
    """(tensor, row stride) of a matrix result: a new one of `dtype`, or `out` checked."""
    if out is None:
        return _new((rows, cols), dtype, device), cols
    if out.shape != (rows, cols) or out.dtype is not dtype or out.device != device or (cols > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be [{rows}][{cols}] of {dtype} on {device} with contiguous columns")
    return out, out.stride(0)


def mx4_dequantize(q: Mx4Tensor, dtype=None, out=None, stream=None):
    """The values of q as a matrix of `dtype` (default: out's, or float16)."""
    torch = _torch or _lazy_torch()
    dtype = dtype or (out.dtype if out is not None else torch.float16)
    code = _dtype(dtype, "dtype")
    if stream is not None:
        return _on(stream, q.device, mx4_dequantize, q, dtype, out=out)
    if out is None:
        y = _fast.mx4_dequantize(q._packed, q._data, q._scales, code)
        if y is not None:
            return y
    y, stride = _output(out, q.rows, q.cols, dtype, q.device)
    _launch(q.device, load().nt_mx4_dequantize, _matrix(q), y.data_ptr(), code, stride)
    return y


def mx4_product(a: Mx4Tensor, b: Mx4Tensor, bias=None, activation: str = "none", alpha: float = 1.0, dtype=None, out=None,
                stream=None):
    """activation(alpha a b^T + bias), [a.rows][b.rows] of `dtype` (default: out's, or float16): a layer's
    output for texels a and weights b [out][in], bias float32 [out] or None."""
    torch = _torch or _lazy_torch()
    dtype = dtype or (out.dtype if out is not None else torch.float16)
    code, act = _dtype(dtype, "dtype"), _activation(activation)
    if stream is not None:
        return _on(stream, a.device, mx4_product, a, b, bias, activation, alpha, dtype, out=out)
    if out is None:
        y = _fast.mx4_product(a._packed, a._data, a._scales, b._packed, b._data, b._scales, bias, act, alpha, code)
        if y is not None:
            return y
    device = a.device
    if b.data.device != device:
        raise ValueError(f"b is on {b.device}, not on {device}")
    y, stride = _output(out, a.rows, b.rows, dtype, device)
    _launch(device, load().nt_mx4_product, _matrix(a), _matrix(b),
            _vector(bias, b.rows, device, "bias"), act, alpha, y.data_ptr(), code, stride)
    return y


# ---------------------------------------------------------------------------------------
# a layer

class TexelLayer:
    """One layer of a network over a channels-last map: group norm, activation, then a product with a
    4-bit weight matrix, texel by texel:  out = act(norm(x)) W^T + bias.

    The fp32 masters are `weight` [out][in], `bias` [out], `gamma` and `beta` [in]; `pack` lays the weights out
    in 4 bits, once after each change.  forward(keep=True) keeps what backward needs.  backward takes the
    gradient of the output and returns that of x; those of the parameters are in `grads`, in `parameters`' order.
    Its products run in 4 bits too, on matrices quantised along the other axis, in blocks of 32: their
    power-of-two scales hold gradients of any size, where E4M3 scales end at 2^-9.  The rounding to 4 bits is
    passed straight through.  The gradient of x, and that of the norm's result before it, have x's type: in fp16 they
    need the factors of backward where gradients are below 10^-4."""

    def __init__(self, channels_in: int, channels_out: int, groups: int, activation: str = "silu", block: int = 16,
                 device="cuda", seed: int = 0):
        torch = _torch or _lazy_torch()
        g = torch.Generator().manual_seed(seed)
        self.groups, self.activation, self.block = groups, activation, block
        f32 = dict(dtype=torch.float32, device=device)
        self.weight = (torch.randn((channels_out, channels_in), generator=g) * channels_in ** -0.5).to(**f32)
        self.bias = torch.zeros(channels_out, **f32)
        self.gamma, self.beta = torch.ones(channels_in, **f32), torch.zeros(channels_in, **f32)
        self.grads = None
        self.pack()

    @property
    def parameters(self):
        return [self.weight, self.bias, self.gamma, self.beta]

    def pack(self):
        self.packed = mx4_quantize(self.weight, block=self.block)

    def forward(self, x, keep: bool = False):
        y, mean, rstd = group_norm(x, self.groups, self.gamma, self.beta, activation=self.activation)
        rows = y.view(-1, y.shape[-1])
        out = mx4_product(mx4_quantize(rows, block=self.block), self.packed, bias=self.bias, dtype=x.dtype)
        if keep:
            self._kept = (x, rows, mean, rstd)
        return out.view(*x.shape[:-1], out.shape[-1])

    def backward(self, dout, scale: float = 1.0, gain: float = 1.0):
        """`dout` holds `scale` times the gradient of the output, the result `scale * gain` times that of x, so that
        fp16 holds it; powers of two cost no digits.  `grads` are the gradients themselves."""
        torch = _torch
        if not 0 < scale < float("inf") or not 0 < gain < float("inf"):
            raise ValueError(f"scale and gain must be positive, not {scale} and {gain}")
        x, rows, mean, rstd = self._kept
        d = dout.reshape(-1, dout.shape[-1])
        dy = mx4_product(mx4_quantize(d), mx4_quantize(self.weight.t()), alpha=float(gain), dtype=x.dtype)
        dweight = mx4_product(mx4_quantize(d.t()), mx4_quantize(rows.t()), alpha=1.0 / scale, dtype=torch.float32)
        dx, dgamma, dbeta = group_norm_backward(dy.view(x.shape), x, mean, rstd, self.groups, self.gamma, self.beta,
                                                activation=self.activation)
        dbias = d.float().sum(dim=0)
        for g, factor in ((dbias, scale), (dgamma, scale * gain), (dbeta, scale * gain)):
            if factor != 1.0:
                g.mul_(1.0 / factor)
        self.grads = [dweight, dbias, dgamma, dbeta]
        return dx
