"""Texel-layer operators: channels-last group normalisation with an activation (forward and
backward), 4-bit microscaled matrices (quantise, read back, product), and TexelLayer, which runs
them as one layer of a network over a feature map.

Every call queues its kernels on `stream` (a torch.cuda.Stream or a raw handle; None: torch's
current stream of the tensors' device) and returns without waiting.  Results are new tensors unless
`out` is given.  Invalid arguments raise: TypeError / ValueError for what only the tensors show
(device, dtype, shape), NtError for what the library rejects.
"""
from __future__ import annotations

import struct

from . import _native as N
from ._native import check, load

ACTIVATIONS = {"none": N.NT_ACT_NONE, "relu": N.NT_ACT_RELU, "silu": N.NT_ACT_SILU, "gelu": N.NT_ACT_GELU}

_torch = None
_DTYPES = {}


def _lazy_torch():
    """torch, imported at the first call as everywhere in this package."""
    global _torch
    if _torch is None:
        import torch
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


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _vector(t, n: int, name: str) -> int | None:
    """Data pointer of an optional contiguous fp32 vector of n elements."""
    if t is None:
        return None
    if t.dtype is not _torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} elements")
    return t.data_ptr()


def _launch(device, stream, made, fn, *args):
    """fn(*args, stream) on `device`.  `made` are tensors of this call: they live in torch's pool of
    the current stream, so when another stream uses them they are recorded on it."""
    torch = _torch
    if device.type != "cuda":
        raise ValueError(f"a CUDA tensor is needed, not one on {device}")
    index = device.index
    current = torch._C._cuda_getCurrentRawStream(index)
    handle = current if stream is None else stream if isinstance(stream, int) else int(stream.cuda_stream)
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, handle)
    else:
        with torch.cuda.device(index):
            status = fn(*args, handle)
    if handle != current:
        other = torch.cuda.ExternalStream(handle, device=device)
        for t in made:
            if t is not None:
                t.record_stream(other)
    if status:
        check(status)


# ---------------------------------------------------------------------------------------
# group normalisation

_GROUP_NORM = struct.Struct("@7if" + "P3q" + "4P" + "P3q" * 3 + "3Pq")
_NO_MAP = (0, 0, 0, 0)
_workspace_sizes = {}


def _map(t, shape, dtype, device, name: str):
    """(pointer, strides) of a channels-last map [N][H][W][C] or [H][W][C]."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} of {dtype} on {device}, not {tuple(t.shape)} of {t.dtype} on {t.device}")
    s = t.stride()
    if s[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the channels must be contiguous (stride 1, not {s[-1]})")
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), 0, s[0], s[1])


def _norm_sizes(x, groups: int):
    if x.dim() not in (3, 4):
        raise ValueError(f"x must be [N][H][W][C] or [H][W][C], not {tuple(x.shape)}")
    n, h, w, c = x.shape if x.dim() == 4 else (1, *x.shape)
    return n, h, w, c, int(groups)


def _norm_call(entry, sizes, dtype: int, act: int, eps: float, x, gamma, beta, mean, rstd, y, dy, dx, dgamma, dbeta,
               device, stream, made):
    L = load()
    backward = int(entry == "nt_group_norm_backward")
    key = (sizes, dtype, backward)
    need = _workspace_sizes.get(key)
    pack = lambda ws, size: _GROUP_NORM.pack(*sizes, dtype, act, eps, *x, gamma or 0, beta or 0, mean, rstd, *y, *dy, *dx,
                                             dgamma, dbeta, ws, size)
    if need is None:
        if len(_workspace_sizes) > 4096:
            _workspace_sizes.clear()
        need = _workspace_sizes[key] = int(L.nt_group_norm_workspace_bytes(pack(0, 0), backward))
    ws = _torch.empty(need, dtype=_torch.uint8, device=device) if need else None
    _launch(device, stream, (ws, *made), getattr(L, entry), pack(ws.data_ptr() if need else 0, need))


def group_norm(x, groups: int, gamma=None, beta=None, activation: str = "none", eps: float = 1e-5, out=None, stream=None):
    """activation(gamma (x - mean) rstd + beta) of a channels-last feature map [N][H][W][C] (or one
    image [H][W][C]) over `groups` groups of consecutive channels; float16, bfloat16 or float32,
    any strides over images, rows and texels.  gamma and beta are float32 [C] or None.  Returns
    (y, mean, rstd) with float32 statistics [N][groups], which group_norm_backward takes.  `out`
    receives y and may be x."""
    torch = _torch or _lazy_torch()
    sizes, dtype = _norm_sizes(x, groups), _dtype(x, "x")
    device, shape = x.device, x.shape
    _same_device(device, gamma=gamma, beta=beta)
    y = torch.empty(shape, dtype=x.dtype, device=device) if out is None else out
    stats = torch.empty((2, sizes[0], max(sizes[4], 0)), dtype=torch.float32, device=device)
    mean, rstd = stats[0], stats[1]
    c = sizes[3]
    _norm_call("nt_group_norm_forward", sizes, dtype, _activation(activation), eps,
               _map(x, shape, x.dtype, device, "x"), _vector(gamma, c, "gamma"), _vector(beta, c, "beta"),
               mean.data_ptr(), rstd.data_ptr(), _map(y, shape, x.dtype, device, "out"), _NO_MAP, _NO_MAP, 0, 0,
               device, stream, (y if out is None else None, stats))
    return y, mean, rstd


def group_norm_backward(dy, x, mean, rstd, groups: int, gamma=None, beta=None, activation: str = "none", out=None, stream=None):
    """Gradients of group_norm at its input x, with the statistics that it returned: (dx, dgamma,
    dbeta).  dx has x's type; dgamma and dbeta are float32 [C], summed over images and texels.
    `out` receives dx and may be dy or x."""
    torch = _torch or _lazy_torch()
    sizes, dtype = _norm_sizes(x, groups), _dtype(x, "x")
    device, shape, c = x.device, x.shape, sizes[3]
    _same_device(device, gamma=gamma, beta=beta, mean=mean, rstd=rstd)
    dx = torch.empty(shape, dtype=x.dtype, device=device) if out is None else out
    grads = torch.empty((2, c), dtype=torch.float32, device=device)
    dgamma, dbeta = grads[0], grads[1]
    stat = sizes[0] * sizes[4]
    _norm_call("nt_group_norm_backward", sizes, dtype, _activation(activation), 1.0,
               _map(x, shape, x.dtype, device, "x"), _vector(gamma, c, "gamma"), _vector(beta, c, "beta"),
               _vector(mean, stat, "mean"), _vector(rstd, stat, "rstd"), _NO_MAP, _map(dy, shape, x.dtype, device, "dy"),
               _map(dx, shape, x.dtype, device, "out"), dgamma.data_ptr(), dbeta.data_ptr(), device, stream,
               (dx if out is None else None, grads))
    return dx, dgamma, dbeta


# ---------------------------------------------------------------------------------------
# 4-bit microscaled matrices

_MATRIX = struct.Struct("@2Pq3i4x")


class Mx4Tensor:
    """A rows x cols matrix in 4-bit microscaled form (NtMx4Matrix): `data`, the uint8 codes
    [rows][pitch], two to a byte, and `scales`, a byte per block of `block` columns (32: powers of
    two, 16: E4M3) in tiles of 128 rows x 4 blocks.  Padding must be zero, as mx4_quantize leaves it."""
    __slots__ = ("data", "scales", "rows", "cols", "block", "_packed")

    def __init__(self, data, scales, rows: int, cols: int, block: int = 32):
        torch = _torch or _lazy_torch()
        L = load()
        if block not in (16, 32):
            raise ValueError(f"block must be 16 or 32, not {block}")
        if rows < 0 or cols < 1:
            raise ValueError(f"{rows} x {cols} is not a matrix size")
        if data.dtype is not torch.uint8 or data.dim() != 2 or data.shape[0] < rows or data.shape[1] < -(-cols // 32) * 16:
            raise ValueError(f"data must be uint8 [{rows}][{-(-cols // 32) * 16}] or larger")
        if data.shape[1] > 1 and data.stride(1) != 1:
            raise ValueError("data: the codes of a row must be contiguous")
        if scales.dtype is not torch.uint8 or not scales.is_contiguous() or scales.numel() < -(-rows // 128) * -(-cols // (4 * block)) * 512:
            raise ValueError(f"scales must be contiguous uint8 of {L.nt_mx4_scales_bytes(rows, cols, block)} bytes")
        _same_device(data.device, scales=scales)
        self.data, self.scales, self.rows, self.cols, self.block = data, scales, int(rows), int(cols), int(block)
        self._packed = _MATRIX.pack(data.data_ptr(), scales.data_ptr(), data.stride(0) if rows > 1 else data.shape[1] // 16 * 16,
                                    self.rows, self.cols, self.block)

    @classmethod
    def empty(cls, rows: int, cols: int, block: int = 32, device="cuda"):
        torch = _torch or _lazy_torch()
        if block not in (16, 32) or rows < 0 or cols < 1:
            raise ValueError(f"{rows} x {cols} in blocks of {block} is not a 4-bit matrix")
        pitch, scales = -(-cols // 32) * 16, -(-rows // 128) * -(-cols // (4 * block)) * 512
        return cls(torch.empty((rows, pitch), dtype=torch.uint8, device=device),
                   torch.empty(scales, dtype=torch.uint8, device=device), rows, cols, block)

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
    dtype = _dtype(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, not {tuple(x.shape)}")
    made = out is None
    if made:
        out = Mx4Tensor.empty(x.shape[0], x.shape[1], block, x.device)
    elif out.shape != tuple(x.shape) or out.block != block or out.device != x.device:
        raise ValueError(f"out must be {tuple(x.shape)} in blocks of {block} on {x.device}")
    rs, cs = x.stride()
    _launch(x.device, stream, (out.data, out.scales) if made else (), load().nt_mx4_quantize, x.data_ptr(), dtype, rs, cs,
            out._packed)
    return out


def _output(out, rows: int, cols: int, dtype, device):
    """(tensor, row stride) of a matrix result: a new one of `dtype`, or `out` checked."""
    if out is None:
        return _torch.empty((rows, cols), dtype=dtype, device=device), cols
    if out.shape != (rows, cols) or out.dtype is not dtype or out.device != device or (cols > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be [{rows}][{cols}] of {dtype} on {device} with contiguous columns")
    return out, out.stride(0)


def mx4_dequantize(q: Mx4Tensor, dtype=None, out=None, stream=None):
    """The values of q as a matrix of `dtype` (default: out's, or float16)."""
    torch = _torch or _lazy_torch()
    dtype = dtype or (out.dtype if out is not None else torch.float16)
    code = _dtype(dtype, "dtype")
    y, stride = _output(out, q.rows, q.cols, dtype, q.device)
    _launch(q.device, stream, (y if out is None else None,), load().nt_mx4_dequantize, q._packed, y.data_ptr(), code, stride)
    return y


def mx4_product(a: Mx4Tensor, b: Mx4Tensor, bias=None, activation: str = "none", alpha: float = 1.0, dtype=None, out=None,
                stream=None):
    """activation(alpha a b^T + bias), [a.rows][b.rows] of `dtype` (default: out's, or float16): a layer's
    output for texels a and weights b [out][in], bias float32 [out] or None."""
    torch = _torch or _lazy_torch()
    dtype = dtype or (out.dtype if out is not None else torch.float16)
    code, act, device = _dtype(dtype, "dtype"), _activation(activation), a.device
    _same_device(device, b=b, bias=bias)
    y, stride = _output(out, a.rows, b.rows, dtype, device)
    _launch(device, stream, (y if out is None else None,), load().nt_mx4_product, a._packed, b._packed,
            _vector(bias, b.rows, "bias"), act, alpha, y.data_ptr(), code, stride)
    return y
