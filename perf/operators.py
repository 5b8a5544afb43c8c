"""Cases of the channels-last group norm and of the 4-bit microscaled tensors: what is timed
and compared, in a plain torch form (`own` false) and through this package (`own` true).

Three operators:
  group_norm   group norm with an activation over [N][H][W][C], forward or backward
  mx4_store    a matrix quantised to 4-bit microscaled values and read back
  mx4_product  act(alpha A B^T + bias) of two such matrices

The packed form that mx4_product takes (and that the package's mx4_quantize writes): codes
are E2M1, two to a byte, the even column in the low nibble, rows of ceil(cols / 32) * 16
bytes; scales (a byte per block of 32: E8M0, or of 16: E4M3) sit in tiles of 128 rows x 4
scales, tile (i, j) at 512 * (i * tiles_per_row + j), in it the scale of row r, block k at
16 * (r % 32) + 4 * (r / 32) + k; what lies past the matrix is zero.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}


# ---- the cases ---------------------------------------------------------------------------

def listed():
    norm = lambda name, way, n, h, w, c, groups, act, dtype, pad=0: dict(  # noqa: E731
        name=name, op="group_norm", way=way, n=n, h=h, w=w, c=c, groups=groups, act=act, dtype=dtype, pad=pad)
    store = lambda name, rows, cols, block, dtype, transposed=False: dict(  # noqa: E731
        name=name, op="mx4_store", rows=rows, cols=cols, block=block, dtype=dtype, transposed=transposed)
    prod = lambda name, m, n, k, block, act, dtype: dict(  # noqa: E731
        name=name, op="mx4_product", m=m, n=n, k=k, block=block, act=act, dtype=dtype)
    return [
        # the last mips of a feature pyramid: one launch's latency
        norm("norm 16x16x64", "forward", 1, 16, 16, 64, 8, "silu", "f16"),
        # a hidden feature map of a 1024 x 1024 material
        norm("norm 1024x1024x64", "forward", 1, 1024, 1024, 64, 8, "silu", "f16"),
        # latent-width maps of odd size, a channel slice of wider texels
        norm("norm odd 3x253x187x12", "forward", 3, 253, 187, 12, 3, "gelu", "bf16", 4),
        # training an encoder of small crops in 32 bits
        norm("norm grad 8x32x32x32", "backward", 8, 32, 32, 32, 4, "relu", "f32"),
        # the same large feature map on the way back
        norm("norm grad 1024x1024x64", "backward", 1, 1024, 1024, 64, 8, "silu", "f16"),
        # a 512 x 512 x 8 latent grid stored row by row, next to its BC6H form
        store("store 512x4096", 512, 4096, 32, "f16"),
        # a large weight or activation matrix
        store("store 16384x8192", 16384, 8192, 16, "bf16"),
        # a ragged 32-bit gradient read along its columns, for the product of a weight's gradient
        store("store odd 1021x1531 turned", 1021, 1531, 16, "f32", True),
        # one token or texel against a layer's weights
        prod("product 1x4096x4096", 1, 4096, 4096, 16, "none", "f16"),
        # the 64-wide hidden layer of every sample of a 512 x 512 lattice
        prod("product 262144x64x64", 262144, 64, 64, 32, "relu", "f16"),
        # ragged everywhere, a fused activation
        prod("product odd 1537x1000x1111", 1537, 1000, 1111, 32, "silu", "f32"),
        # a large layer, where the tensor cores' rate counts
        prod("product 8192x8192x8192", 8192, 8192, 8192, 16, "none", "bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "mx4_store", "mx4_product"])
    dtype = rng.choice(["f16", "f16", "bf16", "f32"])
    if op == "group_norm":
        per, groups = rng.choice([1, 2, 3, 4, 6, 8, 12, 16]), rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = per * groups
        n = rng.choice([1, 1, 2, 3, 5, 8])
        most = (1 << 25) // (n * c)  # elements of half the largest listed map, at most
        texels = _log_int(rng, 16, max(17, min(1 << 20, most)))
        h = max(1, int(math.sqrt(texels) * rng.uniform(0.5, 2.0)))
        w = max(1, texels // h)
        return dict(op=op, way=rng.choice(["forward", "backward"]), n=n, h=h, w=w, c=c, groups=groups,
                    act=rng.choice(["none", "relu", "silu", "gelu"]), dtype=dtype, pad=rng.choice([0, 0, 0, 4, 5]))
    block = rng.choice([16, 32])
    if op == "mx4_store":
        cols = _log_int(rng, 24, 16384)
        rows = _log_int(rng, 16, min(65536, (1 << 26) // cols))
        return dict(op=op, rows=rows, cols=cols, block=block, dtype=dtype, transposed=rng.random() < 0.3)
    k, n = _log_int(rng, 32, 8192), _log_int(rng, 16, 8192)
    m = _log_int(rng, 1, min(1 << 18, (1 << 26) // n, (1 << 37) // (n * k)))
    return dict(op=op, m=m, n=n, k=k, block=block, act=rng.choice(["none", "relu", "silu", "gelu"]), dtype=dtype)


# ---- what a user has in hand ----------------------------------------------------------------

def _normal(shape, seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + salt)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _matrix(rows, cols, seed, salt):
    """Values whose blocks differ in size by a few powers of two, as weights and activations do."""
    return _normal((rows, cols), seed, salt) * torch.exp2(_normal((rows, 1), seed, salt + 1))


def prepare(case, seed):
    op, dtype = case["op"], DTYPES.get(case["dtype"])
    if op == "group_norm":
        n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
        wide = _normal((n, h, w, c + case["pad"]), seed, 0)
        wide = (wide * (0.5 + _normal((c + case["pad"],), seed, 1).abs()) + _normal((c + case["pad"],), seed, 2)).to(dtype)
        state = {"case": case, "x": wide[..., :c], "gamma": 1 + 0.2 * _normal((c,), seed, 3),
                 "beta": 0.2 * _normal((c,), seed, 4)}
        if case["way"] == "backward":
            grouped = state["x"].float().reshape(n, h * w, groups, c // groups)
            state["mean"] = grouped.mean(dim=(1, 3))
            state["rstd"] = torch.rsqrt((grouped - state["mean"][:, None, :, None]).square().mean(dim=(1, 3)) + 1e-5)
            state["dy"] = _normal((n, h, w, c), seed, 5).to(dtype)
        return state
    if op == "mx4_store":
        rows, cols = case["rows"], case["cols"]
        x = _matrix(rows, cols, seed, 0).to(dtype)
        return {"case": case, "x": x.t().contiguous().t() if case["transposed"] else x}
    state = {"case": case, "bias": _normal((case["n"],), seed, 8), "alpha": 1.0 / math.sqrt(case["k"])}
    for name, rows, salt in (("a", case["m"], 0), ("b", case["n"], 4)):
        codes, scales = _quantized(_matrix(rows, case["k"], seed, salt), case["block"])
        state[name + "_data"], state[name + "_scales"] = _packed(codes, scales, case["block"])
    return state


# ---- plain forms -----------------------------------------------------------------------------

def _activation(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _activation_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _norm_forward(x, groups, gamma, beta, act):
    n, h, w, c = x.shape
    v = x.float().reshape(n, h * w, groups, c // groups)
    mean = v.mean(dim=(1, 3))
    centred = v - mean[:, None, :, None]
    rstd = torch.rsqrt(centred.square().mean(dim=(1, 3)) + 1e-5)
    z = (centred * rstd[:, None, :, None]).reshape(n, h, w, c) * gamma + beta
    return {"y": _activation(z, act).to(x.dtype), "mean": mean, "rstd": rstd}


def _norm_backward(dy, x, mean, rstd, groups, gamma, beta, act):
    n, h, w, c = x.shape
    per = (n, h * w, groups, c // groups)
    hat = (x.float().reshape(per) - mean[:, None, :, None]) * rstd[:, None, :, None]
    flat = hat.reshape(n, h, w, c)
    e = dy.float() * _activation_slope(flat * gamma + beta, act)
    ge = (e * gamma).reshape(per)
    s1, s2 = ge.mean(dim=(1, 3), keepdim=True), (ge * hat).mean(dim=(1, 3), keepdim=True)
    dx = (ge - s1 - hat * s2) * rstd[:, None, :, None]
    return {"dx": dx.reshape(n, h, w, c).to(x.dtype), "dgamma": (e * flat).sum(dim=(0, 1, 2)), "dbeta": e.sum(dim=(0, 1, 2))}


def _quantized(x, block):
    """Codes (0 .. 15, uint8) [rows][blocks * block] and scale bytes [rows][blocks] of x."""
    rows, cols = x.shape
    blocks = -(-cols // block)
    v = torch.zeros((rows, blocks * block), dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.reshape(rows, blocks, block)
    most = v.abs().amax(dim=2)
    if block == 32:
        scales = ((most.view(torch.int32) >> 23) - 2).clamp(min=0).to(torch.uint8)
    else:
        scales = (most / 6).clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8)
    s, size = _scale_values(scales, block)[:, :, None], v.abs()
    # each bound between two neighbours, times the scale, is exact in 32 bits; ties go to the even code
    code = ((size > 0.25 * s).to(torch.uint8) + (size >= 0.75 * s) + (size > 1.25 * s) + (size >= 1.75 * s)
            + (size > 2.5 * s) + (size >= 3.5 * s) + (size > 5.0 * s))
    code = torch.where(s > 0, code, torch.zeros_like(code)) + torch.signbit(v).to(torch.uint8) * 8
    return code.reshape(rows, blocks * block), scales


def _scale_values(scales, block):
    if block == 32:
        return torch.exp2(scales.float() - 127)
    return scales.view(torch.float8_e4m3fn).float()


def _values(codes, scales, block):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    rows = codes.shape[0]
    return (table[codes.long()].reshape(rows, -1, block) * _scale_values(scales, block)[:, :, None]).reshape(rows, -1)


def _packed(codes, scales, block):
    rows, blocks = scales.shape
    wide = -(-codes.shape[1] // 32) * 32
    full = torch.zeros((rows, wide), dtype=torch.uint8, device=codes.device)
    full[:, :codes.shape[1]] = codes
    data = full[:, 0::2] | (full[:, 1::2] << 4)
    ti, tj = -(-rows // 128), -(-blocks // 4)
    grid = torch.zeros((ti * 128, tj * 4), dtype=torch.uint8, device=codes.device)
    grid[:rows, :blocks] = scales
    return data.contiguous(), grid.reshape(ti, 4, 32, tj, 4).permute(0, 3, 2, 1, 4).contiguous().reshape(-1)


def _unpacked(data, scales, rows, cols, block):
    codes = torch.stack((data & 15, data >> 4), dim=2).reshape(rows, -1)
    blocks = -(-cols // block)
    ti, tj = -(-rows // 128), -(-blocks // 4)
    grid = scales.reshape(ti, tj, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(ti * 128, tj * 4)
    return _values(codes[:, :blocks * block], grid[:rows, :blocks], block)[:, :cols]


def run(state):
    case = state["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if own:
        import neural_textures_b200 as nt
        if op == "group_norm" and case["way"] == "forward":
            y, mean, rstd = nt.group_norm(state["x"], case["groups"], state["gamma"], state["beta"], activation=case["act"])
            return {"y": y, "mean": mean, "rstd": rstd}
        if op == "group_norm":
            dx, dgamma, dbeta = nt.group_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], case["groups"],
                                                       state["gamma"], state["beta"], activation=case["act"])
            return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
        if op == "mx4_store":
            return nt.mx4_dequantize(nt.mx4_quantize(state["x"], block=case["block"]), dtype)
        a = nt.Mx4Tensor(state["a_data"], state["a_scales"], case["m"], case["k"], case["block"])
        b = nt.Mx4Tensor(state["b_data"], state["b_scales"], case["n"], case["k"], case["block"])
        return nt.mx4_product(a, b, bias=state["bias"], activation=case["act"], alpha=state["alpha"], dtype=dtype)
    if op == "group_norm" and case["way"] == "forward":
        return _norm_forward(state["x"], case["groups"], state["gamma"], state["beta"], case["act"])
    if op == "group_norm":
        return _norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], case["groups"], state["gamma"],
                              state["beta"], case["act"])
    if op == "mx4_store":
        return _values(*_quantized(state["x"].float(), case["block"]), case["block"])[:, :case["cols"]].to(dtype)
    a = _unpacked(state["a_data"], state["a_scales"], case["m"], case["k"], case["block"])
    b = _unpacked(state["b_data"], state["b_scales"], case["n"], case["k"], case["block"])
    return _activation(state["alpha"] * (a @ b.t()) + state["bias"], case["act"]).to(dtype)


# ---- work and 64-bit values -----------------------------------------------------------------

def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "group_norm":
        count, back = case["n"] * case["h"] * case["w"] * case["c"], case["way"] == "backward"
        small = 4 * (2 * case["n"] * case["groups"] + (4 if back else 2) * case["c"])
        return {"bytes": count * size * (3 if back else 2) + small, "flops": count * (24 if back else 12)}
    if case["op"] == "mx4_store":
        count = case["rows"] * case["cols"]
        return {"bytes": 2 * count * (size + 0.5 + 1 / case["block"]), "flops": 4 * count}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": (m + n) * k * (0.5 + 1 / case["block"]) + m * n * size + 4 * n, "flops": 2 * m * n * k}


def _erf_gate(z):
    return torch.special.ndtr(z)  # the normal distribution's integral, (1 + erf(z / sqrt 2)) / 2


def _exact_activation(z, act):
    gate = {"none": torch.ones_like, "relu": lambda t: (t > 0).to(t.dtype), "silu": torch.sigmoid, "gelu": _erf_gate}[act]
    return z * gate(z)


def _exact_e2m1(u):
    """u >= 0 to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6: whole steps of the binade that u lies in."""
    step = torch.exp2(torch.floor(torch.log2(u.clamp(min=1.0))) - 1)
    return (torch.round(u / step) * step).clamp(max=6.0)


def _exact_block_scale(most, block):
    if block == 32:
        _, exponent = torch.frexp(most)  # most = f 2^exponent, f in [1/2, 1)
        return torch.where(most > 0, torch.exp2((exponent.double() - 3).clamp(min=-127)), torch.exp2(torch.full_like(most, -127)))
    v = most / 6
    step = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def _exact_packed(data, scales, rows, cols, block):
    """The matrix that the packed form stands for, by the fields of each code and the place of each scale."""
    column = torch.arange(cols, device=data.device)
    byte = data[:, column // 2].long()
    nibble = torch.where(column % 2 == 0, byte & 15, byte >> 4)
    exponent, mantissa = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    row, k = torch.arange(rows, device=data.device)[:, None], torch.arange(-(-cols // block), device=data.device)[None, :]
    tiles = -(-cols // (4 * block))
    at = ((row // 128) * tiles + k // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + k % 4
    bits = scales[at].long()
    if block == 32:
        s = torch.exp2(bits.double() - 127)
    else:
        e, f = bits >> 3, (bits & 7).double()
        s = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.exp2(e.double() - 10))
    return torch.where(nibble >= 8, -size, size) * s[:, column // block]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "mx4_store":
        rows, cols, block = case["rows"], case["cols"], case["block"]
        v = torch.nn.functional.pad(state["x"].double(), (0, -cols % block)).unflatten(1, (-1, block))
        s = _exact_block_scale(v.abs().amax(dim=2, keepdim=True), block)
        q = torch.where(s > 0, _exact_e2m1(v.abs() / s.clamp(min=2.0 ** -140)) * s, torch.zeros_like(v))
        return torch.copysign(q, v).flatten(1)[:, :cols]
    if case["op"] == "mx4_product":
        a = _exact_packed(state["a_data"], state["a_scales"], case["m"], case["k"], case["block"])
        b = _exact_packed(state["b_data"], state["b_scales"], case["n"], case["k"], case["block"])
        return _exact_activation(torch.addmm(state["bias"].double(), a, b.t(), alpha=state["alpha"]), case["act"])
    x, gamma, beta, groups = state["x"].double(), state["gamma"].double(), state["beta"].double(), case["groups"]
    n, c = x.shape[0], x.shape[3]
    spread = lambda t: t.repeat_interleave(c // groups, dim=1)[:, None, None, :]  # noqa: E731
    if case["way"] == "forward":
        grouped = x.flatten(1, 2).unflatten(2, (groups, -1)).transpose(1, 2).flatten(2)
        mean, rstd = grouped.mean(dim=2), (grouped.var(dim=2, unbiased=False) + 1e-5).rsqrt()
        return {"y": _exact_activation((x - spread(mean)) * spread(rstd) * gamma + beta, case["act"]), "mean": mean, "rstd": rstd}
    # the gradient, with the statistics as given: a function of the sums of e and of e h
    dy, rstd = state["dy"].double(), spread(state["rstd"].double())
    h = (x - spread(state["mean"].double())) * rstd
    z = (h * gamma + beta).requires_grad_()
    (e,) = torch.autograd.grad(_exact_activation(z, case["act"]), z, dy)
    sums = torch.stack((e.sum(dim=(1, 2)), (e * h).sum(dim=(1, 2))))
    of_group = (sums * gamma).reshape(2, n, groups, -1).sum(dim=3) / (x[0].numel() // groups)
    dx = rstd * (e * gamma - spread(of_group[0]) - h * spread(of_group[1]))
    return {"dx": dx, "dgamma": sums[1].sum(dim=0), "dbeta": sums[0].sum(dim=0)}
