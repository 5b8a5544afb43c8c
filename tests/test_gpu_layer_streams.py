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


def test_results_come_from_the_stream_that_writes_them(cuda):
    """A block freed on torch's current stream, where its last user may still be queued, is the next one handed out
    there: no result of a call on another stream lies in it, whether the stream is an object or a handle."""
    import neural_textures_b200 as nt
    x = torch.randn((4, 64, 64, 256), device="cuda").half()
    dy, rows = torch.randn_like(x), x.view(-1, 256)
    gamma, beta = torch.ones(256, device="cuda"), torch.zeros(256, device="cuda")
    y, mean, rstd = nt.group_norm(x, 8, gamma, beta)
    q, w = nt.mx4_quantize(rows), nt.mx4_quantize(torch.randn((256, 256), device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls = {
        "norm": lambda s: nt.group_norm(x, 8, gamma, beta, stream=s),
        "gradient": lambda s: nt.group_norm_backward(dy, x, mean, rstd, 8, gamma, beta, stream=s),
        "quantise": lambda s: (lambda t: (t.data, t.scales))(nt.mx4_quantize(rows, stream=s)),
        "read back": lambda s: (nt.mx4_dequantize(q, stream=s),),
        "product": lambda s: (nt.mx4_product(q, w, stream=s),),
    }
    for name, call in calls.items():
        want = call(None)
        for stream in (side, side.cuda_stream):
            freed = [torch.empty_like(t) for t in want for _ in range(2)]
            spans = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in freed]
            del freed
            got = call(stream)
            for t in got:
                assert not any(lo <= t.data_ptr() < hi for lo, hi in spans), name
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_stream_of_a_call_with_given_results(cuda):
    """`out` together with `stream`; the caller's current stream is what it was."""
    import neural_textures_b200 as nt
    x = torch.randn((2, 9, 7, 24), device="cuda").half()
    want = nt.group_norm(x, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = torch.cuda.current_stream()
    out = torch.zeros_like(x)
    got = nt.group_norm(x, 3, out=out, stream=side)
    side.synchronize()
    assert got[0] is out and all(torch.equal(a, b) for a, b in zip(got, want))
    q = nt.mx4_quantize(x.view(-1, 24))
    back, again = torch.empty((126, 24), device="cuda"), nt.Mx4Tensor.empty(126, 24, device=x.device)
    side.wait_stream(before)
    nt.mx4_dequantize(q, out=back, stream=side.cuda_stream)
    nt.mx4_quantize(x.view(-1, 24), out=again, stream=side)
    side.synchronize()
    assert torch.equal(back, nt.mx4_dequantize(q, torch.float32)) and torch.equal(again.data, q.data)
    assert torch.cuda.current_stream() == before
    same = nt.group_norm(x, 3, stream=before.cuda_stream)
    assert torch.equal(same[0], want[0])
