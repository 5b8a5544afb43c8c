"""LatentEncoder on the host: what a training step calls, in which order and on which stream."""
import types

import pytest
import torch

SIDE = 0x5150  # a stream's handle


class FakeLayer:
    parameters = ()

    def __init__(self, calls):
        self.calls = calls
        self.grads = []

    def forward(self, x, keep=False):
        self.calls.append(("forward", None))
        return x

    def backward(self, d, *args, **kwargs):
        self.calls.append(("backward", None))
        return d

    def pack(self):
        pass


class FakeTexture:
    """The parts of a NeuralTexture that an encoder touches, on the host."""

    def __init__(self, **change):
        self.device, self.C, self.step = torch.device("cpu"), 8, 0
        self.grid_sizes, self.num_mips, self.lattice = [(4, 4), (2, 2)], [1, 1], (8, 8)
        self.latent_format = 0
        self.grids = [torch.zeros(4, 4, 8), torch.zeros(2, 2, 8)]
        self.ggrads = [torch.ones_like(g) for g in self.grids]
        self.__dict__.update(change)

    def params(self, **kwargs):
        return types.SimpleNamespace(num_samples=64)


@pytest.fixture
def step(native, monkeypatch):
    """(encoder, calls): an encoder over fakes whose calls into the library are noted with their stream."""
    from neural_textures_b200 import encoder
    calls = []
    for name in ("InvokeTraining", "InvokeOptimizeNetwork", "InvokeOptimizeFeatures", "InvokeOptimizeAll"):
        monkeypatch.setattr(encoder, name, lambda p, *a, stream=None, name=name: calls.append((name, stream)), raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=SIDE))
    enc = encoder.LatentEncoder.__new__(encoder.LatentEncoder)
    enc.tex, enc.grid, enc.step, enc.adam = FakeTexture(), 0, 0, (1e-3, 0.9, 0.99, 1e-8)
    enc.device = enc.tex.device
    enc.layers = [FakeLayer(calls), FakeLayer(calls)]
    enc.moments = [[], []]
    return enc, calls


def test_a_step_stays_on_the_current_stream(step):
    """The layers run on torch's current stream; the texture's own passes, whose default is another one, run there
    too."""
    enc, calls = step
    enc.train_step(torch.ones(4, 4, 8))
    passes = [c for c in calls if c[0].startswith("Invoke")]
    assert passes and all(stream == SIDE for _, stream in passes), passes
    order = [c[0] for c in calls]
    assert order.index("InvokeTraining") == 2 and order[3:5] == ["backward", "backward"]


@pytest.mark.parametrize("grid", [0, 1])
def test_a_step_optimises_the_other_grid(step, monkeypatch, grid):
    """The texture's Adam sees the other grid's gradient and none of the encoded one, which it leaves alone then."""
    from neural_textures_b200 import encoder
    enc, calls = step
    enc.grid = grid
    enc.tex.grid_sizes, enc.tex.grids[grid] = [(4, 4), (4, 4)], torch.zeros(4, 4, 8)
    enc.tex.ggrads = [torch.ones(4, 4, 8), torch.ones(4, 4, 8)]
    seen = {}

    def note(name):
        return lambda p, *a, stream=None: seen.setdefault(name, [bool(g.any()) for g in enc.tex.ggrads])

    for name in ("InvokeOptimizeNetwork", "InvokeOptimizeFeatures", "InvokeOptimizeAll"):
        monkeypatch.setattr(encoder, name, note(name), raising=False)
    enc.train_step(torch.ones(4, 4, 8))
    features = [v for k, v in seen.items() if k in ("InvokeOptimizeFeatures", "InvokeOptimizeAll")]
    assert features == [[g != grid for g in range(2)]]
    assert enc.tex.step == 1 and not enc.tex.ggrads[grid].any()


@pytest.mark.parametrize("change,needle", [(dict(num_mips=[3, 1]), "one level"), (dict(latent_format=1), "fp16 grids")])
def test_encoder_refuses_textures_that_it_cannot_fill(step, change, needle):
    """Of a chain of mips only the first level would be encoded; block records have no grid to write. Found when the
    encoder is made and, since a texture can change its form, at every call; nothing is written or queued then."""
    from neural_textures_b200 import encoder
    enc, calls = step
    with pytest.raises(ValueError, match=needle):
        encoder.LatentEncoder(FakeTexture(**change))
    enc.tex.__dict__.update(change)
    for call in (enc.encode, enc.train_step):
        with pytest.raises(ValueError, match=needle):
            call(torch.ones(4, 4, 8))
    assert not calls and not enc.tex.grids[0].any()


def test_encoder_takes_a_texture_whose_other_grid_has_mips(step):
    enc, calls = step
    enc.tex.num_mips = [1, 2]
    enc.train_step(torch.ones(4, 4, 8))
    assert enc.tex.step == 1
