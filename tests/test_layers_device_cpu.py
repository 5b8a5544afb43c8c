"""Where a new 4-bit matrix lies when its device is named without an index."""
import pytest
import torch


@pytest.mark.parametrize("device", ["cuda", torch.device("cuda")], ids=str)
def test_an_empty_matrix_lies_on_the_current_device(native, monkeypatch, device):
    """On that of the call, not on the one that was current when the shape was first asked for."""
    from neural_textures_b200 import layers
    import neural_textures_b200 as nt
    asked = []

    def new(shape, dtype, device):
        asked.append(device)
        return torch.empty(shape, dtype=dtype)

    monkeypatch.setattr(layers, "_new", new)
    for index in (1, 0):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: index)
        nt.Mx4Tensor.empty(5, 70, 16, device=device)
        assert asked == [torch.device("cuda", index)] * 2
        asked.clear()


def test_an_empty_matrix_elsewhere(native):
    import neural_textures_b200 as nt
    assert nt.Mx4Tensor.empty(5, 70, 16, device="cpu").device == torch.device("cpu")
