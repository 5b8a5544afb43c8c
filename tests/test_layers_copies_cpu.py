"""A 4-bit matrix always names the memory of the tensors that it holds: after a copy, after loading, after a
tensor got another storage."""
import copy
import io
import pickle

import pytest
import torch


def _memory(q):
    from neural_textures_b200 import _native as N
    m = N.NtMx4Matrix.from_buffer_copy(q._packed)
    return m.data, m.scales, m.pitch, m.rows, m.cols, m.block


def _of_tensors(q):
    pitch = q.data.stride(0) if q.rows > 1 else -(-q.cols // 32) * 16
    return q.data.data_ptr(), q.scales.data_ptr(), pitch, q.rows, q.cols, q.block


def _example():
    import neural_textures_b200 as nt
    q = nt.Mx4Tensor.empty(5, 70, 16, device="cpu")
    q.data.random_(0, 256)
    q.scales.random_(0, 127)
    return q


def _through_torch(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("way", [copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)), _through_torch],
                         ids=["deepcopy", "pickle", "torch.save"])
def test_copies_hold_their_own_memory(native, way):
    q = _example()
    r = way(q)
    assert torch.equal(r.data, q.data) and torch.equal(r.scales, q.scales) and r.shape == q.shape and r.block == q.block
    assert r.data.data_ptr() != q.data.data_ptr()
    assert _memory(r) == _of_tensors(r) and _memory(q) == _of_tensors(q)


def test_a_shallow_copy_shares_its_memory(native):
    q = _example()
    r = copy.copy(q)
    assert r.data is q.data and _memory(r) == _of_tensors(r)


def test_a_copied_layer_packs_its_own_weights(native, monkeypatch):
    import neural_textures_b200 as nt
    from neural_textures_b200 import layers
    monkeypatch.setattr(layers, "mx4_quantize", lambda w, block: nt.Mx4Tensor.empty(*w.shape, block, device="cpu"))
    layer = nt.TexelLayer(32, 16, groups=4, device="cpu")
    other = copy.deepcopy(layer)
    assert other.packed.data.data_ptr() != layer.packed.data.data_ptr()
    assert _memory(other.packed) == _of_tensors(other.packed)


@pytest.mark.parametrize("field", ["data", "scales", "rows", "cols", "block"])
def test_fields_are_read_only(native, field):
    q = _example()
    with pytest.raises(AttributeError):
        setattr(q, field, getattr(q, field))


def test_a_calls_matrix_is_that_of_the_tensors_now(native):
    """Tensors whose storage was replaced in place: the call takes the new memory, or says why it cannot."""
    from neural_textures_b200 import _native as N, layers
    q = _example()
    q.data.set_(torch.zeros(5, 48, dtype=torch.uint8))
    m = N.NtMx4Matrix.from_buffer_copy(layers._matrix(q))
    assert (m.data, m.scales) == (q.data.data_ptr(), q.scales.data_ptr())
    q.scales.set_(torch.zeros(16, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scales must be"):
        layers._matrix(q)
