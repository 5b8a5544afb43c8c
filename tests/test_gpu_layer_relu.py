"""Gradients of the group norm under relu on maps with millions of values, some of which always lie within rounding of
relu's edge: their dy is 0 here, so that either slope gives the same, and everything is compared."""
import numpy as np
import pytest
import torch

from tests import layer_oracle as O
from tests.test_gpu_layers import ALL, SUM, U, close, f64, norm_case, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ALL, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("size", [
    (1, 1, 1, 24, 3, 0), (2, 9, 11, 10, 5, 1), (1, 61, 67, 7, 1, 0), (5, 33, 17, 96, 12, 0), (1, 200, 150, 32, 4, 0),
    (2, 2, 3, 4100, 4, 0),
    (150, 200, 100, 3, 1, 0),   # single channels
    (150, 33, 31, 20, 10, 4),   # vectors across groups, unaligned
    (150, 4, 3, 8192, 16, 0),   # several turns along a texel
    (1, 1000, 1100, 24, 3, 0),  # the whole grid
], ids=lambda s: "x".join(map(str, s)))
def test_group_norm_gradients_under_relu(cuda, size, dtype):
    """The tolerances are those of test_group_norm_forward_and_backward."""
    import neural_textures_b200 as nt
    n, h, w, c, groups, pad = size
    x, gamma, beta, dy = norm_case((n, h, w, c), dtype, 17, pad)
    y, mean, rstd = nt.group_norm(x, groups, gamma, beta, activation="relu", eps=1e-3)
    ga, be, wide = f64(gamma), f64(beta), f64(x)
    hat = (wide - O._spread(f64(mean), c)) * O._spread(f64(rstd), c)
    # z's own rounding and that of x - mean
    size_x = np.abs(wide) + np.abs(O._spread(f64(mean), c))
    edge = np.abs(ga * hat + be) < 16 * U * (np.abs(ga) * (np.abs(hat) + size_x * O._spread(f64(rstd), c)) + np.abs(be)) + 1e-30
    assert edge.mean() < 1e-4
    dy[torch.from_numpy(edge).cuda()] = 0
    dx, dgamma, dbeta = nt.group_norm_backward(dy, x, mean, rstd, groups, gamma, beta, activation="relu")
    wdx, wdg, wdb, sx, sg, sb = O.group_norm_backward(f64(dy), wide, f64(mean), f64(rstd), groups, ga, be, "relu")
    lipschitz = 1.2 * (1 + np.abs(ga).max() + np.abs(be).max())
    close(dx, wdx, rounded(dtype, wdx, SUM * lipschitz * sx + 1e-30), "dx")
    close(dgamma, wdg, SUM * lipschitz * sg + 1e-30, "dgamma")
    close(dbeta, wdb, SUM * lipschitz * sb + 1e-30, "dbeta")
