"""The rows in which a texture's latents are stored in 4 bits: what they cover and what they take."""
import pytest
import torch


def _bytes(native, rows, block):
    r, c = rows.shape
    return r * native.nt_mx4_pitch(c) + native.nt_mx4_scales_bytes(r, c, block)


# grids, channels, mips; the second is that of 512 x 512 with a chain of 8 levels
SIZES = [(((512, 512), (256, 256)), 8, (1, 1)), (((512, 512), (256, 256)), 8, (8, 7)), (((300, 200), (150, 100)), 12, (8, 4)),
         (((511, 257), (129, 67)), 4, (3, 2)), (((3, 900), (1, 4000)), 8, (1, 1)), (((1, 6000), (2, 3000)), 8, (3, 1))]


@pytest.mark.parametrize("block,bits", [(16, 4.5), (32, 4.25)])
@pytest.mark.parametrize("grids,channels,mips", SIZES)
def test_latent_rows_are_small(native, grids, channels, mips, block, bits):
    """Bits a value, and what rows and scale tiles are padded to, at most 127 rows and 255 values: 15% covers it from 20,000
    values on."""
    import neural_textures_b200 as nt
    tex = nt.NeuralTexture(64, 64, grid_sizes=grids, latent_channels=channels, num_mips=mips, device="cpu")
    for g in range(2):
        rows, n = tex._mx4_rows(g), tex.grid_chains[g].numel()
        assert n >= 20000
        assert 8 * _bytes(native, rows, block) <= 1.15 * bits * n, (rows.shape, n)


def test_latent_rows_are_the_grids_memory(native):
    import neural_textures_b200 as nt
    tex = nt.NeuralTexture(64, 64, grid_sizes=((37, 21), (2, 9)), latent_channels=8, num_mips=(3, 1), device="cpu")
    for g in range(2):
        chain, rows = tex.grid_chains[g], tex._mx4_rows(g)
        chain.copy_(torch.arange(chain.numel()).half())
        flat = rows.reshape(-1)
        assert torch.equal(flat[:chain.numel()], chain) and not flat[chain.numel():].any()
        rows.zero_()
        assert not chain.any() and not tex.grids[g].any()


def test_latent_rows_of_a_replaced_chain(native):
    """A chain that another tensor took the place of has nothing behind it to fill a last row: refused."""
    import neural_textures_b200 as nt
    tex = nt.NeuralTexture(64, 64, grid_sizes=((37, 21), (2, 9)), latent_channels=8, num_mips=(3, 1), device="cpu")
    tex.grid_chains[0] = tex.grid_chains[0].clone()
    with pytest.raises(RuntimeError, match="replaced"):
        tex._mx4_rows(0)
