"""Latents from a feature map: a network of TexelLayers whose output is a latent grid of a
NeuralTexture, trained through the texture's own training pass.

    enc = LatentEncoder(tex, grid=0, features=32)
    for _ in range(steps):
        enc.train_step(features)     # features [grid height][grid width][32]
    enc.encode(features)             # tex.grids[0] holds the latents

The training pass (InvokeTraining) leaves dL / dlatents in tex.ggrads; here it goes back through the
layers to their weights.  The other grid and the texture's network are optimised as always.  The encoded grid is
one of fp16 values without mips.
"""
from __future__ import annotations

from . import _native as N
from .api import InvokeOptimizeAll, InvokeTraining, NeuralTexture, _on_device
from .layers import TexelLayer


class LatentEncoder:
    def __init__(self, tex: NeuralTexture, grid: int = 0, features: int = 32, hidden: int = 64, groups: int = 8, block: int = 16,
                 lr: float = 2e-3, beta1: float = 0.9, beta2: float = 0.99, eps: float = 1e-8, seed: int = 0):
        import torch
        self.tex, self.grid, self.device = tex, grid, tex.device
        self._check()
        self.layers = [TexelLayer(features, hidden, groups=1, activation="none", block=block, device=tex.device, seed=seed),
                       TexelLayer(hidden, tex.C, groups=groups, activation="silu", block=block, device=tex.device, seed=seed + 1)]
        self.adam, self.step = (lr, beta1, beta2, eps), 0
        self.moments = [[(torch.zeros_like(p), torch.zeros_like(p)) for p in l.parameters] for l in self.layers]

    def _check(self):
        if self.tex.latent_format != N.NT_LATENT_GRID_F16:
            raise ValueError("a LatentEncoder fills fp16 grids, not block records")
        if self.tex.num_mips[self.grid] > 1:
            raise ValueError(f"a LatentEncoder fills grids of one level, not of {self.tex.num_mips[self.grid]}")

    @_on_device
    def encode(self, features, keep: bool = False):
        """Latents of `features` [h][w][F] (fp16), written into the texture's grid on torch's current stream."""
        self._check()
        x = features
        for layer in self.layers:
            x = layer.forward(x, keep)
        grid = self.tex.grids[self.grid]
        if x.shape != grid.shape:
            raise ValueError(f"features give a grid of {tuple(x.shape)}, the texture's is {tuple(grid.shape)}")
        grid.copy_(x)
        return grid

    @_on_device
    def train_step(self, features) -> None:
        """One step: latents from the features, the texture's training pass, gradients back through the layers,
        Adam on them, on the texture's network and on its other grid.  The loss is added to tex.loss_accum.
        Everything is queued on torch's current stream."""
        import torch
        tex = self.tex
        stream = torch.cuda.current_stream(self.device).cuda_stream
        self.encode(features, keep=True)
        p = tex.params()
        InvokeTraining(p, stream=stream)
        # a latent's gradient is its error over the number of samples, or of latents where they are fewer: times that
        # (a power of two) between the layers, where fp16 would lose it
        w, h = tex.grid_sizes[self.grid]
        d, scale = tex.ggrads[self.grid], 1.0
        gain = 2.0 ** (min(p.num_samples, w * h).bit_length() - 1)
        for layer in reversed(self.layers):
            d = layer.backward(d, scale, gain)
            scale, gain = scale * gain, 1.0
        self._optimize()
        tex.ggrads[self.grid].zero_()  # Adam leaves values without a gradient alone
        InvokeOptimizeAll(p, stream=stream)
        tex.step += 1

    def _optimize(self):
        lr, beta1, beta2, eps = self.adam
        self.step += 1
        for layer, moments in zip(self.layers, self.moments):
            for p, g, (m, v) in zip(layer.parameters, layer.grads, moments):
                m.lerp_(g, 1 - beta1)
                v.lerp_(g * g, 1 - beta2)
                p.addcdiv_(m, (v / (1 - beta2 ** self.step)).sqrt_().add_(eps), value=-lr / (1 - beta1 ** self.step))
            layer.pack()
