"""Modules over the learned-code operators: what a conditioned radiance field has beside the fixed encoders.

A latent code per view (or per object, per frame) is looked up by ``Embedding``, normalised by ``LayerNorm``, regularised by
``Dropout`` and concatenated to the encoded view direction; NeRF's kernels return the gradient of that input, so the codes
train with the networks, also under ``optim.FusedAdam``.  Parameters are named and initialised like torch.nn's modules of the
same names, so their state_dicts are interchangeable.  There is no CPU fallback: the modules raise for tensors off the GPU
(a Dropout that drops nothing launches nothing, and takes any).
"""
import itertools
from typing import Optional

import torch
from torch import nn

from . import ops
from .shard import _mix_int

__all__ = ["Embedding", "LayerNorm", "Dropout"]


class Embedding(nn.Module):
    """scale * weight[ids].  Row `padding_idx` starts at 0 and gets no gradient.  (The third argument is the scale;
    torch.nn.Embedding's is padding_idx.)"""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx: Optional[int] = None,
                 device=None, dtype=None):
        super().__init__()
        if padding_idx is not None and not 0 <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx {padding_idx} is not one of {num_embeddings} rows")
        self.scale, self.padding_idx = float(scale), padding_idx
        self.weight = nn.Parameter(torch.empty((num_embeddings, embedding_dim), device=device, dtype=dtype))
        nn.init.normal_(self.weight)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return ops.EmbeddingFunction.apply(self.weight, ids, self.scale, self.padding_idx)


class LayerNorm(nn.Module):
    """Layer norm over the last axis, of `dim` values."""

    def __init__(self, dim: int, eps: float = 1e-5, affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = int(dim), float(eps)
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.dim:
            raise ValueError(f"Expected rows of {self.dim} values. Got {x.shape[-1]}.")
        return ops.LayerNormFunction.apply(x, self.weight, self.bias, self.eps)


_unseeded = itertools.count()            # Dropout modules made without a seed in this process


class Dropout(nn.Module):
    """Counter-based dropout.  The n-th call in training mode uses key(seed, n).  Modules of one seed drop the same elements, so
    each has its own: without `seed`, one that follows from how many modules were made without one before, the same on
    every rank that builds its model in the same order (a rank passes the flat index of its first element as `first`); a
    program whose ranks or runs build differently names its seeds.  A copy of a module keeps its seed.

    Inside a graph capture the count would be frozen into the graph: pass a key tensor there.  A forward that is run again for
    its gradient (activation checkpointing) would count twice and draw another mask: pass a key there, too.  The count
    (`calls`) is not part of the state_dict, whose keys are torch.nn.Dropout's (none): a resumed run sets it."""

    def __init__(self, p: float = 0.5, seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p must be in [0, 1], got {p}")
        # (mixed, so that it is not one of the small numbers that a program would name)
        self.seed = _mix_int(next(_unseeded) ^ 0x5851F42D4C957F2D) if seed is None else int(seed)
        self.p, self.calls = float(p), 0

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, first: int = 0, key=None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            if residual is None:
                return x
            return x + ops._like(residual, "residual", x, "x")
        if key is None:
            if x.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Dropout inside a graph capture needs a key tensor: its own key would never change")
            key = _mix_int((self.seed * 0x9E3779B97F4A7C15 + self.calls) ^ 0xD6E8FEB86659FD93)
            self.calls += 1
        return ops.DropoutFunction.apply(x, self.p, key, first, residual)
