"""Recurrence module: a gated linear recurrence over the clouds of a sparse tensor."""

from __future__ import annotations

from mlx_lattice_b200.core import SparseTensor
from mlx_lattice_b200.nn._module import Module
from mlx_lattice_b200.ops import recurrence as F

__all__ = ['GatedRecurrence']


class GatedRecurrence(Module):
    def __init__(self, reverse: bool = False) -> None:
        self.reverse = reverse

    def __call__(self, x: SparseTensor, gate, *, initial_state=None, offsets=None, return_state: bool = False):
        return F.gated_recurrence(
            x, gate, initial_state=initial_state, offsets=offsets, reverse=self.reverse, return_state=return_state)
