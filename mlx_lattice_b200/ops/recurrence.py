"""Gated linear recurrence along the rows of a sparse tensor (a sequence per cloud of the
batch, in row order). No counterpart in the reference."""

from __future__ import annotations

import torch

from mlx_lattice_b200 import _ext
from mlx_lattice_b200.core import SparseTensor

__all__ = ['gated_recurrence', 'gated_recurrence_step', 'sequence_offsets']


def sequence_offsets(x: SparseTensor) -> torch.Tensor:
    """The int32 row offsets of the clouds of ``x`` on its device, from ``batch_counts``: one
    entry per cloud and one more. Copies from the host: make them once, outside a capture."""
    if x.batch_counts is None:
        raise ValueError('batch_counts metadata is required for a recurrence without offsets.')
    offsets = [0]
    for count in x.batch_counts:
        offsets.append(offsets[-1] + count)
    return torch.tensor(offsets, dtype=torch.int32, device=x.feats.device)


def gated_recurrence(
    x: SparseTensor, gate, *, initial_state: torch.Tensor | None = None,
    offsets: torch.Tensor | None = None, reverse: bool = False, return_state: bool = False,
):
    """``h_t = a_t h_{t-1} + (1 - a_t) x_t`` with ``a = sigmoid(gate)``, per channel over the
    rows of each sequence; ``reverse`` runs from a sequence's last row to its first.

    ``gate`` is a tensor like ``x.feats``, or a ``SparseTensor`` over the same coordinates; both
    may be column ranges of a wider array. ``offsets`` (int32, rising, sequence ``j`` holds the
    rows ``offsets[j]`` to ``offsets[j + 1] - 1``) defaults to ``sequence_offsets(x)``; rows
    outside all sequences give zeros. ``initial_state`` is float32 ``(sequences, C)``, zero by
    default. Returns the sparse tensor of ``h``, and with ``return_state`` also the float32
    state after every sequence. Differentiable in ``x.feats``, ``gate`` and ``initial_state``."""
    gate = _gate(x, gate)
    if offsets is None:
        offsets = sequence_offsets(x)
    h, final = _ext.recurrence(x.feats, gate, offsets, initial_state, reverse, want_state=return_state)
    h = x.replace(feats=h)
    return (h, final) if return_state else h


def gated_recurrence_step(
    x: SparseTensor, gate, state: torch.Tensor, *, out_state: torch.Tensor | None = None,
) -> tuple[SparseTensor, torch.Tensor]:
    """One new row for each of ``N`` streams: row ``i`` of ``x`` and ``gate`` advances row ``i``
    of the float32 ``state``. Returns the sparse tensor of the new ``h`` and the next state,
    written to ``out_state`` when given (which may be ``state``). For serving: it has no gradient, and
    results that depend on something with one raise when they are differentiated."""
    h, state = _ext.recurrence_step(x.feats, _gate(x, gate), state, out_state)
    return x.replace(feats=h), state


def _gate(x: SparseTensor, gate) -> torch.Tensor:
    if isinstance(gate, SparseTensor):
        if not gate.same_coords(x):
            raise ValueError('gate must share the coordinates of x.')
        return gate.feats
    return gate
