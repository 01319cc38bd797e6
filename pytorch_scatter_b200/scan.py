"""Gated linear recurrence along the segments of a CSR ``indptr``: the running form of ``segment_csr``.

``h[e] = gate[e] * h[e-1] + src[e]`` inside each segment.  Not part of upstream's operator set.
"""
from typing import Optional, Tuple

import torch


def scan_csr(src: torch.Tensor, gate: torch.Tensor, indptr: torch.Tensor,
             state: Optional[torch.Tensor] = None) -> torch.Tensor:
    r"""All ``h`` of ``h[e] = gate[e] * h[e-1] + src[e]`` along the ranges ``[indptr[i], indptr[i+1])`` of dimension
    ``indptr.dim() - 1``; before a range's first row ``h`` is ``state[i]``, or 0.

    Args:
        src: float32, float64, float16 or bfloat16 (CUDA).
        gate: of ``src``'s shape, or 1 in trailing dimensions whose channels share a gate (``[T, heads, 1]`` against
            ``[T, heads, width]``); any other broadcast is expanded.  ``src``'s dtype, or float32 with 16-bit data.
            Products of gates over a few hundred rows have to be finite: meant for magnitudes up to 1.
        indptr: ascending int64 offsets, those beyond the rows ending at them; leading dimensions broadcast against
            ``src``'s.
        state: optional start of each range, ``src``'s shape with one row for each range, float32 (float64 with
            float64 data).

    The recurrence runs in 32 bits (64 for float64) whatever the data's type and is rounded once per output.  Rows
    outside every range are 0 and get no gradient.  With 16-bit data a forward pass that will need the gates' gradient
    keeps ``h`` in float32 as well.  Differentiable (once, in reverse mode) with respect to ``src``, ``gate`` and
    ``state``; bit-reproducible run to run.
    """
    return torch.ops.torch_scatter.scan_csr(src, gate, indptr, state)


def scan_csr_state(src: torch.Tensor, gate: torch.Tensor, indptr: torch.Tensor,
                   state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    r""":func:`scan_csr` that also returns the state after each range's last row, in ``state``'s shape and type (the
    state itself, or 0, for empty ranges): what the next piece of the sequences goes on from."""
    return torch.ops.torch_scatter.scan_csr_state(src, gate, indptr, state)


def scan_step(src: torch.Tensor, gate: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    r"""One token for each of ``n`` running sequences: ``state[i] = gate[i] * state[i] + src[i]`` in place.

    Args:
        src: ``[n, ...]``, one row for each state.
        gate: as in :func:`scan_csr`.
        state: of ``src``'s shape, float32 (float64 with float64 data); each state contiguous, the states possibly apart
            (a slice of a pool).  Must not require a gradient: this is the serving form.  ``src`` and ``gate`` may be the
            state itself, but not overlap it in part.

    Returns the new state rounded to ``src``'s dtype.
    """
    return torch.ops.torch_scatter.scan_step(src, gate, state)
