"""Tokens to experts and back: a router's choice, the sort of tokens by expert, the rows' way there and back.

    weight, index = expert_topk(logits, k)
    slot, order, indptr = expert_sort(index, num_experts)
    rows = expert_dispatch(x, slot, indptr)         # rows of expert e: rows[indptr[e]:indptr[e + 1]], in token order
    y = ...                                         # the experts; segment_csr and scan_csr take the same indptr
    out = expert_combine(y, slot, indptr, weight)

No host synchronisation anywhere: the buffer of rows always holds ``slot.numel()`` rows, those of dropped entries behind
``indptr[-1]``.  Not part of upstream's operator set.
"""
from typing import Optional, Tuple

import torch


def expert_topk(logits: torch.Tensor, k: int, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""The ``k`` experts with the largest logits of each token, and their softmax weights.

    Args:
        logits: ``[..., experts]`` float32, float16 or bfloat16 (CUDA), up to 1024 experts.
        k: experts per token.
        normalize: divide the weights of a token by their sum (a softmax over the chosen experts alone); otherwise
            they are the softmax over all experts.

    Returns ``(weight, index)``, both ``[..., k]``, float32 and int64, in descending order of the logits, ties towards
    the smaller index.  A logit of ``-inf`` is never chosen: where fewer than ``k`` others are left the index is -1 (an
    entry that :func:`expert_sort` drops) and the weight 0.  NaN ranks above everything and makes the token's weights
    NaN.  ``weight`` is differentiable with respect to ``logits`` (once, in reverse mode).
    """
    return torch.ops.torch_scatter.expert_topk(logits, k, normalize)


def expert_sort(index: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    r"""Sort the entries of ``index`` by expert, stably: the order inside an expert is that of the entries.

    Args:
        index: int64 expert of every entry, usually ``[..., k]`` (CUDA); values outside ``[0, num_experts)`` drop the
            entry.
        num_experts: number of experts, up to 4096.

    Returns ``(slot, order, indptr)``, all int64: ``slot`` (of ``index``'s shape) is each entry's place among the sorted
    ones, -1 for dropped entries; ``order`` is the flat entry at each place, dropped ones last; expert ``e`` owns the
    places ``[indptr[e], indptr[e+1])``.
    """
    return torch.ops.torch_scatter.expert_sort(index, num_experts)


def expert_dispatch(src: torch.Tensor, slot: torch.Tensor, indptr: torch.Tensor,
                    weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    r"""Copy each token's row to the places of its ``k`` entries: ``rows[slot[t, j]] = src[t] (* weight[t, j])``.

    Args:
        src: ``[*tokens, ...]`` float32, float64, float16 or bfloat16 (CUDA).
        slot, indptr: as :func:`expert_sort` returned them, ``slot`` ``[*tokens, k]``.  Entries may be dropped afterwards
            by a slot of -1; two entries must not share a slot.
        weight: optional factors of ``slot``'s shape, float32 (float64 with float64 rows).

    Returns ``[slot.numel(), ...]``; rows that no entry names, those behind ``indptr[-1]`` among them, are zero.
    Differentiable (once, in reverse mode) with respect to ``src`` and ``weight``; bit-reproducible run to run.
    """
    return torch.ops.torch_scatter.expert_dispatch(src, slot, indptr, weight)


def expert_combine(rows: torch.Tensor, slot: torch.Tensor, indptr: torch.Tensor,
                   weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    r"""Sum each token's rows: ``out[t] = sum_j rows[slot[t, j]] (* weight[t, j])``, in the order of ``j`` and in 32 bits.

    Args:
        rows: ``[slot.numel(), ...]`` float32, float64, float16 or bfloat16 (CUDA); rows behind ``indptr[-1]`` are not
            read.
        slot, indptr: as :func:`expert_sort` returned them, ``slot`` ``[*tokens, k]``.  Entries may be dropped afterwards
            by a slot of -1 (their rows get a gradient of zero); two entries must not share a slot.
        weight: optional factors of ``slot``'s shape, float32 (float64 with float64 rows).

    Returns ``[*tokens, ...]``; tokens whose entries were all dropped are zero.  Differentiable (once, in
    reverse mode) with respect to ``rows`` and ``weight``; bit-reproducible run to run.
    """
    return torch.ops.torch_scatter.expert_combine(rows, slot, indptr, weight)
