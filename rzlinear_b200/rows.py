"""Rows sorted by the block of the weight they belong to.  No counterpart in the reference, whose only layer is RzLinear."""
from __future__ import annotations

from typing import Tuple

import torch

from . import _lib


def _index_view(t: torch.Tensor, what: str) -> torch.Tensor:
    """Contiguous int64 indices."""
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what} must be int64 or int32, got {t.dtype}")
    return (t if t.dtype == torch.int64 else t.to(torch.int64)).contiguous()


def sort_rows(keys: torch.Tensor, num_bins: int) -> Tuple[torch.Tensor, torch.Tensor]:
    '''
        Stable counting sort of row keys, e.g. the expert of each row: what RzGroupedLinear needs to know.

        Args:
            keys (Tensor): (T), int64 or int32, on the GPU
            num_bins (int): keys are in [0, num_bins); 1 to 1024

        Returns:
            order (Tensor): (T) int32, row numbers by ascending key, equal keys by ascending row.  Rows whose key is outside
                [0, num_bins) (dropped or padding rows, say -1) come last
            offsets (Tensor): (num_bins + 1) int32; the rows of key b are order[offsets[b]:offsets[b + 1]]
    '''
    if keys.dim() != 1:
        raise ValueError(f"sort_rows takes a 1-D tensor of keys, got {keys.dim()} dimensions")
    num_bins = int(num_bins)
    if not 1 <= num_bins <= _lib.SORT_MAX_BINS:
        raise ValueError(f"num_bins must be 1 .. {_lib.SORT_MAX_BINS}, got {num_bins}")
    k = _index_view(keys.detach(), "keys")
    order = torch.empty(k.numel(), dtype=torch.int32, device=k.device)
    offsets = torch.empty(num_bins + 1, dtype=torch.int32, device=k.device)
    _lib.sort_rows(k, num_bins, order, offsets)
    return order, offsets
