"""autograd glue of the RzEmbedding layer (host code only).  No counterpart in the reference, whose only layer is RzLinear."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .RzLinearFunction import DEFAULT_CONFIG, RzConfig
from .impl import launchers
from .RzGroupedLinearFunction import _as, _constant
from .rows import _index_view


def _lookup(ids, hashed_weight, random_numbers, num_embeddings, embedding_dim, init_factor, config, padding_idx, out_dtype,
            gradient):
    """(rows, int64 ids, problem, padding row or -1, plan): the forward pass and what the backward wants of it."""
    cfg = config if config is not None else DEFAULT_CONFIG
    if cfg.relu:
        raise ValueError("RzEmbedding has no ReLU")
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx) + (num_embeddings if padding_idx < 0 else 0)
        if not 0 <= padding < num_embeddings:
            raise ValueError(f"padding_idx {padding_idx} is outside the {num_embeddings} rows")
    dtype = out_dtype if out_dtype is not None else hashed_weight.dtype
    if not dtype.is_floating_point:
        raise TypeError(f"RzEmbedding gives floating-point rows, not {dtype}")
    index = _index_view(ids, "ids")
    hashed = launchers._hashed_f32(hashed_weight)
    # float32 and bfloat16 are written by the kernel; other types are computed in float32 and cast
    compute = dtype if dtype in (torch.float32, torch.bfloat16) else torch.float32
    tokens = index.numel()
    pb = launchers.cached_problem(max(1, tokens), num_embeddings, embedding_dim, hashed.numel(), random_numbers, cfg.block_size_k,
                                  cfg.block_size_n, compute, False, init_factor, cfg.hash_mode)
    _lib._require_together(index, hashed)
    out = torch.empty((*ids.shape, embedding_dim), device=index.device, dtype=compute)
    plan = None
    if tokens:
        plan = _lib.embedding_plan(pb, index.device) if gradient else None
        _lib.embedding_forward(pb, index, padding, hashed, out, plan)
    return (out if compute == dtype else out.to(dtype)), index, pb, padding, plan


class RzEmbeddingFunction(torch.autograd.Function):
    @classmethod
    def apply(cls, *args):
        # nothing to differentiate: the lookup alone, without the autograd machinery (most of a short lookup's time)
        if _constant(args[1]):
            with torch.no_grad():
                return _lookup(*args, *(None,) * (9 - len(args)), False)[0]
        return super().apply(*args, *(None,) * (9 - len(args)))

    @staticmethod
    def forward(ctx, ids: torch.Tensor, hashed_weight: torch.Tensor, random_numbers: torch.Tensor, num_embeddings,
                embedding_dim, init_factor, config: Optional[RzConfig] = None, padding_idx: Optional[int] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        '''
            Args:
                ids (Tensor): any shape, int64 or int32: rows of the virtual num_embeddings x embedding_dim table
                hashed_weight (Tensor): (H), the compressed weight
                random_numbers (Tensor): (8), R[0] the prime, on the CPU
                num_embeddings (int): rows of the table
                embedding_dim (int): entries of a row
                init_factor (float): scale applied to the looked-up rows
                config (RzConfig): hash tile / hash mode (default: the reference's tile and hash)
                padding_idx (int): a row that reads as zeros and gets no gradient; negative counts from the end
                out_dtype (dtype): of the result (default: the hashed weight's)

            Returns:
                output (Tensor): ids.shape + (embedding_dim).  An id outside [0, num_embeddings) gives zeros and no gradient.
        '''
        out, index, pb, padding, plan = _lookup(ids, hashed_weight, random_numbers, num_embeddings, embedding_dim, init_factor,
                                                config, padding_idx, out_dtype, ctx.needs_input_grad[1])
        ctx.save_for_backward(index, plan)
        ctx.pb, ctx.padding = pb, padding
        ctx.weight_shape, ctx.weight_dtype = hashed_weight.shape, hashed_weight.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, plan = ctx.saved_tensors
        weight_grad = None
        if ctx.needs_input_grad[1]:
            grad = _as(grad, torch.bfloat16 if ctx.pb.io_dtype == _lib.BF16 else torch.float32).contiguous()
            dh = torch.empty((ctx.pb.H,), device=index.device, dtype=torch.float32)
            if index.numel():
                _lib.embedding_backward(ctx.pb, index, ctx.padding, grad, dh, plan)   # zeroes dh first
            else:
                dh.zero_()
            weight_grad = _as(dh, ctx.weight_dtype, ctx.weight_shape)
        return None, weight_grad, None, None, None, None, None, None, None
