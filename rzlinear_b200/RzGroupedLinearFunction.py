"""autograd glue of the RzGroupedLinear layer (host code only).  No counterpart in the reference, whose only layer is RzLinear."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .RzLinearFunction import DEFAULT_CONFIG, RzConfig, _compute_view, _unpack, controls
from .impl import launchers


def _offsets_view(offsets: torch.Tensor, rows: int) -> torch.Tensor:
    """Contiguous int32 row offsets."""
    if offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("offsets must be a 1-D tensor of num_groups + 1 row numbers")
    if offsets.dtype == torch.int64:
        return offsets.detach().clamp(0, rows).to(torch.int32)
    if offsets.dtype != torch.int32:
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    return offsets.detach().contiguous()


class RzGroupedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input: torch.Tensor, hashed_weight: torch.Tensor, random_numbers: torch.Tensor, offsets: torch.Tensor,
                output_dim, init_factor, config: Optional[RzConfig] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        '''
            Args:
                input (Tensor): (M, input_dim), rows ordered by group
                hashed_weight (Tensor): (H), the compressed weight of all groups
                random_numbers (Tensor): (8), R[0] the prime, on the CPU
                offsets (Tensor): (num_groups + 1), int32 or int64, on the GPU: rows offsets[g] .. offsets[g + 1) are group g's
                output_dim (int): N
                init_factor (float): scale applied to the product
                config (RzConfig): hash tile / hash mode / ReLU fusion (default: the reference's tile and hash)
                bias (Tensor): (num_groups, N), fused into the kernel epilogue when given

            Returns:
                output (Tensor): (M, output_dim).  Rows that belong to no group (before offsets[0], behind the last offset) are
                zeros and get no gradient.
        '''
        cfg = config if config is not None else DEFAULT_CONFIG
        if input.dim() != 2:
            raise ValueError(f"RzGroupedLinear takes (rows, input_dim) activations, got {input.dim()} dimensions")
        M, K, N, H = input.shape[0], input.shape[1], output_dim, hashed_weight.numel()
        off = _offsets_view(offsets, M)
        groups = off.numel() - 1
        if bias is not None and tuple(bias.shape) != (groups, N):
            raise ValueError(f"bias must have shape {(groups, N)}, got {tuple(bias.shape)}")
        x = _compute_view(input)
        hashed = launchers._hashed_f32(hashed_weight)
        pb = launchers.make_problem(max(1, M), K, N, H, _unpack(random_numbers), cfg.block_size_k, cfg.block_size_n, x.dtype,
                                    controls['triton_allow_tf32'], init_factor, cfg.hash_mode, _lib.FLAG_RELU if cfg.relu else 0)
        _lib._require_together(x, hashed, off, bias)
        copies = launchers.cached_shadow(pb, hashed_weight, hashed, _lib.grouped_copies_bytes(pb)) if M else None
        out = torch.empty((M, N), device=x.device, dtype=x.dtype)
        b = None if bias is None else bias.detach().float().contiguous()
        if M:
            _lib.grouped_forward(pb, groups, off, x, hashed, copies, b, out, _lib.grouped_workspace(pb, groups, x.device))

        # (the saved output keeps the compute dtype: the backward masks with it)
        ctx.save_for_backward(input, hashed_weight, off, out if cfg.relu else None)
        ctx.pb, ctx.groups, ctx.relu = pb, groups, cfg.relu
        ctx.copies = copies  # the backward reads the weights the forward saw
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out if out.dtype == input.dtype else out.to(input.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        input, hashed_weight, off, out = ctx.saved_tensors
        pb, groups = _lib.with_fields(ctx.pb, flags=0), ctx.groups
        M, K, N = input.shape[0], pb.K, pb.N
        input_grad = weight_grad = bias_grad = None
        x = _compute_view(input)
        grad = grad.to(x.dtype).contiguous()
        ws = _lib.grouped_workspace(pb, groups, x.device)
        # one pass over the incoming gradient: ReLU mask from the saved output and the bias gradients (column sums)
        want_bias = ctx.bias_dtype is not None and ctx.needs_input_grad[7]
        if ctx.relu or want_bias:
            masked = torch.empty_like(grad) if ctx.relu else None
            bias_grad = (torch.empty if M else torch.zeros)((groups, N), device=x.device, dtype=torch.float32) if want_bias else None
            if M:
                _lib.grouped_grad_prepare(pb, groups, off, grad, out if ctx.relu else None, masked, bias_grad, ws)
            if ctx.relu:
                grad = masked
            if want_bias:
                bias_grad = bias_grad.to(ctx.bias_dtype)
        if ctx.needs_input_grad[0]:
            input_grad = torch.empty((M, K), device=x.device, dtype=x.dtype)
            if M:
                _lib.grouped_backward_input(pb, groups, off, grad, launchers._hashed_f32(hashed_weight), ctx.copies, input_grad, ws)
            input_grad = input_grad.to(input.dtype)
        if ctx.needs_input_grad[1]:
            dh = torch.empty((pb.H,), device=x.device, dtype=torch.float32)
            if M:
                _lib.grouped_backward_weight(pb, groups, off, x, grad, dh, ws)   # zeroes dh first
            else:
                dh.zero_()
            weight_grad = dh.to(hashed_weight.dtype).view(hashed_weight.shape)
        return input_grad, weight_grad, None, None, None, None, None, bias_grad
