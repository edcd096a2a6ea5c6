"""autograd glue of the RzGroupedLinear layer (host code only).  No counterpart in the reference, whose only layer is RzLinear."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import _lib
from .RzLinearFunction import DEFAULT_CONFIG, RzConfig, _compute_view, controls
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


def _as(t, dtype, shape=None):
    """t in another dtype and shape, where it has others (None stays None)."""
    if t is None:
        return None
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if shape is None or t.shape == shape else t.view(shape)


def _operand(t):
    """t where the kernels can load it 16 bytes at a time; a view that begins elsewhere is copied."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _constant(*tensors) -> bool:
    """None of the tensors wants a gradient or carries a tangent (forward-mode derivatives are left to autograd, which refuses them)."""
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and ((grad and t.requires_grad) or unpack_dual(t).tangent is not None):
            return False
    return True


def _product(input, hashed_weight, random_numbers, offsets, output_dim, init_factor, config, bias):
    """(output in the compute dtype, int32 offsets, problem, groups, shifted copies): the forward pass and what the backward wants of it."""
    cfg = config if config is not None else DEFAULT_CONFIG
    if input.dim() != 2:
        raise ValueError(f"RzGroupedLinear takes (rows, input_dim) activations, got {input.dim()} dimensions")
    M, K, N, H = input.shape[0], input.shape[1], output_dim, hashed_weight.numel()
    off = _offsets_view(offsets, M)
    groups = off.numel() - 1
    if bias is not None and tuple(bias.shape) != (groups, N):
        raise ValueError(f"bias must have shape {(groups, N)}, got {tuple(bias.shape)}")
    x = _operand(_compute_view(input))
    hashed = launchers._hashed_f32(hashed_weight)
    pb = launchers.cached_problem(max(1, M), K, N, H, random_numbers, cfg.block_size_k, cfg.block_size_n, x.dtype,
                                  controls['triton_allow_tf32'], init_factor, cfg.hash_mode, _lib.FLAG_RELU if cfg.relu else 0)
    _lib._require_together(x, hashed, off, bias)
    copies_bytes, ws_bytes = _lib.grouped_sizes(pb, groups)
    copies = launchers.cached_shadow(pb, hashed_weight, hashed, copies_bytes) if M else None
    out = torch.empty((M, N), device=x.device, dtype=x.dtype)
    b = None if bias is None else bias.detach().float().contiguous()
    if M:
        _lib.grouped_forward(pb, groups, off, x, hashed, copies, b, out,
                             torch.empty(ws_bytes, dtype=torch.uint8, device=x.device))
    return out, off, pb, groups, copies


class RzGroupedLinearFunction(torch.autograd.Function):
    @classmethod
    def apply(cls, *args):
        # nothing to differentiate: the product alone, without the autograd machinery
        if _constant(args[0], args[1], *args[7:]):
            with torch.no_grad():
                out = _product(*args, *(None,) * (8 - len(args)))[0]
                return out if out.dtype == args[0].dtype else out.to(args[0].dtype)
        return super().apply(*args, *(None,) * (8 - len(args)))

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
        out, off, pb, groups, copies = _product(input, hashed_weight, random_numbers, offsets, output_dim, init_factor, config, bias)
        # (the saved output keeps the compute dtype: the backward masks with it)
        relu = bool(pb.flags & _lib.FLAG_RELU)
        if copies is not None:   # the backward reads the weights the forward saw; a longer buffer has a linear layer's workspace behind them
            copies = copies[:_lib.grouped_sizes(pb, groups)[0]]
        ctx.save_for_backward(input, hashed_weight, off, out if relu else None, copies)
        ctx.pb, ctx.groups, ctx.relu = pb, groups, relu
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out if out.dtype == input.dtype else out.to(input.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        input, hashed_weight, off, out, copies = ctx.saved_tensors
        pb, groups = ctx.pb, ctx.groups
        x = _operand(_compute_view(input))
        M, make = input.shape[0], torch.empty if input.shape[0] else torch.zeros
        grad = _operand(_as(grad, x.dtype).contiguous())
        dx = make((M, pb.K), device=x.device, dtype=x.dtype) if ctx.needs_input_grad[0] else None
        dh = make((pb.H,), device=x.device, dtype=torch.float32) if ctx.needs_input_grad[1] else None
        bias_grad = make((groups, pb.N), device=x.device, dtype=torch.float32) if ctx.needs_input_grad[7] else None
        if M:
            hashed = None if dx is None else launchers._hashed_f32(hashed_weight)
            _lib.grouped_backward(pb, groups, off, x, grad, out if ctx.relu else None, hashed, copies,
                                  torch.empty_like(grad) if ctx.relu else None, bias_grad, dx, dh,
                                  torch.empty(_lib.grouped_sizes(pb, groups)[1], dtype=torch.uint8, device=x.device))
        return (_as(dx, input.dtype), _as(dh, hashed_weight.dtype, hashed_weight.shape), None, None, None, None, None,
                _as(bias_grad, ctx.bias_dtype))
