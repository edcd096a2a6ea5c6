"""The RzGroupedLinear layer: one virtual, ROBE-Z-hashed weight for each group of rows (the experts of a layer).

No counterpart in the reference, whose only layer is RzLinear.  The groups' input_dim x output_dim weights stand one below the other
in one virtual matrix of the same definition as RzLinear's, every one beginning with a new tile row: group g's weight is that
of an RzLinear layer whose random numbers R[1] and R[4] are advanced by g * ceil(input_dim / block_size_k) times R[3] and R[7].
As there, products of bfloat16 activations on the tensor cores read the hashed array rounded to bfloat16; sums are float32.  Unlike
RzLinear's, the fused ReLU lets a NaN through (forward and backward, like torch.relu); RzLinear's turns it into 0.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.nn.parameter import Parameter

from .RzEmbedding import layer_config, layer_random_numbers
from .RzGroupedLinearFunction import RzGroupedLinearFunction


class RzGroupedLinear(torch.nn.Module):
    def __init__(self, num_groups: int, input_dim: int, output_dim: int, hashed_weight: Parameter = None, seed: int = 1024,
                 bias: bool = True, dtype: torch.dtype = torch.float32, compress_ratio: float = 0.0625, init_factor: float = 1.0, *,
                 block_size_k: int = 32, block_size_n: int = 64, hash_mode: str = 'two_level', prime: Optional[int] = None,
                 random_numbers: Optional[Sequence[int]] = None, relu: bool = False) -> None:
        '''
            num_groups linear layers of input_dim x output_dim over one compressed array.

                num_groups (int): weights (experts); 1 to 4096
                input_dim, output_dim (int): feature counts
                hashed_weight (Parameter): an existing compressed array to share with other layers; when given,
                    compress_ratio plays no part.  A new one is uniform in +-1 / sqrt(input_dim)
                bias (bool): whether the layer owns a (num_groups, output_dim) bias
                compress_ratio (float): length of a new array as a fraction of num_groups * input_dim * output_dim
                seed, dtype, init_factor, block_size_k, block_size_n, hash_mode, prime, random_numbers, relu: as in RzLinear
        '''
        super().__init__()
        assert 0 < input_dim < 10**5 and 0 < output_dim < 10**5
        if not 1 <= num_groups <= 4096:
            raise ValueError(f"num_groups must be 1 .. 4096, got {num_groups}")
        self._num_groups = num_groups
        self._input_dim = input_dim
        self._output_dim = output_dim
        self._seed = seed
        self._init_factor = init_factor
        self._config = layer_config(block_size_k, block_size_n, hash_mode, relu)
        self._random_numbers = layer_random_numbers(seed, prime, random_numbers)
        if hashed_weight is None:
            size = int(num_groups * input_dim * output_dim * compress_ratio)
            hashed_weight = Parameter((torch.rand(size) * 2 - 1).mul_(input_dim ** -0.5).to(dtype))
        self._hashed_weight = hashed_weight
        self._bias = Parameter(torch.zeros(num_groups, output_dim, dtype=dtype)) if bias else None

    def __repr__(self):
        return 'RzGroupedLinear(groups={} mm={}x{} bias={} seed={} hashed_weight_size={}, init_factor={})'.format(
            self._num_groups, self._input_dim, self._output_dim, self._bias is not None, self._seed, self._hashed_weight.size(),
            self._init_factor)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        '''
            x: (rows, input_dim), rows ordered by group -> (rows, output_dim)
            offsets: (num_groups + 1), int32 or int64 on the GPU, as sort_rows returns it: rows offsets[g] .. offsets[g + 1) are
                group g's.  Rows that belong to no group give zeros.
        '''
        if x.dim() != 2 or x.shape[1] != self._input_dim:
            raise ValueError(f"x must be (rows, {self._input_dim}), got {tuple(x.shape)}")
        if offsets.numel() != self._num_groups + 1:
            raise ValueError(f"offsets must have {self._num_groups + 1} entries, got {offsets.numel()}")
        return RzGroupedLinearFunction.apply(x, self._hashed_weight, self._random_numbers, offsets, self._output_dim,
                                             self._init_factor, self._config, self._bias)
