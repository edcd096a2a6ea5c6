"""The RzEmbedding layer: an embedding table whose rows are slices of a ROBE-Z-hashed array.

No counterpart in the reference, whose only layer is RzLinear; the virtual table is defined exactly as RzLinear's virtual
weight (tile hash, random numbers, init_factor), so a table and a linear layer of the same sizes and random numbers share W.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.nn.parameter import Parameter

from . import _lib
from .RzEmbeddingFunction import RzEmbeddingFunction
from .RzLinear import RzLinear
from .RzLinearFunction import RzConfig


def draw_random_numbers(seed: int, prime: int) -> torch.Tensor:
    """The numbers RzLinear draws for this seed and prime, without touching torch's global generator."""
    x = torch.randint(0, prime, (RzLinear.R - 1,), generator=torch.Generator().manual_seed(seed)).type(torch.int32)
    return torch.cat([torch.tensor([prime], dtype=torch.int32), x])


def layer_random_numbers(seed: int, prime: Optional[int], random_numbers: Optional[Sequence[int]]) -> torch.Tensor:
    """Random numbers of a layer, always on the CPU: the ones given, else drawn from the seed."""
    if random_numbers is None:
        return draw_random_numbers(seed, int(prime) if prime is not None else RzLinear.P)
    rn = [int(v) for v in random_numbers]
    assert len(rn) == RzLinear.R
    return torch.tensor(rn, dtype=torch.int64)


def layer_config(block_size_k: int, block_size_n: int, hash_mode: str, relu: bool = False) -> RzConfig:
    if hash_mode not in ('two_level', 'single'):
        raise ValueError("hash_mode must be 'two_level' or 'single'")
    return RzConfig(block_size_k=int(block_size_k), block_size_n=int(block_size_n),
                    hash_mode=_lib.HASH_TWO_LEVEL if hash_mode == 'two_level' else _lib.HASH_SINGLE, relu=bool(relu))


class RzEmbedding(torch.nn.Module):
    def __init__(self, num_embeddings: int, embedding_dim: int, hashed_weight: Parameter = None, seed: int = 1024,
                 dtype: torch.dtype = torch.float32, compress_ratio: float = 0.0625, init_factor: float = 1.0, *,
                 padding_idx: Optional[int] = None, out_dtype: Optional[torch.dtype] = None,
                 block_size_k: int = 32, block_size_n: int = 64, hash_mode: str = 'two_level',
                 prime: Optional[int] = None, random_numbers: Optional[Sequence[int]] = None) -> None:
        '''
            Embedding table of num_embeddings x embedding_dim virtual entries.

                num_embeddings, embedding_dim (int): rows of the table, entries of a row
                hashed_weight (Parameter): an existing compressed array to share with other layers; when given,
                    compress_ratio plays no part.  A new one is drawn from a normal distribution
                seed, dtype, compress_ratio, init_factor: as in RzLinear; init_factor scales the looked-up rows
                padding_idx (int): a row that reads as zeros and gets no gradient (its virtual entries are shared with
                    other rows, so they cannot be zeroed in place)
                out_dtype (dtype): of the looked-up rows (default: the hashed weight's), e.g. torch.bfloat16 activations
                    from a float32 hashed weight
                block_size_k, block_size_n, hash_mode, prime, random_numbers: as in RzLinear
        '''
        super().__init__()
        assert 0 < num_embeddings < 2**31 and 0 < embedding_dim < 2**31
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx {padding_idx} is outside the {num_embeddings} rows")
        self._num_embeddings = num_embeddings
        self._embedding_dim = embedding_dim
        self._seed = seed
        self._init_factor = init_factor
        self._padding_idx = padding_idx
        self._out_dtype = out_dtype
        self._config = layer_config(block_size_k, block_size_n, hash_mode)
        self._random_numbers = layer_random_numbers(seed, prime, random_numbers)
        if hashed_weight is None:
            hashed_weight = Parameter(torch.randn(int(num_embeddings * embedding_dim * compress_ratio), dtype=dtype))
        self._hashed_weight = hashed_weight

    def __repr__(self):
        return 'RzEmbedding(mm={}x{} seed={} hashed_weight_size={}, init_factor={} padding_idx={})'.format(
            self._num_embeddings, self._embedding_dim, self._seed, self._hashed_weight.size(), self._init_factor, self._padding_idx)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        '''
            ids: (...), int64 or int32 -> (..., embedding_dim).  An id outside the table gives zeros and no gradient.
        '''
        return RzEmbeddingFunction.apply(ids, self._hashed_weight, self._random_numbers, self._num_embeddings,
                                         self._embedding_dim, self._init_factor, self._config, self._padding_idx, self._out_dtype)
