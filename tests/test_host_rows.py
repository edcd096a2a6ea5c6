"""Refusals and host logic of the operators that pick rows by an index (no GPU needed)."""
import ctypes

import pytest
import torch

import rzlinear_b200 as rz

LARGE_PRIME = 2038074743


def _pb(rzlib, M=64, K=1000, N=192, H=8192, BK=32, BN=64, io=0, prec=0, **kw):
    return rzlib.make_problem(M, K, N, H, BK, BN, kw.pop("R", [LARGE_PRIME, 5, 7, 11, 13, 17, 19, 23]), kw.pop("mode", 0), io, prec, **kw)


def test_sort_rows_refusals(rzlib):
    lib = rzlib.load()
    some = ctypes.c_void_p(1 << 20)
    assert lib.rz_sort_rows(some, -1, 4, some, some, None, 0, None) == -2
    assert lib.rz_sort_rows(some, 1 << 31, 4, some, some, None, 0, None) == -2
    assert lib.rz_sort_rows(some, 4, 0, some, some, None, 0, None) == -2
    assert lib.rz_sort_rows(some, 4, 1025, some, some, None, 0, None) == -10
    assert lib.rz_sort_rows(None, 4, 4, some, some, None, 0, None) == -1
    assert lib.rz_sort_rows(some, 4, 4, some, None, None, 0, None) == -1
    assert lib.rz_sort_rows(some, 5000, 4, some, some, None, 0, None) == -1            # needs scratch
    need = lib.rz_sort_rows_scratch_bytes(5000, 4)
    assert need == 3 * 5 * 4
    assert lib.rz_sort_rows(some, 5000, 4, some, some, some, need - 1, None) == -11
    assert lib.rz_sort_rows(ctypes.c_void_p((1 << 20) + 4), 4, 4, some, some, None, 0, None) == -5
    assert lib.rz_sort_rows_scratch_bytes(2048, 1024) == 0 and lib.rz_sort_rows_scratch_bytes(1 << 30, 1024) == 148 * 1025 * 4
    with pytest.raises(ValueError):
        rz.sort_rows(torch.zeros(4, dtype=torch.int64), 0)
    with pytest.raises(ValueError):
        rz.sort_rows(torch.zeros(4, dtype=torch.int64), 1025)
    with pytest.raises(ValueError):
        rz.sort_rows(torch.zeros((2, 2), dtype=torch.int64), 4)
    with pytest.raises(TypeError):
        rz.sort_rows(torch.zeros(4), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        rz.sort_rows(torch.zeros(4, dtype=torch.int64), 4)


def test_embedding_refusals(rzlib):
    lib = rzlib.load()
    some = ctypes.c_void_p(1 << 20)
    pb = _pb(rzlib)
    ref = ctypes.byref
    assert lib.rz_embedding_forward(ref(pb), None, -1, some, some, None) == -1
    assert lib.rz_embedding_forward(ref(pb), some, -1, some, None, None) == -1
    assert lib.rz_embedding_forward(ref(pb), ctypes.c_void_p((1 << 20) + 4), -1, some, some, None) == -5
    assert lib.rz_embedding_forward(ref(_pb(rzlib, H=2048)), some, -1, some, some, None) == -3
    assert lib.rz_embedding_forward(ref(_pb(rzlib, K=0)), some, -1, some, some, None) == -2
    assert lib.rz_embedding_forward(ref(_pb(rzlib, io=1, prec=1)), some, -1, some, some, None) == -4
    assert lib.rz_embedding_scratch_bytes(ref(_pb(rzlib, M=256))) == 0
    big = _pb(rzlib, M=257)
    need = lib.rz_embedding_scratch_bytes(ref(big))
    assert need == 257 * 8
    assert lib.rz_embedding_backward(ref(big), some, -1, some, some, None, 0, None) == -1
    assert lib.rz_embedding_backward(ref(big), some, -1, some, some, some, need - 1, None) == -11
    assert lib.rz_embedding_backward(ref(pb), some, -1, some, None, None, 0, None) == -1

    layer = rz.RzEmbedding(1000, 64)
    assert layer._hashed_weight.shape == (4000,) and set(dict(layer.named_parameters())) == {"_hashed_weight"}
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        layer(torch.zeros(4))
    with pytest.raises(AssertionError):
        rz.RzEmbedding(100, 16)(torch.zeros(4, dtype=torch.int64))     # H = 100 <= 32 * 64
    for bad in (1000, -1001):
        with pytest.raises(ValueError):
            rz.RzEmbedding(1000, 64, padding_idx=bad)
    with pytest.raises(ValueError):
        rz.RzEmbedding(1000, 64, hash_mode="other")
    with pytest.raises(ValueError):
        rz.RzEmbeddingFunction.apply(torch.zeros(4, dtype=torch.int64), layer._hashed_weight, layer._random_numbers, 1000, 64, 1.0,
                                     rz.RzConfig(relu=True))
    with pytest.raises(TypeError):
        rz.RzEmbeddingFunction.apply(torch.zeros(4, dtype=torch.int64), layer._hashed_weight, layer._random_numbers, 1000, 64, 1.0,
                                     None, None, torch.int32)


def test_embedding_draws_the_linear_layers_numbers_without_reseeding():
    torch.manual_seed(7)
    want = torch.rand(3)
    torch.manual_seed(7)
    emb = rz.RzEmbedding(1000, 64, hashed_weight=torch.nn.Parameter(torch.zeros(4000)), seed=31)
    assert torch.equal(torch.rand(3), want)
    assert torch.equal(emb._random_numbers, rz.RzLinear(64, 64, seed=31)._random_numbers)
    assert emb._random_numbers.dtype == torch.int32
