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
    def fwd(pb=pb, ids=some, h=some, out=some, plan=None, pbytes=0):
        return lib.rz_embedding_forward(ref(pb), ids, -1, h, out, plan, pbytes, None)

    assert fwd(ids=None) == -1 and fwd(h=None) == -1 and fwd(out=None) == -1
    assert fwd(ids=ctypes.c_void_p((1 << 20) + 4)) == -5 and fwd(out=ctypes.c_void_p((1 << 20) + 2)) == -5
    assert fwd(pb=_pb(rzlib, H=2048)) == -3 and fwd(pb=_pb(rzlib, K=0)) == -2 and fwd(pb=_pb(rzlib, io=1, prec=1)) == -4
    assert lib.rz_embedding_plan_bytes(ref(_pb(rzlib, M=256, N=1 << 20))) == 0            # too few tokens, too few words: not sorted
    assert lib.rz_embedding_plan_bytes(ref(_pb(rzlib, M=1 << 12, N=1 << 10))) == 0
    big = _pb(rzlib, M=1 << 12, N=1025)
    need = lib.rz_embedding_plan_bytes(ref(big))
    assert need == 4096 * 8 and fwd(pb=big, plan=some, pbytes=need - 1) == -11
    assert fwd(pb=big, plan=ctypes.c_void_p((1 << 20) + 2), pbytes=need) == -5
    assert lib.rz_embedding_backward(ref(big), some, -1, some, some, some, need - 1, None) == -11
    assert lib.rz_embedding_backward(ref(pb), some, -1, some, None, None, 0, None) == -1
    assert lib.rz_embedding_backward(ref(pb), some, -1, None, some, None, 0, None) == -1

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


def test_grouped_refusals(rzlib):
    lib = rzlib.load()
    some, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    ref = ctypes.byref
    pb = _pb(rzlib, M=100, K=128, N=192, H=8192, BK=32, BN=64, io=1, prec=2)
    assert rzlib.plan(pb, 0) == rzlib.PATH_TCGEN05
    copies, ws = lib.rz_grouped_copies_bytes(ref(pb)), lib.rz_grouped_workspace_bytes(ref(pb), 4)
    assert copies == 8 * 8192 * 2 and ws > 0 and ws % 256 == 0
    assert lib.rz_grouped_copies_bytes(ref(_pb(rzlib, BK=16))) == 0

    def fwd(pb=pb, groups=4, off=some, x=some, h=some, c=some, cb=copies, y=some, w=some, wb=ws):
        return lib.rz_grouped_forward(ref(pb), groups, off, x, h, c, cb, None, y, w, wb, None)

    assert fwd(groups=0) == -2 and fwd(groups=-1) == -2 and fwd(groups=4097) == -10
    assert fwd(pb=_pb(rzlib, K=1 << 20, BK=32, BN=64), groups=2048) == -2              # stacked rows pass 2^31
    assert fwd(off=None) == -1 and fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(c=None) == -1 and fwd(w=None) == -1
    assert fwd(cb=copies - 1) == -11 and fwd(wb=ws - 1) == -11
    assert fwd(x=odd) == -5 and fwd(y=odd) == -5 and fwd(w=odd) == -5 and fwd(off=ctypes.c_void_p((1 << 20) + 2)) == -5

    half = ctypes.c_void_p((1 << 20) + 2)                                               # bias and hashed array: whole floats
    assert fwd(h=half) == -5
    assert lib.rz_grouped_forward(ref(pb), 4, some, some, some, some, copies, half, some, some, ws, None) == -5

    def bwd(x=some, dy=some, y=None, h=some, c=some, dym=None, db=None, dx=some, dh=some, w=some, wb=ws):
        return lib.rz_grouped_backward(ref(pb), 4, some, x, dy, y, h, c, copies, dym, db, dx, dh, w, wb, None)

    assert bwd(dy=None) == -1 and bwd(x=None) == -1 and bwd(c=None) == -1 and bwd(dx=None, dh=None) == -1 and bwd(w=None) == -1
    assert bwd(y=some) == -1                                                            # a mask, and nowhere to put the masked gradient
    assert bwd(wb=ws - 1) == -11 and bwd(dy=odd) == -5 and bwd(x=odd) == -5 and bwd(dx=odd) == -5 and bwd(y=some, dym=odd) == -5
    assert bwd(h=half) == -5 and bwd(db=half) == -5 and bwd(dh=half) == -5

    layer = rz.RzGroupedLinear(4, 128, 64)
    assert layer._hashed_weight.shape == (2048,) and layer._bias.shape == (4, 64)
    off, x = torch.zeros(5, dtype=torch.int32), torch.randn(6, 128)
    with pytest.raises(AssertionError):
        layer(x, off)                                                                   # H = 2048 <= 32 * 64
    layer = rz.RzGroupedLinear(4, 128, 64, compress_ratio=0.5)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(x, off)
    with pytest.raises(ValueError):
        layer(x, off[:4])
    with pytest.raises(ValueError):
        layer(x[None], off)
    with pytest.raises(ValueError):
        layer(x[:, :64], off)
    with pytest.raises(TypeError):
        layer(x, off.float())
    with pytest.raises(TypeError):
        layer(x.int(), off)
    for bad in (0, 4097):
        with pytest.raises(ValueError):
            rz.RzGroupedLinear(bad, 128, 64)
    with pytest.raises(ValueError):
        rz.RzGroupedLinearFunction.apply(x, layer._hashed_weight, layer._random_numbers, off, 64, 1.0, None, torch.zeros(64))
