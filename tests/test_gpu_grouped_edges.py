"""Grouped products at their edges: where block follows block quickly (many blocks a CTA, two or three contraction stages, last column
blocks that lie mostly past the matrix), as many groups as there may be, few rows, 64-bit activations.

Tolerances: none.  Activations, weights, gradients and bias are small whole numbers, so every product and sum is exact in fp32 (at most
4 * 16384 * 16 / 2 < 2^24 in magnitude) and an output is rounded at most once: the tensor-core kernels and the FMA kernels give the same
bits, in every run.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def rz(rzlib):
    assert torch.cuda.is_available(), "these tests need a GPU"
    rzlib.load()
    import rzlinear_b200
    return rzlinear_b200


@pytest.fixture
def knob(rzlib, monkeypatch):
    def set_(name, value):
        monkeypatch.setenv(name, str(value))
        rzlib.reload_env()
    yield set_
    monkeypatch.undo()
    rzlib.reload_env()


class Whole:
    """A grouped product of small whole numbers, called through the C ABI."""

    def __init__(self, rzlib, sizes, K, N, BK=32, BN=64, behind=0, seed=0):
        self.lib, self.G = rzlib, len(sizes)
        M = int(np.sum(sizes)) + behind
        rng = np.random.RandomState(seed)
        R = [45007] + [int(v) for v in rng.randint(0, 45007, 7)]
        H = max(self.G * K * N // 6, 2 * BK * BN) + 3
        g = torch.Generator(device=DEV).manual_seed(seed)
        whole = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=DEV).float()
        self.x, self.dy, self.h, self.bias = whole(M, K).to(BF16), whole(M, N).to(BF16), whole(H), whole(self.G, N)
        self.offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).to(DEV)
        self.pb = rzlib.make_problem(M, K, N, H, BK, BN, R, 1, rzlib.BF16, rzlib.PREC_BF16, alpha=0.5)
        assert rzlib.plan(self.pb, 0) == rzlib.PATH_TCGEN05

    def __call__(self, simt=False):
        lib = self.lib
        pb = lib.with_fields(self.pb, flags=lib.FLAG_FORCE_SIMT) if simt else self.pb
        copies_bytes, ws_bytes = lib.grouped_sizes(pb, self.G)
        copies = torch.empty(copies_bytes, dtype=torch.uint8, device=DEV) if copies_bytes else None
        if copies is not None:
            lib.shadow_refresh(pb, self.h, copies)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=DEV)
        out = [torch.full_like(t, float("nan")) for t in (self.dy, self.x, self.h, self.bias)]
        lib.grouped_forward(pb, self.G, self.offsets, self.x, self.h, copies, self.bias, out[0], ws)
        lib.grouped_backward(pb, self.G, self.offsets, self.x, self.dy, None, self.h, copies, None, out[3], out[1], out[2], ws)
        return out


def uneven(rows, groups, seed):
    return np.random.RandomState(seed).multinomial(rows, np.random.RandomState(seed + 1).dirichlet(np.full(groups, 3.0)))


@pytest.mark.parametrize("shape", [None, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("K,N", [(128, 1032), (136, 520), (1032, 128), (520, 136)])
def test_blocks_in_quick_succession(rz, rzlib, knob, K, N, shape):
    if shape is not None:
        knob("RZ_TC_CONFIG", shape)
    case = Whole(rzlib, uneven(16384, 16, K), K, N, behind=7)
    want = case(simt=True)
    for _ in range(8):
        for name, got, exact in zip(("output", "input gradient", "hashed gradient", "bias gradient"), case(), want):
            assert torch.equal(got, exact), name
    assert rzlib.device_status()[0] == 0


def agree(case, repeats=2):
    want = case(simt=True)
    for _ in range(repeats):
        for name, got, exact in zip(("output", "input gradient", "hashed gradient", "bias gradient"), case(), want):
            assert torch.equal(got, exact), name
    assert case.lib.device_status()[0] == 0


@pytest.mark.parametrize("kind", ["few each", "last alone", "none"])
def test_as_many_groups_as_there_may_be(rz, rzlib, kind):
    sizes = np.random.RandomState(2).randint(0, 4, 4096) if kind == "few each" else np.zeros(4096, dtype=np.int64)
    if kind == "last alone":
        sizes[-1] = 100
    agree(Whole(rzlib, sizes, 64, 72, behind=5))


@pytest.mark.parametrize("shape", [None, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("sizes", [[64], [1], [0, 0, 37, 0], [5, 0, 60]])
def test_few_rows_in_one_or_two_groups(rz, rzlib, knob, sizes, shape):
    if shape is not None:
        knob("RZ_TC_CONFIG", shape)
    agree(Whole(rzlib, sizes, 1096, 648, BK=64, BN=128))


def test_double_activations_are_computed_in_32_bits(rz):
    layer = rz.RzGroupedLinear(3, 128, 96, compress_ratio=0.5, block_size_n=32).to(DEV)
    off = torch.tensor([0, 30, 30, 77], device=DEV, dtype=torch.int32)
    x = torch.randn(80, 128, device=DEV).double().requires_grad_()
    y = layer(x, off)
    assert y.dtype == torch.float64 and torch.equal(y, layer(x.float(), off).double())
    g = torch.randn_like(y)
    (dx,) = torch.autograd.grad(y, x, g)
    xf = x.detach().float().requires_grad_()
    (dxf,) = torch.autograd.grad(layer(xf, off), xf, g.float())
    assert dx.dtype == torch.float64 and torch.equal(dx, dxf.double())
