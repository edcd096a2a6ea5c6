"""Products grouped by row on the GPU, against 64-bit products with the materialised weights of each group.

Tolerances, element by element.  S is the sum of the magnitudes of an element's terms.
 * Products: bf16 operands multiply exactly in fp32; split tf32 operands drop at most 3 * 2^-20 of a term (10 explicit mantissa bits
   in each part, the product of the low parts is left out); the FMA kernels round once a term.
 * Sums: each tensor-core step (16 bf16 or 8 tf32 terms) and each fp32 addition changes a partial sum, at most S in magnitude, by at
   most 2^-23 (the tensor core truncates), each FMA by 2^-24: steps * 2^-23 * S, where steps counts the steps of the contraction and
   the additions into the hashed gradient, plus 8 for scaling, bias and the handful of partial sums in registers.
 * A bf16 result is rounded once: 2^-8 of its value.  The hashed array is rounded to bf16 for bf16 activations, and the reference uses
   the rounded values (the weight gradient does not read it).
"""
import numpy as np
import pytest
import torch

from oracle import rz_oracle as o

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
LARGE_PRIME = 2038074743
BF16, F32 = torch.bfloat16, torch.float32


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


def numbers(seed, mode):
    rng = np.random.RandomState(seed)
    return [LARGE_PRIME] + [int(v) for v in rng.randint(1, 2**31 - 1, 7)] if mode == 0 else [45007] + [int(v) for v in rng.randint(0, 45007, 7)]


class Case:
    """Inputs of a grouped product and its 64-bit results."""

    def __init__(self, sizes, K, N, BK, BN, mode, dtype, before=0, behind=0, bias=False, relu=False, alpha=0.75, seed=0):
        self.sizes, self.K, self.N, self.dtype, self.alpha, self.relu = sizes, K, N, dtype, float(np.float32(alpha)), relu
        G, nk = len(sizes), -(-K // BK)
        self.H = H = max(G * K * N // 6, 2 * BK * BN) + 3
        self.R = numbers(seed + K + N, mode)
        self.edges = np.concatenate([[before], before + np.cumsum(sizes)])
        self.M = M = int(self.edges[-1]) + behind
        g = torch.Generator(device=DEV).manual_seed(seed + 1)
        self.x = torch.randn((M, K), generator=g, device=DEV).to(dtype)
        self.g = torch.randn((M, N), generator=g, device=DEV).to(dtype)
        self.h = (torch.rand(H, generator=g, device=DEV) * 2 - 1) / K**0.5
        self.bias = torch.randn((G, N), generator=g, device=DEV) if bias else None
        self.offsets = torch.from_numpy(self.edges.astype(np.int32)).to(DEV)
        k = np.arange(K)
        rows = (np.arange(G)[:, None] * nk * BK + k).ravel()
        words = o.element_index_block(G * nk * BK, N, H, BK, BN, self.R, mode, rows, np.arange(N))
        self.words = torch.from_numpy(words).to(DEV).view(G, K, N)

    def exact(self):
        """(y, dx, dh, dbias) and for each the S of its elements, 64 bits."""
        h = (self.h.bfloat16() if self.dtype == BF16 else self.h).double()
        x, g, a = self.x.double(), self.g.double(), self.alpha
        y, ys = torch.zeros_like(g), torch.zeros_like(g)
        dx, dxs = torch.zeros_like(x), torch.zeros_like(x)
        dh = torch.zeros(self.H, dtype=torch.float64, device=DEV)
        dhs, dhn = torch.zeros_like(dh), torch.zeros_like(dh)
        db = torch.zeros((len(self.sizes), self.N), dtype=torch.float64, device=DEV)
        dbs = torch.zeros_like(db)
        for i, (lo, hi) in enumerate(zip(self.edges[:-1], self.edges[1:])):
            r, w, idx = slice(int(lo), int(hi)), h[self.words[i]], self.words[i].flatten()
            v = x[r] @ w * a + (0 if self.bias is None else self.bias[i].double())
            y[r] = v.relu() if self.relu else v
            ys[r] = x[r].abs() @ w.abs() * a + (0 if self.bias is None else self.bias[i].double().abs())
            gi = torch.where(y[r] > 0, g[r], 0.0) if self.relu else g[r]
            dx[r], dxs[r] = gi @ w.T * a, gi.abs() @ w.T.abs() * a
            if hi > lo:
                dh.index_add_(0, idx, (x[r].T @ gi * a).flatten())
                dhs.index_add_(0, idx, (x[r].T.abs() @ gi.abs() * a).flatten())
                dhn.index_add_(0, idx, torch.ones(len(idx), dtype=torch.float64, device=DEV))
            db[i], dbs[i] = gi.sum(0), gi.abs().sum(0)
        return (y, ys), (dx, dxs), (dh, dhs, dhn), (db, dbs)

    def call(self, rz, BK, BN, mode, offsets=None):
        cfg = rz.RzConfig(block_size_k=BK, block_size_n=BN, hash_mode=mode, relu=self.relu)
        x, h = self.x.clone().requires_grad_(), self.h.clone().requires_grad_()
        b = None if self.bias is None else self.bias.clone().requires_grad_()
        y = rz.RzGroupedLinearFunction.apply(x, h, torch.tensor(self.R), self.offsets if offsets is None else offsets, self.N, self.alpha, cfg, b)
        y.backward(self.g)
        return y.detach(), x.grad, h.grad, None if b is None else b.grad


def within(got, exact, size, steps, rounding, what):
    err = (got.double() - exact).abs()
    tol = 1.01 * (steps * 2.0**-23 * size + rounding * exact.abs())
    assert bool((err <= tol).all()), f"{what}: off by {float((err - tol).max())} more than {float(tol.max())} allows"


def check(case, got, split):
    (y, ys), (dx, dxs), (dh, dhs, dhn), (db, dbs) = case.exact()
    per, rounding = (16, 2.0**-8) if case.dtype == BF16 else (1, 0.0)
    lost = 24 if split else 0                                  # 3 * 2^-20 in units of 2^-23
    assert got[0].dtype == case.dtype and got[1].dtype == case.dtype and got[2].dtype == F32
    within(got[0], y, ys, case.K / per + 8 + lost, rounding, "output")
    if case.relu:   # the mask comes from the rounded output: where the exact one is that near 0, either is right
        return
    within(got[1], dx, dxs, case.N / per + 8 + lost, rounding, "input gradient")
    rows = max(max(case.sizes), 1)
    within(got[2], dh, dhs, rows / per + 8 + lost + dhn * (1 + rows // 2048), 0.0, "hashed gradient")
    if case.bias is not None:
        within(got[3], db, dbs, rows + 8, 0.0, "bias gradient")


SIZES = {
    "even": [128, 128, 128, 128],
    "ragged": [1, 200, 0, 63, 64, 65, 0, 300, 7],
    "one": [700],
    "rows": [1, 1, 0, 1, 2, 1],
    "skewed": [0, 0, 900, 0, 33],
    "long": [2500, 31, 1],       # more rows than one accumulation chain takes
}


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N,BK,BN,mode", [(256, 512, 32, 64, 1), (320, 264, 64, 64, 0), (512, 192, 128, 128, 1), (136, 1000, 32, 128, 0)])
def test_bf16(rz, rzlib, sizes, K, N, BK, BN, mode):
    case = Case(SIZES[sizes], K, N, BK, BN, mode, BF16, before=3 if sizes == "ragged" else 0, behind=5, bias=mode == 1)
    pb = rzlib.make_problem(case.M, K, N, case.H, BK, BN, case.R, mode, rzlib.BF16, rzlib.PREC_BF16)
    assert rzlib.plan(pb, 0) == rzlib.PATH_TCGEN05
    check(case, case.call(rz, BK, BN, mode), False)
    assert rzlib.device_status()[0] == 0


@pytest.mark.parametrize("shape", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("sizes", ["ragged", "long"])
def test_every_block_shape(rz, rzlib, knob, shape, sizes):
    knob("RZ_TC_CONFIG", shape)
    case = Case(SIZES[sizes], 576, 832, 64, 64, 1, BF16, behind=40, bias=True)
    check(case, case.call(rz, 64, 64, 1), False)
    assert rzlib.device_status()[0] == 0


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N,BK,BN,mode", [(256, 512, 32, 32, 1), (132, 100, 32, 32, 0)])
def test_fp32_on_the_tensor_cores(rz, rzlib, sizes, K, N, BK, BN, mode):
    case = Case(SIZES[sizes], K, N, BK, BN, mode, F32, behind=2, bias=True)
    pb = rzlib.make_problem(case.M, K, N, case.H, BK, BN, case.R, mode, rzlib.F32, rzlib.PREC_FP32)
    assert rzlib.plan(pb, 0) == rzlib.PATH_TCGEN05
    check(case, case.call(rz, BK, BN, mode), True)


@pytest.mark.parametrize("shape", [4, 5])
def test_fp32_long_contractions_stay_exact(rz, knob, shape):
    # several accumulation chains: beyond 2048, and beyond what the chains hold at 2048 each
    knob("RZ_TC_CONFIG", shape)
    for K, N in ((5000, 64), (64, 5000), (9000, 32)):
        case = Case([130, 1, 64], K, N, 32, 32, 0, F32)
        got = case.call(rz, 32, 32, 0)
        check(case, got, True)
        (y, _), (dx, _), (dh, _, _), _ = case.exact()
        for a, b in ((got[0], y), (got[1], dx), (got[2], dh)):
            assert float((a.double() - b).norm() / b.norm()) < 4e-6


def test_tf32(rz, rzlib):
    rz.controls['triton_allow_tf32'] = True
    try:
        case = Case(SIZES["ragged"], 256, 512, 64, 64, 0, F32, bias=True)
        got = case.call(rz, 64, 64, 0)
    finally:
        rz.controls['triton_allow_tf32'] = False
    (y, _), (dx, _), (dh, _, _), _ = case.exact()
    for a, b in ((got[0], y), (got[1], dx), (got[2], dh)):   # operands with 10 explicit mantissa bits: 2^-11 each at most, the framework's bar
        assert float((a.double() - b).norm() / b.norm()) < 2e-3


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("K,N,BK,BN,mode,dtype", [(37, 53, 8, 5, 0, F32), (37, 53, 8, 5, 0, BF16), (129, 70, 16, 24, 1, F32),
                                                  (129, 70, 16, 24, 1, BF16), (100, 200, 32, 32, 0, BF16)])
def test_fma_kernels(rz, rzlib, sizes, K, N, BK, BN, mode, dtype):
    case = Case(SIZES[sizes], K, N, BK, BN, mode, dtype, before=1, behind=9, bias=True)
    pb = rzlib.make_problem(case.M, K, N, case.H, BK, BN, case.R, mode, rzlib.torch_io_dtype(dtype), 2 if dtype == BF16 else 0)
    assert rzlib.plan(pb, 0) == rzlib.PATH_SIMT
    if dtype == BF16:   # these kernels read the hashed array itself
        case.h = case.h.bfloat16().float()
    got = case.call(rz, BK, BN, mode)
    (y, ys), (dx, dxs), (dh, dhs, dhn), (db, dbs) = case.exact()
    rounding, rows = (2.0**-8 if dtype == BF16 else 0.0), max(case.sizes)
    within(got[0], y, ys, K + 8, rounding, "output")
    within(got[1], dx, dxs, N + 8, rounding, "input gradient")
    within(got[2], dh, dhs, rows + 8 + dhn * 2, 0.0, "hashed gradient")
    within(got[3], db, dbs, rows + 8, 0.0, "bias gradient")


@pytest.mark.parametrize("dtype,K,N,BK,BN", [(BF16, 256, 320, 32, 64), (F32, 37, 53, 8, 5), (F32, 128, 128, 32, 32)])
def test_relu_masks_the_gradient_with_the_saved_output(rz, dtype, K, N, BK, BN):
    case = Case(SIZES["ragged"], K, N, BK, BN, 1, dtype, bias=True, relu=True, behind=4)
    y, dx, dh, db = case.call(rz, BK, BN, 1)
    check(case, (y, dx, dh, db), True)
    # without the ReLU, on a gradient masked by the output: the same kernels on the same operands
    plain = Case(SIZES["ragged"], K, N, BK, BN, 1, dtype, bias=True, behind=4)
    plain.g = torch.where(y > 0, plain.g, 0.0).to(dtype)
    _, dx2, dh2, db2 = plain.call(rz, BK, BN, 1)
    assert torch.equal(dx, dx2)
    assert float((dh - dh2).norm() / dh2.norm()) < 1e-6 and float((db - db2).norm() / db2.norm()) < 1e-6   # order of additions


@pytest.mark.parametrize("dtype,K,N,BK,BN", [(BF16, 256, 320, 32, 64), (F32, 37, 53, 8, 5), (F32, 128, 128, 32, 32)])
def test_relu_lets_nan_through(rz, dtype, K, N, BK, BN):
    case = Case([40, 0, 90], K, N, BK, BN, 0, dtype, bias=True, relu=True)
    clean = case.call(rz, BK, BN, 0)
    case.x[5, 3] = float("nan")
    y, dx, dh, db = case.call(rz, BK, BN, 0)
    assert bool(y[5].isnan().all())
    keep = torch.arange(case.M, device=DEV) != 5
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    # like torch.relu: the gradient of a NaN goes on (and group 0's weights learn of it)
    wanted = case.g[5].double() @ (case.h.bfloat16() if dtype == BF16 else case.h).double()[case.words[0]].T * case.alpha
    assert float((dx[5].double() - wanted).norm() / wanted.norm()) < 2.0**-7
    assert bool(dh.isnan().any()) and bool(db.isfinite().all())


@pytest.mark.parametrize("dtype,K,N,BK,BN", [(BF16, 256, 320, 32, 64), (F32, 37, 53, 8, 5), (F32, 128, 128, 32, 32)])
def test_each_group_is_a_linear_layer(rz, dtype, K, N, BK, BN):
    # group g's weight is an RzLinear's whose R1 and R4 are advanced by its first tile row
    case = Case([70, 0, 130, 5], K, N, BK, BN, 1, dtype)
    y, dx, _, _ = case.call(rz, BK, BN, 1)
    for g, (lo, hi) in enumerate(zip(case.edges[:-1], case.edges[1:])):
        if hi == lo:
            continue
        R, first = list(case.R), g * -(-K // BK)
        R[1], R[4] = (R[1] + first * R[3]) % R[0], (R[4] + first * R[7]) % R[0]
        cfg = rz.RzConfig(block_size_k=BK, block_size_n=BN, hash_mode=1)
        x = case.x[lo:hi].clone().requires_grad_()
        want = rz.RzLinearFunction.apply(x, case.h, torch.tensor(R), N, 1, case.alpha, cfg)
        want.backward(case.g[lo:hi])
        tol = 2.0**-8 if dtype == BF16 else 1e-6
        want = want.detach()
        assert float((y[lo:hi].float() - want.float()).abs().max()) <= tol * float(want.abs().max())
        assert float((dx[lo:hi].float() - x.grad.float()).abs().max()) <= tol * float(x.grad.abs().max())


@pytest.mark.parametrize("dtype,K,N,BK,BN", [(BF16, 256, 320, 32, 64), (F32, 37, 53, 8, 5), (F32, 128, 128, 32, 32)])
def test_rows_of_no_group_and_of_the_next(rz, dtype, K, N, BK, BN):
    # what stands in rows of no group is not looked at, and a group's numbers stay in it: NaN and infinities elsewhere do no harm
    case = Case([40, 100, 3], K, N, BK, BN, 1, dtype, before=2, behind=70, bias=True)
    clean = case.call(rz, BK, BN, 1)
    lo, hi = int(case.edges[1]), int(case.edges[2])
    for t in (case.x, case.g):
        t[:2], t[-70:], t[lo:hi] = float("nan"), float("inf"), float("nan")
    y, dx, dh, db = case.call(rz, BK, BN, 1)
    outside = torch.ones(case.M, dtype=torch.bool, device=DEV)
    outside[2:-70] = False
    assert float(y[outside].abs().sum()) == 0.0 and float(dx[outside].abs().sum()) == 0.0
    keep = ~outside
    keep[lo:hi] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert bool(y[lo:hi].isnan().all()) and bool(db[1].isnan().all()) and not bool(db[[0, 2]].isnan().any())
    others = torch.ones(case.H, dtype=torch.bool, device=DEV)
    others[case.words[1].flatten()] = False
    assert not bool(dh[others].isnan().any())


def test_offsets_out_of_order_or_range_are_clamped(rz):
    case = Case([64, 64, 64], 128, 128, 32, 64, 1, BF16, behind=64)
    wild = torch.tensor([-5, 100, 40, 10**6], dtype=torch.int32, device=DEV)
    tame = torch.tensor([0, 100, 100, 256], dtype=torch.int32, device=DEV)
    got, want = (case.call(rz, 32, 64, 1, offsets=t) for t in (wild, tame))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    as64 = case.call(rz, 32, 64, 1, offsets=torch.tensor([-5, 100, 40, 2**33], device=DEV))
    assert torch.equal(as64[0], want[0])


def test_module_types_and_empty_batches(rz):
    layer = rz.RzGroupedLinear(4, 128, 64, block_size_n=32, compress_ratio=0.5).to(DEV)
    off = torch.tensor([0, 3, 3, 10, 12], device=DEV)
    x = torch.randn(12, 128, device=DEV)
    y = layer(x, off)
    assert y.shape == (12, 64) and y.dtype == F32
    half = layer(x.half(), off).detach()
    assert half.dtype == torch.float16 and float((half.float() - layer(x.half().float(), off).detach()).abs().max()) <= 2.0**-11 * float(half.abs().max())
    assert torch.equal(layer(x.t().contiguous().t(), off), y)                     # strides
    out = layer(x[:0], torch.zeros(5, dtype=torch.int32, device=DEV))
    assert out.shape == (0, 64)
    out.sum().backward()
    assert float(layer._hashed_weight.grad.abs().sum()) == 0.0 and float(layer._bias.grad.abs().sum()) == 0.0
    layer.zero_grad()
    out = layer(x, torch.zeros(5, dtype=torch.int32, device=DEV))                 # rows, but no group has any
    out.sum().backward()
    assert float(out.detach().abs().sum()) == 0.0 and float(layer._hashed_weight.grad.abs().sum()) == 0.0
    wb = torch.nn.Parameter(layer._hashed_weight.detach().bfloat16())
    lb = rz.RzGroupedLinear(4, 128, 64, hashed_weight=wb, bias=False)
    lb(x.bfloat16(), off).float().sum().backward()
    assert wb.grad.dtype == BF16


def test_many_groups_and_gradient_against_differences(rz):
    G, K, N = 1500, 64, 64
    rng = np.random.RandomState(3)
    sizes = rng.randint(0, 4, G)
    case = Case(list(sizes), K, N, 32, 64, 0, BF16)
    check(case, case.call(rz, 32, 64, 0), False)
    # the product is linear in the hashed array: <g, f(v)> = <dh, v>
    small = Case([5, 40, 0, 3], 96, 64, 32, 32, 0, F32)
    _, _, dh, _ = small.call(rz, 32, 32, 0)
    v = torch.randn_like(small.h)
    cfg = rz.RzConfig(block_size_k=32, block_size_n=32, hash_mode=0)
    fv = rz.RzGroupedLinearFunction.apply(small.x, v, torch.tensor(small.R), small.offsets, 64, small.alpha, cfg)
    left, right = (small.g.double() * fv.double()).sum(), (dh.double() * v.double()).sum()
    assert abs(float(left - right)) <= 1e-5 * float(small.g.double().norm() * fv.double().norm())


def test_two_streams_and_a_graph(rz):
    case = Case(SIZES["ragged"], 256, 512, 32, 64, 1, BF16, behind=5)
    cfg = rz.RzConfig(block_size_k=32, block_size_n=64, hash_mode=1)
    R, h = torch.tensor(case.R), case.h.clone().requires_grad_()
    x = case.x.clone().requires_grad_()

    def step(off):
        y = rz.RzGroupedLinearFunction.apply(x, h, R, off, case.N, case.alpha, cfg)
        return y.detach(), torch.autograd.grad(y, x, case.g)[0]

    other = case.offsets.flip(0).neg().add(case.offsets[-1]).contiguous()     # the groups' sizes in reverse order
    want = [step(case.offsets), step(other)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, off in zip(streams, (case.offsets, other)):
            with torch.cuda.stream(s):
                got.append(step(off))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert torch.equal(r[0], want[i % 2][0]) and torch.equal(r[1], want[i % 2][1])

    # two captured graphs, replayed with new offsets, inputs and weights
    off = case.offsets.clone()
    graphs = []
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = step(off)
        graphs.append((graph, held))
    off.copy_(other)
    with torch.no_grad():
        x.mul_(2)
        h.mul_(0.5)
    fresh = step(off)
    for s, (graph, _) in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, held in graphs:
        assert torch.equal(held[0], fresh[0]) and torch.equal(held[1], fresh[1])


def test_copies_replaced_while_another_stream_reads_them(rz):
    # a linear layer over the same array wants a larger buffer than a grouped call: the smaller one, still read by a call that waits on
    # another stream, must not be handed out again before that call has run
    case = Case([200, 0, 90], 256, 512, 32, 64, 1, BF16)
    cfg = rz.RzConfig(block_size_k=32, block_size_n=64, hash_mode=1)
    R, h = torch.tensor(case.R), case.h.clone()
    grouped = lambda: rz.RzGroupedLinearFunction.apply(case.x, h, R, case.offsets, case.N, case.alpha, cfg)
    want = grouped()
    before = h._rz_shadow_cache[next(iter(h._rz_shadow_cache))]["shadow"].numel()
    wide = torch.randn(64, 1024, device=DEV).bfloat16()
    linear = lambda weight: rz.RzLinearFunction.apply(wide, weight, R, 4096, 0, case.alpha, cfg)
    fill = lambda: torch.full((before,), 0x7f, dtype=torch.uint8, device=DEV)
    linear(h.clone()), fill()                  # (load their kernels, which would wait for the device later)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grouped()                              # (gets this stream its memory)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)         # some 0.1 s
        got = grouped()
    linear(h)
    entry, = h._rz_shadow_cache.values()
    assert entry["shadow"].numel() > before    # replaced
    garbage = [fill() for _ in range(16)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(garbage) == 16

def test_an_expert_model_end_to_end(rz):
    # tokens -> table -> rows sorted by expert -> two grouped products -> weighted sum per token, forward and backward, all weights
    # slices of one hashed array; against the same model with materialised weights in 64 bits.  Five products deep, each within the
    # 1e-5 of the framework's fp32 path.
    V, D, F, E, T, top = 500, 128, 192, 6, 333, 2
    torch.manual_seed(0)
    w = torch.nn.Parameter((torch.rand(20011, device=DEV) * 2 - 1) * 0.3)
    emb = rz.RzEmbedding(V, D, hashed_weight=w, seed=1, init_factor=2.0, padding_idx=0, block_size_n=32)
    up = rz.RzGroupedLinear(E, D, F, hashed_weight=w, seed=2, init_factor=0.2, block_size_n=32).to(DEV)
    down = rz.RzGroupedLinear(E, F, D, hashed_weight=w, seed=3, init_factor=0.2, bias=False, block_size_n=32)
    with torch.no_grad():
        up._bias.normal_()
    ids = torch.randint(0, V, (T,), device=DEV)
    ids[-20:] = 0
    scores = torch.rand(T, E, device=DEV)
    scores[:, 4] = 0                                              # an expert without rows
    weight, choice = scores.topk(top)
    keys = torch.where(ids[:, None] == 0, -1, choice).flatten()   # padding goes to no expert
    g = torch.randn(T, D, device=DEV)

    order, offsets = rz.sort_rows(keys, E)
    token = order // top
    h = emb(ids)
    y = down(torch.nn.functional.silu(up(h[token], offsets)), offsets)
    out = torch.zeros_like(h).index_add(0, token, y * weight.flatten()[order, None])
    out.backward(g)

    def materialised(layer, rows, cols, groups=1):
        BK, BN = layer._config.block_size_k, layer._config.block_size_n
        nk = -(-rows // BK)
        at = (np.arange(groups)[:, None] * nk * BK + np.arange(rows)).ravel()
        words = o.element_index_block(groups * nk * BK, cols, w.numel(), BK, BN, layer._random_numbers.tolist(), layer._config.hash_mode, at, np.arange(cols))
        return torch.from_numpy(words).to(DEV).view(groups, rows, cols)

    wd = w.detach().double().requires_grad_()
    bd = up._bias.detach().double().requires_grad_()
    table, w1, w2 = wd[materialised(emb, V, D)][0] * 2.0, wd[materialised(up, D, F, E)] * float(np.float32(0.2)), wd[materialised(down, F, D, E)] * float(np.float32(0.2))
    hd = torch.where(ids[:, None] == 0, 0.0, table[ids])
    want = torch.zeros_like(hd)
    for t in range(top):
        e = choice[:, t]
        mid = torch.nn.functional.silu(torch.einsum("td,tdf->tf", hd, w1[e]) + bd[e])
        part = torch.einsum("tf,tfd->td", mid, w2[e]) * weight[:, t, None].double()
        want = want + torch.where(ids[:, None] == 0, 0.0, part)
    want.backward(g.double())
    for got, exact in ((out.detach(), want.detach()), (w.grad, wd.grad), (up._bias.grad, bd.grad)):
        assert float((got.double() - exact).norm() / exact.norm()) < 5e-5


def test_offsets_beyond_32_bits(rz):
    # 4.6e9 entries of output: rows at the end are computed, stored and differentiated like the first
    M, K, N, G = 70000, 64, 65536, 2
    x = torch.randn(M, K, device=DEV).bfloat16()
    layer = rz.RzGroupedLinear(G, K, N, hashed_weight=torch.nn.Parameter((torch.rand(1 << 20, device=DEV) - 0.5)), bias=False)
    off = torch.tensor([0, 40, M - 3], device=DEV, dtype=torch.int32)
    xs = x.clone().requires_grad_()
    y = layer(xs, off)
    assert y.numel() > 2**32
    g = torch.ones((), device=DEV, dtype=BF16).expand(M, N)
    dx, dh = torch.autograd.grad(y, (xs, layer._hashed_weight), g)
    sample = torch.tensor([0, 39, 40, 41, M // 2, M - 5, M - 4], device=DEV)
    few = x[sample].clone().requires_grad_()
    few_off = torch.tensor([0, 2, 7], device=DEV, dtype=torch.int32)
    yf = layer(few, few_off)
    (dxf,) = torch.autograd.grad(yf, few, torch.ones_like(yf))
    assert float(y[M - 3:].detach().abs().sum()) == 0.0 and float(dx[M - 3:].abs().sum()) == 0.0
    # the same sums in blocks of other shapes: at most one rounding to bf16 apart
    assert bool(((y[sample] - yf).detach().float().abs() <= 2.0**-7 * yf.detach().float().abs() + 1e-6).all())
    assert float((dx[sample] - dxf).float().norm() / dxf.float().norm()) <= 2.0**-7
    # every word of a group's weight gradient is alpha * (sum over rows of x): check one tile row of group 1 against it
    want = x[40:M - 3].double().sum(0)
    words = o.element_index_block(G * K, N, 1 << 20, 32, 64, layer._random_numbers.tolist(), 1, np.arange(G * K), np.arange(N))
    total = torch.zeros(1 << 20, dtype=torch.float64, device=DEV)
    w = torch.from_numpy(words).to(DEV)
    first = x[:40].double().sum(0)
    total.index_add_(0, w[:K].flatten(), first[:, None].expand(K, N).flatten())
    total.index_add_(0, w[K:].flatten(), want[:, None].expand(K, N).flatten())
    assert float((dh.double() - total).norm() / total.norm()) < 1e-5      # the framework's bar for fp32 results


@pytest.mark.parametrize("dtype,K,N,BK,BN", [(BF16, 256, 320, 32, 64), (F32, 128, 160, 32, 32)])
def test_call_options_give_the_same_bits(rz, rzlib, dtype, K, N, BK, BN):
    # small whole numbers: every product and sum is exact in fp32 (and rounded once to bf16), whatever computes them in whatever order
    case = Case([300, 0, 33, 1], K, N, BK, BN, 1, dtype, before=2, behind=3)
    g = torch.Generator(device=DEV).manual_seed(5)
    whole = lambda t: torch.randint(-2, 3, t.shape, generator=g, device=DEV).to(t.dtype)
    x, dy, h, bias = whole(case.x), whole(case.g), whole(case.h), torch.randint(-2, 3, (4, N), generator=g, device=DEV).float()
    io, prec = (rzlib.BF16, rzlib.PREC_BF16) if dtype == BF16 else (rzlib.F32, rzlib.PREC_FP32)
    pb = rzlib.make_problem(case.M, K, N, case.H, BK, BN, case.R, 1, io, prec, alpha=0.5)
    assert rzlib.plan(pb, 0) == rzlib.PATH_TCGEN05

    def run(pb, want=("dx", "dh", "db"), dh=None, db=None):
        copies_bytes, ws_bytes = rzlib.grouped_sizes(pb, 4)
        copies = torch.empty(copies_bytes, dtype=torch.uint8, device=DEV) if copies_bytes else None
        if copies is not None:
            rzlib.shadow_refresh(pb, h, copies)
        y, ws = torch.empty_like(dy), torch.empty(ws_bytes, dtype=torch.uint8, device=DEV)
        rzlib.grouped_forward(pb, 4, case.offsets, x, h, copies, bias, y, ws)
        out = {"dx": torch.empty_like(x), "dh": torch.empty_like(h) if dh is None else dh, "db": torch.empty_like(bias) if db is None else db}
        rzlib.grouped_backward(pb, 4, case.offsets, x, dy, None, h, copies, None, *(out[k] if k in want else None for k in ("db", "dx", "dh")), ws)
        return {"y": y, **{k: out[k] for k in want}}

    first = run(pb)
    assert float(first["dh"].abs().max()) > 0 and float(first["dx"].abs().max()) > 0
    others = [run(rzlib.with_fields(pb, flags=rzlib.FLAG_FORCE_SIMT)), run(rzlib.with_fields(pb, sm_reserve=100)),
              run(pb, ("dx",)), run(pb, ("dh",)), run(pb, ("db",)), run(pb, ("dh", "db"))]
    others += [run(pb, ("db",), db=torch.empty(4 * N + 1, device=DEV)[1:].view(4, N))]     # (begins at an odd word)
    for other in others:
        for k, v in other.items():
            assert torch.equal(v, first[k]), k
    twice = run(rzlib.with_fields(pb, flags=rzlib.FLAG_ACCUMULATE_DH), dh=first["dh"].clone())["dh"]
    assert torch.equal(twice, 2 * first["dh"])


def test_views_that_begin_anywhere(rz):
    case = Case([70, 0, 130, 5], 256, 320, 32, 64, 1, BF16)
    clean = case.call(rz, 32, 64, 1)
    for name in ("x", "g"):
        t = getattr(case, name)
        buf = torch.empty(t.numel() + 8, device=DEV, dtype=t.dtype)
        setattr(case, name, buf[3:3 + t.numel()].view(t.shape).copy_(t))
        assert getattr(case, name).data_ptr() % 16
    cfg = rz.RzConfig(block_size_k=32, block_size_n=64, hash_mode=1)
    x = case.x.detach().requires_grad_()
    y = rz.RzGroupedLinearFunction.apply(x, case.h, torch.tensor(case.R), case.offsets, case.N, case.alpha, cfg)
    (dx,) = torch.autograd.grad(y, x, case.g)
    assert torch.equal(y, clean[0]) and torch.equal(dx, clean[1])
