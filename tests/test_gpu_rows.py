"""Row sort, embedding lookup and its gradient on the GPU, against plain 64-bit forms on the CPU.

Tolerances.  Lookup: one fp32 product, then at most one rounding to bf16 - the same two operations in torch, so the bits are
equal.  Gradient: a word of dH is a sum of n products (one fp32 rounding each, 2^-24 relative) added in fp32 in some order, whose
error is at most (n - 1) 2^-24 (1 + small) times the sum of the magnitudes; scaling and the running sums in registers add no
more than two roundings a term.  Hence |dH - exact| <= 1.01 (n + 2) 2^-24 sum |terms|, word by word.  Sorts are exact.
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


def numbers(seed, mode):
    rng = np.random.RandomState(seed)
    return [LARGE_PRIME] + [int(v) for v in rng.randint(1, 2**31 - 1, 7)] if mode == 0 else [45007] + [int(v) for v in rng.randint(0, 45007, 7)]


# ---- sort ---------------------------------------------------------------------------------------------------------------
def exact_sort(keys, bins):
    k = np.where((keys < 0) | (keys >= bins), bins, keys)
    order = np.argsort(k, kind="stable")
    return order.astype(np.int32), np.searchsorted(k[order], np.arange(bins + 1)).astype(np.int32)


@pytest.mark.parametrize("rows", [0, 1, 31, 33, 512, 2047, 2048, 2049, 5000, 40961, 700001])
@pytest.mark.parametrize("bins,kind", [(1, "even"), (7, "even"), (128, "skewed"), (1024, "even"), (1000, "one"), (16, "outside")])
def test_sort_rows(rz, rows, bins, kind):
    rng = np.random.RandomState(rows + bins)
    keys = {"even": lambda: rng.randint(0, bins, rows), "skewed": lambda: (rng.rand(rows) ** 4 * bins).astype(np.int64),
            "one": lambda: np.full(rows, bins - 1), "outside": lambda: rng.randint(-3, bins + 3, rows) * rng.choice([1, 2**33], rows)}[kind]()
    keys = keys.astype(np.int64)
    order, offsets = rz.sort_rows(torch.from_numpy(keys).to(DEV), bins)
    want_order, want_offsets = exact_sort(keys, bins)
    assert order.dtype == torch.int32 and offsets.dtype == torch.int32
    assert np.array_equal(offsets.cpu().numpy(), want_offsets)
    assert np.array_equal(order.cpu().numpy(), want_order)


def test_sort_rows_strided_and_int32(rz):
    keys = torch.randint(0, 9, (3000, 2), device=DEV)
    for k in (keys[:, 1], keys[:, 0].int()):
        order, offsets = rz.sort_rows(k, 9)
        want = exact_sort(k.cpu().numpy().astype(np.int64), 9)
        assert np.array_equal(order.cpu().numpy(), want[0]) and np.array_equal(offsets.cpu().numpy(), want[1])


# ---- embedding ------------------------------------------------------------------------------------------------------------
def words_of(ids, live, V, D, H, BK, BN, R, mode):
    """Index into the hashed array of every entry of the selected rows, [tokens, D] (row 0's words where not live)."""
    off = o.tile_offsets(V, D, H, BK, BN, R, mode)
    k = np.where(live, ids, 0).astype(np.int64)[:, None]
    n = np.arange(D)[None, :]
    return off[k // BK, n // BN] + (k % BK) * BN + n % BN


CASES = [
    # tokens, V, D, BK, BN, mode, padding, kind;  more than 2^22 entries: tokens are sorted before the gradient
    (1, 1000, 64, 32, 64, 1, None, "text"),
    (1, 33, 1, 4, 3, 0, None, "text"),
    (7, 500, 130, 16, 24, 1, 3, "text"),
    (64, 5000, 256, 32, 32, 0, -1, "even"),
    (255, 128, 63, 32, 64, 1, None, "text"),       # odd row length: no pairs
    (256, 777, 96, 32, 96, 0, None, "one"),
    (257, 777, 96, 32, 32, 0, 0, "text"),
    (1000, 50021, 1000, 16, 24, 1, 50020, "text"),
    (2048, 70000, 64, 64, 128, 0, None, "even"),   # row shorter than a hash tile
    (2049, 300, 320, 128, 64, 1, 5, "one"),
    (8193, 131072, 72, 64, 64, 0, 7, "outside"),   # rows of no table entry
    (20000, 2, 50, 1, 50, 0, None, "even"),
    (5000, 2**31 - 2**13, 64, 2048, 64, 0, None, "outside"),   # the largest ids
    (257, 3000, 16400, 32, 64, 1, 2, "text"),      # first length that is sorted
    (2048, 60000, 2052, 32, 32, 1, 9, "even"),     # one chunk, full; a ragged last piece
    (2049, 3000, 2056, 32, 8, 0, None, "text"),    # a chunk of one token
    (4097, 5000, 1090, 16, 109, 0, 17, "text"),    # odd segments
    (6000, 900, 770, 16, 96, 0, None, "one"),      # halves of a piece apart
    (8193, 131072, 520, 64, 64, 0, 7, "outside"),
    (16385, 100000, 1024, 32, 64, 1, 5, "text"),   # the longest chunks, and one of one token
    (70000, 65536, 64, 32, 64, 1, None, "text"),   # many chunks
    (100000, 40, 47, 4, 2, 0, None, "outside"),    # most tokens of no row
    (90000, 2, 50, 1, 50, 0, None, "even"),
]


def make_ids(kind, T, V, padding, rng):
    if kind == "text":
        ids = np.minimum(np.exp(rng.rand(T) * np.log(V)).astype(np.int64), V - 1)
    elif kind == "one":
        ids = np.full(T, V - 2, dtype=np.int64)
    elif kind == "even":
        ids = rng.randint(0, V, T).astype(np.int64)
    else:
        ids = rng.randint(-V, 2 * V, T).astype(np.int64)
        ids[:: 97] = 2**40 + 1
    if padding is not None:
        ids[-(T // 7 + 1):] = padding % V
    return ids


@pytest.mark.parametrize("T,V,D,BK,BN,mode,padding,kind", CASES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding(rz, T, V, D, BK, BN, mode, padding, kind, dtype):
    rng = np.random.RandomState(T + V + D)
    R = numbers(T + D, mode)
    H = min(max(V * D // 8, 2 * BK * BN), 1 << 22) + 5
    ids = make_ids(kind, T, V, padding, rng)
    live = (ids >= 0) & (ids < V) & (ids != (padding % V if padding is not None else -1))
    words = words_of(ids, live, V, D, H, BK, BN, R, mode)
    h = torch.from_numpy(rng.randn(H).astype(np.float32))
    cfg = rz.RzConfig(block_size_k=BK, block_size_n=BN, hash_mode=mode)
    scale = 1.7
    hd = h.to(DEV).requires_grad_()
    out = rz.RzEmbeddingFunction.apply(torch.from_numpy(ids).to(DEV), hd, torch.tensor(R), V, D, scale, cfg, padding, dtype)
    want = torch.where(torch.from_numpy(live)[:, None], h[torch.from_numpy(words)] * np.float32(scale), torch.zeros(())).to(dtype)
    assert out.dtype == dtype and torch.equal(out.detach().cpu(), want)

    g = torch.from_numpy(rng.randn(T, D).astype(np.float32)).to(dtype)
    g[torch.from_numpy(~live)] = float("nan")          # what stands at tokens without a row is not looked at
    (dh,) = torch.autograd.grad(out, hd, g.to(DEV))
    gl = g[torch.from_numpy(live)].double().numpy() * np.float64(np.float32(scale))
    wl = words[live].ravel()
    exact = np.bincount(wl, weights=gl.ravel(), minlength=H)
    terms = np.bincount(wl, minlength=H)
    size = np.bincount(wl, weights=np.abs(gl).ravel(), minlength=H)
    err = np.abs(dh.cpu().double().numpy() - exact)
    assert (err <= 1.01 * (terms + 2) * 2.0**-24 * size).all(), float((err - 1.01 * (terms + 2) * 2.0**-24 * size).max())


def test_embedding_is_linear_in_the_hashed_array(rz):
    # the gradient against differences: E(h + v) - E(h) = E(v) exactly, so <dOut, E(v)> = <dH, v>
    T, V, D = 3000, 900, 192
    layer = rz.RzEmbedding(V, D, init_factor=0.5, padding_idx=4, block_size_k=32, block_size_n=64).to(DEV)
    ids = torch.randint(0, V, (3, T // 3), device=DEV)
    out = layer(ids)
    assert out.shape == (3, T // 3, D) and out.dtype == F32
    g = torch.randn_like(out)
    out.backward(g)
    v = torch.randn_like(layer._hashed_weight)
    shared = rz.RzEmbedding(V, D, hashed_weight=torch.nn.Parameter(v), init_factor=0.5, padding_idx=4)
    left = (shared(ids).double() * g.double()).sum()
    right = (layer._hashed_weight.grad.double() * v.double()).sum()
    # both sides are sums of T * D products of unit-size numbers with fp32 roundings: far below 1e-5 of the norms' product
    assert abs(float((left - right).detach())) <= 1e-5 * float((g.double().norm() * shared(ids).double().norm()).detach())


def test_embedding_row_is_the_linear_layers_weight_row(rz):
    # a table and a linear layer with the same sizes and random numbers share the virtual matrix
    V, D = 96, 128
    w = torch.nn.Parameter(torch.randn(4096 + 77, device=DEV))
    emb = rz.RzEmbedding(V, D, hashed_weight=w)
    lin = rz.RzLinear(V, D, hashed_weight=w, bias=False)
    got = lin(torch.eye(V, device=DEV))
    assert torch.allclose(got, emb(torch.arange(V, device=DEV)), rtol=0, atol=1e-6 * float(w.detach().abs().max()))


def test_embedding_types_and_views(rz):
    V, D = 300, 64
    w = torch.nn.Parameter(torch.randn(4096, device=DEV))
    ids = torch.randint(0, V, (50, 4), device=DEV)
    base = rz.RzEmbedding(V, D, hashed_weight=w)(ids)
    strided = rz.RzEmbedding(V, D, hashed_weight=w)(ids.t())
    assert torch.equal(strided, base.transpose(0, 1))
    assert torch.equal(rz.RzEmbedding(V, D, hashed_weight=w)(ids.int()), base)
    half = rz.RzEmbedding(V, D, hashed_weight=w, out_dtype=torch.float16)(ids)
    assert half.dtype == torch.float16 and torch.equal(half, base.half())
    half.sum().backward()
    # an expanded gradient (stride 0) and a transposed one give what their contiguous copies give, to the order of additions
    grads = []
    for g in (torch.ones((), device=DEV).expand(50, 4, D), torch.ones(D, 50, 4, device=DEV).permute(1, 2, 0)):
        (dh,) = torch.autograd.grad(rz.RzEmbedding(V, D, hashed_weight=w)(ids), w, g)
        grads.append(dh)
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], w.grad)       # (sums of ones are exact in any order)
    wb = torch.nn.Parameter(w.detach().bfloat16())
    out = rz.RzEmbedding(V, D, hashed_weight=wb)(ids)
    assert out.dtype == BF16 and torch.equal(out, wb.detach().float()[torch.from_numpy(
        words_of(ids.cpu().numpy().ravel(), np.ones(200, bool), V, D, 4096, 32, 64,
                 rz.RzEmbedding(V, D, hashed_weight=w)._random_numbers.tolist(), 1)).to(DEV)].view(50, 4, D).bfloat16())
    (dwb,) = torch.autograd.grad(out.float().sum(), wb)
    assert dwb.dtype == BF16


def test_embedding_gradient_without_a_plan(rz, rzlib):
    T, V, D, BK, BN, H = 5000, 300, 1024, 32, 64, 9000
    R = numbers(5, 1)
    ids = torch.randint(0, V, (T,), device=DEV)
    g = torch.ones(T, D, device=DEV)                                               # (sums of ones are exact in any order)
    pb = rzlib.make_problem(T, V, D, H, BK, BN, R, 1, rzlib.F32, rzlib.PREC_FP32)
    alone = torch.empty(H, device=DEV)
    rzlib.embedding_backward(pb, ids, -1, g, alone)
    plan, out, planned = rzlib.embedding_plan(pb, torch.device(DEV)), torch.empty(T, D, device=DEV), torch.empty(H, device=DEV)
    rzlib.embedding_forward(pb, ids, -1, torch.randn(H, device=DEV), out, plan)
    rzlib.embedding_backward(pb, ids, -1, g, planned, plan)
    assert torch.equal(alone, planned)
    rzlib.embedding_backward(rzlib.with_fields(pb, flags=rzlib.FLAG_ACCUMULATE_DH), ids, -1, g, planned, plan)
    assert torch.equal(planned, 2 * alone)


def test_embedding_empty_and_no_tokens(rz):
    layer = rz.RzEmbedding(100, 64, compress_ratio=0.5).to(DEV)
    out = layer(torch.empty((0, 5), dtype=torch.int64, device=DEV))
    assert out.shape == (0, 5, 64)
    out.sum().backward()
    assert float(layer._hashed_weight.grad.abs().sum()) == 0.0
    out = layer(torch.full((3,), 100, device=DEV))     # ids that select nothing
    layer._hashed_weight.grad = None
    out.sum().backward()
    assert float(out.detach().abs().sum()) == 0.0 and float(layer._hashed_weight.grad.abs().sum()) == 0.0


@pytest.mark.parametrize("T", [1500, 40000])
def test_embedding_on_another_stream_and_in_a_graph(rz, T):
    V, D = 2000, 128
    layer = rz.RzEmbedding(V, D).to(DEV)
    w = layer._hashed_weight
    ids = torch.randint(0, V, (T,), device=DEV)
    g = torch.ones(T, D, device=DEV)                    # (sums of ones: any order gives the same bits)

    def step():
        out = layer(ids)
        return out.detach(), torch.autograd.grad(out, w, g)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    side.synchronize()
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    ids.copy_(torch.randint(0, V, (T,), device=DEV))
    with torch.no_grad():
        w.mul_(0.5)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_embedding_beyond_32_bit_offsets(rz):
    # 4.3e9 entries of output and gradient: the last rows are looked up, and their gradients added, as the first
    T, V, D = 33000, 300, 131072
    assert T * D > 2**32
    layer = rz.RzEmbedding(V, D, hashed_weight=torch.nn.Parameter(torch.randn(1 << 20, device=DEV)), out_dtype=BF16)
    ids = torch.randint(0, V, (T,), device=DEV)
    out = layer(ids)
    for t in (0, T // 2, T - 2, T - 1):
        assert torch.equal(out[t], layer(ids[t:t + 1])[0])
    (whole,) = torch.autograd.grad(out, layer._hashed_weight, torch.ones((), device=DEV, dtype=BF16).expand(T, D))
    count = torch.bincount(ids, minlength=V)
    rows = layer(torch.arange(V, device=DEV))
    (each,) = torch.autograd.grad(rows, layer._hashed_weight, count[:, None].to(BF16).expand(V, D))
    # counts up to 256 are whole in bf16 and every word's sum is a whole number below 2^24: exact in any order
    assert int(count.max()) <= 256 and float(whole.max()) < 2**24 and torch.equal(whole, each)
