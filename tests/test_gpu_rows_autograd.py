"""Lookup and grouped products under autograd's hooks: saved tensors that leave the GPU, checkpoints, graphs used twice.

Tolerances: none.  Gradients, activations and weights are small whole numbers, so sums are exact in any order (below 2^24).
"""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def rz(rzlib):
    assert torch.cuda.is_available(), "these tests need a GPU"
    rzlib.load()
    import rzlinear_b200
    return rzlinear_b200


def whole(*shape, dtype=torch.float32):
    return torch.randint(-2, 3, shape, device=DEV).to(dtype)


def lookup(rz):
    T, V, D = 5000, 700, 1024                                  # long enough for a plan
    weight = whole(20000).requires_grad_()
    ids, g = torch.randint(-2, V, (T,), device=DEV), whole(T, D)
    args = (torch.tensor([45007, 5, 7, 11, 13, 17, 19, 23]), V, D, 1.0)
    return lambda w: rz.RzEmbeddingFunction.apply(ids, w, *args), [weight], g


def products(rz):
    M, K, N = 300, 128, 192
    x, weight, bias = (t.requires_grad_() for t in (whole(M, K, dtype=BF16), whole(9000), whole(3, N)))
    off, g = torch.tensor([0, 100, 100, 290], dtype=torch.int32, device=DEV), whole(M, N, dtype=BF16)
    R, cfg = torch.tensor([45007, 5, 7, 11, 13, 17, 19, 23]), rz.RzConfig(relu=True)
    return lambda x, w, b: rz.RzGroupedLinearFunction.apply(x, w, R, off, N, 1.0, cfg, b), [x, weight, bias], g


@pytest.mark.parametrize("make", [lookup, products])
def test_saved_tensors_may_leave_the_gpu(rz, make):
    call, leaves, g = make(rz)
    out = call(*leaves)
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    again = torch.autograd.grad(out, leaves, g)
    with torch.autograd.graph.save_on_cpu():
        out = call(*leaves)
    moved = torch.autograd.grad(out, leaves, g)
    kept = checkpoint(call, *leaves, use_reentrant=False)
    once_more = torch.autograd.grad(kept, leaves, g)
    for got in (again, moved, once_more):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_checkpoint_around_a_layer_that_wants_a_longer_buffer(rz):
    # the linear layer replaces the weight's buffer of shifted copies by a longer one between a grouped call and its recomputation
    call, (x, weight, bias), g = products(rz)
    want = torch.autograd.grad(call(x, weight, bias), (x, weight, bias), g)
    rz.impl.launchers.drop_shadow_cache(weight)
    kept = checkpoint(call, x, weight, bias, use_reentrant=False)
    R = torch.tensor([45007, 5, 7, 11, 13, 17, 19, 23])
    rz.RzLinearFunction.apply(whole(64, 1024, dtype=BF16), weight.detach(), R, 4096, 0, 1.0)
    before = [e["shadow"].numel() for e in weight._rz_shadow_cache.values()]
    rz.RzLinearFunction.apply(whole(64, 1024, dtype=BF16), weight, R, 4096, 0, 1.0)
    assert [e["shadow"].numel() for e in weight._rz_shadow_cache.values()] > before
    got = torch.autograd.grad(kept, (x, weight, bias), g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_plan_goes_with_the_backward(rz):
    call, leaves, g = lookup(rz)
    for _ in range(2):                                         # (the first pass gets the caching allocator its blocks)
        out = call(*leaves)
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(out, leaves, g)
        freed = before + sum(-(-t.numel() * t.element_size() // 512) * 512 for t in grads) - torch.cuda.memory_allocated()
    assert freed >= 8 * 5000                                   # though the output lives
