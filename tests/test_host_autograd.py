"""What the layers that pick rows by an index tell autograd, with the kernels replaced by host functions (no GPU needed)."""
import weakref

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import rzlinear_b200 as rz
from rzlinear_b200 import _lib
from rzlinear_b200.impl import launchers


@pytest.fixture
def on_the_host(rzlib, monkeypatch):
    """Kernels that fill their results with ones."""
    def fill(*tensors):
        for t in tensors:
            if t is not None:
                t.fill_(1)
    monkeypatch.setattr(rzlib, "_require_together", lambda *tensors: None)
    monkeypatch.setattr(rzlib, "embedding_forward", lambda pb, ids, padding, hashed, out, plan=None: fill(out, plan))
    monkeypatch.setattr(rzlib, "embedding_backward", lambda pb, ids, padding, dout, dh, plan=None: fill(dh))
    monkeypatch.setattr(launchers, "cached_shadow", lambda pb, weight, hashed, nbytes=None: torch.zeros(nbytes or 1, dtype=torch.uint8))
    monkeypatch.setattr(rzlib, "grouped_forward", lambda pb, groups, off, x, hashed, copies, bias, y, ws: fill(y))
    monkeypatch.setattr(rzlib, "grouped_backward",
                        lambda pb, groups, off, x, dy, y, hashed, copies, dym, db, dx, dh, ws: fill(db, dx, dh))


def embedding_call(weight=None):
    layer = rz.RzEmbedding(1000, 64)
    ids = torch.randint(0, 1000, (5,))
    args = [ids, layer._hashed_weight if weight is None else weight, layer._random_numbers, 1000, 64, 1.0]
    return args


def grouped_call():
    layer = rz.RzGroupedLinear(4, 128, 64, compress_ratio=0.5)
    off = torch.tensor([0, 1, 1, 4, 6], dtype=torch.int32)
    return [torch.randn(6, 128), layer._hashed_weight, layer._random_numbers, off, 64, 1.0, None, layer._bias]


@pytest.mark.parametrize("function,make,which", [(rz.RzEmbeddingFunction, embedding_call, 1), (rz.RzGroupedLinearFunction, grouped_call, 0),
                                                 (rz.RzGroupedLinearFunction, grouped_call, 1), (rz.RzGroupedLinearFunction, grouped_call, 7)])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("leaf", [True, False])
def test_tangents_are_refused_not_dropped(on_the_host, function, make, which, grad_mode, leaf):
    # forward-mode derivatives are not offered: a call that carries one has to say so, since a result without a tangent counts as constant
    args = [a.detach() if isinstance(a, torch.Tensor) else a for a in make()]
    primal = args[which].clone().requires_grad_(leaf)
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(primal, torch.ones_like(primal))
        with torch.set_grad_enabled(grad_mode), pytest.raises(NotImplementedError):
            function.apply(*args)
        args[which] = primal.detach()      # without one, inside a level: an ordinary call
        out = function.apply(*args)
        assert forward_ad.unpack_dual(out).tangent is None and float(out.min()) == 1.0


class Held:
    """What a saved-tensor hook keeps of a tensor."""

    def __init__(self, tensor):
        self.tensor = tensor


@pytest.mark.parametrize("function", [rz.RzEmbeddingFunction, rz.RzGroupedLinearFunction])
@pytest.mark.parametrize("retain", [False, True])
def test_buffers_of_the_backward_are_saved_tensors(on_the_host, function, retain):
    # the plan of a lookup and the shifted copies of a grouped product are seen by hooks (offloading, checkpoints), and go when the
    # backward has run, like all that autograd saves
    if function is rz.RzEmbeddingFunction:
        tokens, V, D = 4100, 1000, 1024                       # long enough for a plan
        weight = torch.randn(V * D // 16).requires_grad_()
        args = [torch.randint(0, V, (tokens,)), weight, rz.RzEmbedding(V, D)._random_numbers, V, D, 1.0]
        nbytes = 8 * tokens
    else:
        args = grouped_call()
        weight = args[1]
        pb = launchers.cached_problem(6, 128, 64, weight.numel(), args[2], 32, 64, torch.float32, False, 1.0, 1)
        nbytes = _lib.grouped_sizes(pb, 4)[0] or 1
    held = weakref.WeakSet()

    def pack(tensor):
        kept = Held(tensor)
        held.add(kept)
        return kept

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda kept: kept.tensor):
        out = function.apply(*args)
    assert [k.tensor.numel() for k in held if k.tensor.dtype == torch.uint8] == [nbytes]
    for _ in range(2 if retain else 1):
        (grad,) = torch.autograd.grad(out, weight, torch.ones_like(out), retain_graph=retain)
        assert float(grad.min()) == 1.0
    assert bool(len(held)) == retain
