"""Forward-mode derivatives, which no function of the library has: asked for, they are refused and never lost, also where nothing asks
for a gradient and a call would pass its autograd function by."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import oracle  # noqa: F401  (the test double's)
from scattermoe_amd import ParallelAdapters, parallel_adapters
from scattermoe_amd.mlp import GLUMLP, RoutedGLUMLP, routed_glu_mlp
from test_few_tokens_and_adapters import _Backend
from scattermoe_amd.kernels import ops


class _Pointers(_Backend):
    """A backend as the library is one: it sees the tensors' memory, and no derivative comes out of it."""

    def __getattribute__(self, name):
        call = object.__getattribute__(self, name)

        def without(*args):
            return call(*(a.detach() if isinstance(a, torch.Tensor) else a for a in args))
        return without if callable(call) else call


@pytest.fixture
def backend(monkeypatch):
    monkeypatch.setattr(ops, "_backend", _Pointers())


def _cases():
    torch.manual_seed(0)
    rows, ids = torch.randn(5, 16), torch.tensor([0, 2, -1, 1, 1])
    a = dict(x=rows, weight=torch.randn(12, 16), lora_a=torch.randn(3, 4, 16), lora_b=torch.randn(3, 12, 4), bias=torch.randn(12),
             scales=torch.ones(3))
    layer = dict(x=rows, router_weight=torch.randn(6, 16), w1=torch.randn(6, 16, 16), w2=torch.randn(6, 16, 8), b1=torch.randn(6, 16),
                 b2=torch.randn(6, 16))
    return {"adapters": (lambda **kw: parallel_adapters(adapter_idxs=ids, **kw), a),
            "layer": (lambda **kw: routed_glu_mlp(k=2, **kw), layer)}


CASES = [("adapters", n) for n in ("x", "weight", "lora_a", "lora_b", "bias", "scales")]
CASES += [("layer", n) for n in ("x", "router_weight", "w1", "w2", "b1", "b2")]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which,name", CASES)
def test_tangents_are_refused(which, name, grad, backend):
    call, kw = _cases()[which]
    call(**kw)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        call(**kw)                                       # (nothing asks for one)
        dual = forward_ad.make_dual(kw[name], torch.randn(kw[name].shape))
        with pytest.raises(NotImplementedError):
            call(**dict(kw, **{name: dual}))


@pytest.mark.parametrize("which", ["adapters", "layer"])
def test_transforms_are_refused(which, backend):
    call, kw = _cases()[which]
    x = kw.pop("x")
    out = lambda x: (lambda y: y[0] if isinstance(y, tuple) else y)(call(x=x, **kw))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(out, (x,), (torch.ones_like(x),))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda x: out(x).sum())(x)


@pytest.mark.parametrize("grad", [True, False])
def test_modules(grad, backend):
    x, ids = torch.randn(3, 16), torch.tensor([0, 1, -1])
    gates, experts = torch.rand(3, 2), torch.tensor([[0, 1], [2, 3], [1, 0]])
    adapters, layer, mlp = ParallelAdapters(2, 16, 8, 4), RoutedGLUMLP(16, 8, 4, 2), GLUMLP(16, 8, 4, 2)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: adapters(dual, ids), lambda: layer(dual), lambda: mlp(dual, gates, experts)):
            with pytest.raises(NotImplementedError):
                call()
