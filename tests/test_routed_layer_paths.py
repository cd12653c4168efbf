"""Which way a layer with its router goes, and that both give the same, without a GPU."""
import pytest
import torch

import oracle  # noqa: F401  (the test double's)
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import routed_glu_mlp
from test_few_tokens_and_adapters import _Backend, _layer


class _Library(_Backend):
    """The library's kernels know nothing of autocast, the double's products do."""

    def __getattribute__(self, name):
        call = object.__getattribute__(self, name)

        def plain(*args):
            with torch.autocast("cpu", enabled=False):
                return call(*args)
        return plain if callable(call) else call

    # (the double's views have no shape without rows)
    @staticmethod
    def combine(Y, gates, out, k):
        if out.numel():
            _Backend.combine(Y, gates, out, k)

    @staticmethod
    def gate_grad(Y, d_out, d_gates, k):
        if d_out.numel():
            _Backend.gate_grad(Y, d_out, d_gates, k)


@pytest.fixture
def backend(monkeypatch):
    monkeypatch.setattr(ops, "_backend", _Library())


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("T", [5, 100])
def test_autocast_leaves_the_logits(T, train, backend):
    """float32 logits, of every way, whatever autocast would make of a product."""
    m, x = _layer(), torch.randn(T, 16)
    with torch.set_grad_enabled(train):
        want, want_logits = m(x)
        with torch.autocast("cpu", dtype=torch.bfloat16):
            out, logits = m(x)
    assert logits.dtype == torch.float32 and torch.equal(logits, want_logits) and torch.equal(out, want)


def test_autocast_in_a_compiled_step(backend):
    m, x = _layer(), torch.randn(100, 16)
    want = m(x)
    torch._dynamo.reset()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        out, logits = torch.compile(m, fullgraph=True, backend="aot_eager")(x)
    assert logits.dtype == torch.float32
    torch.testing.assert_close(logits, want[1], rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(out, want[0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("turned", [(), ("w1",), ("w2",), ("w1", "w2")])
@pytest.mark.parametrize("T,d,F,one_call", [(1, 16, 24, True), (64, 128, 64, True), (64, 512, 160, False), (5, 2048, 512, False)])
def test_weights_of_a_strided_contraction(T, d, F, one_call, turned, backend, monkeypatch):
    """(E, in, out) weights, which the general path takes as they lie, go there unless they are small: the few-token kernels that take
    any layout read a line of memory per element."""
    E, k, calls = 4, 2, []
    plain = ops._backend.routed_glu_mlp
    monkeypatch.setattr(_Library, "routed_glu_mlp", staticmethod(lambda *a: calls.append(a[0]) or plain(*a)))
    g = torch.Generator().manual_seed(T)
    x, wr = torch.randn(T, d, generator=g), torch.randn(E, d, generator=g)
    w = {"w1": torch.randn(E, 2 * F, d, generator=g) * d ** -0.5, "w2": torch.randn(E, d, F, generator=g) * F ** -0.5}
    want = routed_glu_mlp(x, wr, w["w1"], w["w2"], k)
    assert len(calls) == 1
    s = {n: t.transpose(1, 2).contiguous().transpose(1, 2) if n in turned else t for n, t in w.items()}
    got = routed_glu_mlp(x, wr, s["w1"], s["w2"], k)
    assert len(calls) == (2 if one_call or not turned else 1)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


def test_columns_of_the_tokens_are_contiguous_in_the_library(backend, monkeypatch):
    calls = []
    plain = ops._backend.routed_glu_mlp
    monkeypatch.setattr(_Library, "routed_glu_mlp", staticmethod(lambda *a: calls.append(a[0]) or plain(*a)))
    m, x = _layer(), torch.randn(5, 16)
    with torch.no_grad():
        want, got = m(x), m(x.t().contiguous().t())
        rows = m(torch.cat([x, x], 1)[:, :16])
    assert [t.stride() for t in calls] == [(16, 1), (16, 1), (32, 1)]
    assert all(torch.equal(a, b) for other in (got, rows) for a, b in zip(other, want))


def test_a_training_step_without_tokens(backend):
    m, x = _layer(), torch.randn(0, 16, requires_grad=True)
    out, logits = m(x)
    assert out.requires_grad and logits.requires_grad and out.shape == (0, 16) and logits.shape == (0, 6)
    (out.sum() + logits.sum()).backward()
    assert x.grad.shape == (0, 16)
    assert all(p.grad is not None and not bool(p.grad.any()) for p in m.parameters())
