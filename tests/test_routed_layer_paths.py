"""Which way a layer with its router goes, and that both give the same, without a GPU."""
import pytest
import torch

import oracle  # noqa: F401  (the test double's)
from scattermoe_amd.kernels import ops
from test_few_tokens_and_adapters import _Backend, _layer


class _Library(_Backend):
    """The library's kernels know nothing of autocast, the double's products do."""

    def __getattribute__(self, name):
        call = object.__getattribute__(self, name)

        def plain(*args):
            with torch.autocast("cpu", enabled=False):
                return call(*args)
        return plain if callable(call) else call


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
