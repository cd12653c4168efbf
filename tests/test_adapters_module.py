"""ParallelAdapters as a module: its factors keep their type and value, without a GPU."""
import copy

import pytest
import torch

import oracle  # noqa: F401  (the test double's)
from scattermoe_amd import ParallelAdapters
from scattermoe_amd.kernels import ops
from test_few_tokens_and_adapters import _Backend


@pytest.mark.parametrize("change", [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.type(torch.float16),
                                    lambda m: torch.nn.Sequential(m).to(torch.bfloat16)[0], lambda m: m.half().float(),
                                    lambda m: copy.deepcopy(m).to("cpu", torch.bfloat16), lambda m: m.double(), lambda m: m.cpu()])
def test_scales_keep_type_and_value(change):
    m = ParallelAdapters(3, 16, 8, 4, scale=0.7)
    m.scales[1] = 1.2345678
    want = m.scales.clone()
    got = change(m)
    assert got.scales.dtype == torch.float32 and torch.equal(got.scales, want)
    assert "scales" in got.state_dict() and "scales" in dict(got.named_buffers())


def test_scales_of_a_low_default_type_and_of_the_meta_device():
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        m = ParallelAdapters(3, 16, 8, 4, scale=0.7)
    finally:
        torch.set_default_dtype(before)
    assert m.weight.dtype == torch.bfloat16 and m.scales.dtype == torch.float32 and abs(float(m.scales[0]) - 0.7) < 1e-7
    with torch.device("meta"):
        m = ParallelAdapters(3, 16, 8, 4)
    m = m.to(torch.bfloat16)
    assert m.scales.is_meta and m.scales.dtype == torch.float32
    m = m.to_empty(device="cpu")
    assert m.scales.dtype == torch.float32 and m.weight.dtype == torch.bfloat16


def test_state_of_another_type(monkeypatch):
    m = ParallelAdapters(3, 16, 8, 4, scale=0.7).bfloat16()
    m.load_state_dict({k: v.to(torch.bfloat16) for k, v in ParallelAdapters(3, 16, 8, 4, scale=0.5).state_dict().items()})
    assert m.scales.dtype == torch.float32 and bool((m.scales == 0.5).all())


def test_a_call_hands_the_buffer_on_as_it_is(monkeypatch):
    seen = []

    class Spy(_Backend):
        @classmethod
        def adapter_forward(cls, X, W, bias, A, B, ids, scales, idx, off, U, Y):
            seen.append(scales)
            Y.zero_()
    monkeypatch.setattr(ops, "_backend", Spy())
    m = ParallelAdapters(3, 16, 8, 4, scale=0.7).bfloat16()
    with torch.no_grad():
        m(torch.randn(5, 16, dtype=torch.bfloat16), torch.tensor([0, 1, 2, -1, 0]))
    assert seen[0] is m.scales
