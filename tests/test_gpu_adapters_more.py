"""Adapters: a table beyond 32-bit counts as it lies, gradients of float32 low-rank values, a training step's values."""
import pytest
import torch

import _bounds
from scattermoe_amd import ParallelAdapters
from test_gpu_adapters import DEV, DTYPES, _inputs, _step, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [40, 400])
def test_a_table_of_more_elements_than_32_bits_count(T):
    """2047 adapters of 512 x 2112 in one contiguous tensor of 2.2e9 elements, the used ones at both ends and in the middle; what the others hold is
    not met (the first factor's; it is too large to copy for nothing)."""
    R, r, d, n = 2047, 512, 2112, 64
    i, dy = _inputs(T, d, n, 4, r, torch.bfloat16, seed=16)
    want = _want(i, dy)
    used = torch.tensor([0, 1023, 2045, 2046], device=DEV)
    ids = i["adapter_idxs"]
    inside = (ids >= 0) & (ids < 4)
    s = dict(i, adapter_idxs=torch.where(inside, used[ids.clamp(0, 3)], torch.full_like(ids, R)))
    for name, shape in (("lora_a", (R, r, d)), ("lora_b", (R, n, r))):
        s[name] = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=DEV)
        s[name][used] = i[name]
        assert s[name].is_contiguous()
    assert s["lora_a"].numel() > 2 ** 31 and (R - 1) * r * d > 2 ** 31
    s["scales"] = torch.ones(R, device=DEV)
    s["scales"][used] = i["scales"]
    y, grads = _step(s, dy, ["x"])
    _bounds.check("y", y, *want["y"])
    _bounds.check("dx", grads["x"], *want["dx"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d,n,R,r", [(50, 128, 96, 3, 8), (500, 256, 512, 4, 16), (3000, 1856, 1024, 3, 24)])
def test_gradients_of_the_factors_take_float32_values(T, d, n, R, r, dtype):
    """Not the two parts of 16 bits that the products take."""
    i, dy = _inputs(T, d, n, R, r, dtype, seed=T)
    _, grads = _step(i, dy, ["lora_a", "lora_b"])
    want = _bounds.adapters(i["x"], i["weight"], i["lora_a"], i["lora_b"], i["adapter_idxs"], i["scales"], None, dy, held_in_gradients=False)
    _bounds.check("da", grads["lora_a"], *want["da"])
    _bounds.check("db", grads["lora_b"], *want["db"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_training_step(dtype):
    """An optimizer's step over the adapters of a frozen projection: the gradients of the module's output and the step they make."""
    g = torch.Generator().manual_seed(0)
    m = ParallelAdapters(3, 64, 48, 8, bias=True, scale=0.7).to(DEV).to(dtype)
    m.weight.requires_grad_(False), m.bias.requires_grad_(False)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, generator=g) * 0.25)
    opt = torch.optim.SGD([m.lora_a, m.lora_b], lr=0.5)
    x = torch.randn(40, 64, generator=g).to(dtype).to(DEV)
    ids, dy = torch.randint(-1, 3, (40,), generator=g).to(DEV), torch.randn(40, 48, generator=g).to(dtype).to(DEV)
    before = m.lora_a.detach().clone(), m.lora_b.detach().clone()
    assert m.scales.dtype == torch.float32
    y = m(x, ids)
    y.backward(dy)
    want = _bounds.adapters(x, m.weight, *before, ids, m.scales, m.bias, dy)
    _bounds.check("y", y, *want["y"])
    assert m.weight.grad is None and m.bias.grad is None
    for p, old, key in ((m.lora_a, before[0], "da"), (m.lora_b, before[1], "db")):
        _bounds.check(key, p.grad, *want[key])
    opt.step()
    for p, old in zip((m.lora_a, m.lora_b), before):
        assert torch.equal(p.detach(), torch.add(old, p.grad, alpha=-0.5)) and not torch.equal(p.detach(), old)
