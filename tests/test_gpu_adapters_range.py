"""Low-rank values (u in the forward pass, v in the backward one) beyond what the operands' type holds, large and small: they are
float32 whatever the number of rows, in the row kernels and in the tiles."""
import pytest
import torch

import _bounds
from scattermoe_amd import ParallelAdapters, parallel_adapters
from test_gpu_adapters import DEV, _inputs, _step, _want

pytestmark = pytest.mark.gpu


def _scaled(i, adapters, factors):
    """Low-rank values `adapters` times as large, the factor behind them `factors` times (both powers of two)."""
    return dict(i, scales=i["scales"] * adapters, **{n: (i[n].float() * f).to(i[n].dtype) for n, f in factors.items()})


# 64 rows: row by row; 65 and 100: by the work; 400 and 3000: tiles of every class (3000 x 1856: one wave per SIMD)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("r", [8, 16, 40])
@pytest.mark.parametrize("T,d,n", [(64, 128, 96), (65, 2048, 2048), (400, 128, 96), (700, 1024, 1024), (3000, 1856, 4096), (3000, 520, 3584)])
@pytest.mark.parametrize("log", [17, -24])
def test_large_and_small_low_values(log, T, d, n, r, dtype):
    i, dy = _inputs(T, d, n, 5, r, dtype, bias=True, seed=T + r)
    # u is scales * A x: large against a small B, small against a large one
    s = _scaled(i, 2.0 ** log, {"lora_b": 2.0 ** (-10 if log > 0 else 8)})
    y, _ = _step(s, dy, ["x"])
    want = _want(s)["y"]
    assert float(want[0].abs().max()) < 60000
    _bounds.check("y", y, *want)
    # v is scales * B^T dy: the same with A behind it
    s = _scaled(i, 2.0 ** log, {"lora_a": 2.0 ** (-10 if log > 0 else 8)})
    _, grads = _step(s, dy, ["x"])
    want = _want(s, dy)["dx"]
    assert float(want[0].abs().max()) < 60000
    _bounds.check("dx", grads["x"], *want)


@pytest.mark.parametrize("T", [64, 400, 3000])
def test_large_low_values_beside_a_factor_of_zeros(T):
    """A module as it is initialised: W x alone, whatever A x is."""
    i, dy = _inputs(T, 256, 192, 4, 16, torch.float16, bias=True, seed=T)
    s = _scaled(i, 2.0 ** 17, {})
    s["lora_b"] = torch.zeros_like(i["lora_b"])
    y, _ = _step(s, dy, ["x"])
    _bounds.check("y", y, *_want(s)["y"])
    assert torch.equal(y, parallel_adapters(**dict(s, adapter_idxs=torch.full_like(s["adapter_idxs"], -1))))


@pytest.mark.parametrize("T", [65, 400, 3000])
def test_one_large_rank_among_small_ones(T):
    """A row's ranks far apart, in one block of 16 and in several; the largest beside zeros of B, which leaves the others."""
    i, dy = _inputs(T, 1024, 4096 if T == 65 else 192, 4, 40, torch.float16, seed=T + 1)
    for rank in (3, 20, 39):
        s = dict(i, lora_a=i["lora_a"].clone())
        s["lora_a"][:, rank] *= 2.0 ** 12
        s["scales"] = i["scales"] * 2.0 ** 5
        s["lora_b"] = (i["lora_b"].float() * 2.0 ** -8).half()
        s["lora_b"][:, :, rank] = 0.0
        y, _ = _step(s, dy, ["x"])
        _bounds.check("y", y, *_want(s)["y"])


@pytest.mark.parametrize("T", [400, 3000])
@pytest.mark.parametrize("log", range(-34, 1, 2))
def test_small_ranks_beside_ordinary_ones(log, T):
    """A block of 16 ranks far below the row's largest: what is left of it counts as long as float16 can hold it beside the others."""
    i, dy = _inputs(T, 128 if T == 400 else 1856, 192, 4, 40, torch.float16, seed=T - log)
    for block in (slice(0, 16), slice(16, 32), slice(32, 40)):
        s = dict(i, lora_a=i["lora_a"].clone(), lora_b=i["lora_b"].clone())
        up = min(8, -log)                                # (a small value in front of a large factor)
        s["lora_a"][:, block] = (s["lora_a"][:, block].float() * 2.0 ** log).half()
        s["lora_b"][:, :, block] = (s["lora_b"][:, :, block].float() * 2.0 ** up).half()
        y, _ = _step(s, dy, ["x"])
        _bounds.check("y", y, *_want(s)["y"])


@pytest.mark.parametrize("T", [65, 400, 3000])
def test_an_infinite_low_value(T):
    """... makes the outputs infinite that it adds to, and those of its row alone."""
    i, dy = _inputs(T, 1024, 4096 if T == 65 else 192, 4, 40, torch.float16, bare=0.0, seed=T + 2)
    want = parallel_adapters(**i)
    s = dict(i, scales=i["scales"].clone(), lora_a=i["lora_a"].clone(), lora_b=i["lora_b"].clone())
    s["lora_a"][1, 7] = 60000.0
    s["scales"][1] = 3e38
    s["lora_b"][1, :, :] = 0.5
    s["x"] = i["x"].abs() + 0.125                     # (one sign: infinity, no difference of infinities)
    s["lora_a"][1] = s["lora_a"][1].abs() + 0.125
    got, rows = parallel_adapters(**s), i["adapter_idxs"] == 1
    assert bool(rows.any()) and bool(torch.isinf(got[rows]).all())
    assert torch.equal(got[~rows], parallel_adapters(**dict(s, adapter_idxs=torch.where(rows, -1, i["adapter_idxs"])))[~rows])
    assert bool(torch.isfinite(want).all())


def test_module_with_loss_scaling():
    """float16 training as it is done: the loss, and with it v, times 2^16; B at its initial zeros but for a few values."""
    torch.manual_seed(0)
    m = ParallelAdapters(3, 128, 192, 8).to(DEV).half()
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        m.lora_b[:, ::7] = (torch.randn(m.lora_b[:, ::7].shape, generator=g) * 8).half()
        m.lora_a.mul_(2.0 ** -10)
    x = torch.randn(400, 128, generator=g).half().to(DEV).requires_grad_()
    ids = torch.randint(0, 3, (400,), generator=g).to(DEV)
    dy = (torch.randn(400, 192, generator=g) * 2.0 ** 13).half().to(DEV)
    (dx,) = torch.autograd.grad(m(x, ids), x, dy)
    want = _bounds.adapters(x.detach(), m.weight, m.lora_a, m.lora_b, ids, m.scales, None, dy)["dx"]
    assert float((dy.double() @ m.lora_b[0].double()).abs().max()) > 65504
    _bounds.check("dx", dx, *want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_more_columns_in_a_tile_row_than_a_round(dtype):
    """A projection to a vocabulary: the tiles of one row are more than the CUs."""
    i, dy = _inputs(200, 160, 65800, 3, 8, dtype, seed=5)
    y, grads = _step(i, dy, ["x"])
    want = _want(i, dy)
    _bounds.check("y", y, *want["y"])
    _bounds.check("dx", grads["x"], *want["dx"])
