"""float32 products beside adapters in tiles: both sizes of tile, forward and, with the weight as it lies, for the input's gradient."""
import pytest
import torch

import _bounds
from scattermoe_amd import parallel_adapters
from test_gpu_adapters import DEV, _compare, _inputs, _step, _want

pytestmark = pytest.mark.gpu


# 64 x 64 and, with 2048 rows and more, 128 x 128; rows, columns and contractions that no tile or slice divides; ranks beyond a block of 16
@pytest.mark.parametrize("T,d,n,R,r,grouped", [(1024, 1024, 1024, 8, 16, False), (1000, 1003, 1517, 5, 7, False), (700, 1500, 1501, 40, 33, True),
                                                (1030, 2050, 1000, 1, 1, False), (2048, 1536, 2000, 3, 40, False), (2047, 1999, 2001, 64, 16, True),
                                                (300, 4099, 2300, 300, 8, False), (4100, 600, 1100, 7, 20, False)])
def test_values_and_gradients(T, d, n, R, r, grouped):
    i, dy = _inputs(T, d, n, R, r, torch.float32, bias=T % 2 == 0, grouped=grouped, seed=T + d)
    _compare(i, dy)


@pytest.mark.parametrize("which", ["none", "one", "last"])
def test_rows_without_and_with_one_adapter(which):
    i, dy = _inputs(1024, 1100, 1000, 6, 8, torch.float32, seed=7)
    ids = torch.full((1024,), -1 if which != "one" else 4, dtype=torch.int64, device=DEV)
    if which == "last":
        ids[-1] = 5
    i["adapter_idxs"] = ids
    _compare(i, dy)


def test_strided_operands():
    """Rows apart, factors stored the other way round, a weight and rows that start at any multiple of four bytes."""
    T, d, n = 900, 1030, 1201
    i, dy = _inputs(T, d, n, 4, 12, torch.float32, bias=True, seed=8)
    wide = torch.cat([i["x"], i["x"]], 1)
    flat = torch.empty(n * d + 1, device=DEV)
    s = dict(i, x=wide[:, 515:515 + d], weight=flat[1:].view(n, d), lora_a=i["lora_a"].transpose(1, 2).contiguous().transpose(1, 2),
             lora_b=i["lora_b"].transpose(1, 2).contiguous().transpose(1, 2))
    s["weight"].copy_(i["weight"])
    _compare(s, dy.t().contiguous().t())
    _compare(dict(i, weight=i["weight"].t().contiguous().t(), x=i["x"][:1].expand(T, d)), dy[:1].expand(T, n))


def test_values_that_are_not_finite_stay_in_their_rows():
    i, dy = _inputs(1024, 1024, 1100, 5, 8, torch.float32, bare=0.2, seed=21)
    y, grads = _step(i, dy)
    ids = i["adapter_idxs"]
    for a in (0, 2, 4):
        s = dict(i, x=i["x"].clone(), lora_a=i["lora_a"].clone(), lora_b=i["lora_b"].clone())
        s["lora_a"][a, 2] = float("inf")
        s["lora_b"][a, 9] = float("nan")
        row = int((ids != a).nonzero()[3])
        s["x"][row, 700] = float("nan")
        got, g = _step(s, dy, ["x"])
        keep = ids != a
        assert torch.equal(g["x"][keep], grads["x"][keep])
        keep[row] = False
        assert torch.equal(got[keep], y[keep]) and bool(torch.isnan(got[ids == a, 9]).all()) and bool(torch.isnan(got[row]).all())


def test_same_bits_every_time_on_another_stream_and_from_a_graph():
    i, dy = _inputs(1024, 1024, 1000, 6, 16, torch.float32, seed=13)
    y, grads = _step(i, dy)
    side = torch.cuda.Stream()
    for _ in range(2):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2, grads2 = _step(i, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = parallel_adapters(**i)
    for r in range(3):
        g = torch.Generator().manual_seed(r)
        i["x"].copy_(torch.randn(1024, 1024, generator=g))
        i["adapter_idxs"].copy_(torch.randint(-1, 7, (1024,), generator=g))
        graph.replay()
        want = parallel_adapters(**i)
        torch.cuda.synchronize()
        assert torch.equal(out, want), r


def test_a_row_is_the_same_among_others():
    """... in tiles of either size: its values depend neither on its place nor on the other rows."""
    i, _ = _inputs(2048, 1024, 2000, 4, 16, torch.float32, bare=0.1, seed=14)
    whole = parallel_adapters(**i)
    order = torch.randperm(2048, generator=torch.Generator().manual_seed(0)).to(DEV)
    assert torch.equal(parallel_adapters(**dict(i, x=i["x"][order], adapter_idxs=i["adapter_idxs"][order])), whole[order])
    y, bound = _want(dict(i, x=i["x"][:1000], adapter_idxs=i["adapter_idxs"][:1000]))["y"]
    _bounds.check("fewer rows", parallel_adapters(**dict(i, x=i["x"][:1000], adapter_idxs=i["adapter_idxs"][:1000])), y, bound)
