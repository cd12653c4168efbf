"""float32 products beside adapters in tiles: both sizes of tile, forward and, with the weight as it lies, for the input's gradient."""
import pytest
import torch

import _bounds
from scattermoe_amd import parallel_adapters
from test_gpu_adapters import DEV, _compare, _inputs, _step, _want

pytestmark = pytest.mark.gpu


# Tiles of 64 x 64 and 128 x 128, whole or their slices dealt out; rows, columns and contractions that no tile or slice divides; ranks beyond
# a block of 16; adapters of less than a block of 16 rows and of many tiles
SHAPES = [(1024, 1024, 1024, 8, 16, False), (1000, 1003, 1517, 5, 7, False), (700, 1500, 1501, 40, 33, True), (1030, 2050, 1000, 1, 1, False),
          (2048, 1536, 2000, 3, 40, False), (2047, 1999, 2001, 64, 16, True), (300, 4099, 2300, 300, 8, False), (4100, 600, 1100, 7, 20, False),
          (65, 4096, 4096, 3, 8, False), (320, 4100, 2051, 9, 40, True), (1020, 1472, 2051, 1, 64, True), (520, 2999, 3001, 200, 5, False),
          (129, 8200, 1030, 4, 130, False), (300, 4, 4, 5, 3, False)]


@pytest.mark.parametrize("T,d,n,R,r,grouped", SHAPES)
def test_values_and_gradients(T, d, n, R, r, grouped):
    i, dy = _inputs(T, d, n, R, r, torch.float32, bias=T % 2 == 0, grouped=grouped, seed=T + d)
    _compare(i, dy)


# slices dealt out, and whole tiles of 64 x 64 and 128 x 128
WHOLE = [(1024, 1024, 1024), (2048, 1024, 2000)]
SIZES = [(80, 4096, 4096), (400, 2048, 3000), (1024, 1024, 1100)] + WHOLE


@pytest.mark.parametrize("T,d,n", SIZES)
@pytest.mark.parametrize("which", ["none", "one", "last"])
def test_rows_without_and_with_one_adapter(which, T, d, n):
    i, dy = _inputs(T, d, n, 6, 8, torch.float32, seed=7)
    ids = torch.full((T,), -1 if which != "one" else 4, dtype=torch.int64, device=DEV)
    if which == "last":
        ids[-1] = 5
    i["adapter_idxs"] = ids
    _compare(i, dy)


@pytest.mark.parametrize("T,d,n", [(900, 1030, 1201), (300, 2062, 2003), (2048, 1022, 1985)])
def test_strided_operands(T, d, n):
    """Rows apart, factors stored the other way round, a weight and rows that start at any multiple of four bytes."""
    i, dy = _inputs(T, d, n, 4, 12, torch.float32, bias=True, seed=8)
    wide = torch.cat([i["x"], i["x"]], 1)
    flat = torch.empty(n * d + 1, device=DEV)
    s = dict(i, x=wide[:, d // 2:d // 2 + d], weight=flat[1:].view(n, d), lora_a=i["lora_a"].transpose(1, 2).contiguous().transpose(1, 2),
             lora_b=i["lora_b"].transpose(1, 2).contiguous().transpose(1, 2))
    s["weight"].copy_(i["weight"])
    _compare(s, dy.t().contiguous().t())
    _compare(dict(i, weight=i["weight"].t().contiguous().t(), x=i["x"][:1].expand(T, d)), dy[:1].expand(T, n))


@pytest.mark.parametrize("T,d,n", SIZES)
@pytest.mark.parametrize("grouped", [False, True])
def test_values_that_are_not_finite_stay_in_their_rows(T, d, n, grouped):
    i, dy = _inputs(T, d, n, 5, 8, torch.float32, bare=0.2, grouped=grouped, seed=21)
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


@pytest.mark.parametrize("T,d,n", SIZES)
def test_same_bits_every_time_on_another_stream_and_from_a_graph(T, d, n):
    i, dy = _inputs(T, d, n, 6, 16, torch.float32, seed=13)
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
        i["x"].copy_(torch.randn(T, d, generator=g))
        i["adapter_idxs"].copy_(torch.randint(-1, 7, (T,), generator=g))
        graph.replay()
        want = parallel_adapters(**i)
        torch.cuda.synchronize()
        assert torch.equal(out, want), r


@pytest.mark.parametrize("T,d,n", SIZES)
def test_a_row_is_the_same_among_others(T, d, n):
    """In whole tiles its values depend neither on its place among the rows nor on its neighbours' adapters; where slices are dealt out its place
    decides where its sums are cut."""
    i, _ = _inputs(T, d, n, 4, 16, torch.float32, bare=0.1, seed=14)
    whole = parallel_adapters(**i)
    order = torch.randperm(T, generator=torch.Generator().manual_seed(0)).to(DEV)
    got = parallel_adapters(**dict(i, x=i["x"][order], adapter_idxs=i["adapter_idxs"][order]))
    if (T, d, n) in WHOLE:
        assert torch.equal(got, whole[order])
    _bounds.check("other places", got, *_want(dict(i, x=i["x"][order], adapter_idxs=i["adapter_idxs"][order]))["y"])
    y, bound = _want(dict(i, x=i["x"][:T // 2], adapter_idxs=i["adapter_idxs"][:T // 2]))["y"]
    _bounds.check("fewer rows", parallel_adapters(**dict(i, x=i["x"][:T // 2], adapter_idxs=i["adapter_idxs"][:T // 2])), y, bound)


def test_two_calls_at_once():
    """Runs of slices leave their parts in a workspace of each call's own."""
    i, dy = _inputs(320, 2048, 3000, 6, 16, torch.float32, seed=18)
    j = dict(i, x=torch.randn(320, 2048, generator=torch.Generator().manual_seed(3)).to(DEV))
    want = [_step(s, dy, ["x", "lora_a", "lora_b"]) for s in (i, j)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        got = []
        for st, s in zip(streams, (i, j)):
            with torch.cuda.stream(st):
                got.append(_step(s, dy, ["x", "lora_a", "lora_b"]))
        torch.cuda.synchronize()
        for (y, grads), (y2, grads2) in zip(got, want):
            assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads2)
