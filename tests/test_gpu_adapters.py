"""Low-rank adapters beside a shared projection (adapters.parallel_adapters, ParallelAdapters): values and gradients against
the formulas in 64 bits, with bounds that follow from the roundings (_bounds.py)."""
import pytest
import torch

import _bounds
from scattermoe_amd import ParallelAdapters, parallel_adapters
from scattermoe_amd.mlp import RoutedGLUMLP

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(T, d, n, R, r, dtype, bias=False, bare=0.2, grouped=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(DEV)
    ids = torch.randint(0, R, (T,), generator=g)
    if grouped:
        ids = torch.sort(ids).values
    drop = torch.rand(T, generator=g) < bare
    ids = torch.where(drop, torch.tensor([-1, R, R + 7])[torch.randint(0, 3, (T,), generator=g)], ids)
    return dict(x=f(T, d), weight=f(n, d, std=d ** -0.5), lora_a=f(R, r, d, std=d ** -0.5), lora_b=f(R, n, r, std=r ** -0.5),
                adapter_idxs=ids.to(DEV), scales=(torch.rand(R, generator=g) + 0.5).to(DEV), bias=f(n, std=0.3) if bias else None,
                ), f(T, n)


def _want(i, dy=None):
    return _bounds.adapters(i["x"], i["weight"], i["lora_a"], i["lora_b"], i["adapter_idxs"], i["scales"], i["bias"], dy)


LEAVES = [("dx", "x"), ("dw", "weight"), ("da", "lora_a"), ("db", "lora_b"), ("dbias", "bias")]


def _step(i, dy, names=None):
    names = [n for _, n in LEAVES if i[n] is not None and (names is None or n in names)]
    s = {n: (t.detach().requires_grad_() if n in names else t) for n, t in i.items()}
    y = parallel_adapters(**s)
    return y.detach(), dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], dy)))


def _compare(i, dy):
    y, grads = _step(i, dy)
    want = _want(i, dy)
    _bounds.check("y", y, *want["y"])
    for key, name in LEAVES:
        if name in grads:
            _bounds.check(key, grads[name], *want[key])
    return y, grads


# rows, widths, adapters, rank: one row to several tiles, widths that no tile divides, ranks of one and of more than a tile
SHAPES = [(1, 64, 64, 1, 1), (1, 128, 256, 4, 16), (2, 40, 24, 3, 5), (7, 131, 77, 5, 3), (16, 256, 128, 16, 8), (17, 96, 200, 2, 64),
          (33, 520, 136, 40, 4), (64, 128, 96, 64, 16), (65, 64, 320, 7, 8), (100, 200, 72, 3, 17), (130, 256, 256, 1, 32),
          (257, 192, 264, 9, 16), (300, 72, 520, 30, 24), (400, 64, 64, 2, 130), (513, 136, 128, 100, 8), (3, 1, 1, 2, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d,n,R,r", SHAPES)
def test_values_and_gradients(T, d, n, R, r, dtype):
    i, dy = _inputs(T, d, n, R, r, dtype, bias=T % 2 == 1, grouped=T % 3 == 0, seed=T + d)
    _compare(i, dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,n,R,r,grouped", [(2600, 1856, 4096, 5, 8, True), (2600, 4104, 1800, 40, 24, False), (3000, 1016, 3584, 3, 40, False),
                                                (4096, 1792, 4096, 9, 8, False), (700, 2048, 1800, 20, 12, False), (330, 264, 1000, 6, 33, True)])
def test_large_tiles(T, d, n, R, r, grouped, dtype):
    """Tiles of every class: contractions of whole slices of 64 and others, forward and, transposed, backward; more than a round of
    256 x 256 tiles by less than half, in two launches."""
    i, dy = _inputs(T, d, n, R, r, dtype, bias=True, grouped=grouped, seed=T + n)
    _compare(i, dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,n,R,r", [(65, 4096, 1024, 6, 16), (130, 2056, 2048, 9, 5), (319, 2048, 2050, 200, 40)])
def test_few_rows_beside_a_large_weight(T, d, n, R, r, dtype):
    """The gradient of the input in tiles, the output row by row or in tiles too."""
    i, dy = _inputs(T, d, n, R, r, dtype, bias=False, grouped=False, seed=T + d)
    _compare(i, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 64, 200])
@pytest.mark.parametrize("which", ["none", "one", "last"])
def test_rows_without_and_with_one_adapter(which, T, dtype):
    """No row has an adapter; all rows have the same one; only the last row has one."""
    i, dy = _inputs(T, 96, 80, 6, 8, dtype, seed=7)
    ids = torch.full((T,), -1 if which != "one" else 4, dtype=torch.int64, device=DEV)
    if which == "last":
        ids[-1] = 5
    i["adapter_idxs"] = ids
    y, grads = _compare(i, dy)
    used = set(ids[ids >= 0].tolist())
    for a in range(6):
        if a not in used:
            assert not bool(grads["lora_a"][a].any()) and not bool(grads["lora_b"][a].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [6, 150])
def test_strided_operands(T, dtype):
    """Rows apart from each other, factors stored the other way round, a weight of a larger one, a bias of one value, rows
    that start at any multiple of the element's size."""
    i, dy = _inputs(T, 72, 88, 4, 8, dtype, bias=True, seed=8)
    s = dict(i)
    s["x"] = torch.cat([i["x"], i["x"]], 1)[:, 36:108]
    s["weight"] = i["weight"].t().contiguous().t()
    s["lora_a"] = i["lora_a"].transpose(1, 2).contiguous().transpose(1, 2)
    s["lora_b"] = i["lora_b"].transpose(1, 2).contiguous().transpose(1, 2)
    s["bias"] = i["bias"][:1].expand(88)
    y, grads = _step(s, dy, ["x", "weight", "lora_a", "lora_b"])
    want = _want(s, dy)
    _bounds.check("y", y, *want["y"])
    for key, name in LEAVES[:4]:
        _bounds.check(key, grads[name], *want[key])
    flat = torch.empty(88 * 72 + 1, dtype=dtype, device=DEV)
    s = dict(i, weight=flat[1:].view(88, 72))
    s["weight"].copy_(i["weight"])
    _compare(s, dy)
    s = dict(i, x=i["x"][:, :1].expand(T, 72).t().contiguous().t())
    _compare(s, dy.t().contiguous().t())


@pytest.mark.parametrize("itype", [torch.int32, torch.int16, torch.uint8, torch.int64])
def test_id_types_and_leading_dimensions(itype):
    i, dy = _inputs(24, 64, 48, 5, 8, torch.bfloat16, bare=0.0, seed=9)
    want = parallel_adapters(**i)
    s = dict(i, x=i["x"].view(2, 3, 4, 64), adapter_idxs=i["adapter_idxs"].view(2, 3, 4).to(itype))
    got = parallel_adapters(**s)
    assert got.shape == (2, 3, 4, 48) and torch.equal(got.view(24, 48), want)


def test_without_scales_and_ids_of_one_byte():
    i, dy = _inputs(70, 64, 48, 5, 8, torch.bfloat16, seed=15)
    i["scales"] = None
    i["adapter_idxs"] = torch.where(i["adapter_idxs"] < 0, torch.full_like(i["adapter_idxs"], 255), i["adapter_idxs"]).to(torch.uint8)
    _compare(i, dy)


@pytest.mark.parametrize("T", [40, 300, 1000])
def test_as_many_adapters_as_there_may_be(T):
    """2047 adapters, most of them without rows, in a table of more elements than 32 bits count: what holds nothing is not read."""
    R, r, d, n = 2047, 8, 64, 32
    i, dy = _inputs(T, d, n, 4, r, torch.bfloat16, seed=16)
    used = torch.tensor([0, 1023, 1024, 2046], device=DEV)
    want = _want(i, dy)
    ids = i["adapter_idxs"]
    inside = (ids >= 0) & (ids < 4)
    s = dict(i, adapter_idxs=torch.where(inside, used[ids.clamp(0, 3)], torch.full_like(ids, R)))
    wide = torch.full((R, r, 1 << 18), float("nan"), dtype=torch.bfloat16, device=DEV)       # 4.3e9 elements, d of each row used
    s["lora_a"] = wide[:, :, :d]
    s["lora_a"][used] = i["lora_a"]
    s["lora_b"] = torch.full((R, n, r), float("nan"), dtype=torch.bfloat16, device=DEV)
    s["lora_b"][used] = i["lora_b"]
    s["scales"] = torch.ones(R, device=DEV)
    s["scales"][used] = i["scales"]
    y, grads = _step(s, dy, ["x", "lora_a", "lora_b"])
    _bounds.check("y", y, *want["y"])
    _bounds.check("dx", grads["x"], *want["dx"])
    for key, name in (("da", "lora_a"), ("db", "lora_b")):
        _bounds.check(key, grads[name][used], *want[key])
        rest = torch.ones(R, dtype=torch.bool, device=DEV)
        rest[used] = False
        assert not bool(grads[name][rest].any())


def test_no_rows():
    i, _ = _inputs(4, 64, 48, 5, 8, torch.bfloat16)
    s = dict(i, x=i["x"][:0].requires_grad_(), adapter_idxs=i["adapter_idxs"][:0], lora_a=i["lora_a"].clone().requires_grad_(),
             weight=i["weight"].clone().requires_grad_())
    y = parallel_adapters(**s)
    assert y.shape == (0, 48)
    gx, ga, gw = torch.autograd.grad(y.sum(), [s["x"], s["lora_a"], s["weight"]])
    assert gx.shape == (0, 64) and not bool(ga.any()) and not bool(gw.any())


def test_some_gradients_only():
    i, dy = _inputs(70, 64, 48, 5, 8, torch.bfloat16, bias=True, seed=10)
    _, every = _step(i, dy)
    for names in (["x"], ["lora_a"], ["lora_b"], ["bias"], ["weight"], ["lora_b", "x"]):
        _, some = _step(i, dy, names)
        assert sorted(some) == sorted(names) and all(torch.equal(some[n], every[n]) for n in names)


def test_gradients_against_differences():
    i, dy = _inputs(70, 48, 40, 3, 4, torch.float32, bias=True, seed=11)
    _, grads = _step(i, dy)

    def value(s):
        return float((_want(s)["y"][0] * dy.double()).sum())
    h = 2.0 ** -10
    for name, at in (("x", (3, 5)), ("x", (69, 47)), ("weight", (7, 9)), ("lora_a", (1, 2, 30)), ("lora_b", (2, 11, 3)), ("bias", (4,))):
        pair = []
        for sign in (h, -h):
            t = i[name].double()
            t[at] += sign
            pair.append(value(dict(i, **{name: t})))
        # (each factor enters linearly: a central difference has no error of its own but the rounding of the sums)
        want = (pair[0] - pair[1]) / (2 * h)
        assert abs(float(grads[name][at]) - want) <= 1e-4 * max(1.0, abs(want)), (name, at)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [12, 300])
def test_values_that_are_not_finite_stay_in_their_rows(T, dtype):
    i, dy = _inputs(T, 64, 48, 4, 8, dtype, bare=0.1, seed=12)
    i["adapter_idxs"][:6] = torch.tensor([0, 1, 2, 3, -1, 2])
    want = parallel_adapters(**i)
    s = dict(i, x=i["x"].clone(), lora_a=i["lora_a"].clone())
    s["x"][3, 7] = float("nan")
    a = int((i["adapter_idxs"][5]))
    s["lora_a"][a, 2] = float("inf")
    s["lora_b"] = i["lora_b"].clone()
    s["lora_b"][a, 9] = float("nan")
    got = parallel_adapters(**s)
    keep = i["adapter_idxs"] != a
    keep[3] = False
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[5]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,n,grouped", [(700, 1024, 1024, False), (700, 1024, 1024, True), (3000, 1792, 4096, True), (3000, 256, 4096, False)])
def test_values_that_are_not_finite_stay_in_their_rows_of_tiles(T, d, n, grouped, dtype):
    """Tiles of every class; the adapter beside, before and behind others and rows without one, in runs of its own or alone."""
    i, dy = _inputs(T, d, n, 5, 8, dtype, bare=0.2, grouped=grouped, seed=21)
    y, grads = _step(i, dy)
    ids = i["adapter_idxs"]
    for a in (0, 2, 4):
        s = dict(i, lora_a=i["lora_a"].clone(), lora_b=i["lora_b"].clone())
        s["lora_a"][a, 2] = float("inf")
        s["lora_b"][a, 9] = float("nan")
        got, g = _step(s, dy)
        keep, others = ids != a, [j for j in range(5) if j != a]
        assert torch.equal(got[keep], y[keep]) and bool(torch.isnan(got[~keep, 9]).all())
        assert torch.equal(g["x"][keep], grads["x"][keep])
        for name in ("lora_a", "lora_b"):
            assert torch.equal(g[name][others], grads[name][others])


@pytest.mark.parametrize("T", [5, 100, 700])
def test_broadcast_rows_and_a_broadcast_gradient(T):
    """One row for all, and the gradient of a sum: strides of zero either way."""
    i, _ = _inputs(T, 256, 192, 4, 8, torch.bfloat16, bias=True, seed=22)
    i["x"] = i["x"][:1].expand(T, 256)
    dy = torch.ones(1, 1, dtype=torch.bfloat16, device=DEV).expand(T, 192)
    y, grads = _step(i, dy)
    want, grads_want = _step(dict(i, x=i["x"].contiguous()), dy.contiguous())
    assert torch.equal(y, want) and all(torch.equal(grads[n], grads_want[n]) for n in grads)
    _bounds.check("y", y, *_want(i)["y"])


@pytest.mark.parametrize("T", [9, 200])
def test_same_bits_every_time_and_on_another_stream(T):
    i, dy = _inputs(T, 128, 96, 6, 16, torch.bfloat16, seed=13)
    y, grads = _step(i, dy)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2, grads2 = _step(i, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)


def test_captured_steps_and_eager_work_between():
    """A forward of few rows and one of many with its products' launches, replayed with new rows and new ids."""
    for T in (8, 160):
        i, _ = _inputs(T, 96, 64, 5, 8, torch.bfloat16, seed=14)
        parallel_adapters(**i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = parallel_adapters(**i)
        for r in range(3):
            g = torch.Generator().manual_seed(r)
            i["x"].copy_(torch.randn(T, 96, generator=g))
            i["adapter_idxs"].copy_(torch.randint(-1, 6, (T,), generator=g))
            graph.replay()
            want = parallel_adapters(**i)
            torch.cuda.synchronize()
            assert torch.equal(y, want), (T, r)


@pytest.mark.parametrize("T", [20, 150, 700])
def test_captured_gradients(T):
    """The backward call by itself, captured and replayed with eager work between the replays."""
    from scattermoe_amd.kernels import ops
    i, dy = _inputs(T, 96, 64, 5, 8, torch.bfloat16, seed=17)
    args = (i["x"], i["weight"], i["lora_a"], i["lora_b"], i["adapter_idxs"], i["scales"])

    def both():
        y, u, order = ops.adapter_forward(*args)
        return (y,) + ops.adapter_backward(dy, *args, u, order, need_bias=True)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for r in range(3):
        g = torch.Generator().manual_seed(r)
        i["x"].copy_(torch.randn(T, 96, generator=g))
        dy.copy_(torch.randn(T, 64, generator=g))
        i["adapter_idxs"].copy_(torch.randint(-1, 6, (T,), generator=g))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r


def test_two_calls_at_once():
    """On two streams, over the same weights, while neither waits for the other."""
    i, dy = _inputs(500, 256, 192, 6, 16, torch.bfloat16, seed=18)
    j = dict(i, x=torch.randn_like(i["x"]))
    want = [_step(s, dy) for s in (i, j)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        got = []
        for st, s in zip(streams, (i, j)):
            with torch.cuda.stream(st):
                got.append(_step(s, dy))
        torch.cuda.synchronize()
        for (y, grads), (y2, grads2) in zip(got, want):
            assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 24, 64])
def test_projection_with_adapters_then_routed_layer(T, dtype):
    """The two together, as in a block of a decode step: the requests' projections, the residual sum, the routed layer; twice, the second time
    from a captured graph."""
    torch.manual_seed(0)
    proj = ParallelAdapters(4, 64, 64, 8, scale=0.5).to(DEV).to(dtype)
    proj.scales = proj.scales.float()
    layer = RoutedGLUMLP(64, 96, 8, 2, bias=True).to(DEV).to(dtype)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for p in list(proj.parameters()) + list(layer.parameters()):
            p.copy_(torch.randn(p.shape, generator=g) * 0.1)
    x = torch.randn(T, 64, generator=g).to(dtype).to(DEV)
    ids = torch.randint(-1, 4, (T,), generator=g).to(DEV)

    def block():
        with torch.no_grad():
            y = proj(x, ids)
            mid = x + y
            return y, mid, layer(mid)
    y, mid, (out, logits) = block()
    want = _bounds.adapters(x, proj.weight, proj.lora_a, proj.lora_b, ids, proj.scales)
    _bounds.check("projection", y, *want["y"])
    ref, bound, ref_logits, logits_bound, clear = _bounds.layer(mid, layer.router.weight, layer.experts.weight, layer.output_experts.weight, 2,
                                                                 layer.experts.bias, layer.output_experts.bias)
    assert bool(clear.all())
    _bounds.check("logits", logits, ref_logits, logits_bound)
    _bounds.check("layer", out, ref, bound)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = block()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[0], y) and torch.equal(again[2][0], out) and torch.equal(again[2][1], logits)
        block()


def test_training_step_lowers_nothing_but_runs():
    """An optimizer's step over the adapters of a frozen projection."""
    torch.manual_seed(0)
    m = ParallelAdapters(3, 64, 48, 8, bias=True).to(DEV)
    m.weight.requires_grad_(False)
    opt = torch.optim.SGD([m.lora_a, m.lora_b], lr=0.1)
    x, ids = torch.randn(40, 64, device=DEV), torch.randint(0, 3, (40,), device=DEV)
    before = m.lora_b.detach().clone()
    m(x, ids).square().sum().backward()
    assert m.weight.grad is None and m.lora_a.grad.shape == m.lora_a.shape
    opt.step()
    assert not torch.equal(before, m.lora_b)


def test_refusals():
    i, _ = _inputs(4, 64, 48, 5, 8, torch.bfloat16)
    for change, error in ((dict(x=i["x"].float()), TypeError), (dict(adapter_idxs=i["adapter_idxs"].float()), TypeError),
                          (dict(adapter_idxs=i["adapter_idxs"][:3]), ValueError), (dict(lora_b=i["lora_b"][:, :, :7]), ValueError),
                          (dict(scales=i["scales"][:4]), ValueError), (dict(weight=i["weight"].cpu()), RuntimeError),
                          (dict(scales=i["scales"].clone().requires_grad_()), ValueError), (dict(x=i["x"][:, :63]), ValueError)):
        with pytest.raises(error):
            parallel_adapters(**dict(i, **change))
