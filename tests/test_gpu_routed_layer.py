"""A whole gated layer for a few tokens (ops.routed_glu_mlp, mlp.routed_glu_mlp, mlp.RoutedGLUMLP) against the formulas in 64
bits, with bounds that follow from the roundings (_bounds.py)."""
import pytest
import torch

import _bounds
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import RoutedGLUMLP, routed_glu_mlp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(T, d, F, E, dtype, bias=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(DEV)
    return dict(x=r(T, d), wr=r(E, d, std=1.5 * d ** -0.5), w1=r(E, 2 * F, d, std=d ** -0.5), w2=r(E, d, F, std=F ** -0.5),
                b1=r(E, 2 * F, std=0.3) if bias else None, b2=r(E, d, std=0.3) if bias else None)


def _call(i, k, **kw):
    with torch.no_grad():
        return routed_glu_mlp(i["x"], i["wr"], i["w1"], i["w2"], k, b1=i["b1"], b2=i["b2"], **kw)


def _compare(i, k, got, least=0.9, **kw):
    out, bound, logits, logits_bound, clear = _bounds.layer(i["x"], i["wr"], i["w1"], i["w2"], k, i["b1"], i["b2"], **kw)
    assert int(clear.sum()) >= least * len(clear)
    _bounds.check("logits", got[1], logits, logits_bound)
    _bounds.check("out", got[0].cpu().reshape(out.shape)[clear], out[clear], bound[clear])


SHAPES = [(1, 64, 64, 4, 2), (1, 256, 96, 128, 8), (2, 2048, 64, 5, 1), (3, 72, 40, 8, 8), (5, 131, 77, 13, 3), (7, 520, 264, 16, 2),
          (16, 128, 512, 6, 2), (17, 192, 320, 32, 4), (33, 65, 129, 3, 2), (64, 128, 128, 8, 8), (64, 256, 80, 128, 8),
          (48, 64, 96, 2, 1), (64, 64, 64, 1, 1), (1, 1, 1, 1, 1), (9, 8, 24, 512, 5), (4, 32, 16, 64, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d,F,E,k", SHAPES)
def test_layer(T, d, F, E, k, dtype):
    i = _inputs(T, d, F, E, dtype, bias=(T + k) % 2 == 1, seed=T + d)
    _compare(i, k, _call(i, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d,F,E,k", [(5, 2048, 72, 32, 4), (16, 2500, 40, 20, 2), (9, 2051, 33, 64, 3), (3, 2880, 1440, 16, 4), (11, 2056, 264, 6, 1)])
def test_long_weight_rows(T, d, F, E, k, dtype):
    """Workgroups of fewer or more weight rows, widths that no block of the contraction divides."""
    i = _inputs(T, d, F, E, dtype, bias=T % 2 == 1, seed=T + d)
    # (of so few tokens one or two whose k-th and next logits lie within twice the logits' own bound of each other - sums of
    # 2051 products and 64 experts to choose from - are more than a tenth; which of them is taken is then no error)
    _compare(i, k, _call(i, k), least=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize,gate_first", [(False, False), (True, True), (False, True)])
def test_conventions(renormalize, gate_first, dtype):
    i = _inputs(6, 96, 72, 10, dtype, bias=True, seed=3)
    kw = dict(renormalize=renormalize, gate_first=gate_first)
    _compare(i, 3, _call(i, 3, **kw), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_all_tokens_to_the_same_experts(dtype):
    """One expert takes 64 rows, the others none."""
    i = _inputs(64, 96, 160, 12, dtype, bias=True, seed=4)
    i["x"] = (i["x"].abs() + 0.5).to(dtype)
    i["wr"][3] = 1.0
    i["wr"][7] = 0.75
    _compare(i, 2, _call(i, 2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_operands(dtype):
    """Rows apart from each other, widths of a larger tensor, weights whose contraction axis is strided, shared biases."""
    i = _inputs(5, 80, 48, 6, dtype, bias=True, seed=5)
    want = _call(i, 2)
    s = dict(i)
    s["x"] = torch.cat([i["x"], i["x"]], 1)[:, :80]
    s["wr"] = torch.cat([i["wr"], i["wr"]], 0)[:6]
    s["w1"] = torch.cat([i["w1"], i["w1"]], 2)[:, :, :80]
    s["w2"] = i["w2"].transpose(1, 2).contiguous().transpose(1, 2)
    s["b1"] = torch.cat([i["b1"], i["b1"]], 1)[:, :96]
    got = _call(s, 2)
    _compare(s, 2, got)
    assert torch.equal(got[1], want[1])
    s["w1"] = i["w1"].transpose(1, 2).contiguous().transpose(1, 2)
    s["x"] = i["x"].t().contiguous().t()
    s["wr"] = i["wr"].t().contiguous().t()
    s["b2"] = i["b2"][:, :1].expand(6, 80)
    _compare(s, 2, _call(s, 2))
    # one odd element in front: rows that start at any multiple of the element's size
    flat = torch.empty(6 * 96 * 80 + 1, dtype=dtype, device=DEV)
    s = dict(i, w1=flat[1:].view(6, 96, 80))
    s["w1"].copy_(i["w1"])
    _compare(s, 2, _call(s, 2))


def test_leading_dimensions_and_no_tokens():
    i = _inputs(6, 64, 32, 8, torch.bfloat16)
    want = _call(i, 2)
    got = _call(dict(i, x=i["x"].view(2, 3, 64)), 2)
    assert got[0].shape == (2, 3, 64) and torch.equal(got[0].view(6, 64), want[0]) and torch.equal(got[1], want[1])
    none = _call(dict(i, x=i["x"][:0]), 2)
    assert none[0].shape == (0, 64) and none[1].shape == (0, 8)


def test_equal_logits_take_the_lowest_experts():
    i = _inputs(3, 64, 32, 9, torch.float32)
    i["wr"].zero_()
    same = dict(i, wr=i["wr"][:4], w1=i["w1"][:4], w2=i["w2"][:4])
    a, b = _call(i, 4), _call(same, 4)
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_broken_router_row(bad):
    """A logit that is not a number counts as minus infinity; the ids stay valid and the other tokens what they were."""
    i = _inputs(4, 64, 32, 8, torch.float32, seed=9)
    want = _call(i, 2)
    x = i["x"].clone()
    x[2, 5] = bad
    got = _call(dict(i, x=x), 2)
    keep = [0, 1, 3]
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
    wr = i["wr"].clone()
    wr[6] = float("nan")
    rest = [0, 1, 2, 3, 4, 5, 7]
    got = _call(dict(i, wr=wr), 2)
    assert bool(torch.isnan(got[1][:, 6]).all())
    _compare(dict(i, wr=i["wr"][rest], w1=i["w1"][rest], w2=i["w2"][rest]), 2, (got[0], got[1][:, rest]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_of_very_different_size(dtype):
    """Hidden values far below and far above one: what a row is multiplied with does not depend on the others."""
    i = _inputs(4, 64, 64, 4, dtype, seed=11)
    for scale in (2.0 ** -6, 2.0 ** 3):
        s = dict(i, w1=(i["w1"].float() * scale).to(dtype))
        _compare(s, 2, _call(s, 2))


def test_same_bits_every_time_and_on_another_stream():
    i = _inputs(40, 128, 96, 16, torch.bfloat16, bias=True, seed=12)
    want = _call(i, 4)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _call(i, 4)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_captured_graphs_with_eager_work_between():
    a, b = _inputs(3, 128, 96, 16, torch.bfloat16, seed=13), _inputs(21, 64, 160, 8, torch.float16, bias=True, seed=14)
    graphs = []
    for i, k in ((a, 4), (b, 2)):
        _call(i, k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _call(i, k)
        graphs.append((graph, out, i, k))
    for r in range(3):
        for graph, out, i, k in graphs:
            i["x"].copy_(torch.randn(i["x"].shape, generator=torch.Generator().manual_seed(r)).to(i["x"].dtype))
        for graph, _, _, _ in graphs:
            graph.replay()
        for graph, out, i, k in graphs:
            want = _call(i, k)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_general_path_and_few_token_path(dtype):
    """The module with autograd, or with more tokens, and without it: the same layer, each within the bound of its own
    roundings."""
    torch.manual_seed(0)
    m = RoutedGLUMLP(96, 128, 8, 2, bias=True).to(DEV).to(dtype)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())) * 0.1)
    x = torch.randn(9, 96, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    with torch.no_grad():
        few, few_logits = m(x)
        many = m(x.repeat(12, 1))
    trained = m(x.clone().requires_grad_())
    args = (x, m.router.weight, m.experts.weight, m.output_experts.weight, 2, m.experts.bias, m.output_experts.bias)
    out, bound, logits, logits_bound, clear = _bounds.layer(*args)
    assert bool(clear.all())
    slack = _bounds.layer(*args, stored=True)[1]
    _bounds.check("few tokens", few, out, bound)
    _bounds.check("with autograd", trained[0], out, slack)
    _bounds.check("many tokens", many[0][:9], out, slack)
    _bounds.check("few tokens, logits", few_logits, logits, logits_bound)
    _bounds.check("logits", trained[1], logits, logits_bound)
    grads = torch.autograd.grad(trained[0].float().sum() + trained[1].sum(), [x_ for x_ in m.parameters()])
    assert all(bool(torch.isfinite(g).all()) and float(g.float().abs().max()) > 0 for g in grads)


def test_router_gradient_of_the_general_path():
    """Against differences of the formula in 64 bits, at a router weight and an input value."""
    torch.manual_seed(0)
    i = _inputs(5, 32, 24, 6, torch.float32, seed=21)
    x, wr = i["x"].clone().requires_grad_(), i["wr"].clone().requires_grad_()
    out, _ = routed_glu_mlp(x, wr, i["w1"], i["w2"], 2)
    dy = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    gx, gw = torch.autograd.grad(out, (x, wr), dy)
    h = 2.0 ** -12
    for leaf, grad, at in ((i["x"], gx, (1, 3)), (i["x"], gx, (4, 30)), (i["wr"], gw, (2, 7)), (i["wr"], gw, (5, 1))):
        up, down = leaf.double(), leaf.double()
        up[at] += h
        down[at] -= h
        pair = [(u, i["wr"].double()) if leaf is i["x"] else (i["x"].double(), u) for u in (up, down)]
        want = (value64(*pair[0], i, dy) - value64(*pair[1], i, dy)) / (2 * h)
        assert abs(float(grad[at]) - want) <= 1e-4 * max(1.0, abs(want)), (at, float(grad[at]), want)


def value64(x, wr, i, dy):
    """sum(out * dy) with every tensor in 64 bits."""
    x, wr, w1, w2 = (t.double().cpu() for t in (x, wr, i["w1"], i["w2"]))
    p = torch.softmax(x @ wr.t(), -1)
    g, e = torch.topk(p, 2)
    g = g / g.sum(-1, keepdim=True)
    total = torch.zeros(x.shape, dtype=torch.double)
    for j in range(2):
        pre = (w1[e[:, j]] @ x.unsqueeze(2)).squeeze(2)
        lin, gate = pre.chunk(2, -1)
        total += g[:, j:j + 1] * (w2[e[:, j]] @ (lin * torch.nn.functional.silu(gate)).unsqueeze(2)).squeeze(2)
    return float((total * dy.double().cpu()).sum())


def test_weights_of_more_elements_than_32_bits_count():
    """512 experts in 10.5 GB: the chosen ones lie far apart, and nothing else is read."""
    E, F, d, k = 512, 1664, 2048, 2
    chosen = [1, 300, 510, 511]
    i = _inputs(6, d, 64, E, torch.bfloat16, seed=31)
    g = torch.Generator(DEV).manual_seed(0)
    w1 = torch.full((E, 2 * F, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    w2 = torch.full((E, d, F), float("nan"), dtype=torch.bfloat16, device=DEV)
    wr = torch.zeros(E, d, dtype=torch.bfloat16, device=DEV)
    wr[:, 0] = -4.0
    i["x"][:, 0] = 1.0
    for e in chosen:
        w1[e] = torch.randn(2 * F, d, generator=g, device=DEV) * d ** -0.5
        w2[e] = torch.randn(d, F, generator=g, device=DEV) * F ** -0.5
        wr[e] = (torch.randn(d, generator=g, device=DEV) * d ** -0.5).bfloat16()
    for T in (1, 6):
        s = dict(i, x=i["x"][:T], wr=wr, w1=w1, w2=w2)
        out, logits = _call(s, k)
        small = dict(s, wr=wr[chosen], w1=w1[chosen], w2=w2[chosen])
        # (the other experts' share of the softmax drops out of the renormalised gates)
        _compare(small, k, (out, logits[:, chosen]))


def test_two_calls_at_once():
    i, j = _inputs(30, 256, 192, 16, torch.bfloat16, seed=32), _inputs(3, 256, 192, 16, torch.bfloat16, seed=33)
    want = [_call(s, 2) for s in (i, j)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, s in zip(streams, (i, j)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(_call(s, 2))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


def test_refusals():
    i = _inputs(4, 64, 32, 8, torch.bfloat16)
    with torch.no_grad():
        with pytest.raises(TypeError):
            routed_glu_mlp(i["x"].float(), i["wr"], i["w1"], i["w2"], 2)
        with pytest.raises(RuntimeError):
            routed_glu_mlp(i["x"].cpu(), i["wr"], i["w1"], i["w2"], 2)
        with pytest.raises(ValueError):
            ops.routed_glu_mlp(i["x"].repeat(17, 1), i["wr"], i["w1"], None, i["w2"], None, 2)
