"""The few-token layer's rows in another order: what a token gets does not depend on its place among the tokens, also where an
expert's rows take several passes, of which the last is not full."""
import pytest
import torch

import _bounds
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import RoutedGLUMLP, routed_glu_mlp
from test_gpu_routed_layer import DEV, DTYPES, _call, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
# tokens, experts, experts per token: passes of 8, 16 and 32 rows of an expert, the hot one's last pass of 1 to 16 rows
@pytest.mark.parametrize("T,E,k", [(20, 16, 2), (21, 8, 2), (17, 8, 2), (24, 8, 2), (33, 4, 1), (37, 8, 4), (41, 4, 2), (48, 4, 2), (64, 8, 2)])
def test_order_of_the_tokens(T, E, k, dtype):
    i = _inputs(T, 2048, 1024, E, dtype, seed=T + E)
    i["x"] = (i["x"].abs() + 0.25).to(dtype)
    i["wr"][1] = 1.0                                     # every token's first expert
    want = _call(i, k)
    g = torch.Generator().manual_seed(0)
    for order in [torch.arange(T).flip(0)] + [torch.randperm(T, generator=g) for _ in range(3)]:
        order = order.to(DEV)
        got = _call(dict(i, x=i["x"][order]), k)
        assert torch.equal(got[1], want[1][order])
        assert torch.equal(got[0], want[0][order]), "%d values differ" % int((got[0] != want[0][order]).sum())
    again = _call(i, k)
    assert torch.equal(again[0], want[0])


def _layouts(i):
    """The same weights in both layouts, and without the weights' streams."""
    turned = {n: i[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("w1", "w2")}
    return [i, dict(i, w2=turned["w2"]), dict(i, w1=turned["w1"]), dict(i, **turned)]


@pytest.mark.parametrize("T", [3, 9])
def test_hidden_values_beyond_float16(T):
    """float16 hidden values above 65504 are infinite, whatever the weights' layout and as where they are stored: the rows that have one
    are not finite, and the others are what they are without them."""
    i = _inputs(T, 64, 96, 4, torch.float16, seed=T)
    large = dict(i, x=i["x"].clone(), w1=(i["w1"].float() * 16).half())
    large["x"][1] = (i["x"][1].float() * 24).half()
    _, _, _, _, clear = _bounds.layer(large["x"], large["wr"], large["w1"], large["w2"], 2)
    assert bool(clear.all())
    others = [t for t in range(T) if t != 1]
    for s in _layouts(large):
        got = ops.routed_glu_mlp(s["x"], s["wr"], s["w1"], None, s["w2"], None, 2)
        assert not bool(torch.isfinite(got[0][1]).any())
        out, bound, _, _, _ = _bounds.layer(s["x"], s["wr"], s["w1"], s["w2"], 2)
        _bounds.check("others", got[0][others], out[others], bound[others])
    general = routed_glu_mlp(large["x"].clone().requires_grad_(), large["wr"], large["w1"], large["w2"], 2)[0]
    assert not bool(torch.isfinite(general[1]).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [3, 9, 40])
def test_small_hidden_values(T, dtype):
    """Hidden values of about 2^-20, a part of the smallest step of float16 away from their sum: every layout within the same bound."""
    i = _inputs(T, 64, 96, 4, dtype, seed=T + 1)
    s = dict(i, w1=(i["w1"].float() * 2.0 ** -9).to(dtype), w2=(i["w2"].float() * 2.0 ** 10).to(dtype))
    out, bound, _, _, clear = _bounds.layer(s["x"], s["wr"], s["w1"], s["w2"], 2)
    assert bool(clear.all())
    for of in _layouts(s):
        got = ops.routed_glu_mlp(of["x"], of["wr"], of["w1"], None, of["w2"], None, 2)
        _bounds.check("out", got[0], out, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2, 30])
def test_larger_weights_of_a_strided_contraction(T, dtype):
    """The general path, within the bound of its own roundings, and columns of the tokens that lie apart."""
    i = _inputs(T, 512, 520, 8, dtype, bias=True, seed=T + 2)
    args = (i["x"], i["wr"], i["w1"], i["w2"], 4, i["b1"], i["b2"])
    out, bound, logits, logits_bound, clear = _bounds.layer(*args, stored=True)
    assert int(clear.sum()) >= 0.9 * T
    for s in _layouts(i)[1:]:
        got = _call(s, 4)
        _bounds.check("logits", got[1], logits, logits_bound)
        _bounds.check("out", got[0].cpu()[clear], out[clear], bound[clear])
    want = _call(i, 4)
    got = _call(dict(i, x=i["x"].t().contiguous().t()), 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_training_step_without_tokens(dtype):
    """... as on a rank that got none: the outputs are part of the graph, and every gradient is zeros."""
    m = RoutedGLUMLP(64, 96, 8, 2, bias=True).to(DEV).to(dtype)
    x = torch.randn(0, 3, 64, device=DEV).to(dtype).requires_grad_()
    out, logits = m(x)
    assert out.shape == x.shape and logits.shape == (0, 8) and out.requires_grad and logits.requires_grad
    (out.float().sum() + logits.sum()).backward()
    assert x.grad.shape == x.shape
    for name, p in m.named_parameters():
        assert p.grad is not None and p.grad.shape == p.shape and not bool(p.grad.any()), name
    with torch.no_grad():
        out, logits = m(x)
    assert out.shape == x.shape and logits.shape == (0, 8) and logits.dtype == torch.float32
