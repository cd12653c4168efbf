"""Training through the layer with its router in 16 bits: gradients of the experts' weights and biases against the chain rule in 64 bits.

The general path rounds gates, pre-activations, hidden rows, the output's gradient times its gate, the pre-activations' gradient and the
result, each by at most half a step u of the type.  A gradient is a sum of products of these, so it is off by at most the number of
roundings that a term passes through (six; a pre-activation enters through both halves and through the activation's slope, two more) times
u times the same sum over magnitudes: |silu(b)| <= |b| and its change at most 1.1 of b's, |silu'(b)| <= 1.1 and its change at most half
of b's.  float32 sums of a few hundred terms add nothing that counts beside 2^-11; a tenth is left for them."""
import pytest
import torch

import _bounds
from scattermoe_amd.mlp import routed_glu_mlp
from test_gpu_routed_layer import DEV, _inputs

pytestmark = pytest.mark.gpu
ROUNDINGS = 8 * 1.1


def _chain(i, k, dout, chosen, g, sizes):
    """Gradients of w1, b1, w2, b2 by the formulas, or (`sizes`) the same sums over magnitudes."""
    x, w1, w2, b1, b2 = (i[n].double() for n in ("x", "w1", "w2", "b1", "b2"))
    dout = dout.double()
    if sizes:
        x, w1, w2, b1, b2, dout = (t.abs() for t in (x, w1, w2, b1, b2, dout))
    grads = {n: torch.zeros_like(t) for n, t in (("w1", w1), ("b1", b1), ("w2", w2), ("b2", b2))}
    for e in range(w1.size(0)):
        for j in range(k):
            rows = (chosen[:, j] == e).nonzero().squeeze(1)
            if not len(rows):
                continue
            pre = x[rows] @ w1[e].t() + b1[e]
            a, b = pre.chunk(2, -1)
            s = torch.sigmoid(b)
            act, slope = (b, 1.1 + 0.5 * b) if sizes else (b * s, s * (1 + b * (1 - s)))
            dy = dout[rows] * g[rows, j:j + 1]
            dh = dy @ w2[e]
            dpre = torch.cat([dh * act, dh * a * slope], -1)
            grads["w2"][e] += dy.t() @ (a * act)
            grads["b2"][e] += dy.sum(0)
            grads["w1"][e] += dpre.t() @ x[rows]
            grads["b1"][e] += dpre.sum(0)
    return grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,F,E,k", [(5, 64, 96, 4, 2), (70, 128, 64, 8, 2), (300, 96, 160, 6, 3)])
def test_gradients_of_the_experts(T, d, F, E, k, dtype):
    i = _inputs(T, d, F, E, dtype, bias=True, seed=T)
    leaves = {n: i[n].clone().requires_grad_() for n in ("w1", "b1", "w2", "b2")}
    dout = torch.randn(T, d, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    out, logits = routed_glu_mlp(i["x"], i["wr"], leaves["w1"], leaves["w2"], k, b1=leaves["b1"], b2=leaves["b2"])
    exact = i["x"].double() @ i["wr"].double().t()
    p = torch.softmax(exact, -1)
    chosen = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, :k]
    order = torch.sort(exact, dim=-1, descending=True).values
    # (the selection is the same for float32 logits and exact ones)
    assert bool(((order[:, k - 1] - order[:, k]) > 2 * (d + 8) * 2.0 ** -24 * (i["x"].double().abs() @ i["wr"].double().abs().t()).max()).all())
    g = p.gather(1, chosen)
    g = g / g.sum(-1, keepdim=True)
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)))
    want, size = _chain(i, k, dout, chosen, g, False), _chain(i, k, dout, chosen, g, True)
    for name in leaves:
        _bounds.check(name, got[name], want[name], ROUNDINGS * torch.finfo(dtype).eps / 2 * size[name] + _bounds.TINY[dtype])
