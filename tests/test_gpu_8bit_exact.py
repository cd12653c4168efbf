"""Layers in float16 on weights in 8 bits are as exact as in float32 but for the rounding of their results: a hidden value taken to the other of two
neighbouring 8-bit values, a step of up to 2^-4, would stand out.  Bounds are those of the float32 layer of the same numbers (no matrix
instruction's cut: sums of exact products in float32), and a rounding to float16."""
import pytest
import torch

import _ref_8bit as ref
from scattermoe_amd import eight_bit
from test_gpu_8bit import _ids, _layer_reference, _normal, _weight

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# by the ids, streams (up to 16 rows per expert), tiles with the unit behind the product and its gradient, tiles without
CASES = [(5, 2, 4, 512, 256, "any"), (48, 2, 8, 520, 384, "any"), (96, 2, 12, 384, 200, "gap"), (130, 2, 6, 512, 512, "any"), (150, 3, 5, 392, 328, "any"),
         (90, 1, 2, 1032, 264, "one")]


@pytest.mark.parametrize("float_scales", [False, True])
@pytest.mark.parametrize("T,k,E,d,F,kind", CASES)
def test_float16_layers(float_scales, T, k, E, d, F, kind):
    g = torch.Generator().manual_seed(T + d)
    x, dout, ids = _normal(g, T, d, dtype=torch.float16), _normal(g, T, d, dtype=torch.float16), _ids(g, T, E, k, kind)
    p = (torch.rand((T, k), generator=g) + 0.2).half()
    q1, s1, t1, w1 = _weight(g, E, 2 * F, d, d ** -0.5, float_scales)
    q2, s2, t2, w2 = _weight(g, E, d, F, F ** -0.5, float_scales)
    b1, b2 = _normal(g, E, 2 * F, dtype=torch.float16), _normal(g, E, d, dtype=torch.float16)
    xg, pg = x.to(DEV).requires_grad_(), p.to(DEV).requires_grad_()
    call = lambda a, b, **kw: eight_bit.glu_mlp_8bit(a, b, ids.to(DEV), q1, s1, q2, s2, b1=b1.to(DEV), b2=b2.to(DEV), **kw)
    out = call(xg, pg, w1_t=t1, w2_t=t2)
    dx, dp = torch.autograd.grad(out, (xg, pg), dout.to(DEV))
    with torch.no_grad():
        plain = call(xg, pg)
    want = _layer_reference(x.float(), p.float(), ids, w1, w2, b1, b2, dout.float(), False, float_scales, False, torch.float32)
    for name, got, (v, bound) in zip(("out", "dx", "dgates", "out, forward only"), (out, dx, dp, plain), want + want[:1]):
        ref.check(name, got, v, ref.rounded(v, bound, torch.float16))


@pytest.mark.parametrize("T,k,E,d,F,kind", [(130, 2, 6, 512, 512, "any"), (96, 2, 12, 384, 200, "gap"), (256, 2, 4, 1024, 256, "any")])
def test_float16_layers_as_a_whole(T, k, E, d, F, kind):
    """In the Euclidean norm rounding to float16 costs at most 2^-11.  Sums in float32, off by some 2^-22 of their size, take a share of 2 * 2^-22 / 2^-4 =
    2^-17 of the values that go to 8 bits over a border, each by 2^-4 to 2^-3 of itself: 2^-8.5 * 0.09 = 2.5e-4 for each such step (one in the output,
    two in the gradient).  With sums that are 1.3e-5 off it is 1.3e-3."""
    g = torch.Generator().manual_seed(T + F)
    x, dout, ids = _normal(g, T, d, dtype=torch.float16), _normal(g, T, d, dtype=torch.float16), _ids(g, T, E, k, kind)
    p = (torch.rand((T, k), generator=g) + 0.2).half()
    q1, s1, t1, w1 = _weight(g, E, 2 * F, d, d ** -0.5, False)
    q2, s2, t2, w2 = _weight(g, E, d, F, F ** -0.5, False)
    xg = x.to(DEV).requires_grad_()
    out = eight_bit.glu_mlp_8bit(xg, p.to(DEV), ids.to(DEV), q1, s1, q2, s2, w1_t=t1, w2_t=t2)
    (dx,) = torch.autograd.grad(out, xg, dout.to(DEV))
    want = _layer_reference(x.float(), p.float(), ids, w1, w2, None, None, dout.float(), False, False, False, torch.float32)
    for name, got, (v, _), steps in zip(("out", "dx"), (out, dx), want, (1, 2)):
        off = float((got.detach().cpu().double() - v).norm() / v.norm())
        assert off <= 2.0 ** -11 + steps * 2.5e-4, "%s: %.3g" % (name, off)
