"""Gated layers on weights in 8 bits whose rows pass what 32-bit offsets reach: forward passes and training steps, rows of both ends and of the
places that a wrapped offset would take instead."""
import pytest
import torch

import _ref_8bit as ref
from scattermoe_amd import eight_bit
from test_gpu_8bit import _layer_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# 2^20 tokens of 4096 are 4 GiB in 8 bits: tokens that are copied in the experts' order (one expert per token, two), and tokens that are looked up while
# their gradients times the gates, one row per slot, are copied
@pytest.mark.parametrize("T,k,step", [((1 << 20) + 64, 1, True), ((1 << 20) + 64, 2, False), ((1 << 19) + 64, 2, True)])
def test_layer_of_rows_beyond_32_bits(T, k, step):
    E, d, F = 4, 4096, 128
    g = torch.Generator(device=DEV).manual_seed(T + k)
    w1, w2 = (torch.randn(s, device=DEV, generator=g) * s[2] ** -0.5 for s in ((E, 2 * F, d), (E, d, F)))
    (q1, s1, t1), (q2, s2, t2) = (eight_bit.quantize_blocks(w, 128, transposed=True) for w in (w1, w2))
    x = torch.empty(T, d, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    ids = (torch.randint(0, E, (T, 1), device=DEV, generator=g) + torch.arange(k, device=DEV)) % E
    p = (torch.randint(1, 4, (T, k), device=DEV, generator=g) / 4).bfloat16()
    some = torch.tensor([0, 1, 63, 64, T // 2, T - 129, T - 65, T - 64, T - 2, T - 1])
    at = some.to(DEV)
    if step:
        dout = torch.empty(T, d, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
        x.requires_grad_(), p.requires_grad_()
        out = eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2, w1_t=t1, w2_t=t2)
        got = [out.detach(), *torch.autograd.grad(out, (x, p), dout)]
    else:
        dout = x
        got = [eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2)]
    want = _layer_reference(x.detach()[at].cpu(), p.detach()[at].cpu(), ids[at].cpu(), ref.stands_for(q1, s1, d), ref.stands_for(q2, s2, F), None, None,
                            dout[at].cpu(), True, False, False, torch.bfloat16)
    for name, g, (v, bound) in zip(("out", "dx", "dgates"), got, want):
        ref.check(name, g[at], v, bound)
