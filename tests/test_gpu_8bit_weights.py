"""Weights in 8 bits whose experts lie apart are read where they are: the same bits as contiguous ones give, and no copy."""
import pytest
import torch

from scattermoe_amd import eight_bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _apart(q):
    """Every second expert of twice as many, the ones between no numbers."""
    full = torch.full((2 * q.size(0), *q.shape[1:]), 0x7f, dtype=torch.uint8, device=DEV)
    full[::2] = q.view(torch.uint8)
    return full.view(q.dtype)[::2]


# by the ids, streams, tiles with and without the unit behind the product
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k,E,d,F", [(2, 2, 4, 512, 256), (40, 2, 32, 528, 384), (200, 2, 4, 512, 512), (90, 2, 3, 136, 72)])
def test_layer(dtype, T, k, E, d, F):
    g = torch.Generator().manual_seed(T)
    w1, w2 = (torch.randn(s, generator=g).to(DEV) * s[2] ** -0.5 for s in ((E, 2 * F, d), (E, d, F)))
    (q1, s1, t1), (q2, s2, t2) = (eight_bit.quantize_blocks(w, 128, transposed=True) for w in (w1, w2))
    x, dout = (torch.randn(T, d, generator=g).to(DEV, dtype) for _ in range(2))
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(DEV)
    p = torch.rand(T, k, generator=g).to(DEV, dtype)

    def step(q1, t1, q2, t2):
        a, b = x.clone().requires_grad_(), p.clone().requires_grad_()
        with torch.no_grad():
            plain = eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2)
        out = eight_bit.glu_mlp_8bit(a, b, ids, q1, s1, q2, s2, w1_t=t1, w2_t=t2)
        return [plain, out.detach(), *torch.autograd.grad(out, (a, b), dout)]

    want = step(q1, t1, q2, t2)
    held = [_apart(q) for q in (q1, t1, q2, t2)]
    assert all(torch.equal(a, b) for a, b in zip(step(*held), want))


def test_nothing_is_copied():
    E, d, F = 8, 1024, 2048
    q1, q2 = (_apart(torch.zeros(s, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)) for s in ((E, 2 * F, d), (E, d, F)))
    s1, s2 = torch.ones(E, 32, 8, device=DEV), torch.ones(E, 8, 16, device=DEV)
    x, p, ids = torch.randn(64, d, device=DEV).bfloat16(), torch.ones(64, 1, device=DEV).bfloat16(), torch.arange(64, device=DEV).view(64, 1) % E
    for _ in range(2):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2)
        torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < q2.numel() // 2
