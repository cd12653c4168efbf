"""What a token's slots add up to on weights in 8 bits: rows stay float32 until they are added up, in every way that a call goes.  The numbers are
chosen so that every product, hidden value and gradient is exact: a row is 1 + eps, which the rows' type does not hold, another one 1, and
their difference eps."""
import pytest
import torch

import _ref_8bit as ref
from scattermoe_amd import eight_bit, flatten_sort_count

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# a value beside 1 that the type would round away: half of its last place, or less
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -12, torch.float32: 2.0 ** -12}
DTYPES = list(EPS)


def _weights(E, N, K):
    return torch.zeros(E, N, K, device=DEV)


def _ids(T, E):
    """Every token goes to experts E - 2 and E - 1."""
    return torch.tensor([[E - 2, E - 1]], device=DEV).expand(T, 2).contiguous()


def _gates(T, dtype):
    return torch.tensor([[1.0, -1.0]], device=DEV, dtype=dtype).expand(T, 2).contiguous()


def _all(t, value):
    assert bool((t == value).all()), "%s instead of %s" % (t.flatten()[:4].tolist(), value)


# few rows per expert: streams over the weights; more: tiles; long contractions: tiles whose contraction is cut into parts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,K,N", [(1, 2, 128, 128), (3, 2, 160, 132), (100, 2, 128, 128), (90, 3, 8320, 128), (100, 2, 128, 67)])
def test_sums_over_the_slots_of_products(dtype, T, E, K, N):
    eps = EPS[dtype]
    ids, gates = _ids(T, E), _gates(T, dtype)
    eid, idx, off = flatten_sort_count(ids, E)
    # rows that come grouped, weighed by the gates: y = 1 + eps, 1
    w = _weights(E, N, K)
    w[:, :, 0] = 1.0
    w[E - 2, :, 64] = 1.0
    q, s, qt = eight_bit.quantize_blocks(w, 128, transposed=True)
    x = torch.zeros(2 * T, K, device=DEV, dtype=dtype)
    x[:, 0], x[:, 64] = 1.0, eps
    y = eight_bit.parallel_linear_8bit(x, q, s, 1, eid, idx, off, gates=gates, grouped_in=True)
    _all(y, eps)
    # their gates' gradient: of one column 1 + eps, of another one -1
    w = w.clone()
    w[:, 1, 0], w[:, 1, 64] = -1.0, 0.0
    q2, s2 = eight_bit.quantize_blocks(w, 128)
    p = gates.clone().requires_grad_()
    dout = torch.zeros(T, N, device=DEV, dtype=dtype)
    dout[:, :2] = 1.0
    y = eight_bit.parallel_linear_8bit(x, q2, s2, 1, eid, idx, off, gates=p, grouped_in=True)
    (dp,) = torch.autograd.grad(y, p, dout)
    _all(dp[:, 0], eps)
    _all(dp[:, 1], 0.0)
    # the gradient of tokens, one row of it per slot: dx = 1 + eps, -1
    if N > 64:
        w = _weights(E, N, K)
        w[E - 2, 0], w[E - 2, 64], w[E - 1, 0] = 1.0, eps, -1.0
        q, s, qt = eight_bit.quantize_blocks(w, 128, transposed=True)
        x = torch.randn(T, K, device=DEV).to(dtype).requires_grad_()
        y = eight_bit.parallel_linear_8bit(x, q, s, 2, eid, idx, off, weight_t=qt)
        dy = torch.zeros(2 * T, N, device=DEV, dtype=dtype)
        dy[:, 0] = dy[:, 64] = 1.0
        (dx,) = torch.autograd.grad(y, x, dy)
        _all(dx, eps)


def _layer(E, d, F, eps, top=1.0):
    """silu(64) = 64: hidden values are 1 and eps; y = top (1 + eps) of one expert and top of the other, in column 0, 0 in the others.  Column 1 of the
    tokens reaches the linear half alone: its gradient of dout = 1 in column 0 is 1 + eps times the one gate, and the other gate."""
    w1, w2 = _weights(E, 2 * F, d), _weights(E, d, F)
    w1[:, 0, :2], w1[:, 64, :2] = 2.0 ** -6, 2.0 ** -6 * eps
    w1[:, F:, 0] = 64.0
    w2[:, 0, 0] = top
    w2[E - 2, 0, 64] = top
    return (*eight_bit.quantize_blocks(w1, 128, transposed=True), *eight_bit.quantize_blocks(w2, 128, transposed=True))


# by the ids; in the experts' order: streams, tiles with and without the unit behind the product, tiles whose contraction is cut into parts
LAYERS = [(1, 2, 128, 128), (3, 2, 160, 96), (3, 2, 160, 160), (100, 2, 128, 160), (40, 40, 128, 128), (100, 2, 128, 128), (100, 2, 130, 129), (60, 2, 128, 8320)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,d,F", LAYERS)
def test_sums_over_the_slots_of_layers(dtype, T, E, d, F):
    eps = EPS[dtype]
    q1, s1, t1, q2, s2, t2 = _layer(E, d, F, eps)
    # (what the weight of the second hidden value stands for: with F below 128 its block of 128 rows holds gates of 64 too, whose scale 2^-2 leaves
    # nothing of 2^-6 eps; hidden values are 1 and 0 then)
    eps = float(ref.stands_for(q1, s1, d)[0, 64, 0]) * 2.0 ** 6
    assert eps == (EPS[dtype] if F >= 128 else 0.0)
    ids, gates = _ids(T, E), _gates(T, dtype)
    x = torch.zeros(T, d, device=DEV, dtype=dtype)
    x[:, 0] = 1.0
    want = torch.zeros(T, d, device=DEV, dtype=dtype)
    want[:, 0] = eps
    with torch.no_grad():
        out = eight_bit.glu_mlp_8bit(x, gates, ids, q1, s1, q2, s2)
    assert torch.equal(out, want)
    x.requires_grad_()
    out = eight_bit.glu_mlp_8bit(x, gates, ids, q1, s1, q2, s2, w1_t=t1, w2_t=t2)
    assert torch.equal(out, want)
    dout = torch.zeros_like(want)
    dout[:, 0] = 1.0
    (dx,) = torch.autograd.grad(out, x, dout)
    _all(dx[:, 1], eps)


@pytest.mark.parametrize("T,E,d,F", LAYERS)
def test_rows_of_experts_beyond_float16(T, E, d, F):
    """131072 from an expert, weighed by 1/4 and -1/8: 16384 + 32768 eps, which float16 rounds to 16384; 131072 it would not hold."""
    q1, s1, t1, q2, s2, t2 = _layer(E, d, F, 2.0 ** -12, top=2.0 ** 17)
    ids = _ids(T, E)
    p = torch.tensor([[0.25, -0.125]], device=DEV, dtype=torch.float16).expand(T, 2).contiguous()
    x = torch.zeros(T, d, device=DEV, dtype=torch.float16)
    x[:, 0] = 1.0
    for a in (p, p.clone().requires_grad_()):
        out = eight_bit.glu_mlp_8bit(x, a, ids, q1, s1, q2, s2)
        _all(out[:, 0], 16384.0)
        _all(out[:, 1:], 0.0)
    dout = torch.zeros(T, d, device=DEV, dtype=torch.float16)
    dout[:, 0] = 2.0 ** -4
    (dp,) = torch.autograd.grad(out, a, dout)
    _all(dp, 8192.0)
