"""Expert ids outside [0, E) (padding, sentinels) on weights in 8 bits: their slots add nothing and have no gradient, in every way that a call goes and
whatever the memory of its buffers held before; the rest has the bits of the call in which those slots go to expert 0 with a gate of zero."""
import pytest
import torch

from scattermoe_amd import eight_bit, flatten_sort_count

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _stale():
    """What later allocations find: no numbers."""
    torch.cuda.synchronize()
    for n in (1 << 12, 1 << 16, 1 << 19, 1 << 20, 1 << 22, 1 << 24, 1 << 26):
        [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for _ in range(6)]


def _ids(T, k, E, share, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    drop = torch.rand(T, k, generator=g) < share
    out = torch.tensor([-1, E, E + 5, 1 << 33])[torch.randint(0, 4, (T, k), generator=g)]
    return torch.where(drop, out, ids).to(DEV), drop.to(DEV)


def _weights(E, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    return eight_bit.quantize_blocks((torch.randn(E, N, K, generator=g) * K ** -0.5).to(DEV), 128, transposed=True)


# by the ids (forward only), streams, tiles with and without the unit behind the product, rows of odd widths
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,d,F,share", [(5, 2, 4, 128, 96, 0.4), (40, 3, 48, 136, 64, 0.3), (150, 2, 5, 256, 128, 0.2), (130, 3, 4, 203, 117, 0.2),
                                             (90, 2, 3, 144, 80, 1.0), (1, 1, 2, 67, 33, 1.0)])
def test_layer(dtype, T, k, E, d, F, share):
    ids, drop = _ids(T, k, E, share, T)
    (q1, s1, t1), (q2, s2, t2) = _weights(E, 2 * F, d, 1), _weights(E, d, F, 2)
    g = torch.Generator().manual_seed(d)
    x, dout = (torch.randn(T, d, generator=g).to(DEV, dtype) for _ in range(2))
    p = (torch.rand(T, k, generator=g) + 0.2).to(DEV, dtype)

    def step(ids, p):
        a, b = x.clone().requires_grad_(), p.clone().requires_grad_()
        with torch.no_grad():
            _stale()
            plain = eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2)
        _stale()
        out = eight_bit.glu_mlp_8bit(a, b, ids, q1, s1, q2, s2, w1_t=t1, w2_t=t2)
        _stale()
        return [plain, out.detach(), *torch.autograd.grad(out, (a, b), dout)]

    want = step(torch.where(drop, 0, ids), torch.where(drop, 0.0, p).to(dtype))
    want[3] = torch.where(drop, 0.0, want[3]).to(dtype)
    got = step(ids, torch.where(drop, float("nan"), p).to(dtype))
    for name, a, b in zip(("out, forward only", "out", "dx", "dgates"), got, want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,N,share", [(5, 2, 4, 128, 96, 0.4), (150, 2, 5, 256, 128, 0.2), (130, 3, 4, 203, 117, 0.2), (20, 2, 3, 144, 80, 1.0)])
def test_products(dtype, T, k, E, K, N, share):
    ids, drop = _ids(T, k, E, share, K)
    q, s, qt = _weights(E, N, K, 3)
    g = torch.Generator().manual_seed(N)
    x, dy = torch.randn(T, K, generator=g).to(DEV, dtype), torch.randn(T * k, N, generator=g).to(DEV, dtype)
    eid, idx, off = flatten_sort_count(ids, E)
    n = int(off[-1])
    a = x.clone().requires_grad_()
    _stale()
    y = eight_bit.parallel_linear_8bit(a, q, s, k, eid, idx, off, weight_t=qt)
    _stale()
    (dx,) = torch.autograd.grad(y, a, dy)
    _stale()
    grouped = eight_bit.parallel_linear_8bit(x, q, s, k, eid, idx, off, grouped_out=True)
    order = flatten_sort_count(torch.where(drop, 0, ids), E)
    b = x.clone().requires_grad_()
    z = eight_bit.parallel_linear_8bit(b, q, s, k, *order, weight_t=qt)
    none = drop.reshape(-1, 1)
    (db,) = torch.autograd.grad(z, b, torch.where(none, 0.0, dy).to(dtype))
    assert torch.equal(y, torch.where(none, 0.0, z).to(dtype)) and torch.equal(dx, db)
    assert torch.equal(grouped[:n], y[idx[:n]]) and not bool(grouped[n:].any())
    # rows that come grouped, weighed by the gates
    h, p = torch.randn(T * k, K, generator=g).to(DEV, dtype), torch.rand(T, k, generator=g).to(DEV, dtype)
    rows = torch.zeros(T * k, N, device=DEV)
    _stale()
    rows[idx[:n]] = eight_bit.parallel_linear_8bit(h.float(), q, s, 1, eid, idx, off, grouped_in=True, grouped_out=True)[:n]
    _stale()
    got = eight_bit.parallel_linear_8bit(h.float(), q, s, 1, eid, idx, off, gates=p.float(), grouped_in=True)
    want = (rows.view(T, k, N) * p.float().unsqueeze(-1)).double().sum(1)
    assert bool(((got - want).abs() <= (k + 2) * 2.0 ** -24 * (rows.view(T, k, N).abs() * p.float().unsqueeze(-1)).sum(1) + 1e-30).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,E,d,F", [(5, 2, 4, 128, 96), (40, 3, 48, 136, 64), (150, 2, 5, 256, 128)])
def test_replayed_with_other_padding(dtype, T, k, E, d, F):
    """A captured forward pass and a captured step, replayed with no, some and only dropped slots, and none again: each the eager call's bits."""
    (q1, s1, t1), (q2, s2, t2) = _weights(E, 2 * F, d, 1), _weights(E, d, F, 2)
    g = torch.Generator().manual_seed(d)
    x, dout = (torch.randn(T, d, generator=g).to(DEV, dtype) for _ in range(2))
    p = (torch.rand(T, k, generator=g) + 0.2).to(DEV, dtype)
    ids = _ids(T, k, E, 0.0, 1)[0]

    def step():
        a, b = x.detach().requires_grad_(), p.detach().requires_grad_()
        out = eight_bit.glu_mlp_8bit(a, b, ids, q1, s1, q2, s2, w1_t=t1, w2_t=t2)
        return [out.detach(), *torch.autograd.grad(out, (a, b), dout)]

    def forward():
        with torch.no_grad():
            return eight_bit.glu_mlp_8bit(x, p, ids, q1, s1, q2, s2)

    forward(), step()
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        out = forward()
    with torch.cuda.graph(two, pool=one.pool()):
        got = step()
    for r, share in enumerate((0.0, 0.3, 1.0, 0.2, 0.0)):
        ids.copy_(_ids(T, k, E, share, r)[0])
        x.copy_(torch.randn(T, d, generator=g))
        one.replay()
        want = forward()
        torch.cuda.synchronize()
        assert torch.equal(out, want), r
        two.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r
