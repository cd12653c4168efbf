"""Host side of the few-token layer and of the adapters, without a GPU: refusals, shapes, the general path, what a tracing
compiler sees, and the library's own argument checks."""
import ctypes

import pytest
import torch

import oracle  # noqa: F401  (the test double's)
from _cpu_backend import OracleBackend
from scattermoe_amd import ParallelAdapters, _C, parallel_adapters
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import RoutedGLUMLP, routed_glu_mlp


class _Backend(OracleBackend):
    @staticmethod
    def route(flat_ids, num_experts, eid, idx, off):
        """With ids outside [0, num_experts) dropped: behind the others, expert num_experts, slot -1."""
        ids = flat_ids.long()
        on = (ids >= 0) & (ids < num_experts)
        slots = on.nonzero().squeeze(1)
        order = torch.sort(ids[slots], stable=True)
        eid.fill_(num_experts), idx.fill_(-1)
        eid[:len(slots)] = order.values
        idx[:len(slots)] = slots[order.indices]
        off.copy_(torch.bincount(ids[slots], minlength=num_experts).cumsum(0))

    @staticmethod
    def routed_glu_mlp(x, wr, w1, b1, w2, b2, out, logits, k, renormalize, act):
        l = x.double() @ wr.double().t()
        p = torch.softmax(l, -1)
        order = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, :k]
        g = p.gather(1, order)
        g = g / g.sum(-1, keepdim=True) if renormalize else g
        total = torch.zeros(x.shape, dtype=torch.double)
        for j in range(k):
            e = order[:, j]
            pre = (w1[e].double() @ x.double().unsqueeze(2)).squeeze(2) + (0 if b1 is None else b1[e].double())
            lin, gate = pre.chunk(2, -1)
            if act & 1:
                lin, gate = gate, lin
            y = (w2[e].double() @ (lin * torch.nn.functional.silu(gate)).unsqueeze(2)).squeeze(2)
            total += g[:, j:j + 1] * (y + (0 if b2 is None else b2[e].double()))
        out.copy_(total)
        logits.copy_(l)

    @staticmethod
    def _picked(factor, ids):
        on = (ids >= 0) & (ids < factor.size(0))
        return factor[ids.clamp(0, factor.size(0) - 1)].double() * on.view(-1, 1, 1)

    @classmethod
    def _product(cls, X, W, A, B, ids, scales):
        s = torch.ones(A.size(0)) if scales is None else scales
        u = (cls._picked(A, ids) @ X.double().unsqueeze(2)).squeeze(2) * s[ids.clamp(0, A.size(0) - 1)].unsqueeze(1)
        return u, X.double() @ W.double().t() + (cls._picked(B, ids) @ u.unsqueeze(2)).squeeze(2)

    @classmethod
    def adapter_forward(cls, X, W, bias, A, B, ids, scales, idx, off, U, Y):
        u, y = cls._product(X, W, A, B, ids, scales)
        U.copy_(u)
        Y.copy_(y if bias is None else y + bias.double())
        if idx is not None:
            groups = torch.where((ids >= 0) & (ids < A.size(0)), ids, torch.full_like(ids, A.size(0)))
            idx.copy_(torch.sort(groups, stable=True).indices)
            off.copy_(torch.bincount(groups, minlength=A.size(0) + 1).cumsum(0))

    @classmethod
    def adapter_backward(cls, DY, X, W, A, B, ids, scales, idx, off, U, DX, DA, DB, DBIAS):
        v, dx = cls._product(DY, W.t(), B.transpose(1, 2), A.transpose(1, 2), ids, scales)
        if DX is not None:
            DX.copy_(dx)
        for a in range(A.size(0)):
            rows = ids == a
            if DA is not None:
                DA[a] = (v[rows].t() @ X[rows].double()).to(DA.dtype)
            if DB is not None:
                DB[a] = (DY[rows].double().t() @ U[rows].double()).to(DB.dtype)
        if DBIAS is not None:
            DBIAS.copy_(DY.double().sum(0))


@pytest.fixture
def backend(monkeypatch):
    monkeypatch.setattr(ops, "_backend", _Backend())


def _layer(dtype=torch.float32):
    torch.manual_seed(0)
    m = RoutedGLUMLP(16, 24, 6, 2, bias=True)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape) * 0.3)
    return m.to(dtype)


def test_layer_paths_agree(backend):
    m, x = _layer(), torch.randn(5, 16)
    with torch.no_grad():
        few, logits = m(x)
        many = m(x.repeat(20, 1))
    trained = m(x)
    assert few.shape == (5, 16) and logits.shape == (5, 6) and logits.dtype == torch.float32
    for other in (many[0][:5], trained[0]):
        torch.testing.assert_close(few, other, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(logits, trained[1], rtol=1e-5, atol=1e-5)
    assert set(m.state_dict()) == {"router.weight", "experts.weight", "experts.bias", "output_experts.weight", "output_experts.bias"}


def test_layer_of_leading_dimensions(backend):
    m, x = _layer(), torch.randn(2, 3, 16)
    with torch.no_grad():
        out, logits = m(x)
        assert out.shape == x.shape and logits.shape == (6, 6)
        assert m(x[:0])[0].shape == (0, 3, 16)


def test_layer_refusals():
    m = _layer()
    args = (m.router.weight, m.experts.weight, m.output_experts.weight)
    x = torch.randn(5, 16)
    with torch.no_grad():
        for bad in (0, 7, 65):
            with pytest.raises(ValueError):
                routed_glu_mlp(x, *args, bad)
        with pytest.raises(ValueError):
            routed_glu_mlp(x[:, :15], *args, 2)
        with pytest.raises(ValueError):
            routed_glu_mlp(x, args[0], args[1][:, 1:], args[2], 2)
        with pytest.raises(ValueError):
            routed_glu_mlp(x, *args, 2, b1=torch.zeros(6, 24))
        with pytest.raises(TypeError):
            routed_glu_mlp(x.half(), *args, 2)
        with pytest.raises(RuntimeError, match="no CPU path"):
            routed_glu_mlp(x, *args, 2)
    assert ops.few_tokens(64, 8, 128) and not ops.few_tokens(65, 1, 8) and not ops.few_tokens(64, 9, 128) and not ops.few_tokens(0, 1, 1)


@pytest.mark.parametrize("times", [1, 10])
def test_adapters_values_and_gradients(backend, times):
    """Row by row, and with the rows in order."""
    torch.manual_seed(0)
    m = ParallelAdapters(3, 10, 7, 4, bias=True, scale=0.5)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape))
    x = torch.randn(2, 6 * times, 10, requires_grad=True)
    ids = torch.tensor([[0, 1, -1, 2, 2, 3], [1, 1, 0, 9, 2, 0]]).repeat(1, times)
    y = m(x, ids)
    flat = ids.reshape(-1)
    on = ((flat >= 0) & (flat < 3)).float()
    safe = flat.clamp(0, 2)

    def plain(x, w, b, la, lb):
        rows = x.reshape(-1, 10)
        low = (la[safe] @ rows.unsqueeze(2)).squeeze(2) * 0.5 * on.unsqueeze(1)
        return (rows @ w.t() + b + (lb[safe] @ low.unsqueeze(2)).squeeze(2)).view(2, 6 * times, 7)
    leaves = [x, m.weight, m.bias, m.lora_a, m.lora_b]
    want = plain(*leaves)
    torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-5)
    dy = torch.randn(2, 6 * times, 7)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


def test_adapters_refusals():
    x, w, la, lb, ids = torch.randn(4, 10), torch.randn(7, 10), torch.randn(3, 4, 10), torch.randn(3, 7, 4), torch.zeros(4, dtype=torch.int64)
    for args, kw, error in (((x[:, :9], w, la, lb, ids), {}, ValueError), ((x, w, la, lb[:2], ids), {}, ValueError),
                            ((x, w, la, lb, ids[:3]), {}, ValueError), ((x, w, la, lb, ids.float()), {}, TypeError),
                            ((x, w, la, lb, ids.bool()), {}, TypeError), ((x.half(), w, la, lb, ids), {}, TypeError),
                            ((x, w, la, lb, ids), {"scales": torch.ones(2)}, ValueError),
                            ((x, w, la, lb, ids), {"scales": torch.ones(3, requires_grad=True)}, ValueError),
                            ((x, w, la, lb, ids), {"bias": torch.ones(6)}, ValueError),
                            ((x, w, la.expand(3, 4, 10)[:0], lb[:0], ids), {}, ValueError)):
        with pytest.raises(error):
            parallel_adapters(*args, **kw)
    with pytest.raises(ValueError, match="2047"):
        parallel_adapters(x, w, la[:1].expand(2048, 4, 10), lb[:1].expand(2048, 7, 4), ids)
    with pytest.raises(RuntimeError, match="no CPU path"):
        parallel_adapters(x, w, la, lb, ids)


def test_fullgraph_trace(backend):
    m, layer = ParallelAdapters(3, 16, 16, 4).requires_grad_(), _layer()
    with torch.no_grad():
        m.lora_b.normal_()
    x, ids = torch.randn(5, 16, requires_grad=True), torch.tensor([0, 2, -1, 1, 1])

    def block(x):
        return layer(m(x, ids))[0]
    want = block(x)
    torch._dynamo.reset()
    compiled = torch.compile(block, fullgraph=True, backend="aot_eager")
    got = compiled(x)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    leaves = [x] + list(m.parameters())
    for a, b in zip(torch.autograd.grad(got.sum(), leaves, allow_unused=True), torch.autograd.grad(want.sum(), leaves, allow_unused=True)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        torch.testing.assert_close(torch.compile(block, fullgraph=True, backend="aot_eager")(x), block(x), rtol=1e-5, atol=1e-6)


def test_library_refuses_before_it_launches():
    lib = _C.load()
    one = ctypes.c_void_p(256)

    def layer(T=4, k=2, d=64, F=64, E=8, act=0, dtype=1, x=one, ws=one, ws_bytes=1 << 30):
        return lib.smoe_routed_glu_mlp(x, d, 1, one, d, 1, one, 2 * F * d, d, 1, None, 0, 0, one, F * d, F, 1, None, 0, 0, one, d, one,
                                       T, k, d, F, E, 1, act, dtype, ws, ws_bytes, None)
    assert layer(dtype=5) == -3 and layer(k=0) == -2 and layer(k=9) == -2 and layer(F=0) == -2 and layer(act=3) == -2
    assert layer(T=ops.FEW_TOKENS + 1) == -5 and layer(F=1 << 29) == -5 and layer(T=64, k=9, E=16) == -5 and layer(E=513) == -5
    assert layer(x=None) == -1 and layer(ws=None) == -4 and layer(ws_bytes=1000) == -4 and layer(ws=ctypes.c_void_p(264)) == -4
    assert b"workspace" in lib.smoe_last_error()
    assert layer(T=0) == 0
    assert lib.smoe_routed_glu_mlp_workspace_bytes(0, 2, 64, 64) == 0 and lib.smoe_routed_glu_mlp_workspace_bytes(4, 2, 64, 64) >= 8 * 64 * 4
    bytes_ = lib.smoe_adapter_workspace_bytes
    assert bytes_(0, 64, 64, 8, 3, 0, 1) == 0 and bytes_(4, 64, 64, 0, 3, 0, 1) == 0 and bytes_(4, 64, 64, 8, 2048, 0, 1) == 0

    def forward(T=100, K=64, N=64, r=8, R=3, x=one, idx=one, dtype=1, ws=one, ws_bytes=1 << 30):
        return lib.smoe_adapter_forward(x, K, one, None, one, one, one, None, idx, one, one, one, T, K, N, r, R, dtype, ws, ws_bytes, None)
    assert forward(r=0) == -2 and forward(R=0) == -2 and forward(K=0) == -2 and forward(T=-1) == -2 and forward(dtype=7) == -3
    assert forward(R=2048) == -5 and forward(r=513) == -5 and forward(T=1 << 31) == -5 and forward(x=None) == -1
    assert forward(idx=None) == -1 and forward(ws=None) == -4 and forward(ws_bytes=1000) == -4 and forward(ws=ctypes.c_void_p(264)) == -4

    def backward(T=100, K=64, N=64, dy=one, idx=one, ws=one, ws_bytes=1 << 30):
        return lib.smoe_adapter_backward(dy, one, K, one, one, one, one, None, idx, one, one, one, one, one, one, T, K, N, 8, 3, 1, ws,
                                         ws_bytes, None)
    assert backward(T=0) == -2 and backward(N=0) == -2 and backward(dy=None) == -1 and backward(idx=None) == -1
    assert backward(T=ops.ADAPTER_FEW_ROWS, idx=None, ws=None) == -4 and backward(T=ops.ADAPTER_FEW_ROWS + 1, idx=None, ws=None) == -1
    assert backward(ws=None) == -4 and backward(ws_bytes=1000) == -4 and backward(T=4, ws=None) == -4
    assert forward(T=0) == 0 and lib.smoe_last_error() == b""
