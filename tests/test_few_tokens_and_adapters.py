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
        return factor[ids.clamp(0, factor.size(0) - 1)].double() * on.view(-1, 1, 1), on

    @staticmethod
    def adapter_order(ids, R, idx, off):
        groups = torch.where((ids >= 0) & (ids < R), ids, torch.full_like(ids, R))
        idx.copy_(torch.sort(groups, stable=True).indices)
        off.copy_(torch.bincount(groups, minlength=R + 1).cumsum(0))

    @staticmethod
    def adapter_pack(src, dst, off):
        dst.zero_()
        dst[:, :, :src.size(2)] = src

    @classmethod
    def adapter_low(cls, X, A, ids, scales, idx, off, U, planes, slots):
        f, _ = cls._picked(A, ids)
        s = torch.ones(A.size(0)) if scales is None else scales
        U.copy_((f @ X.double().unsqueeze(2)).squeeze(2) * s[ids.clamp(0, A.size(0) - 1)].unsqueeze(1))
        if planes is not None:
            planes.zero_()
            planes[:, 0, :U.size(1)] = U.to(planes.dtype)
            planes[:, 1, :U.size(1)] = (U - planes[:, 0, :U.size(1)].float()).to(planes.dtype)

    @classmethod
    def adapter_project(cls, X, W, bias, U, planes, slots, B, ids, Y):
        f, _ = cls._picked(B[:, :, :U.size(1)], ids)
        u = U.double() if planes is None else planes.double().sum(1)[:, :U.size(1)]
        Y.copy_(X[:, :W.size(1)].double() @ W.double().t() + (f @ u.unsqueeze(2)).squeeze(2) + (0 if bias is None else bias.double()))

    @staticmethod
    def adapter_grad(P, M, idx, off, out):
        lo = 0
        for a, hi in enumerate(off[:out.size(0)].tolist()):
            rows = torch.arange(lo, hi) if idx is None else idx[lo:hi]
            out[a] = (P[rows].double().t() @ M[rows].double()).to(out.dtype)
            lo = hi


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
    assert layer(T=65) == -5 and layer(T=64, k=9, E=16) == -5 and layer(E=513) == -5
    assert layer(x=None) == -1 and layer(ws=None) == -4 and layer(ws_bytes=1000) == -4 and layer(ws=ctypes.c_void_p(264)) == -4
    assert b"workspace" in lib.smoe_last_error()
    assert layer(T=0) == 0
    assert lib.smoe_routed_glu_mlp_workspace_bytes(0, 2, 64, 64) == 0 and lib.smoe_routed_glu_mlp_workspace_bytes(4, 2, 64, 64) >= 8 * 64 * 4
    def low(r=8, R=3, T=4, x=one, idx=None, off=None, planes=None, dtype=1, K=64):
        return lib.smoe_adapter_low(x, 64, one, 64, 64, 1, one, None, idx, off, one, planes, planes, T, K, r, R, dtype, None)
    assert low(r=0) == -2 and low(R=2048) == -5 and low(r=513) == -5 and low(x=None) == -1 and low(dtype=7) == -3
    assert low(idx=one) == -6 and low(planes=one) == -6 and low(idx=one, off=one, planes=one, dtype=0) == -6
    assert low(idx=one, off=one, planes=one, K=7) == -6

    def project(r=8, ids=one, slots=None, T=4):
        return lib.smoe_adapter_project(one, 64, one, 64, 1, None, 0, one, None, slots, one, 8, 8, 1, ids, one, 64, T, 64, 64, r, 3, 1, None)
    assert project(r=513) == -5 and project(ids=None) == -1 and project(slots=one) == -1 and project(T=-1) == -2
    for T, R in ((1, 1), (15, 3), (16, 1), (1777, 16), (100, 2047)):
        assert lib.smoe_adapter_slots(T, R) == 17 * max(1, min(T, T // 16 + R + 1))
    assert lib.smoe_adapter_slots(0, 3) == 0 and lib.smoe_adapter_slots(4, 0) == 0

    def grad(off=one, T=4, C=64, ws=None, ws_bytes=0):
        return lib.smoe_adapter_grad(one, one, 64, None, off, one, 8, 8, 1, T, C, 8, 1, 1, ws, ws_bytes, None)
    assert grad(off=None) == -1 and grad(T=0) == -1 and grad(T=-1) == -2
    assert lib.smoe_adapter_grad_workspace_bytes(8192, 4096, 16, 1, 1) > 0 and lib.smoe_adapter_grad_workspace_bytes(64, 4096, 16, 1, 1) == 0
    assert grad(T=8192, C=4096) == -4 and grad(T=8192, C=4096, ws=one, ws_bytes=64) == -4
    order = lambda ids=one, T=4, R=3, off=one, ws=one, ws_bytes=1 << 20: lib.smoe_adapter_order(ids, T, R, one, off, ws, ws_bytes, None)
    assert order(ids=None) == -1 and order(R=0) == -2 and order(off=None) == -1 and order(ws=None) == -4 and order(ws_bytes=16) == -4
    assert order(R=2048) == -5 and order(ws=ctypes.c_void_p(264)) == -4
    assert lib.smoe_adapter_pack(one, 64, 8, 1, one, 2, 8, 9, 8, None, 1, None) == -2
    assert lib.smoe_adapter_pack(one, 64, 8, 1, None, 2, 8, 8, 8, None, 1, None) == -1
    assert low(T=0) == 0 and lib.smoe_last_error() == b""
