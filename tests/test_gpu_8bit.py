"""8-bit rows and weights, the products on them, the gated layer and the gated unit's 8-bit checkpoint against the same in 64 bits."""
import pytest
import torch

import _ref_8bit as ref
from scattermoe_amd import eight_bit, flatten_sort_count
from scattermoe_amd.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * std).to(dtype)


def _bits(t):
    return t.cpu().view(torch.uint8)


# ---- rows ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (5, 16), (2, 127), (7, 128), (4, 129), (130, 1003), (65, 2880), (0, 64), (3, 0)])
def test_rows_in_8_bits_are_exact(dtype, rows, K):
    g = torch.Generator().manual_seed(rows * 10007 + K)
    x = _normal(g, rows, K) * torch.exp(3 * _normal(g, rows, 1))
    x = x.to(dtype)
    q, s = eight_bit.quantize_blocks(x.to(DEV))
    assert q.shape == (rows, -(-K // 16) * 16) and s.shape == (rows, -(-K // 128))
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu
    if rows == 0 or K == 0:
        return
    want, ex = ref.q8(x.double())
    assert torch.equal(s.cpu().float().double(), torch.ldexp(torch.ones_like(ex, dtype=torch.double), ex))
    assert torch.equal(ref.stands_for(q, s, K, 1), want)
    assert not bool(_bits(q)[:, K:].any())
    back = eight_bit.dequantize_blocks(q, s, size=K, dtype=torch.float32)
    assert torch.equal(back.cpu().double(), want)


def test_rows_with_every_kind_of_value():
    big = torch.finfo(torch.float32).max
    x = torch.zeros(8, 300)
    x[1, 0], x[1, 200] = big, -big
    x[2, :128] = torch.arange(128) * 2.0 ** -149                     # subnormal numbers
    x[3, :256] = 448.0 * torch.ldexp(torch.ones(256), torch.arange(256, dtype=torch.int32) % 2)
    x[4, 5], x[4, 6] = float("nan"), 3.0
    x[5, 128], x[5, 3] = float("inf"), 2.0
    x[6, 7] = 448.0000305                                           # one step above what scale 1 holds
    x[7, ::3] = -0.0
    q, s = eight_bit.quantize_blocks(x.to(DEV))
    v = ref.stands_for(q, s, 300, 1)
    clean = x.clone()
    clean[4, 5], clean[5, 128:256] = 0, 0
    want, ex = ref.q8(clean.double())
    assert bool(torch.isnan(v[4, 5])) and float(v[4, 6]) == 3.0
    assert bool(torch.isnan(v[5, 128])) and float(v[5, 3]) == 2.0
    v[4, 5], v[5, 128] = 0, 0
    assert torch.equal(v, want)
    assert float(s.cpu().float()[6, 0]) == 2.0 and float(s.cpu().float()[3, 0]) == 2.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_strides(dtype):
    g = torch.Generator().manual_seed(3)
    wide = _normal(g, 9, 401, dtype=dtype).to(DEV)
    for x in (wide[:, 1:300], wide[::2, :256], wide.t(), wide[:1].expand(5, -1), wide.view(3, 3, 401)):
        q, s = eight_bit.quantize_blocks(x)
        flat = x.reshape(-1, x.size(-1)).cpu().double()
        assert torch.equal(ref.stands_for(q.reshape(-1, q.size(-1)), s.reshape(-1, s.size(-1)), x.size(-1), 1), ref.q8(flat)[0])
        back = eight_bit.dequantize_blocks(q, s, size=x.size(-1), dtype=torch.float32)
        assert back.shape == x.shape and torch.equal(back.reshape(flat.shape).cpu().double(), ref.q8(flat)[0])


# ---- weights -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,N,K", [(1, 1, 1), (2, 130, 127), (3, 128, 256), (2, 203, 300), (1, 17, 2880)])
def test_weights_in_8_bits_are_exact(dtype, E, N, K):
    g = torch.Generator().manual_seed(E + N + K)
    w = (_normal(g, E, N, K) * torch.exp(_normal(g, E, N, 1))).to(dtype)
    q, s, qt = eight_bit.quantize_blocks(w.to(DEV), 128, transposed=True)
    want, ex = ref.q8(w.double(), 128)
    assert torch.equal(s.cpu().float().double(), torch.ldexp(torch.ones_like(ex, dtype=torch.double), ex))
    assert torch.equal(ref.stands_for(q, s, K), want)
    assert torch.equal(ref.stands_for(qt, s.transpose(1, 2), N), want.transpose(1, 2))
    assert not bool(_bits(q)[:, :, K:].any()) and not bool(_bits(qt)[:, :, N:].any())
    assert torch.equal(eight_bit.dequantize_blocks(q, s, 128, size=K, dtype=torch.float32).cpu().double(), want)
    view = w.to(DEV).transpose(1, 2)                                 # not contiguous
    q2, s2 = eight_bit.quantize_blocks(view, 128)
    assert torch.equal(_bits(q2), _bits(qt)) and torch.equal(_bits(s2), _bits(s).transpose(1, 2))


def _weight(g, E, N, K, std, float_scales):
    """A weight on the GPU with its transpose, and its values in 64 bits."""
    w = _normal(g, E, N, K, std=std) * torch.exp(0.5 * _normal(g, E, N, 1))
    q, s, qt = eight_bit.quantize_blocks(w.to(DEV), 128, transposed=True)
    if float_scales:
        s = s.float() * (0.5 + torch.rand(s.shape, generator=g)).to(DEV)
    return q, s, qt, ref.stands_for(q, s, K)


def _ids(g, T, E, k, kind):
    if kind == "one":                                                # everything to the last expert
        return torch.full((T, k), E - 1)
    if kind == "same":                                               # a token's slots name one expert several times
        return torch.randint(0, E, (T, 1), generator=g).expand(T, k).contiguous()
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T else torch.zeros(0, k, dtype=torch.long)
    return ids.clamp(max=max(0, E - 2)) if kind == "gap" else ids    # the last expert without rows


PRODUCTS = [
    # T, k, E, K, N, ids
    (1, 1, 1, 16, 1, "any"), (1, 2, 3, 64, 40, "any"), (5, 3, 13, 203, 117, "any"), (37, 2, 5, 300, 203, "gap"), (64, 4, 8, 128, 256, "any"),
    (130, 1, 2, 129, 257, "any"), (150, 2, 4, 520, 300, "one"), (90, 2, 6, 1000, 72, "same"), (0, 2, 3, 64, 32, "any"), (300, 2, 3, 272, 513, "any"),
    (50, 2, 16, 144, 200, "any"), (24, 4, 12, 208, 72, "same"),                                  # 4 to 8 rows per expert
    (22, 2, 4, 4104, 136, "any"),                                                                # 11, of a long contraction
    (300, 1, 2, 8208, 100, "any"), (400, 2, 3, 144, 264, "gap"),                                   # 150 and 270 rows per expert
    (50, 1, 2, 8400, 260, "any"), (30, 2, 3, 72, 8320, "gap"), (70, 1, 4, 9000, 17, "one"),      # long contractions of few tiles
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("float_scales", [False, True])
@pytest.mark.parametrize("T,k,E,K,N,kind", PRODUCTS)
def test_product_and_its_gradient(dtype, float_scales, T, k, E, K, N, kind):
    g = torch.Generator().manual_seed(T * 31 + K)
    x, ids = _normal(g, T, K, dtype=dtype), _ids(g, T, E, k, kind)
    q, s, qt, w = _weight(g, E, N, K, K ** -0.5, float_scales)
    b = _normal(g, E, N, dtype=dtype) if T % 2 else None
    dy = _normal(g, T * k, N, dtype=dtype)
    eid, idx, off = flatten_sort_count(ids.to(DEV), E)
    xg = x.to(DEV).requires_grad_()
    y = eight_bit.parallel_linear_8bit(xg, q, s, k, eid, idx, off, expert_biases=None if b is None else b.to(DEV), grouped_out=True, weight_t=qt)
    (dx,) = torch.autograd.grad(y, xg, dy.to(DEV))
    assert y.dtype == dtype and dx.dtype == dtype
    rows16 = dtype != torch.float32
    x8, dy8 = (ref.q8(t.double())[0] if t.numel() else t.double() for t in (x, dy))
    eid, idx = eid.cpu(), idx.cpu()
    want, bound = torch.zeros(T * k, N, dtype=torch.double), torch.zeros(T * k, N, dtype=torch.double)
    back, berr = torch.zeros(T * k, K, dtype=torch.double), torch.zeros(T * k, K, dtype=torch.double)
    for e in range(E):
        mine = eid == e
        if not bool(mine.any()):
            continue
        v, err = ref.product(x8[idx[mine] // k], torch.zeros(int(mine.sum()), K, dtype=torch.double), w[e], rows16, float_scales)
        if b is not None:
            v = v + b[e].double()
            err = err + 2 * ref.U * v.abs()
        want[mine], bound[mine] = v, ref.rounded(v, err, dtype)
        v, err = ref.product(dy8[mine], torch.zeros(int(mine.sum()), N, dtype=torch.double), w[e].t(), rows16, float_scales)
        back[idx[mine]], berr[idx[mine]] = v, ref.rounded(v, err, dtype)
    ref.check("y", y, want, bound)
    v, err = back.view(T, k, K).sum(1), berr.view(T, k, K).sum(1) + k * ref.U * back.view(T, k, K).abs().sum(1)
    ref.check("dx", dx, v, ref.rounded(v, err, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,N", [(3, 2, 4, 96, 80), (70, 3, 5, 260, 144)])
def test_product_with_gates_and_grouped_rows(dtype, T, k, E, K, N):
    """x grouped -> weighted sum over the slots, with the gradients of rows and gates (the second product of a layer)."""
    g = torch.Generator().manual_seed(T)
    ids = _ids(g, T, E, k, "any")
    x, dy = _normal(g, T * k, K, dtype=dtype), _normal(g, T, N, dtype=dtype)
    p = torch.rand((T, k), generator=g).to(dtype)
    q, s, qt, w = _weight(g, E, N, K, K ** -0.5, False)
    eid, idx, off = flatten_sort_count(ids.to(DEV), E)
    xg, pg = x.to(DEV).requires_grad_(), p.to(DEV).requires_grad_()
    y = eight_bit.parallel_linear_8bit(xg, q, s, 1, eid, idx, off, gates=pg, grouped_in=True, weight_t=qt)
    dx, dp = torch.autograd.grad(y, (xg, pg), dy.to(DEV))
    rows16 = dtype != torch.float32
    x8 = ref.q8(x.double())[0]
    eid, idx = eid.cpu(), idx.cpu()
    rows, rerr = torch.zeros(T * k, N, dtype=torch.double), torch.zeros(T * k, N, dtype=torch.double)
    dgate = (dy.double()[idx // k] * p.double().reshape(-1)[idx].unsqueeze(1))
    d8, d8err = ref.q8_known(dgate, ref.U * dgate.abs() if dtype == torch.float32 else 0 * dgate)
    back, berr = torch.zeros(T * k, K, dtype=torch.double), torch.zeros(T * k, K, dtype=torch.double)
    for e in range(E):
        mine = eid == e
        v, err = ref.product(x8[mine], torch.zeros(int(mine.sum()), K, dtype=torch.double), w[e], rows16, False)
        rows[idx[mine]], rerr[idx[mine]] = v, ref.rounded(v, err, dtype)
        v, err = ref.product(d8[mine], d8err[mine], w[e].t(), rows16, False)
        back[mine], berr[mine] = v, ref.rounded(v, err, dtype)
    p64 = p.double().unsqueeze(-1)
    v = (rows.view(T, k, N) * p64).sum(1)
    err = (rerr.view(T, k, N) * p64).sum(1) + (k + 2) * ref.U * (rows.view(T, k, N).abs() * p64).sum(1)
    ref.check("y", y, v, ref.rounded(v, err, dtype))
    ref.check("dx", dx, back, berr)
    v = (rows.view(T, k, N) * dy.double().unsqueeze(1)).sum(-1)
    size = (rows.view(T, k, N).abs() * dy.double().abs().unsqueeze(1)).sum(-1)
    err = (rerr.view(T, k, N) * dy.double().abs().unsqueeze(1)).sum(-1) + 2 * (N + 8) * ref.U * size
    ref.check("dgates", dp, v, ref.rounded(v, err, dtype))


# ---- the layer -----------------------------------------------------------------------------------------
def _layer_reference(x, p, ids, w1, w2, b1, b2, dout, rows16, float_scales, gate_first, dtype):
    """out, dx, dgates with bounds; w1 (E, 2F, d), w2 (E, d, F) float64."""
    (T, k), d, F = ids.shape, x.size(1), w2.size(2)
    x8 = ref.q8(x.double())[0]
    zero = lambda *s: torch.zeros(*s, dtype=torch.double)
    y, yerr, back, berr = zero(T * k, d), zero(T * k, d), zero(T * k, d), zero(T * k, d)
    p64, do = p.double(), dout.double()
    for e in ids.unique().tolist():
        mine = (ids.reshape(-1) == e).nonzero().squeeze(1)
        tok = mine // k
        pre, err = ref.product(x8[tok], zero(len(mine), d), w1[e], rows16, float_scales)
        if b1 is not None:
            pre = pre + b1[e].double()
            err = err + 2 * ref.U * pre.abs()
        (lin, lerr), (gate, gerr) = (pre[:, :F], err[:, :F]), (pre[:, F:], err[:, F:])
        if gate_first:
            (lin, lerr), (gate, gerr) = (gate, gerr), (lin, lerr)
        h8, herr = ref.q8_known(*ref.unit(lin, lerr, gate, gerr))
        v, err = ref.product(h8, herr, w2[e], rows16, float_scales)
        if b2 is not None:
            v = v + b2[e].double()
            err = err + 2 * ref.U * v.abs()
        y[mine], yerr[mine] = v, ref.rounded(v, err, dtype)
        dgate = do[tok] * p64.reshape(-1)[mine].unsqueeze(1)
        d8, d8err = ref.q8_known(dgate, (0 if rows16 else ref.U) * dgate.abs())
        dh, derr = ref.product(d8, d8err, w2[e].t(), rows16, float_scales)
        lin8, l8err = ref.q8_known(lin, lerr)
        gat8, g8err = ref.q8_known(gate, gerr)
        dl, dlerr, dg, dgerr = ref.unit_grad(dh, derr, lin8, gat8)
        # (a half whose 8 bits may be one step further: the gradient's largest change over that step, silu' <= 1.1, silu'' <= 0.5)
        dlerr = dlerr + (dh.abs() + derr) * 1.1 * g8err
        dgerr = dgerr + (dh.abs() + derr) * (1.1 * l8err + 0.5 * (lin8.abs() + l8err) * g8err)
        parts = [(dg, dgerr), (dl, dlerr)] if gate_first else [(dl, dlerr), (dg, dgerr)]
        dp8, dp8err = ref.q8_known(torch.cat([t for t, _ in parts], 1), torch.cat([t for _, t in parts], 1))
        v, err = ref.product(dp8, dp8err, w1[e].t(), rows16, float_scales)
        back[mine], berr[mine] = v, ref.rounded(v, err, dtype)
    g3 = p64.unsqueeze(-1)
    out = (y.view(T, k, d) * g3).sum(1)
    oerr = (yerr.view(T, k, d) * g3).sum(1) + (k + 2) * ref.U * (y.view(T, k, d).abs() * g3).sum(1)
    dx = back.view(T, k, d).sum(1)
    dxerr = berr.view(T, k, d).sum(1) + (k + 2) * ref.U * back.view(T, k, d).abs().sum(1)
    dg = (y.view(T, k, d) * do.unsqueeze(1)).sum(-1)
    dgerr = ((yerr.view(T, k, d) + 2 * (d + 8) * ref.U * y.view(T, k, d).abs()) * do.abs().unsqueeze(1)).sum(-1)
    return [(out, ref.rounded(out, oerr, dtype)), (dx, ref.rounded(dx, dxerr, dtype)), (dg, ref.rounded(dg, dgerr, dtype))]


LAYERS = [
    # T, k, E, d, F, ids, bias, gate_first
    (1, 1, 1, 32, 16, "any", False, False), (1, 2, 4, 128, 96, "any", True, False), (3, 4, 6, 203, 117, "any", False, True),
    (8, 2, 3, 256, 128, "same", True, False), (33, 2, 5, 130, 203, "gap", True, True), (70, 2, 4, 256, 160, "one", False, False),
    (140, 3, 4, 160, 256, "any", True, False), (0, 2, 3, 64, 32, "any", False, False),
    (16, 2, 8, 144, 80, "one", True, False), (10, 4, 12, 203, 117, "same", False, True), (32, 2, 3, 136, 200, "any", True, True),
    (45, 2, 4, 144, 96, "any", True, True), (30, 2, 3, 144, 80, "one", True, False), (25, 2, 8, 200, 72, "any", True, True),
    (200, 2, 2, 144, 384, "any", True, True), (60, 1, 2, 8208, 128, "any", False, True), (150, 2, 3, 200, 96, "any", False, False),
    (40, 1, 2, 8208, 128, "any", True, True), (20, 2, 1, 96, 8200, "same", False, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("float_scales", [False, True])
@pytest.mark.parametrize("T,k,E,d,F,kind,bias,gate_first", LAYERS)
def test_layer_and_its_gradients(dtype, float_scales, T, k, E, d, F, kind, bias, gate_first):
    g = torch.Generator().manual_seed(T * 17 + d)
    x, ids = _normal(g, T, d, dtype=dtype), _ids(g, T, E, k, kind)
    p = (torch.rand((T, k), generator=g) + 0.2).to(dtype)
    q1, s1, t1, w1 = _weight(g, E, 2 * F, d, d ** -0.5, float_scales)
    q2, s2, t2, w2 = _weight(g, E, d, F, F ** -0.5, float_scales)
    b1, b2 = (_normal(g, E, n, dtype=dtype) if bias else None for n in (2 * F, d))
    dout = _normal(g, T, d, dtype=dtype)
    up = lambda t: None if t is None else t.to(DEV)
    xg, pg = up(x).requires_grad_(), up(p).requires_grad_()
    call = lambda a, b, **kw: eight_bit.glu_mlp_8bit(a, b, up(ids), q1, s1, q2, s2, b1=up(b1), b2=up(b2), gate_first=gate_first, **kw)
    out = call(xg, pg, w1_t=t1, w2_t=t2)
    dx, dp = torch.autograd.grad(out, (xg, pg), up(dout))
    with torch.no_grad():
        plain = call(xg, pg)
    if T == 0:
        assert out.shape == (0, d) and dx.shape == (0, d) and dp.shape == (0, k) and plain.shape == (0, d)
        return
    want = _layer_reference(x, p, ids, w1, w2, b1, b2, dout, dtype != torch.float32, float_scales, gate_first, dtype)
    for name, got, (v, bound) in zip(("out", "dx", "dgates"), (out, dx, dp), want):
        ref.check(name, got, v, bound)
    ref.check("out, forward only", plain, *want[0])
    if T * k <= ops.FEW_ROWS_8BIT:
        act = ops.ACT_SILU_GATE_FIRST if gate_first else ops.ACT_SILU
        by_ids = ops.glu_mlp_8bit(up(x), up(p), q1, s1, up(b1), q2, s2, up(b2), experts=up(ids), act=act)[0]
        ref.check("out, by the ids", by_ids, *want[0])
    (dp2,) = torch.autograd.grad(call(xg.detach(), pg), pg, up(dout))      # gates alone: no transposed weights
    ref.check("dgates alone", dp2, *want[2])


# ---- the gated unit --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,F,gate_first", [(1, 1, False), (3, 8, True), (5, 127, False), (4, 128, True), (7, 129, False), (33, 1411, False), (130, 256, True),
                                               (0, 16, False), (2, 0, False)])
def test_unit_with_its_checkpoint(dtype, rows, F, gate_first):
    g = torch.Generator().manual_seed(rows + F)
    pre, dh = _normal(g, rows, 2 * F, std=2.0, dtype=dtype), _normal(g, rows, F, dtype=dtype)
    a = pre.to(DEV).requires_grad_()
    h = eight_bit.checkpointed_glu(a, gate_first=gate_first)
    (da,) = torch.autograd.grad(h, a, dh.to(DEV))
    assert h.shape == (rows, F) and da.shape == (rows, 2 * F)
    if rows == 0 or F == 0:
        return
    with torch.no_grad():
        assert torch.equal(eight_bit.checkpointed_glu(a, gate_first=gate_first), h)
    one, two = pre.double()[:, :F], pre.double()[:, F:]
    zero = torch.zeros_like(one)
    lin, gate = (two, one) if gate_first else (one, two)
    v, err = ref.unit(lin, zero, gate, zero)
    ref.check("h", h, v, ref.rounded(v, err, dtype))
    dl, dlerr, dg, dgerr = ref.unit_grad(dh.double(), zero, ref.q8(lin)[0], ref.q8(gate)[0])
    parts = [(dg, dgerr), (dl, dlerr)] if gate_first else [(dl, dlerr), (dg, dgerr)]
    v, err = torch.cat([t for t, _ in parts], 1), torch.cat([t for _, t in parts], 1)
    ref.check("dpre", da, v, ref.rounded(v, err, dtype))


def test_unit_keeps_half_the_memory_and_takes_strided_rows():
    pre = torch.randn(512, 2048, device=DEV, dtype=torch.bfloat16)
    a = torch.zeros(512, 2049, device=DEV, dtype=torch.bfloat16)[:, 1:].copy_(pre).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = eight_bit.checkpointed_glu(a)
    kept = torch.cuda.memory_allocated() - before - h.numel() * 2
    assert kept <= 512 * 2048 + 512 * 16 + 2048
    b = pre.clone().requires_grad_()
    h2 = eight_bit.checkpointed_glu(b)
    dh = torch.randn(1024, 512, device=DEV, dtype=torch.bfloat16).t()
    (da,), (db,) = torch.autograd.grad(h, a, dh), torch.autograd.grad(h2, b, dh.contiguous())
    assert torch.equal(h, h2) and torch.equal(da, db)
