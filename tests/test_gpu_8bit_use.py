"""Layers, modules and steps on 8 bits as a program has them: strides, codes that are no numbers, streams, graphs, compiled programs, the operators one after
the other, and `GLUMLP` with its checkpoint in 8 bits against the same in 64 bits."""
import pytest
import torch
from torch import nn

import _ref_8bit as ref
import scattermoe_amd
from scattermoe_amd import eight_bit, flatten_sort_count
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import GLUMLP

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


class _Layer:
    """A layer's arguments on the GPU, its weights in 8 bits."""

    def __init__(self, T, k, E, d, F, dtype, bias=True, seed=0):
        g = torch.Generator().manual_seed(seed + T + d)
        up = lambda t: t.to(dtype).to(DEV)
        self.x, self.dout = up(torch.randn(T, d, generator=g)), up(torch.randn(T, d, generator=g))
        self.ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(DEV)
        self.p = up(torch.rand(T, k, generator=g) + 0.2)
        w1, w2 = torch.randn(E, 2 * F, d, generator=g) * d ** -0.5, torch.randn(E, d, F, generator=g) * F ** -0.5
        self.w1, self.s1, self.w1_t = eight_bit.quantize_blocks(w1.to(DEV), 128, transposed=True)
        self.w2, self.s2, self.w2_t = eight_bit.quantize_blocks(w2.to(DEV), 128, transposed=True)
        self.b1, self.b2 = (up(torch.randn(E, n, generator=g)) if bias else None for n in (2 * F, d))
        self.E = E

    def new_rows(self, r):
        g = torch.Generator().manual_seed(100 + r)
        self.x.copy_(torch.randn(self.x.shape, generator=g))
        self.dout.copy_(torch.randn(self.x.shape, generator=g))
        self.ids.copy_(torch.randint(0, self.E, self.ids.shape, generator=g))

    def forward(self, x=None, p=None, **kw):
        return eight_bit.glu_mlp_8bit(self.x if x is None else x, self.p if p is None else p, self.ids, self.w1, self.s1, self.w2, self.s2,
                                      b1=self.b1, b2=self.b2, w1_t=self.w1_t, w2_t=self.w2_t, **kw)

    def step(self):
        x, p = self.x.detach().requires_grad_(), self.p.detach().requires_grad_()
        out = self.forward(x, p)
        return [out.detach(), *torch.autograd.grad(out, (x, p), self.dout)]


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


# sizes: by ids (up to 64 rows), few rows per expert, tiles with the unit behind the product, tiles without
SIZES = [(3, 2, 4, 200, 96), (40, 2, 16, 144, 128), (120, 3, 4, 256, 256), (90, 2, 3, 136, 72)]


@pytest.mark.parametrize("T,k,E,d,F", SIZES)
def test_operators_one_after_the_other_are_the_layer(T, k, E, d, F):
    """In float32, where nothing is rounded between them: the two products, the unit with its checkpoint and their gradients give the layer's own bits."""
    i = _Layer(T, k, E, d, F, torch.float32)
    x, p = i.x.detach().requires_grad_(), i.p.detach().requires_grad_()
    eid, idx, off = flatten_sort_count(i.ids, E)
    pre = eight_bit.parallel_linear_8bit(x, i.w1, i.s1, k, eid, idx, off, expert_biases=i.b1, grouped_out=True, weight_t=i.w1_t)
    h = eight_bit.checkpointed_glu(pre)
    out = eight_bit.parallel_linear_8bit(h, i.w2, i.s2, 1, eid, idx, off, expert_biases=i.b2, gates=p, grouped_in=True, weight_t=i.w2_t)
    got = [out.detach(), *torch.autograd.grad(out, (x, p), i.dout)]
    want = i.step()
    # (of few rows per expert the layer's step takes tiles, the products by themselves streams: sums in another order, up to a step of
    # 8 bits where a value lies at a border)
    if T * k > 12 * E:
        assert _same(got, want)
    else:
        for a, b in zip(got, want):
            assert float((a - b).norm()) <= 2.0 ** -4 * float(b.norm())


@pytest.mark.parametrize("T,k,E,d,F", [(6, 1, 1, 4096, 4100), (9, 2, 2, 4100, 4096), (9, 2, 6, 200, 96)])
def test_forwards_one_after_the_other_are_the_layer(T, k, E, d, F):
    """The same of forward passes whose rows are few: 5 to 12 rows per expert of long contractions, and fewer."""
    i = _Layer(T, k, E, d, F, torch.float32)
    if T * k <= 4 * E:
        i.ids = torch.arange(T * k, device=DEV).view(T, k) % E
    eid, idx, off = flatten_sort_count(i.ids, E)
    with torch.no_grad():
        pre = eight_bit.parallel_linear_8bit(i.x, i.w1, i.s1, k, eid, idx, off, expert_biases=i.b1, grouped_out=True)
        out = eight_bit.parallel_linear_8bit(eight_bit.checkpointed_glu(pre), i.w2, i.s2, 1, eid, idx, off, expert_biases=i.b2, gates=i.p, grouped_in=True)
        want = i.forward()
    # (in float32 the rows are not rounded before gates weigh them in either form; what is left is the sums' order over a token's slots)
    bound = (k + 2) * ref.U * (out.abs() + want.abs()).double().cpu() + 2.0 ** -20 * float(want.abs().max())
    ref.check("out", out, want.double().cpu(), bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,d,F", SIZES)
def test_same_bits_on_other_streams_and_twice(dtype, T, k, E, d, F):
    i, j = _Layer(T, k, E, d, F, dtype), _Layer(T, k, E, d, F, dtype, seed=5)
    want = [i.step() + [i.forward()], j.step() + [j.forward()]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(2):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        got = []
        for st, s in zip(streams, (i, j)):
            with torch.cuda.stream(st):
                got.append(s.step() + [s.forward().detach()])
        torch.cuda.synchronize()
        assert _same(got[0], want[0]) and _same(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k,E,d,F", SIZES)
def test_captured_steps_and_eager_work_between(dtype, T, k, E, d, F):
    """Two captured graphs in one memory pool, a forward and a whole step, replayed in turn with new rows, ids and gradients."""
    i = _Layer(T, k, E, d, F, dtype)
    with torch.no_grad():
        i.forward()
    i.step()
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one), torch.no_grad():
        out = i.forward()
    with torch.cuda.graph(two, pool=one.pool()):
        step = i.step()
    for r in range(3):
        i.new_rows(r)
        one.replay()
        with torch.no_grad():
            want = i.forward()
        torch.cuda.synchronize()
        assert torch.equal(out, want), r
        two.replay()
        want = i.step()
        torch.cuda.synchronize()
        assert _same(step, want), r


@pytest.mark.parametrize("dtype", DTYPES)
def test_unit_on_streams_and_in_graphs(dtype):
    pre = torch.randn(300, 2 * 200, device=DEV).to(dtype).requires_grad_()
    dh = torch.randn(300, 200, device=DEV).to(dtype)

    def step():
        x = pre.detach().requires_grad_()
        h = eight_bit.checkpointed_glu(x)
        return [h.detach(), *torch.autograd.grad(h, x, dh)]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.synchronize()
    assert _same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for r in range(3):
        with torch.no_grad():
            pre.copy_(torch.randn(300, 400, generator=torch.Generator().manual_seed(r)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert _same(got, want), r


@pytest.mark.parametrize("T,k,E,d,F", SIZES)
def test_codes_that_are_no_numbers_stay_where_they_are(T, k, E, d, F):
    """NaN in every second weight row of the second product, whose slices end inside a row's 16 bytes or 128 columns: every other output as before;
    NaN in one token: the other tokens as before."""
    i = _Layer(T, k, E, d, F, torch.bfloat16)
    with torch.no_grad():
        want = i.forward()
        keep = i.w2.clone()
        i.w2.view(torch.uint8)[:, 1::2, :F] = 0x7F
        got = i.forward()
        assert torch.equal(got[:, ::2], want[:, ::2]) and bool(torch.isnan(got[:, 1::2]).all())
        i.w2 = keep
        i.x[1, 3] = float("nan")
        got = i.forward()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:]) and bool(torch.isnan(got[1]).all())


def test_weights_of_other_strides():
    i = _Layer(40, 2, 4, 160, 96, torch.bfloat16)
    want = i.step() + [i.forward()]
    w1, w2, s1 = i.w1, i.w2, i.s1
    i.w1 = w1.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(w1.dtype)
    i.w2 = torch.zeros(w2.numel() + 8, dtype=torch.uint8, device=DEV)[8:].view(w2.shape).copy_(w2.view(torch.uint8)).view(w2.dtype)   # not at 16 bytes
    i.s1 = s1.view(torch.uint8).permute(2, 1, 0).contiguous().permute(2, 1, 0).view(s1.dtype)
    i.b1 = i.b1.t().contiguous().t()
    wide = torch.zeros(40, 2 * 160 + 1, dtype=torch.bfloat16, device=DEV)
    i.x = wide[:, 1::2].copy_(i.x)
    i.dout = i.dout.t().contiguous().t()
    i.ids = i.ids.int()
    assert _same(i.step() + [i.forward()], want)
    one = _Layer(40, 1, 1, 160, 96, torch.bfloat16)                  # one expert's weights for all of four
    four = _Layer(40, 1, 4, 160, 96, torch.bfloat16)
    with torch.no_grad():
        a = eight_bit.glu_mlp_8bit(one.x, one.p, four.ids, *(t.expand(4, -1, -1) for t in (one.w1, one.s1, one.w2, one.s2)))
        b = eight_bit.glu_mlp_8bit(one.x, one.p, one.ids, one.w1, one.s1, one.w2, one.s2)
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [2, 30, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_of_any_byte(T, dtype):
    """A weight's e8m0 scale may be anything from 2^-127 to 2^127, or no number."""
    E, k, K, N = 4, 2, 256, 256
    g = torch.Generator().manual_seed(T)
    q = torch.randint(0, 127, (E, N, K), generator=g, dtype=torch.uint8).to(DEV).view(torch.float8_e4m3fn)
    byte = torch.full((E, 2, 2), 127, dtype=torch.uint8)
    byte[0, 0], byte[1, 1] = torch.tensor([0, 1], dtype=torch.uint8), torch.tensor([117, 255], dtype=torch.uint8)
    s = byte.to(DEV).view(torch.float8_e8m0fnu)
    want = q.float().double() * ref.spread(s.float().double(), N, K, 128)
    back = eight_bit.dequantize_blocks(q, s, 128, dtype=torch.float32)
    assert torch.equal(torch.nan_to_num(back.double(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))
    x = (torch.randn(T, K, generator=g) * 2.0 ** 70).to(dtype).to(DEV)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    eid, idx, off = flatten_sort_count(ids.to(DEV), E)
    y = eight_bit.parallel_linear_8bit(x, q, s, k, eid, idx, off, grouped_out=True).cpu()
    x8 = ref.q8(x.cpu().double())[0]
    w = want.cpu()
    for r in range(T * k):
        e, tok = int(eid[r]), int(idx[r]) // k
        v, err = ref.product(x8[tok:tok + 1], torch.zeros(1, K, dtype=torch.double), torch.nan_to_num(w[e]), dtype != torch.float32, False)
        bad = torch.isnan(w[e]).any(1)
        assert bool(torch.isnan(y[r][bad]).all())
        ref.check("row %d" % r, y[r:r + 1, ~bad], v[:, ~bad], ref.rounded(v, err, dtype)[:, ~bad])


def test_compiled_steps_are_the_eager_ones():
    i = _Layer(60, 2, 4, 128, 96, torch.bfloat16)
    eid, idx, off = flatten_sort_count(i.ids, 4)

    def step(x, p):
        out = i.forward(x, p)
        pre = eight_bit.parallel_linear_8bit(x, i.w1, i.s1, 2, eid, idx, off, grouped_out=True, weight_t=i.w1_t)
        return out, eight_bit.checkpointed_glu(pre), eight_bit.dequantize_blocks(*eight_bit.quantize_blocks(x))
    results = []
    for fn in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        x, p = i.x.detach().requires_grad_(), i.p.detach().requires_grad_()
        out, h, back = fn(x, p)
        results.append([out.detach(), h.detach(), back, *torch.autograd.grad((out, h), (x, p), (i.dout, torch.ones_like(h)))])
    assert _same(*results)
    torch._dynamo.reset()


def test_compiled_step_of_a_gated_layer_with_its_checkpoint():
    torch.manual_seed(2)
    with torch.device(DEV):
        m = GLUMLP(64, 96, 4, 2, checkpoint_8bit=True).bfloat16()
    x, p = torch.randn(30, 64, device=DEV).bfloat16().requires_grad_(), torch.rand(30, 2, device=DEV).bfloat16()
    ids = torch.randint(0, 4, (30, 2), device=DEV)
    results = []
    for fn in (m, torch.compile(m, fullgraph=True, backend="aot_eager")):
        out = fn(x, p, ids)
        results.append([out.detach(), *torch.autograd.grad(out, [x] + list(m.parameters()), torch.ones_like(out))])
    assert _same(*results)
    torch._dynamo.reset()


# ---- modules -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_module_from_a_gated_layer(dtype, bias):
    torch.manual_seed(1)
    with torch.device(DEV):
        m = GLUMLP(160, 96, 5, 2, bias=bias).to(dtype)
    if bias:
        nn.init.normal_(m.experts.bias), nn.init.normal_(m.output_experts.bias)
    q = scattermoe_amd.GLUMLP8bit.from_module(m, input_gradients=True)
    x = torch.randn(3, 11, 160, device=DEV).to(dtype).requires_grad_()
    p, ids = torch.rand(33, 2, device=DEV).to(dtype), torch.randint(0, 5, (33, 2), device=DEV)
    y = q(x, p, ids)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    w1, w2 = (eight_bit.quantize_blocks(w.detach(), 128, transposed=True) for w in (m.experts.weight, m.output_experts.weight))
    a = x.detach().requires_grad_()
    want = eight_bit.glu_mlp_8bit(a, p, ids, w1[0], w1[1], w2[0], w2[1], b1=m.experts.bias.detach() if bias else None,
                                  b2=m.output_experts.bias.detach() if bias else None, w1_t=w1[2], w2_t=w2[2])
    assert y.shape == x.shape and torch.equal(y, want) and torch.equal(dx, torch.autograd.grad(want, a, torch.ones_like(want))[0])
    copy = scattermoe_amd.GLUMLP8bit(160, 96, 5, 2, bias=bias, dtype=dtype, input_gradients=True).to(DEV)
    copy.load_state_dict(q.state_dict())
    assert torch.equal(copy(x, p, ids), y) and not list(q.parameters())


def _glumlp_reference(m, x, p, ids, dout, pre, dtype):
    """{name: (gradient, bound)} of a GLUMLP whose backward pass has `pre` (rows by expert, as stored) in 8 bits."""
    eid, idx, _ = flatten_sort_count(ids, m.num_experts)
    eid, idx = eid.cpu(), idx.cpu()
    w1, w2 = m.experts.weight.detach().cpu().double(), m.output_experts.weight.detach().cpu().double()
    (T, k), F = ids.shape, w2.size(2)
    x64, p64, do = x.cpu().double(), p.cpu().double().reshape(-1), dout.cpu().double()
    pre = pre.cpu().double()
    U, out = ref.U, {}
    tok = idx // k
    dy = do[tok] * p64[idx].unsqueeze(1)
    dyerr = ref.rounded(dy, U * dy.abs(), dtype)
    lin8, gat8 = ref.q8(pre[:, :F])[0], ref.q8(pre[:, F:])[0]
    zero = torch.zeros_like(lin8)
    h, herr = ref.unit(lin8, zero, gat8, zero)
    herr = ref.rounded(h, herr, dtype)
    drow, drerr = torch.zeros(T * k, x.size(1), dtype=torch.double), torch.zeros(T * k, x.size(1), dtype=torch.double)
    dw1, dw1e, dw2, dw2e = torch.zeros_like(w1), torch.zeros_like(w1), torch.zeros_like(w2), torch.zeros_like(w2)
    db1, db1e = torch.zeros_like(w1[:, :, 0]), torch.zeros_like(w1[:, :, 0])

    def product(a, aerr, b, berr):
        size = (a.abs() + aerr) @ (b.abs() + berr)
        return a @ b, size - a.abs() @ b.abs() + 2 * (a.size(1) + 8) * U * size
    for e in eid.unique().tolist():
        mine = eid == e
        none = torch.zeros_like(w2[e])
        dh, derr = product(dy[mine], dyerr[mine], w2[e], none)
        derr = ref.rounded(dh, derr, dtype)
        dl, dlerr, dg, dgerr = ref.unit_grad(dh, derr, lin8[mine], gat8[mine])
        dp, dperr = torch.cat([dl, dg], 1), torch.cat([dlerr, dgerr], 1)
        dperr = ref.rounded(dp, dperr, dtype)
        v, err = product(dp, dperr, w1[e], torch.zeros_like(w1[e]))
        drow[idx[mine]], drerr[idx[mine]] = v, ref.rounded(v, err, dtype)
        dw1[e], err = product(dp.t(), dperr.t(), x64[tok[mine]], torch.zeros_like(x64[tok[mine]]))
        dw1e[e] = ref.rounded(dw1[e], err, dtype)
        dw2[e], err = product(dy[mine].t(), dyerr[mine].t(), h[mine], herr[mine])
        dw2e[e] = ref.rounded(dw2[e], err, dtype)
        db1[e] = dp.sum(0)
        db1e[e] = ref.rounded(db1[e], dperr.sum(0) + 2 * (dp.size(0) + 8) * U * (dp.abs() + dperr).sum(0), dtype)
    dx = drow.view(T, k, -1).sum(1)
    out["x"] = dx, ref.rounded(dx, drerr.view(T, k, -1).sum(1) + k * U * drow.view(T, k, -1).abs().sum(1), dtype)
    out["experts.weight"], out["output_experts.weight"], out["experts.bias"] = (dw1, dw1e), (dw2, dw2e), (db1, db1e)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,d,F,bias", [(1, 1, 1, 16, 8, True), (6, 2, 3, 64, 96, True), (90, 2, 5, 136, 200, False), (150, 3, 4, 128, 256, True)])
def test_glumlp_with_its_checkpoint_in_8_bits(dtype, T, k, E, d, F, bias):
    torch.manual_seed(T)
    with torch.device(DEV):
        m, plain = (GLUMLP(d, F, E, k, bias=bias, checkpoint_8bit=c).to(dtype) for c in (True, False))
    if bias:
        nn.init.normal_(m.experts.bias), nn.init.normal_(m.output_experts.bias)
    plain.load_state_dict(m.state_dict())
    x = torch.randn(T, d, device=DEV).to(dtype).requires_grad_()
    p = (torch.rand(T, k, device=DEV) + 0.2).to(dtype).requires_grad_()
    ids = torch.stack([torch.randperm(E)[:k] for _ in range(T)]).to(DEV)
    dout = torch.randn(T, d, device=DEV).to(dtype)
    names = ["x", "p"] + [n for n, _ in m.named_parameters()]
    out = m(x, p, ids)
    got = dict(zip(names, torch.autograd.grad(out, [x, p] + list(m.parameters()), dout)))
    want_out = plain(x, p, ids)
    want = dict(zip(names, torch.autograd.grad(want_out, [x, p] + list(plain.parameters()), dout)))
    assert torch.equal(out, want_out) and torch.equal(got["p"], want["p"])
    if bias:
        assert torch.equal(got["output_experts.bias"], want["output_experts.bias"])
    eid, idx, off = flatten_sort_count(ids, E)
    with torch.no_grad():
        pre = m.experts(x, k, eid, idx, off, grouped_out=True)
    for name, (v, bound) in _glumlp_reference(m, x.detach(), p.detach(), ids, dout, pre, dtype).items():
        if name in got:
            ref.check(name, got[name], v, bound)
    # parts of the gradient alone
    (dw2,) = torch.autograd.grad(m(x.detach(), p.detach(), ids), m.output_experts.weight, dout)
    _, (v, bound) = None, _glumlp_reference(m, x.detach(), p.detach(), ids, dout, pre, dtype)["output_experts.weight"]
    ref.check("output_experts.weight alone", dw2, v, bound)
    m.requires_grad_(False)
    (dx,) = torch.autograd.grad(m(x, p.detach(), ids), x, dout)
    assert torch.equal(dx, got["x"])


def test_glumlp_keeps_a_third():
    with torch.device(DEV):
        mlps = [GLUMLP(64, 1024, 4, 2, checkpoint_8bit=c).bfloat16() for c in (False, True)]
    x, p = torch.randn(1000, 64, device=DEV).bfloat16(), torch.rand(1000, 2, device=DEV).bfloat16()
    ids = torch.randint(0, 4, (1000, 2), device=DEV)
    kept = []
    for m in mlps:
        m(x, p, ids)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = m(x, p, ids)
        torch.cuda.synchronize()
        kept.append(torch.cuda.memory_allocated() - before)
        del out
    assert kept[0] - kept[1] >= 2000 * 1024 * (6 - 2 - 0.1)


def _some_rows(name, got, x, w, which, experts, dtype):
    """Rows `which` of got against x8[which] w[expert]^T; x (rows, K) float64 of those rows."""
    for r, e in zip(range(len(which)), experts):
        v, err = ref.product(ref.q8(x[r:r + 1])[0], torch.zeros_like(x[r:r + 1]), w[e], True, False)
        ref.check("%s, row %d" % (name, int(which[r])), got[which[r]].unsqueeze(0), v, ref.rounded(v, err, dtype))


def test_rows_that_pass_32_bit_offsets():
    """More than 4 GiB of rows in 8 bits: tokens, and rows scaled one by one, in and out of the experts' order."""
    E, d, n, k = 8, 4096, 16, 8
    T = (1 << 20) + 64
    g = torch.Generator(device=DEV).manual_seed(3)
    w = torch.randn(E, n, d, device=DEV, generator=g) * d ** -0.5
    q, s, qt = eight_bit.quantize_blocks(w, 128, transposed=True)
    w64 = ref.stands_for(q, s, d)
    some = torch.tensor([0, 1, 77777, 524288, T - 65, T - 2, T - 1])
    x = torch.empty(T, d, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    ids = torch.randint(0, E, (T, 1), device=DEV, generator=g)
    eid, idx, off = flatten_sort_count(ids, E)
    y = eight_bit.parallel_linear_8bit(x, q, s, 1, eid, idx, off)
    _some_rows("by token", y, x[some.to(DEV)].cpu().double(), w64, some, ids[some.to(DEV), 0].tolist(), torch.bfloat16)
    del x, y
    # the second product of a layer, 2^20 rows of 16 -> 4096, and its gradient from the tokens' times their gates
    tokens = T // k
    h = torch.randn(T, n, device=DEV, generator=g).bfloat16().requires_grad_()
    gates = (torch.randint(1, 3, (tokens, k), device=DEV, generator=g) / 2).bfloat16()
    dout = torch.empty(tokens, d, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    eid, idx, off = flatten_sort_count(ids.view(tokens, k), E)
    out = eight_bit.parallel_linear_8bit(h, qt, s.transpose(1, 2), 1, eid, idx, off, gates=gates, grouped_in=True, weight_t=q)
    (dh,) = torch.autograd.grad(out, h, dout)
    slots = idx[some.to(DEV)].cpu()
    scaled = dout[(slots // k).to(DEV)].cpu().double() * gates.view(-1)[slots.to(DEV)].cpu().double().unsqueeze(1)
    _some_rows("scaled", dh, scaled, w64, some, eid[some.to(DEV)].tolist(), torch.bfloat16)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    i = _Layer(40, 2, 4, 160, 96, torch.bfloat16)
    eid, idx, off = flatten_sort_count(i.ids, 4)
    with fwad.dual_level():
        x = fwad.make_dual(i.x, torch.ones_like(i.x))
        for call in (lambda: i.forward(x), lambda: eight_bit.checkpointed_glu(x),
                     lambda: eight_bit.parallel_linear_8bit(x, i.w1, i.s1, 2, eid, idx, off, weight_t=i.w1_t)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
