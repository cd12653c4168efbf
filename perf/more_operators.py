"""Experts whose weights are held in 8 bits, and what a training step keeps in 8 bits, as their users call them: the expert
products, a whole gated expert layer, both forward and as a training step with the weights frozen, and the gated unit of a
layer in training, which keeps its input in 8 bits for the backward pass.

8 bits are e4m3 with a scale for each block of 128.  Rows (activations, gradients) are cut into blocks of 128 columns, whose
scale is the smallest power of two, 2^-126 or more, by which the block's largest magnitude divided is at most 448.  Weights
(E, N, K) come with a scale for every 128 x 128 block: powers of two (8 bits) or any numbers (float32).

A case is a dict of
  op      "product" (`eight_bit.parallel_linear_8bit`), "product_step" (the same, with the gradient of the input),
          "layer" (`eight_bit.glu_mlp_8bit`), "layer_step" (the same, with the gradients of the input and the gates),
          "unit_step" (`eight_bit.checkpointed_glu`, forward and backward)
  dtype   "bf16", "fp16", "fp32" of activations and results
  T       tokens; E, k: experts, and experts per token; d: model width
  n       a product's output columns; f: a layer's, or a unit's, hidden width
  scales  "e8m0" or "fp32" of the weights; bias; skew: whether some experts get most of the tokens
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda:0"
BLOCK = 128

# Expert shapes of the benchmark's workloads
WIDE = {"d": 4096, "f": 14336, "E": 8, "k": 2}
SQUARE = {"d": 2880, "f": 2880, "E": 32, "k": 4}
FINE = {"d": 2048, "f": 768, "E": 128, "k": 8}


def _layer(name, shape, T, dtype="bf16", scales="e8m0", bias=False, skew=False, step=False):
    return dict(shape, name=name, op="layer_step" if step else "layer", T=T, dtype=dtype, scales=scales, bias=bias, skew=skew)


def _product(name, T, d, n, E, k, dtype="bf16", scales="e8m0", bias=False, skew=False, step=False):
    return {"name": name, "op": "product_step" if step else "product", "T": T, "d": d, "n": n, "E": E, "k": k, "dtype": dtype,
            "scales": scales, "bias": bias, "skew": skew}


def _unit(name, T, f, dtype="bf16"):
    return {"name": name, "op": "unit_step", "T": T, "f": f, "dtype": dtype}


def listed():
    return [
        # one token of one user, fine-grained experts: the latency of a layer in a decode step
        _layer("layer_1_fine", FINE, 1),
        # a small serving batch of the widest experts, scales as a checkpoint holds them: a stream over 1.4 GB of weights
        _layer("layer_16_wide_fp32scales", WIDE, 16, scales="fp32"),
        # a serving batch of ragged size with biases, half precision
        _layer("layer_65_square_fp16", SQUARE, 65, dtype="fp16", bias=True),
        # prompts of several requests, the widest experts
        _layer("layer_4099_wide", WIDE, 4099),
        # fine-tuning what stands around frozen experts, loads uneven
        _layer("layer_step_2051_square", SQUARE, 2051, bias=True, skew=True, step=True),
        # the same over many small experts
        _layer("layer_step_8192_fine", FINE, 8192, step=True),
        # a toy product of odd widths in full precision
        _product("product_5_odd_fp32", 5, 1003, 1517, 13, 3, dtype="fp32", scales="fp32", bias=True),
        # the first product of a training batch: the largest
        _product("product_16384_wide", 16384, 4096, 28672, 8, 2),
        # a product with its input's gradient over a ragged batch, scales as a checkpoint holds them
        _product("product_step_3001_fp16", 3001, 2048, 1536, 64, 4, dtype="fp16", scales="fp32", step=True),
        # the hidden rows of a training batch
        _unit("unit_step_16384", 16384, 14336),
        # a ragged batch of an odd width, half precision
        _unit("unit_step_1777_odd_fp16", 1777, 1411, dtype="fp16"),
        # a toy in full precision
        _unit("unit_step_256_fp32", 256, 256, dtype="fp32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Three of four widths are whole numbers of 64; the others are any."""
    w = _spread(rng, low, high)
    return max(64, w // 64 * 64) if rng.random() < 0.75 else w


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kind = rng.choice(["layer", "layer", "layer_step", "product", "product_step", "unit_step"])
    if kind == "unit_step":
        T, f = _spread(rng, 1, 16384), _width(rng, 64, 14336)
        return {"op": kind, "dtype": dtype, "T": T, "f": f}
    E = _spread(rng, 2, 128)
    k = rng.randint(1, min(8, E))
    T = _spread(rng, 1, 4096)
    d = _width(rng, 128, 4096)
    case = {"op": kind, "dtype": dtype, "T": T, "E": E, "k": k, "d": d, "scales": rng.choice(["e8m0", "e8m0", "fp32"]),
            "bias": rng.random() < 0.4, "skew": rng.random() < 0.3}
    wide = _width(rng, 128, 8192)
    if kind.startswith("product"):
        case["n"] = max(64, min(wide, 1_000_000_000 // (E * d)))
    else:
        # (what a layer rounds to 8 bits between its products is compared in the 16-bit types)
        case["dtype"] = "bf16" if dtype == "fp32" else dtype
        case["f"] = max(64, min(wide, 400_000_000 // (E * d)))
    return case


def _weights(g, E, N, K, std, scales, transposed):
    """A weight (E, N, K) in 8 bits with K filled up to a multiple of 16 by zeros, its scales, and its transpose (E, K, N) likewise."""
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    w = torch.randn((E, nb * BLOCK, kb * BLOCK), generator=g, device=DEVICE, dtype=torch.float32)
    w[:, N:], w[:, :, K:] = 0, 0
    w = w.view(E, nb, BLOCK, kb, BLOCK)
    w *= std * torch.exp(0.4 * torch.randn((E, nb, 1, kb, 1), generator=g, device=DEVICE))       # blocks of unlike size
    top = w.abs().amax((2, 4), keepdim=True)
    if scales == "fp32":
        s = top / 448.0
    else:
        m, e = torch.frexp(top)
        s = torch.ldexp(torch.ones_like(top), e - 9 + (m > 0.875).to(torch.int32))
    q = (w / s).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(E, nb * BLOCK, kb * BLOCK)

    def cut(t, rows, cols):
        full = -(-cols // 16) * 16
        return t.view(torch.uint8)[:, :rows, :full].contiguous().view(torch.float8_e4m3fn)

    s = s.view(E, nb, kb)
    s = s.contiguous() if scales == "fp32" else s.to(torch.float8_e8m0fnu)
    return cut(q, N, K), s, cut(q.view(torch.uint8).transpose(1, 2).contiguous(), K, N) if transposed else None


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=dt if dt != torch.float16 else torch.float32) * std).to(dt)

    op, T = case["op"], case["T"]
    s = {"op": op}
    if op == "unit_step":
        s["pre"] = normal(T, 2 * case["f"], std=1.5).requires_grad_()
        s["dh"] = normal(T, case["f"])
        return s
    E, k, d = case["E"], case["k"], case["d"]
    step = op.endswith("step")
    s["x"], s["k"], s["E"] = normal(T, d), k, E
    keys = torch.rand((T, E), generator=g, device=DEVICE).log()
    if case["skew"]:
        keys = keys * torch.arange(1, E + 1, device=DEVICE) ** 0.5           # (the largest of E exponential races)
    s["experts"] = keys.argsort(1, descending=True)[:, :k].contiguous()
    # the routing, as a layer of two products holds it: rows by expert, where each comes from, where each expert ends
    eid, s["idx"] = torch.sort(s["experts"].reshape(-1), stable=True)
    counts = torch.bincount(eid, minlength=E)
    s["eid"], s["off"], s["most"] = eid, counts.cumsum(0), int(counts.max())
    bias = case["bias"]
    if op.startswith("product"):
        n = case["n"]
        s["w"], s["s"], s["wt"] = _weights(g, E, n, d, d ** -0.5, case["scales"], step)
        s["b"] = normal(E, n, std=0.1) if bias else None
        if step:
            s["dy"] = normal(T * k, n)
            s["x"].requires_grad_()
        return s
    f = case["f"]
    s["w1"], s["s1"], s["w1t"] = _weights(g, E, 2 * f, d, d ** -0.5, case["scales"], step)
    s["w2"], s["s2"], s["w2t"] = _weights(g, E, d, f, f ** -0.5, case["scales"], step)
    s["b1"] = normal(E, 2 * f, std=0.1) if bias else None
    s["b2"] = normal(E, d, std=0.1) if bias else None
    p = torch.rand((T, k), generator=g, device=DEVICE) + 0.2
    s["gates"] = (p / p.sum(1, keepdim=True)).to(dt)
    if step:
        s["dout"] = normal(T, d)
        s["x"].requires_grad_()
        s["gates"].requires_grad_()
    return s


def _in_blocks(v):
    """The numbers that the float32 rows v (..., K) stand for in 8 bits."""
    K = v.size(-1)
    b = torch.nn.functional.pad(v, (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = torch.clamp(e - 9 + (m > 0.875), min=-126).to(torch.int32)
    s = ((e + 127) << 23).view(torch.float32)
    return ((b / s).to(torch.float8_e4m3fn).float() * s).flatten(-2)[..., :K]


def _stood_for(w, s, K):
    """The float32 numbers (E, N, K) of a weight in 8 bits."""
    s = s.float().repeat_interleave(BLOCK, 1)[:, :w.size(1)].repeat_interleave(BLOCK, 2)[:, :, :K]
    return w.float()[:, :, :K] * s


def _by_expert(s, rows, w, scales, back=False):
    """The product of every row (sorted by expert) and its expert's weight: w (E, N, K), or K x N of it, `back`."""
    L, E = s["eid"].numel(), s["E"]
    K = rows.size(1)
    scales = scales.float().transpose(1, 2) if back else scales.float()
    if L <= E:                                                       # the weights of the rows' experts
        return torch.bmm(_stood_for(w.view(torch.uint8)[s["eid"]].view(w.dtype), scales[s["eid"]], K), rows.unsqueeze(-1)).squeeze(-1)
    starts = s["off"] - torch.bincount(s["eid"], minlength=E)        # every expert's rows, filled up to the most that one has
    at = s["eid"] * s["most"] + torch.arange(L, device=rows.device) - starts[s["eid"]]
    full = rows.new_zeros(E * s["most"], K)
    full[at] = rows
    y = torch.bmm(_stood_for(w, scales, K), full.view(E, s["most"], K).transpose(1, 2).contiguous())
    return y.transpose(1, 2).reshape(E * s["most"], -1)[at]


def _plain_product(s):
    x = s["x"].detach()
    T, d = x.shape
    y = _by_expert(s, _in_blocks(x.float())[s["idx"] // s["k"]], s["w"], s["s"])
    if s["b"] is not None:
        y = y + s["b"].float()[s["eid"]]
    if s["op"] == "product":
        return y.to(x.dtype)
    back = _by_expert(s, _in_blocks(s["dy"].float()), s["wt"], s["s"], back=True)
    dx = torch.empty_like(back)
    dx[s["idx"]] = back
    return y.to(x.dtype), dx.view(T, s["k"], d).sum(1).to(x.dtype)


def _plain_layer(s):
    x, gates = s["x"].detach(), s["gates"].detach().float()
    T, d = x.shape
    k, idx, dt = s["k"], s["idx"], x.dtype
    pre = _by_expert(s, _in_blocks(x.float())[idx // k], s["w1"], s["s1"])
    if s["b1"] is not None:
        pre = pre + s["b1"].float()[s["eid"]]
    lin, gate = pre.chunk(2, dim=1)
    y = _by_expert(s, _in_blocks(lin * (gate / (1.0 + torch.exp(-gate)))), s["w2"], s["s2"])
    if s["b2"] is not None:
        y = y + s["b2"].float()[s["eid"]]
    rows = torch.empty_like(y)
    rows[idx] = y
    out = (rows.view(T, k, d) * gates.unsqueeze(-1)).sum(1).to(dt)
    if s["op"] == "layer":
        return out
    dout = s["dout"].float()
    dgates = (rows.view(T, k, d) * dout.unsqueeze(1)).sum(-1).to(dt)
    dh = _by_expert(s, _in_blocks(dout[idx // k] * gates.view(-1, 1)[idx]), s["w2t"], s["s2"], back=True)
    lin, gate = _in_blocks(lin), _in_blocks(gate)
    c = 1.0 / (1.0 + torch.exp(-gate))
    dpre = torch.cat([dh * gate * c, dh * lin * c * (1.0 + gate * (1.0 - c))], dim=1)
    back = _by_expert(s, _in_blocks(dpre), s["w1t"], s["s1"], back=True)
    dx = torch.empty_like(back)
    dx[idx] = back
    return out, dx.view(T, k, d).sum(1).to(dt), dgates


def _plain_unit(s):
    pre, dh = s["pre"].detach(), s["dh"].float()
    lin, gate = pre.float().chunk(2, dim=1)
    h = lin * (gate / (1.0 + torch.exp(-gate)))
    lin, gate = _in_blocks(lin), _in_blocks(gate)
    c = 1.0 / (1.0 + torch.exp(-gate))
    return h.to(pre.dtype), torch.cat([dh * gate * c, dh * lin * c * (1.0 + gate * (1.0 - c))], dim=1).to(pre.dtype)


def run(state):
    s = state
    op = s["op"]
    if own:
        from scattermoe_amd import eight_bit
        if op == "unit_step":
            h = eight_bit.checkpointed_glu(s["pre"])
            return h.detach(), torch.autograd.grad(h, s["pre"], s["dh"])[0]
        if op.startswith("product"):
            y = eight_bit.parallel_linear_8bit(s["x"], s["w"], s["s"], s["k"], s["eid"], s["idx"], s["off"], expert_biases=s["b"],
                                               grouped_out=True, weight_t=s["wt"])
            if op == "product":
                return y
            return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
        out = eight_bit.glu_mlp_8bit(s["x"], s["gates"], s["experts"], s["w1"], s["s1"], s["w2"], s["s2"], b1=s["b1"], b2=s["b2"],
                                     w1_t=s["w1t"], w2_t=s["w2t"])
        if op == "layer":
            return out
        return (out.detach(),) + torch.autograd.grad(out, (s["x"], s["gates"]), s["dout"])
    if op == "unit_step":
        return _plain_unit(s)
    return _plain_product(s) if op.startswith("product") else _plain_layer(s)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op, T = case["op"], case["T"]
    if op == "unit_step":
        f = case["f"]
        kept = 2 * f + 2 * -(-f // BLOCK)                # a row in 8 bits with its scales: written, and read again
        return {"bytes": T * (6 * f * size + 2 * kept), "flops": 20.0 * T * f}
    E, k, d = case["E"], case["k"], case["d"]
    rows = T * k
    hit = E * (1.0 - (1.0 - k / E) ** T)                 # experts that T tokens reach on average
    if op.startswith("product"):
        n = case["n"]
        reads = hit * n * (d + (size if case["bias"] else 0)) + size * T * d + 16 * rows + size * rows * n
        if op == "product":
            return {"bytes": reads, "flops": 2.0 * rows * d * n}
        return {"bytes": reads + hit * n * d + size * (rows * n + T * d), "flops": 4.0 * rows * d * n}
    f = case["f"]
    reads = hit * (3 * d * f + (size * (2 * f + d) if case["bias"] else 0)) + 2 * size * T * d + (8 + size) * rows
    if op == "layer":
        return {"bytes": reads, "flops": 6.0 * rows * d * f}
    return {"bytes": reads + hit * 3 * d * f + 2 * size * T * d + size * rows, "flops": 12.0 * rows * d * f}


def _exact_blocks(v):
    """Blocks of 128 of the float64 rows, divided by their scale and rounded to four significant bits (or to 2^-9), ties to even."""
    out = torch.empty_like(v)
    for at in range(0, v.size(1), BLOCK):
        b = v[:, at:at + BLOCK]
        top = b.abs().amax(1, keepdim=True).clamp_min(2.0 ** -140)
        s = torch.exp2(torch.ceil(torch.log2(top / 448.0) - 1e-13).clamp_min(-126.0))
        s = torch.where(top > 448.0 * s, 2.0 * s, s)
        s = torch.where((top <= 224.0 * s) & (s > 2.0 ** -126), 0.5 * s, s)
        b = b / s
        step = torch.exp2(torch.floor(torch.log2(b.abs().clamp_min(2.0 ** -6)) + 1e-13) - 3.0)
        step = torch.where(b.abs().clamp_min(2.0 ** -6) < 8.0 * step, 0.5 * step, step)
        out[:, at:at + BLOCK] = torch.round(b / step) * step * s
    return out


def _exact_weight(w, s, e, K):
    w, s = w[e].double()[:, :K], s[e].float().double()
    n = torch.arange(w.size(0), device=w.device) // BLOCK
    c = torch.arange(K, device=w.device) // BLOCK
    return w * s[n][:, c]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "unit_step":
        f = case["f"]
        pre, dh = s["pre"].detach().double(), s["dh"].double()
        h = pre[:, :f] * torch.nn.functional.silu(pre[:, f:])
        lin, gate = _exact_blocks(pre[:, :f]), _exact_blocks(pre[:, f:])
        c = torch.sigmoid(gate)
        return h, torch.cat([dh * gate * c, dh * lin * (c + gate * c * (1.0 - c))], dim=1)
    k, d, T = case["k"], case["d"], case["T"]
    x8 = _exact_blocks(s["x"].detach().double())
    ends = s["off"].tolist()
    parts = [(e, a, b) for e, (a, b) in enumerate(zip([0] + ends[:-1], ends)) if b > a]
    token = s["idx"] // k
    if op.startswith("product"):
        y = x8.new_empty(T * k, case["n"])
        dx = torch.zeros_like(x8) if op == "product_step" else None
        dy8 = _exact_blocks(s["dy"].double()) if op == "product_step" else None
        for e, a, b in parts:
            w = _exact_weight(s["w"], s["s"], e, d)
            y[a:b] = x8[token[a:b]].matmul(w.t())
            if s["b"] is not None:
                y[a:b] += s["b"][e].double()
            if dx is not None:
                dx.index_add_(0, token[a:b], dy8[a:b].matmul(w))
        return y if dx is None else (y, dx)
    f = case["f"]
    gates = s["gates"].detach().double().reshape(-1)
    out = torch.zeros_like(x8)
    step = op == "layer_step"
    dx, dg = torch.zeros_like(x8), torch.zeros_like(gates)
    for e, a, b in parts:
        w1, w2 = _exact_weight(s["w1"], s["s1"], e, d), _exact_weight(s["w2"], s["s2"], e, f)
        rows, mine = token[a:b], s["idx"][a:b]
        pre = x8[rows].matmul(w1.t())
        if s["b1"] is not None:
            pre += s["b1"][e].double()
        y = _exact_blocks(pre[:, :f] * torch.nn.functional.silu(pre[:, f:])).matmul(w2.t())
        if s["b2"] is not None:
            y += s["b2"][e].double()
        out.index_add_(0, rows, y * gates[mine].unsqueeze(1))
        if step:
            dout = s["dout"].double()[rows]
            dg[mine] = (dout * y).sum(1)
            dh = _exact_blocks(dout * gates[mine].unsqueeze(1)).matmul(w2)
            lin, gate = _exact_blocks(pre[:, :f]), _exact_blocks(pre[:, f:])
            c = torch.sigmoid(gate)
            dpre = torch.cat([dh * gate * c, dh * lin * (c + gate * c * (1.0 - c))], dim=1)
            dx.index_add_(0, rows, _exact_blocks(dpre).matmul(w1))
    return (out, dx, dg.view(T, k)) if step else out
