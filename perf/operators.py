"""Two operators as their users call them: a whole mixture-of-experts layer for a few tokens - router product, softmax,
selection, the gated experts, the weighted sum - and low-rank adapters of many requests beside a shared projection,
forward and as a training step.

A case is a dict of
  op      "layer" (`mlp.routed_glu_mlp`), "adapters" (`adapters.parallel_adapters`), "adapters_step" (the same, with the
          gradients of the input and of both halves of the adapters)
  dtype   "bf16", "fp16", "fp32"
  T       tokens; bias: whether the products have biases
  layer   d (model width), f (expert width), E (experts), k (experts per token)
  adapters  d (input width), n (output width), R (adapters held), r (rank), bare (the share of rows without an adapter),
          sorted (whether the rows of an adapter stand side by side, as the tokens of a prompt do)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda:0"

# Expert shapes of the benchmark's workloads
WIDE = {"d": 4096, "f": 14336, "E": 8, "k": 2}
SQUARE = {"d": 2880, "f": 2880, "E": 32, "k": 4}
FINE = {"d": 2048, "f": 768, "E": 128, "k": 8}


def _layer(name, shape, T, dtype="bf16", bias=False):
    return dict(shape, name=name, op="layer", T=T, dtype=dtype, bias=bias)


def _adapters(name, T, d, n, R, r, dtype="bf16", bias=False, bare=0.0, grouped=True, step=False):
    return {"name": name, "op": "adapters_step" if step else "adapters", "T": T, "d": d, "n": n, "R": R, "r": r,
            "dtype": dtype, "bias": bias, "bare": bare, "sorted": grouped}


def listed():
    return [
        # one token of one user, fine-grained experts: the latency of a layer in a decode step
        _layer("layer_1_fine", FINE, 1),
        # one token, the widest experts: a stream over 705 MB of weights
        _layer("layer_1_wide", WIDE, 1),
        # a small serving batch of ragged size, biases, half precision
        _layer("layer_17_square_fp16", SQUARE, 17, dtype="fp16", bias=True),
        # the largest batch of the few-token range over many experts
        _layer("layer_64_fine", FINE, 64),
        # a prototype in full precision, of odd widths
        _layer("layer_5_odd_fp32", {"d": 1003, "f": 1411, "E": 13, "k": 3}, 5, dtype="fp32", bias=True),
        # a decode step of one request with its adapter
        _adapters("adapters_1", 1, 4096, 4096, 8, 16),
        # a decode step of many requests, nearly each with an adapter of its own, one in eight with none
        _adapters("adapters_48_many_fp16", 48, 2880, 4096, 64, 32, dtype="fp16", bias=True, bare=0.125, grouped=False),
        # prompts of several requests in one ragged batch
        _adapters("adapters_1777_prompts", 1777, 2048, 4096, 16, 64, bare=0.1),
        # a ragged batch of odd widths in full precision
        _adapters("adapters_203_odd_fp32", 203, 1003, 1517, 5, 7, dtype="fp32", bias=True, bare=0.2, grouped=False),
        # fine-tuning one adapter
        _adapters("adapters_step_8192", 8192, 4096, 4096, 1, 16, step=True),
        # fine-tuning adapters of several tenants in one batch whose rows are mixed
        _adapters("adapters_step_4099_mixed_fp16", 4099, 2880, 2880, 24, 24, dtype="fp16", bias=True, bare=0.05,
                  grouped=False, step=True),
        # a toy step in full precision
        _adapters("adapters_step_300_fp32", 300, 512, 768, 3, 8, dtype="fp32", step=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Three of four widths are whole numbers of 64; the others are any."""
    w = _spread(rng, low, high)
    return max(64, w // 64 * 64) if rng.random() < 0.75 else w


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    bias = rng.random() < 0.4
    if rng.random() < 0.4:
        E = _spread(rng, 4, 128)
        T = _spread(rng, 1, 64)
        k = rng.randint(1, min(8, E))
        d, f = _width(rng, 256, 4096), _width(rng, 256, 8192)
        f = max(64, min(f, 300_000_000 // (E * d)))
        return {"op": "layer", "dtype": dtype, "T": T, "bias": bias, "d": d, "f": f, "E": E, "k": k}
    step = rng.random() < 0.4
    T = _spread(rng, 1, 4096)
    d, n = _width(rng, 256, 4096), _width(rng, 256, 4096)
    if dtype == "fp32":
        T = min(T, 1024)
    r = rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)])
    R = _spread(rng, 1, 64)
    return {"op": "adapters_step" if step else "adapters", "dtype": dtype, "T": T, "bias": bias, "d": d, "n": n, "R": R,
            "r": r, "bare": rng.choice([0.0, 0.1, 0.5]), "sorted": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=dt if dt != torch.float16 else torch.float32) * std).to(dt)

    T, d = case["T"], case["d"]
    s = {"op": case["op"], "x": normal(T, d)}
    if case["op"] == "layer":
        E, f = case["E"], case["f"]
        s["k"] = case["k"]
        s["router"] = normal(E, d, std=1.5 * d ** -0.5)
        s["w1"] = normal(E, 2 * f, d, std=d ** -0.5)
        s["w2"] = normal(E, d, f, std=f ** -0.5)
        s["b1"] = normal(E, 2 * f, std=0.1) if case["bias"] else None
        s["b2"] = normal(E, d, std=0.1) if case["bias"] else None
        return s
    n, R, r = case["n"], case["R"], case["r"]
    s["weight"] = normal(n, d, std=d ** -0.5)
    s["bias"] = normal(n, std=0.1) if case["bias"] else None
    s["a"] = normal(R, r, d, std=d ** -0.5)
    s["b"] = normal(R, n, r, std=r ** -0.5)
    s["scales"] = torch.rand(R, generator=g, device=DEVICE) * 1.5 + 0.5
    ids = torch.randint(0, R, (T,), generator=g, device=DEVICE)
    if case["sorted"]:
        ids = torch.sort(ids).values
    bare = torch.rand(T, generator=g, device=DEVICE) < case["bare"]
    s["ids"] = torch.where(bare, torch.full_like(ids, -1), ids)
    if case["op"] == "adapters_step":
        s["dy"] = normal(T, n)
        for name in ("x", "a", "b"):
            s[name].requires_grad_()
    return s


def _plain_layer(s):
    x, k = s["x"], s["k"]
    T, E = x.size(0), s["router"].size(0)
    logits = x.double() @ s["router"].double().t()
    p = torch.exp(logits - logits.max(-1, keepdim=True).values)
    p = p / p.sum(-1, keepdim=True)
    order = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, :k]
    g = p.gather(1, order)
    g = (g / g.sum(-1, keepdim=True)).float()
    f = s["w2"].size(2)
    if T * k <= E:                                   # the selected experts' weights
        e = order.reshape(-1)
        w1, w2, rows = s["w1"][e].float(), s["w2"][e].float(), x.float().repeat_interleave(k, 0).unsqueeze(1)
        b1 = 0.0 if s["b1"] is None else s["b1"][e].float().unsqueeze(1)
        b2 = 0.0 if s["b2"] is None else s["b2"][e].float().unsqueeze(1)
    else:                                            # every expert on every token, weighted by its gate or by zero
        w1, w2, rows = s["w1"].float(), s["w2"].float(), x.float().unsqueeze(0).expand(E, -1, -1).contiguous()
        b1 = 0.0 if s["b1"] is None else s["b1"].float().unsqueeze(1)
        b2 = 0.0 if s["b2"] is None else s["b2"].float().unsqueeze(1)
    pre = torch.matmul(rows, w1.transpose(1, 2).contiguous()) + b1
    lin, gate = pre[..., :f], pre[..., f:]
    y = torch.matmul(lin * (gate / (1.0 + torch.exp(-gate))), w2.transpose(1, 2).contiguous()) + b2
    if T * k <= E:
        out = (y.view(T, k, -1) * g.unsqueeze(-1)).sum(1)
    else:
        weight = torch.zeros(T, E, device=x.device).scatter_(1, order, g)
        out = (y * weight.t().unsqueeze(-1)).sum(0)
    return out.to(x.dtype), logits.float()


def _plain_adapters(s, step):
    x, a, b, w = (s[name].detach() for name in ("x", "a", "b", "weight"))
    R, r, n = a.size(0), a.size(1), w.size(0)
    dt, T = x.dtype, x.size(0)
    x32, a32 = x.float(), a.float().reshape(R * r, -1)
    b32 = b.float().permute(0, 2, 1).reshape(R * r, n)                                  # rows: (adapter, rank)
    mine = (s["ids"].unsqueeze(1) == torch.arange(R, device=x.device)).float() * s["scales"]      # (T, R), scaled
    mine = mine.repeat_interleave(r, 1)
    u = (x32 @ a32.t()) * mine
    y = x32 @ w.float().t() + u @ b32
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if not step:
        return y.to(dt)
    dy = s["dy"].float()
    v = (dy @ b32.t()) * mine
    dx = dy @ w.float() + v @ a32
    da = (v.t() @ x32).view(R, r, -1)
    db = (u.t() @ dy).view(R, r, n).permute(0, 2, 1)
    return y.to(dt), dx.to(dt), da.to(dt), db.to(dt).contiguous()


def run(state):
    s = state
    if own:
        if s["op"] == "layer":
            from scattermoe_amd.mlp import routed_glu_mlp
            return routed_glu_mlp(s["x"], s["router"], s["w1"], s["w2"], s["k"], b1=s["b1"], b2=s["b2"])
        from scattermoe_amd.adapters import parallel_adapters
        y = parallel_adapters(s["x"], s["weight"], s["a"], s["b"], s["ids"], scales=s["scales"], bias=s["bias"])
        if s["op"] == "adapters":
            return y
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])
    if s["op"] == "layer":
        return _plain_layer(s)
    return _plain_adapters(s, s["op"] == "adapters_step")


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    T, d = case["T"], case["d"]
    if case["op"] == "layer":
        E, f, k = case["E"], case["f"], case["k"]
        hit = E * (1.0 - (1.0 - k / E) ** T)         # experts that T tokens reach on average
        weights = hit * (3 * d * f + (2 * f + d if case["bias"] else 0)) + E * d
        return {"bytes": size * (weights + 2 * T * d) + 4 * T * E, "flops": 2.0 * T * E * d + 6.0 * T * k * d * f}
    n, R, r = case["n"], case["R"], case["r"]
    rows = T * (1.0 - case["bare"])
    hit = R * (1.0 - (1.0 - 1.0 / R) ** rows)
    reads = n * d + (n if case["bias"] else 0) + T * d + hit * r * (n + d)
    low = 2.0 * rows * r * (n + d)
    flops = 2.0 * T * n * d + low
    if case["op"] == "adapters":
        return {"bytes": size * (reads + T * n) + 8 * T, "flops": flops}
    # the step: the output's gradient read, y, dx and the adapters' gradients written
    return {"bytes": size * (reads + T * n + T * n + T * d + R * r * (n + d)) + 8 * T, "flops": 2.0 * flops + low}


def exact(case, seed):
    s = prepare(case, seed)
    T = case["T"]
    x = s["x"].detach().double()
    if case["op"] == "layer":
        if T * case["k"] * case["d"] * case["f"] > 2e10:
            return None
        logits = torch.einsum("td,ed->te", x, s["router"].double())
        p = torch.softmax(logits, -1)
        out = torch.zeros_like(x)
        chosen = torch.argsort(p, dim=-1, descending=True, stable=True)[:, :case["k"]]
        total = p.gather(1, chosen).sum(-1)
        for e in torch.unique(chosen).tolist():
            rows = (chosen == e).any(-1).nonzero().squeeze(-1)
            pre = torch.nn.functional.linear(x[rows], s["w1"][e].double(), None if s["b1"] is None else s["b1"][e].double())
            lin, gate = pre.chunk(2, dim=-1)
            y = torch.nn.functional.linear(torch.nn.functional.silu(gate) * lin, s["w2"][e].double(),
                                           None if s["b2"] is None else s["b2"][e].double())
            out[rows] += y * (p[rows, e] / total[rows]).unsqueeze(-1)
        return out, logits
    w, ids = s["weight"].double(), s["ids"]
    y = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
    dx = da = db = None
    if case["op"] == "adapters_step":
        dy = s["dy"].double()
        dx, da, db = dy.matmul(w), torch.zeros_like(s["a"].detach(), dtype=torch.double), torch.zeros_like(s["b"].detach(), dtype=torch.double)
    for j in torch.unique(ids[ids >= 0]).tolist():
        rows = (ids == j).nonzero().squeeze(-1)
        a, b, scale = s["a"][j].detach().double(), s["b"][j].detach().double(), s["scales"][j].double()
        low = x[rows].matmul(a.t()) * scale
        y[rows] += low.matmul(b.t())
        if dx is not None:
            back = dy[rows].matmul(b) * scale
            dx[rows] += back.matmul(a)
            da[j] = back.t().matmul(x[rows])
            db[j] = dy[rows].t().matmul(low)
    return y if dx is None else (y, dx, da, db)
