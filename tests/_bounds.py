"""References in 64 bits, with an elementwise bound of the error of a float32 computation, for the few-token layer and the adapters.

u = 2^-24 is half a step of float32.  A sum of n products in float32, in any order, is off by at most n u times the sum
of the products' magnitudes (one rounding per product or multiply-add and one per addition a term passes through; `n + 8`
leaves room for the joins of partial sums).  A value that is kept as the sum of two 16-bit ones is off by half a step of the
second, whose magnitude is at most half a step of the first: SPLIT of its magnitude (half-steps 2^-9 squared for
bfloat16, 2^-12 squared for float16, where the second also ends at half the smallest number, 2^-25).  The result is rounded once to its type: eps / 2 of its magnitude, at least
half the type's smallest number."""
import torch

U = 2.0 ** -24
SPLIT = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 2.0 ** -18, torch.float16: 2.0 ** -24}
SPLIT_ABS = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def rounded(value, err, dtype):
    """Bound of a result of magnitude |value| known up to `err`, rounded once to `dtype`."""
    return err + torch.finfo(dtype).eps / 2 * (value.abs() + err) + TINY[dtype]


def held(value, err, dtype):
    """Bound of a factor known up to `err` that a product of `dtype` holds in two parts."""
    return err + SPLIT[dtype] * (value.abs() + err) + SPLIT_ABS[dtype]


def layer(x, wr, w1, w2, k, b1=None, b2=None, renormalize=True, gate_first=False, stored=False):
    """(out, bound, logits, bound of the logits, the rows whose selection the errors of the logits leave
    no doubt about).  `stored`: of the general path,
    which rounds gates, pre-activations, hidden and expert rows to the type."""
    e_ = torch.finfo(x.dtype).eps / 2 if stored else 0.0
    dtype, (T, d), E, F = x.dtype, x.shape, wr.size(0), w2.size(2)
    x, wr, w1, w2 = (t.detach().double().cpu() for t in (x, wr, w1, w2))
    b1 = None if b1 is None else b1.detach().double().cpu()
    b2 = None if b2 is None else b2.detach().double().cpu()
    logits = x @ wr.t()
    logits_err = (d + 8) * U * (x.abs() @ wr.abs().t())
    p = torch.softmax(logits, -1)
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    chosen = order[:, :k]
    clear = torch.ones(T, dtype=torch.bool)
    if k < E:
        gap = logits.gather(1, order[:, k - 1:k]) - logits.gather(1, order[:, k:k + 1])
        clear = gap.squeeze(1) > 2 * logits_err.max(-1).values
    g = p.gather(1, chosen)
    total = g.sum(-1, keepdim=True) if renormalize else torch.ones(T, 1, dtype=torch.double)
    g = g / total
    # a softmax changes by at most twice the largest change of its logits, relatively; E + 16 roundings in its sums and quotients,
    # and the exponent's own: |l - max| u for the difference
    spread = (logits.max(-1).values - logits.min(-1).values).unsqueeze(1)
    g_err = g * (4 * logits_err.max(-1, keepdim=True).values + (E + 16 + 4 * spread) * U)
    g_err = g_err + e_ * (g + g_err)
    out, err = torch.zeros(T, d, dtype=torch.double), torch.zeros(T, d, dtype=torch.double)
    for j in range(k):
        for t in range(T):
            e = int(chosen[t, j])
            pre = w1[e] @ x[t]
            size = w1[e].abs() @ x[t].abs()
            if b1 is not None:
                pre, size = pre + b1[e], size + b1[e].abs()
            pre_err = (d + 8) * U * size
            pre_err = pre_err + e_ * (pre.abs() + pre_err)
            lin, gate = pre.chunk(2)
            lin_err, gate_err = pre_err.chunk(2)
            if gate_first:
                lin, gate, lin_err, gate_err = gate, lin, gate_err, lin_err
            act = gate * torch.sigmoid(gate)
            # |silu'| <= 1.1; the sigmoid in float32: the hardware's exponential and reciprocal, a few units of the last place and
            # |gate| u of the argument
            act_err = 1.1 * gate_err + act.abs() * (8 + gate.abs()) * U
            h = lin * act
            h_err = act.abs() * lin_err + lin.abs() * act_err + lin_err * act_err + 2 * U * h.abs()
            h_err = h_err + e_ * (h.abs() + h_err) if stored else held(h, h_err, dtype)
            y = w2[e] @ h
            y_err = w2[e].abs() @ h_err + (F + 8) * U * (w2[e].abs() @ h.abs())
            if b2 is not None:
                y = y + b2[e]
                y_err = y_err + U * b2[e].abs()
            y_err = y_err + e_ * (y.abs() + y_err)
            out[t] += g[t, j] * y
            err[t] += g[t, j] * y_err + g_err[t, j] * (y.abs() + y_err) + (k + 2) * U * (g[t, j] * y).abs()
    return out, rounded(out, err, dtype), logits, logits_err, clear


def adapters(x, w, la, lb, ids, scales=None, bias=None, dy=None, held_in_gradients=True):
    """{name: (value, bound)} of y and, with dy, of dx, da, db, dw, dbias.  `held_in_gradients`: whether the low-rank values may have been
    held in two parts for the factors' gradients, as they may for y and dx."""
    dtype = x.dtype
    x, w, la, lb = (t.detach().double() for t in (x, w, la, lb))
    ids = ids.long()
    (T, K), N, (R, r) = x.shape, w.size(0), la.shape[:2]
    s = torch.ones(R, dtype=torch.double, device=x.device) if scales is None else scales.detach().double()
    on = ((ids >= 0) & (ids < R)).double().unsqueeze(1)
    safe = ids.clamp(0, R - 1)
    A, B, sc = la[safe] * on.unsqueeze(2), lb[safe] * on.unsqueeze(2), (s[safe] * on.squeeze(1)).unsqueeze(1)

    def low(rows, factor, n):                   # factor (T, r, n)
        v = (factor @ rows.unsqueeze(2)).squeeze(2) * sc
        size = (factor.abs() @ rows.abs().unsqueeze(2)).squeeze(2) * sc.abs()
        return v, (n + 9) * U * size

    def project(rows, weight, v, v_err, factor, n):      # factor (T, n_out, r)
        v_err = held(v, v_err, dtype)
        y = rows @ weight.t() + (factor @ v.unsqueeze(2)).squeeze(2)
        size = rows.abs() @ weight.abs().t() + (factor.abs() @ v.abs().unsqueeze(2)).squeeze(2)
        return y, (n + 2 * r + 8) * U * size + (factor.abs() @ v_err.unsqueeze(2)).squeeze(2)

    u, u_err = low(x, A, K)
    y, y_err = project(x, w, u, u_err, B, K)
    if bias is not None:
        b = bias.detach().double()
        y, y_err = y + b, y_err + U * (y.abs() + b.abs())
    found = {"y": (y, rounded(y, y_err, dtype))}
    if dy is None:
        return found
    dy = dy.detach().double()
    v, v_err = low(dy, B.transpose(1, 2), N)
    dx, dx_err = project(dy, w.t(), v, v_err, A.transpose(1, 2), N)
    found["dx"] = (dx, rounded(dx, dx_err, dtype))

    def grad(p, p_err, m):                      # (R, r, C)
        out, err = torch.zeros(R, r, m.size(1), dtype=torch.double, device=m.device), torch.zeros(R, r, m.size(1), dtype=torch.double, device=m.device)
        for a in range(R):
            rows = (ids == a).nonzero().squeeze(1)
            out[a] = p[rows].t() @ m[rows]
            p_held = held(p[rows], p_err[rows], dtype) if held_in_gradients else p_err[rows]
            err[a] = p_held.t() @ m[rows].abs() + (2 * len(rows) + 8) * U * (p[rows].abs().t() @ m[rows].abs())
        return out, rounded(out, err, dtype)

    found["da"] = grad(v, v_err, x)
    db, db_bound = grad(u, u_err, dy)
    found["db"] = (db.transpose(1, 2), db_bound.transpose(1, 2))
    dw = dy.t() @ x
    found["dw"] = (dw, rounded(dw, (T + 8) * U * (dy.abs().t() @ x.abs()), dtype))
    found["dbias"] = (dy.sum(0), rounded(dy.sum(0), (T + 8) * U * dy.abs().sum(0), dtype))
    return found


def check(name, got, want, bound):
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, "%s: shape %s, %s wanted" % (name, tuple(got.shape), tuple(want.shape))
    err = (got - want).abs()
    assert bool(torch.isfinite(got).all()), "%s: %d values are not finite" % (name, int((~torch.isfinite(got)).sum()))
    off = err > bound
    assert not bool(off.any()), "%s: %d of %d values off by more than their bound, worst %.3g against %.3g" % (
        name, int(off.sum()), off.numel(), float(err[off].max()), float(bound[off].max()))
