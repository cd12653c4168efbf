"""8 bits (e4m3 with a scale for each block of 128) in 64 bits, with elementwise bounds of what the kernels may be off by.

u = 2^-24 is half a step of float32.  A product of rows in 8 bits is exact but for
  - its sums: n + 8 roundings of the products' magnitudes, as for any float32 sum (half a step each, a whole one where the matrix cores may cut);
  - where the rows are 16-bit ones, what the matrix cores cut: eight neighbouring products are added after each has lost what lies
    below 2^-13 of the largest one's binade, so at most 8 * 2^-13 of the largest product of every eight;
  - the weights' float32 scale: its product with the values, one rounding;
  - rounding the result: eps / 2 of its magnitude, at least half the type's smallest number.
A value that is taken to 8 bits and known up to an error lands on what the interval's ends land on, or between."""
import torch

U = 2.0 ** -24
CUT = 8 * 2.0 ** -13
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def scale_exponent(top):
    """The exponent of the scale of blocks whose largest magnitudes are `top` (float64)."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126), torch.full_like(e, -126))


def nearest(v, ex):
    """v / 2^ex to the nearest of e4m3, ties to even, times 2^ex."""
    b = torch.ldexp(v, -ex)
    _, e = torch.frexp(b)
    step = (e - 4).clamp(min=-9)
    return torch.ldexp(torch.round(torch.ldexp(b, -step)), step + ex)


def blocked(v, block_rows=1):
    """v (..., N, K) float64 with its blocks' largest magnitudes, spread over the blocks."""
    N, K = v.shape[-2:]
    full = torch.nn.functional.pad(v.abs(), (0, -K % 128, 0, -N % block_rows))
    top = full.unflatten(-1, (-1, 128)).amax(-1).unflatten(-2, (-1, block_rows)).amax(-2)
    return top


def spread(s, N, K, block_rows=1):
    return s.repeat_interleave(block_rows, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]


def q8(v, block_rows=1):
    """(the values that v (..., N, K) stands for in 8 bits, the scales' exponents)."""
    ex = scale_exponent(blocked(v, block_rows))
    return nearest(v, spread(ex, *v.shape[-2:], block_rows)), ex


def q8_known(v, err):
    """(q8(v), bound) for rows v (..., N, K) known up to err."""
    N, K = v.shape[-2:]
    got = q8(v)[0]
    bound = torch.zeros_like(v)
    low, high = scale_exponent(blocked((v.abs() - err).clamp(min=0))), scale_exponent(blocked(v.abs() + err))
    for ex in (low, high):                                   # a power of two more or less where the largest is at the border
        ex = spread(ex, N, K)
        for w in (v - err, v, v + err):
            bound = torch.maximum(bound, (nearest(w, ex) - got).abs())
    return got, bound


def rounded(value, err, dtype):
    return err + torch.finfo(dtype).eps / 2 * (value.abs() + err) + TINY[dtype]


def held(value, err, dtype):
    """bound of a value stored as dtype on the way (the same, for readers)."""
    return rounded(value, err, dtype)


def stands_for(q, s, K, block_rows=128):
    """Float64 values of e4m3 weights (E, N, >= K) with their scales (8 bits or float32)."""
    return q.cpu().float().double()[..., :K] * spread(s.cpu().float().double(), q.size(-2), K, block_rows)


def product(x, xerr, w, rows16, float_scales):
    """(x w^T, bound) for x (M, K) known up to xerr and w (N, K), float64; rows16: of rows that came in 16 bits."""
    K = x.size(1)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    err = xerr @ w.abs().t() + (2 * (K + 8) + (2 if float_scales else 0)) * U * (size + xerr @ w.abs().t())
    if rows16:
        pad = (0, -K % 8)
        top = ((x.abs() + xerr).unsqueeze(1) * w.abs().unsqueeze(0))                       # (M, N, K)
        err = err + CUT * torch.nn.functional.pad(top, pad).unflatten(-1, (-1, 8)).amax(-1).sum(-1)
    return y, err


def sigmoid(g, gerr):
    """(sigmoid, bound): the exponent's argument is rounded (|g| u, twice), the exponential, the sum and the reciprocal are off by two steps each."""
    s = torch.sigmoid(g)
    return s, s * (1 - s) * gerr * 1.0001 + s * (4 * g.abs() + 16) * U + 2.0 ** -126


def unit(lin, lerr, gate, gerr):
    """(lin silu(gate), bound)."""
    s, serr = sigmoid(gate, gerr)
    a = gate * s
    aerr = gate.abs() * serr + gerr * (s + serr) + 2 * U * a.abs()
    h = a * lin
    return h, aerr * (lin.abs() + lerr) + a.abs() * lerr + 4 * U * h.abs() + 2.0 ** -140


def unit_grad(dh, derr, lin, gate):
    """(d lin, bound, d gate, bound) of exact lin and gate."""
    zero = torch.zeros_like(gate)
    s, serr = sigmoid(gate, zero)
    a = gate * s
    dlin = dh * a
    dlin_err = derr * a.abs() + (dh.abs() + derr) * (gate.abs() * serr + 2 * U * a.abs()) + 4 * U * dlin.abs()
    c = 1 + gate * (1 - s)
    dgate = dh * lin * s * c
    cerr = gate.abs() * serr + 4 * U * (1 + gate.abs())
    inner = (lin * s * c).abs()
    ierr = lin.abs() * (serr * (c.abs() + cerr) + s * cerr) + 6 * U * inner
    return dlin, dlin_err + 2.0 ** -140, dgate, derr * inner + (dh.abs() + derr) * ierr + 4 * U * dgate.abs() + 2.0 ** -140


def check(name, got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, "%s: shape %s, not %s" % (name, tuple(got.shape), tuple(want.shape))
    over = ~((got - want).abs() <= bound)
    assert not bool(over.any()), "%s: %d of %d values off, by up to %.3g of the bound (|value| up to %.3g)" % (
        name, int(over.sum()), over.numel(), float(((got - want).abs() / bound.clamp_min(1e-300)).max()), float(want.abs().max()))
