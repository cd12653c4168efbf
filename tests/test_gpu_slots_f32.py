"""Sums over a token's float32 rows and their gates' gradient against the same in 64 bits: widths and strides that are and are not whole 16-byte pieces,
one slot and many, without gates, ids outside of the experts.  Bounds: a sum of n terms in float32 is off by at most n + 1 roundings (2^-24 each) of
the terms' magnitudes, the gates' gradient as much of its N terms; then one rounding to the type."""
import pytest
import torch

import _ref_8bit as ref
from scattermoe_amd import _C
from scattermoe_amd.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 1, 1), (1, 9, 64), (3, 2, 7), (5, 4, 260), (17, 5, 1028), (2, 8, 4096), (300, 3, 130), (33, 1, 2048), (4, 64, 12), (0, 2, 8)]


def _rows(T, k, N, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T * k, N, generator=g), torch.rand(T, k, generator=g) - 0.3, torch.randn(T, N, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,N", SIZES)
def test_sums_and_gradients(dtype, T, k, N):
    rows, p, dout = _rows(T, k, N, T + N)
    p, dout = p.to(dtype), dout.to(dtype)
    y = rows.to(DEV).view(T, k, N)
    y64, p64, d64 = rows.double().view(T, k, N), p.double().unsqueeze(-1), dout.double().unsqueeze(1)
    got = ops.combine(y, p.to(DEV), dtype=dtype)
    assert got.dtype == dtype
    ref.check("weighed", got, (y64 * p64).sum(1), ref.rounded((y64 * p64).sum(1), (k + 1) * ref.U * (y64 * p64).abs().sum(1), dtype))
    got = ops.slot_sum(y.view(T * k, N), T, k, dtype=dtype)
    if k > 1:
        ref.check("sum", got, y64.sum(1), ref.rounded(y64.sum(1), k * ref.U * y64.abs().sum(1), dtype))
    got = ops.gate_grad(y, dout.to(DEV))
    v = (y64 * d64).sum(-1)
    assert got.dtype == dtype
    ref.check("gates", got, v, ref.rounded(v, (N + 1) * ref.U * (y64 * d64).abs().sum(-1), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (4, 0), (1, 0), (4, 1), (0, 2)])
def test_strides_and_ids_through_the_library(dtype, pad, shift):
    """Rows and results of other strides, not at 16 bytes; gates of strides of their own; ids outside [0, E) leave out their slots, no numbers in either."""
    T, k, N, E = 11, 3, 68, 5
    rows, p, dout = _rows(T, k, N, pad + shift)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-2, E + 2, (T, k), generator=g)
    ids[0], ids[1, 0] = -1, 1 << 32
    kept = (ids >= 0) & (ids < E)
    wide = torch.full((T * k * (N + pad) + 4,), float("nan"))
    y = wide[shift:shift + T * k * (N + pad)].view(T * k, N + pad)[:, :N]
    y.copy_(torch.where(kept.view(-1, 1), rows, torch.tensor(float("nan"))))
    y = wide.to(DEV)[shift:shift + T * k * (N + pad)].view(T * k, N + pad)[:, :N]
    gates = torch.where(kept, p, torch.tensor(float("inf"))).to(dtype).t().contiguous().to(DEV).t()
    out = torch.full((T, N + pad), 7.0, dtype=dtype, device=DEV)
    lib, code, st = _C.load(), _C.float_code(dtype), _C.stream_ptr(torch.device(DEV))
    ids = ids.to(DEV)
    assert lib.smoe_combine_f32(_C.ptr(y), y.stride(0), _C.ptr(gates), gates.stride(0), gates.stride(1), _C.ptr(ids), E, _C.ptr(out), out.stride(0), T, k, N,
                                code, st) == 0
    y64 = torch.where(kept.view(T, k, 1), rows.double().view(T, k, N) * p.to(dtype).double().unsqueeze(-1), torch.zeros((), dtype=torch.double))
    ref.check("weighed", out[:, :N], y64.sum(1), ref.rounded(y64.sum(1), (k + 1) * ref.U * y64.abs().sum(1), dtype))
    assert bool((out[:, N:] == 7.0).all()) and not bool(out[0, :N].any())
    d = torch.zeros(T, N + pad, dtype=dtype)
    d[:, :N] = dout.to(dtype)
    d = d.to(DEV)
    dg = torch.zeros(k, T, dtype=dtype, device=DEV).t()
    assert lib.smoe_gate_grad_f32(_C.ptr(y), y.stride(0), _C.ptr(d), d.stride(0), _C.ptr(dg), dg.stride(0), dg.stride(1), T, k, N, code, st) == 0
    v = rows.double().view(T, k, N) * dout.to(dtype).double().unsqueeze(1)
    ref.check("gates", dg[kept.to(DEV)], v.sum(-1)[kept], ref.rounded(v.sum(-1), (N + 1) * ref.U * v.abs().sum(-1), dtype)[kept])
    assert bool(dg[~kept.to(DEV)].isnan().all())
