"""Low-rank adapters of many requests beside a shared projection.

`ParallelExperts` holds E weights and every row picks one by its id; here all rows share one weight and each picks a
low-rank addition to it by its id: the projections around the expert layer of fine-tuned requests served, or trained, in
one batch.  The reference has no counterpart (its rows pick whole weights, scattermoe/parallel_experts.py:148-182).
"""
import torch
from torch import nn

from .kernels import ops


_ID_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class _ParallelAdapters(torch.autograd.Function):
    """y = x W^T (+ bias) + u B[a]^T with u = scales[a] x A[a]^T kept in float32.  The backward pass is the same two
    products on the transposed factors, v = scales[a] dy B[a] and dx = dy W + v A[a], and the sums of v x^T and dy u^T
    over each adapter's rows."""

    @staticmethod
    def forward(ctx, x, weight, bias, lora_a, lora_b, ids, scales):
        y, u, order = ops.adapter_forward(x, weight, lora_a, lora_b, ids, scales, bias)
        ctx.save_for_backward(x, weight, lora_a, lora_b, ids, scales, u, *order)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, lora_a, lora_b, ids, scales, u, *order = ctx.saved_tensors
        need_x, need_w, need_bias, need_a, need_b = ctx.needs_input_grad[:5]
        dx = da = db = dbias = dw = None
        if need_x or need_a or need_b or need_bias:
            dx, da, db, dbias = ops.adapter_backward(dy, x, weight, lora_a, lora_b, ids, scales, u, order, need_x, need_a,
                                                     need_b, need_bias)
        if need_w:
            rows = torch.full((1,), x.size(0), dtype=torch.int64, device=x.device)
            dw = ops.group_bwd_W(DY=dy.contiguous(), X=x, expert_offsets=rows, E=1)[0][0].t()
        return dx, dw, dbias, da, db, None, None


def parallel_adapters(x, weight, lora_a, lora_b, adapter_idxs, scales=None, bias=None):
    """y[t] = weight @ x[t] (+ bias) + scales[a] * lora_b[a] @ (lora_a[a] @ x[t]),  a = adapter_idxs[t].

    x (..., d), weight (n, d), bias (n) or None, lora_a (R, r, d), lora_b (R, n, r): float32, bfloat16 or float16, all the
    same; adapter_idxs: integers of x's leading shape, and a row whose id lies outside [0, R) (-1, say) gets the shared
    projection alone; scales (R) or None (ones), a constant.  Adapters of a smaller rank are padded with zeros.  Everything but
    the output is summed and kept in float32.  Gradients go to x, weight, bias, lora_a and lora_b; forward-mode derivatives are refused."""
    dtype, device, shape = x.dtype, x.device, x.shape
    tensors = (weight, lora_a, lora_b) if bias is None else (weight, lora_a, lora_b, bias)
    if weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3 or not shape:
        raise ValueError("parallel_adapters: x (..., d), weight (n, d), lora_a (R, r, d) and lora_b (R, n, r)")
    n, d = weight.shape
    R, r, _ = lora_a.shape
    if shape[-1] != d or lora_a.size(2) != d or lora_b.shape != (R, n, r) or (bias is not None and bias.shape != (n,)):
        raise ValueError("parallel_adapters: sizes of x %s, weight %s, lora_a %s, lora_b %s%s do not fit"
                         % (tuple(shape), tuple(weight.shape), tuple(lora_a.shape), tuple(lora_b.shape),
                            "" if bias is None else ", bias %s" % (tuple(bias.shape),)))
    if not 0 < R <= ops.ADAPTERS_MAX or not 0 < r <= ops.ADAPTER_MAX_RANK or d == 0:
        raise ValueError("parallel_adapters: 1..%d adapters of rank 1..%d" % (ops.ADAPTERS_MAX, ops.ADAPTER_MAX_RANK))
    if adapter_idxs.shape != shape[:-1]:
        raise ValueError("parallel_adapters: adapter_idxs %s for rows %s" % (tuple(adapter_idxs.shape), tuple(shape[:-1])))
    if adapter_idxs.dtype not in _ID_TYPES:
        raise TypeError("parallel_adapters: adapter_idxs must be integers, got %s" % adapter_idxs.dtype)
    if adapter_idxs.device != device or (scales is not None and scales.device != device):
        raise RuntimeError("parallel_adapters: all tensors on the device of x (%s)" % device)
    trained = x.requires_grad
    for t in tensors:
        if t.dtype != dtype:
            raise TypeError("parallel_adapters: dtype mismatch (%s vs %s)" % (dtype, t.dtype))
        if t.device != device:
            raise RuntimeError("parallel_adapters: all tensors on the device of x (%s)" % device)
        trained = trained or t.requires_grad
    if scales is not None:
        if scales.shape != (R,):
            raise ValueError("parallel_adapters: scales %s for %d adapters" % (tuple(scales.shape), R))
        if scales.requires_grad:
            raise ValueError("parallel_adapters: scales are constants (no gradient goes to them)")
        if scales.dtype != torch.float32 or not scales.is_contiguous():
            scales = scales.to(torch.float32).contiguous()
    ids = adapter_idxs
    if len(shape) != 2:
        x, ids = x.reshape(-1, d), ids.reshape(-1)
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        ids = ids.to(torch.int64).contiguous()
    if (trained and torch.is_grad_enabled()) or ops.has_tangents(x, scales, *tensors):
        y = _ParallelAdapters.apply(x, weight, bias, lora_a, lora_b, ids, scales)
    else:
        y = ops.adapter_forward(x, weight, lora_a, lora_b, ids, scales, bias)[0]
    return y if len(shape) == 2 else y.view(*shape[:-1], n)


class ParallelAdapters(nn.Module):
    """A linear map (weight (out, in), optional bias) shared by all rows, with R low-rank adapters beside it:
    lora_a (R, rank, in), drawn like a weight, lora_b (R, out, rank), zeros, and their factors `scales` (R), which are float32
    whatever type the module is taken to."""

    def __init__(self, num_adapters, input_size, output_size, rank, bias=False, scale=1.0) -> None:
        super().__init__()
        self.num_adapters = num_adapters
        self.input_size = input_size
        self.output_size = output_size
        self.rank = rank
        self.weight = nn.Parameter(torch.empty(output_size, input_size))
        self.bias = nn.Parameter(torch.empty(output_size)) if bias else None
        self.lora_a = nn.Parameter(torch.empty(num_adapters, rank, input_size))
        self.lora_b = nn.Parameter(torch.empty(num_adapters, output_size, rank))
        self.register_buffer("scales", torch.full((num_adapters,), float(scale), dtype=torch.float32))
        self.reset_parameters()

    def _apply(self, fn, recurse=True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:                       # (eight bits of them would be left in bfloat16)
            self.scales = scales.to(device=self.scales.device, dtype=torch.float32)
        return self

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=0.02)
        nn.init.normal_(self.lora_a, std=0.02)
        nn.init.zeros_(self.lora_b)
        if self.bias is not None:
            nn.init.zeros_(self.bias)

    def extra_repr(self):
        return "num_adapters={}, input_size={}, output_size={}, rank={}".format(
            self.num_adapters, self.input_size, self.output_size, self.rank)

    def forward(self, x, adapter_idxs):
        return parallel_adapters(x, self.weight, self.lora_a, self.lora_b, adapter_idxs, scales=self.scales, bias=self.bias)
