"""Low-rank adapters of many requests beside a shared projection.

`ParallelExperts` holds E weights and every row picks one by its id; here all rows share one weight and each picks a
low-rank addition to it by its id: the projections around the expert layer of fine-tuned requests served, or trained, in
one batch.  The reference has no counterpart (its rows pick whole weights, scattermoe/parallel_experts.py:148-182).
"""
import torch
from torch import nn

from .kernels import ops


class _ParallelAdapters(torch.autograd.Function):
    """y = x W^T (+ bias) + u B[a]^T with u = scales[a] x A[a]^T kept in float32.  The backward pass is the same two
    products on the transposed factors, v = scales[a] dy B[a] and dx = dy W + v A[a], and the sums of v x^T and dy u^T
    over each adapter's rows."""

    @staticmethod
    def forward(ctx, x, weight, bias, lora_a, lora_b, ids, scales):
        order = ops.adapter_order(ids, lora_a.size(0)) if x.size(0) > ops.ADAPTER_FEW_ROWS else None
        u, planes = ops.adapter_low(x, lora_a, ids, scales, order)
        y = ops.adapter_project(x, weight, u, lora_b, ids, bias, planes, order)
        ctx.save_for_backward(x, weight, lora_a, lora_b, ids, scales, u, *(order or ()))
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, lora_a, lora_b, ids, scales, u = ctx.saved_tensors[:7]
        order = ctx.saved_tensors[7:] or None
        need_x, need_w, need_b, need_la, need_lb = ctx.needs_input_grad[:5]
        R = lora_a.size(0)
        dx = dw = db = da = dlb = None
        if not dy.is_contiguous():
            dy = dy.contiguous()
        if need_x or need_la:
            v, planes = ops.adapter_low(dy, lora_b.transpose(1, 2), ids, scales, order)
            if need_x:
                dx = ops.adapter_project(dy, weight.t(), v, lora_a.transpose(1, 2), ids, None, planes, order)
        if need_la or need_lb:
            idx, off = order or ops.adapter_order(ids, R)
            if need_la:
                da = ops.adapter_grad(v, x, idx, off, R)
            if need_lb:
                dlb = ops.adapter_grad(u, dy, idx, off, R, transposed=True)
        if need_w or (need_b and ctx.has_bias):
            rows = torch.full((1,), x.size(0), dtype=torch.int64, device=x.device)
            if need_w:
                dw = ops.group_bwd_W(DY=dy, X=x, expert_offsets=rows, E=1)[0][0].t()
            if need_b and ctx.has_bias:
                ones = torch.ones((x.size(0), 1), dtype=torch.float32, device=x.device)
                db = ops.adapter_grad(ones, dy, None, rows, 1).view(-1)
        return dx, dw, db, da, dlb, None, None


def parallel_adapters(x, weight, lora_a, lora_b, adapter_idxs, scales=None, bias=None):
    """y[t] = weight @ x[t] (+ bias) + scales[a] * lora_b[a] @ (lora_a[a] @ x[t]),  a = adapter_idxs[t].

    x (..., d), weight (n, d), bias (n) or None, lora_a (R, r, d), lora_b (R, n, r): float32, bfloat16 or float16, all the
    same; adapter_idxs: integers of x's leading shape, and a row whose id lies outside [0, R) (-1, say) gets the shared
    projection alone; scales (R) or None (ones), a constant.  Adapters of a smaller rank are padded with zeros.  Everything but
    the output is summed and kept in float32.  Gradients go to x, weight, bias, lora_a and lora_b."""
    if weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3 or x.dim() < 1:
        raise ValueError("parallel_adapters: x (..., d), weight (n, d), lora_a (R, r, d) and lora_b (R, n, r)")
    n, d = weight.shape
    R, r = lora_a.shape[:2]
    if x.size(-1) != d or lora_a.size(2) != d or lora_b.shape != (R, n, r) or (bias is not None and bias.shape != (n,)):
        raise ValueError("parallel_adapters: sizes of x %s, weight %s, lora_a %s, lora_b %s%s do not fit"
                         % (tuple(x.shape), tuple(weight.shape), tuple(lora_a.shape), tuple(lora_b.shape),
                            "" if bias is None else ", bias %s" % (tuple(bias.shape),)))
    if not 0 < R <= ops.ADAPTERS_MAX or not 0 < r <= ops.ADAPTER_MAX_RANK or d == 0:
        raise ValueError("parallel_adapters: 1..%d adapters of rank 1..%d" % (ops.ADAPTERS_MAX, ops.ADAPTER_MAX_RANK))
    if adapter_idxs.shape != x.shape[:-1]:
        raise ValueError("parallel_adapters: adapter_idxs %s for rows %s" % (tuple(adapter_idxs.shape), tuple(x.shape[:-1])))
    if adapter_idxs.is_floating_point() or adapter_idxs.is_complex() or adapter_idxs.dtype == torch.bool:
        raise TypeError("parallel_adapters: adapter_idxs must be integers, got %s" % adapter_idxs.dtype)
    ops._same_dtype("parallel_adapters", x, weight, lora_a, lora_b, bias)
    for t in (weight, lora_a, lora_b, adapter_idxs, scales, bias):
        if t is not None and t.device != x.device:
            raise RuntimeError("parallel_adapters: tensors on %s and %s" % (x.device, t.device))
    if scales is not None:
        if scales.shape != (R,):
            raise ValueError("parallel_adapters: scales %s for %d adapters" % (tuple(scales.shape), R))
        if scales.requires_grad:
            raise ValueError("parallel_adapters: scales are constants (no gradient goes to them)")
        scales = scales.to(torch.float32).contiguous()
    ids = ops._as_i64(adapter_idxs.reshape(-1)).contiguous()
    y = _ParallelAdapters.apply(x.reshape(-1, d), weight, bias, lora_a, lora_b, ids, scales)
    return y.view(*x.shape[:-1], n)


class ParallelAdapters(nn.Module):
    """A linear map (weight (out, in), optional bias) shared by all rows, with R low-rank adapters beside it:
    lora_a (R, rank, in), drawn like a weight, lora_b (R, out, rank), zeros, and their factors `scales` (R)."""

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
        self.register_buffer("scales", torch.full((num_adapters,), float(scale)))
        self.reset_parameters()

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
