"""Experts whose weights are held in 8 bits, and training steps that keep their activations in 8 bits.

8 bits are `torch.float8_e4m3fn` with a scale for each block of 128: of a row's columns for activations and gradients, 128 x 128
values for weights.  Scales made here are powers of two (`torch.float8_e8m0fnu`); weights may bring float32 scales of any
positive size.  Half of bfloat16's memory, and products at up to twice its rate.  The reference has no counterpart: its expert weights
are float tensors (scattermoe/parallel_experts.py:148-182).
"""
import torch
from torch import nn

from .kernels import ops
from .parallel_experts import flatten_sort_count


def quantize_blocks(x, block_rows=1, transposed=False):
    """(q, scales) of x in 8 bits.  block_rows 1: x (..., K), a scale for every 128 values of a row, scales (..., ceil(K / 128));
    block_rows 128: weights x (E, N, K), a scale for every 128 x 128 values, scales (E, ceil(N / 128), ceil(K / 128)); `transposed`: (q, scales, q of the
    transposed weights (E, K, N)), which take the same scales.

    q's rows are filled with zeros to a multiple of 16.  A scale is the smallest power of two, 2^-126 or more, by which the block's
    largest magnitude divided is at most 448; values are rounded to nearest, ties to even.  NaN and infinities become NaN, and a block that
    holds an infinity keeps nothing of its other values.  No gradient passes."""
    if block_rows not in (1, ops.BLOCK_8BIT):
        raise ValueError("quantize_blocks: blocks of 1 or %d rows" % ops.BLOCK_8BIT)
    if block_rows == 1:
        if x.dim() < 1 or transposed:
            raise ValueError("quantize_blocks: rows x (..., K), not transposed")
        K = x.size(-1)
        with torch.no_grad():
            q, s = ops.quantize_rows(x.detach().reshape(-1, K) if K else x.detach().reshape(x.shape[:-1].numel(), 0))
        return q.view(*x.shape[:-1], q.size(1)), s.reshape(*x.shape[:-1], s.size(1))
    if x.dim() != 3:
        raise ValueError("quantize_blocks: weights x (E, N, K)")
    with torch.no_grad():
        q, s, qt = ops.quantize_weights(x.detach(), transposed)
    return (q, s, qt) if transposed else (q, s)


def dequantize_blocks(q, scales, block_rows=1, size=None, dtype=torch.bfloat16):
    """The values, of `dtype`, that q and its scales stand for (as `quantize_blocks` returns them; scales of float32 too).  `size`:
    how many columns they are, q's without it."""
    if block_rows not in (1, ops.BLOCK_8BIT):
        raise ValueError("dequantize_blocks: blocks of 1 or %d rows" % ops.BLOCK_8BIT)
    K = q.size(-1) if size is None else size
    if q.dtype != ops.TYPE_8BIT or scales.dtype not in (ops.SCALE_8BIT, torch.float32):
        raise TypeError("dequantize_blocks: float8_e4m3fn values with float8_e8m0fnu or float32 scales, got %s, %s" % (q.dtype, scales.dtype))
    if scales.device != q.device:
        raise RuntimeError("dequantize_blocks: all tensors on the device of q (%s)" % q.device)
    if not 0 <= K <= q.size(-1):
        raise ValueError("dequantize_blocks: %d columns of %s" % (K, tuple(q.shape)))
    if block_rows == 1:
        lead = q.shape[:-1]
        if scales.shape != (*lead, ops.blocks_8bit(K)):
            raise ValueError("dequantize_blocks: scales %s for rows %s of %d" % (tuple(scales.shape), tuple(lead), K))
        rows = lead.numel()
        y = ops.dequantize(q.reshape(1, rows, q.size(-1)), scales.reshape(1, rows, scales.size(-1)), 1, K, dtype)
        return y.view(*lead, K)
    if q.dim() != 3 or scales.shape != (q.size(0), ops.blocks_8bit(q.size(1)), ops.blocks_8bit(K)):
        raise ValueError("dequantize_blocks: scales %s for weights %s of %d columns" % (tuple(scales.shape), tuple(q.shape), K))
    return ops.dequantize(q, scales, ops.BLOCK_8BIT, K, dtype)


def _experts_in_place(q):
    """q (E, N, K) where each expert's values are contiguous and experts lie multiples of 16 bytes apart (every second one, one for all); else a copy."""
    if q.stride(2) == 1 and q.stride(1) == q.size(2) and (q.size(0) == 1 or q.stride(0) % 16 == 0):
        return q
    return q.contiguous()


def _weight(what, name, q, s, device, E, N, K, t=None):
    """The weight (E, N, K), its scales and its transpose as the kernels take them, or an error."""
    if q.dtype != ops.TYPE_8BIT or (t is not None and t.dtype != ops.TYPE_8BIT):
        raise TypeError("%s: %s is held in float8_e4m3fn, got %s" % (what, name, q.dtype if q.dtype != ops.TYPE_8BIT else t.dtype))
    if s.dtype not in (ops.SCALE_8BIT, torch.float32):
        raise TypeError("%s: scales of %s are float8_e8m0fnu or float32, got %s" % (what, name, s.dtype))
    if q.shape != (E, N, ops.row_8bit(K)):
        raise ValueError("%s: %s is (E, N, K) = (%d, %d, %d), K filled with zeros to a multiple of 16, got %s"
                         % (what, name, E, N, ops.row_8bit(K), tuple(q.shape)))
    if s.shape != (E, ops.blocks_8bit(N), ops.blocks_8bit(K)):
        raise ValueError("%s: a scale for every 128 x 128 of %s is %s, got %s"
                         % (what, name, (E, ops.blocks_8bit(N), ops.blocks_8bit(K)), tuple(s.shape)))
    if t is not None and t.shape != (E, K, ops.row_8bit(N)):
        raise ValueError("%s: the transpose of %s is (E, K, N) = (%d, %d, %d), N filled with zeros to a multiple of 16, got %s"
                         % (what, name, E, K, ops.row_8bit(N), tuple(t.shape)))
    for u in (q, s, t):
        if u is not None and u.device != device:
            raise RuntimeError("%s: all tensors on the device of the rows (%s)" % (what, device))
    if s.size(1) * s.stride(1) + s.size(2) * s.stride(2) > 1 << 28:
        s = s.contiguous()
    return _experts_in_place(q), s, None if t is None else _experts_in_place(t)


def _rows_and_bias(what, x, b, name, shape):
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("%s: rows of float32, bfloat16 or float16, got %s" % (what, x.dtype))
    if b is None:
        return
    if b.shape != shape:
        raise ValueError("%s: %s %s, got %s" % (what, name, shape, tuple(b.shape)))
    if b.dtype != x.dtype:
        raise TypeError("%s: dtype mismatch (%s vs %s)" % (what, x.dtype, b.dtype))
    if b.device != x.device:
        raise RuntimeError("%s: all tensors on the device of the rows (%s)" % (what, x.device))
    if b.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s: %s is held constant beside weights in 8 bits (no gradient goes to it)" % (what, name))


class _Linear8bit(torch.autograd.Function):
    """y = Q(x) W^T, combined with the gates; backward dx = Q(gate dy) W from the transposed weights, nothing to the weights."""

    @staticmethod
    def rows(x, gates, w, s, b, idx, off, k, grouped_in, grouped_out):
        """(y, the experts' rows where gates weigh them)"""
        y = ops.linear_8bit(x, w, s, idx, off, k, b=b, x_grouped=grouped_in, y_grouped=grouped_out, dtype=None if gates is None else torch.float32)
        if gates is None:
            return y, None
        kept = y.view(gates.size(0), gates.size(1), y.size(1))
        return ops.combine(kept, gates, dtype=x.dtype), kept

    @staticmethod
    def forward(ctx, x, gates, w, s, wt, b, idx, off, k, grouped_in, grouped_out):
        y, kept = _Linear8bit.rows(x, gates, w, s, b, idx, off, k, grouped_in, grouped_out)
        ctx.save_for_backward(gates, kept if gates is not None and ctx.needs_input_grad[1] else None, wt, s, idx, off)
        ctx.k, ctx.rows, ctx.grouped = k, x.size(0), (grouped_in, grouped_out)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        gates, kept, wt, s, idx, off = ctx.saved_tensors
        grouped_in, grouped_out = ctx.grouped
        dx = d_gates = None
        if not dy.is_contiguous():
            dy = dy.contiguous()
        if kept is not None:
            d_gates = ops.gate_grad(kept, dy)
        if ctx.needs_input_grad[0]:
            fan, coeff = 1, None
            if gates is not None:
                fan, coeff = gates.size(1), gates.to(dy.dtype).contiguous()
            d_rows = ops.linear_8bit(dy, wt, s, idx, off, fan, coeff=coeff, transposed=True, x_grouped=grouped_out, y_grouped=grouped_in,
                                     dtype=dy.dtype if ctx.k == 1 else torch.float32)
            dx = ops.slot_sum(d_rows, ctx.rows, ctx.k, dtype=dy.dtype)
        return dx, d_gates, None, None, None, None, None, None, None, None, None


def parallel_linear_8bit(inputs, weight, weight_scales, k, sorted_expert_idxs, sorted_scattered_idxs, expert_offsets,
                         expert_biases=None, gates=None, grouped_in=False, grouped_out=False, weight_t=None):
    """`parallel_linear` on weights in 8 bits: inputs (tokens, K), or (rows, K) with `grouped_in`, float32, bfloat16 or float16, are taken to
    8 bits with a scale for every 128 of a row, multiplied by weight (E, N, K rounded up to 16, the rest zeros) of float8_e4m3fn with weight_scales
    (E, ceil(N / 128), ceil(K / 128)) of float8_e8m0fnu or float32, and rounded once: rows that gates weigh, and the gradients of a token's
    slots, are added up in float32.  A product's own sums are those of the 8-bit matrix instruction, 1.3e-5 of the result off, where rows of 16 bits
    are many, and float32 ones where they are float32 (`inputs.float()` chooses those, at half the rate).  Biases (E, N) and gates (tokens, k) of
    the inputs' type.  Routing as for `parallel_linear`; gates go with `grouped_out=False`.

    Slots that the routing dropped (ids outside [0, E)) have rows of zeros; gates that weigh those are finite numbers.

    Weights, scales and biases are constants.  The inputs' gradient, Q(gate dy) W, needs weight_t (E, K, N rounded up to 16), the transposed
    weight (`quantize_blocks(w, 128, transposed=True)`); gates have theirs without it."""
    what = "parallel_linear_8bit"
    if inputs.dim() != 2 or weight.dim() != 3 or k < 1:
        raise ValueError("%s: inputs (rows, K) and weight (E, N, K)" % what)
    E, N, _ = weight.shape
    rows, K = inputs.shape
    L = sorted_scattered_idxs.numel()
    if K == 0 or N == 0 or E == 0 or L != (rows if grouped_in and k == 1 else rows * k) or expert_offsets.numel() != E:
        raise ValueError("%s: %d rows of %d for %d (token, slot) pairs, k = %d, %d offsets for %d experts"
                         % (what, rows, K, L, k, expert_offsets.numel(), E))
    if grouped_in and k != 1:
        raise ValueError("%s: rows that come grouped have k = 1" % what)
    _rows_and_bias(what, inputs, expert_biases, "expert_biases", (E, N))
    weight, scales, weight_t = _weight(what, "weight", weight, weight_scales, inputs.device, E, N, K, weight_t)
    if sorted_scattered_idxs.device != inputs.device or expert_offsets.device != inputs.device:
        raise RuntimeError("%s: all tensors on the device of the rows (%s)" % (what, inputs.device))
    if gates is not None:
        if grouped_out or gates.dim() != 2 or gates.numel() != L:
            raise ValueError("%s: gates (tokens, k) weigh rows by slot (grouped_out=False)" % what)
        if gates.device != inputs.device:
            raise RuntimeError("%s: all tensors on the device of the rows (%s)" % (what, inputs.device))
    if inputs.requires_grad and torch.is_grad_enabled() and weight_t is None:
        raise ValueError("%s: the gradient of the inputs needs weight_t, the transposed weight" % what)
    idx, off = ops._as_i64(sorted_scattered_idxs).contiguous(), ops._as_i64(expert_offsets).contiguous()
    trained = torch.is_grad_enabled() and (inputs.requires_grad or (gates is not None and gates.requires_grad))
    if not trained and not ops.has_tangents(inputs, gates, expert_biases):
        return _Linear8bit.rows(inputs, gates, weight, scales, expert_biases, idx, off, k, grouped_in, grouped_out)[0]
    return _Linear8bit.apply(inputs, gates, weight, scales, weight_t, expert_biases, idx, off, k, grouped_in, grouped_out)


class _GluMLP8bit(torch.autograd.Function):
    """The whole layer; keeps its pre-activation in 8 bits where the tokens' gradient is asked for."""

    @staticmethod
    def forward(ctx, x, gates, experts, w1, s1, w1t, b1, w2, s2, w2t, b2, idx, off, act):
        need_x, need_g = ctx.needs_input_grad[:2]
        out, rows, p8, ps = ops.glu_mlp_8bit(x, gates.to(x.dtype), w1, s1, b1, w2, s2, b2, experts=experts, order=(idx, off), act=act, keep=need_x)
        ctx.save_for_backward(gates, rows if need_g else None, w1t, s1, w2t, s2, p8, ps, idx, off)
        ctx.act = act
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        gates, rows, w1t, s1, w2t, s2, p8, ps, idx, off = ctx.saved_tensors
        d_out = ops._rows_contiguous(d_out)
        dx = d_gates = None
        if rows is not None:
            d_gates = ops.gate_grad(rows.view(gates.size(0), gates.size(1), rows.size(1)), d_out)
        if p8 is not None:
            dx = ops.glu_mlp_8bit_bwd(d_out, gates.to(d_out.dtype), w1t, s1, w2t, s2, p8, ps, idx, off, ctx.act)
        return (dx, d_gates) + (None,) * 12


def glu_mlp_8bit(x, expert_p, expert_idxs, w1, s1, w2, s2, b1=None, b2=None, gate_first=False, w1_t=None, w2_t=None):
    """GLUMLP.forward on weights in 8 bits: x (..., d), expert_p and expert_idxs (tokens, k), w1 (E, 2F, d rounded up to 16) and w2 (E, d, F
    rounded up to 16) of float8_e4m3fn, the rest zeros, with scales s1, s2 for every 128 x 128, float8_e8m0fnu or float32; biases (E, 2F), (E, d) or
    None of x's type; SiLU on the second half of the first product's columns, on the first when `gate_first`.

    The tokens and the hidden rows are taken to 8 bits; pre-activations, the experts' rows and sums stay in float32, and the result is rounded
    once.  Sums whose results go to 8 bits again (hidden values, their gradients) are those of the 8-bit matrix instruction for bfloat16, where a value
    next to a border of 8 bits may fall to its other side (2.0e-3 to 2.2e-3 of the result against 64 bits, bfloat16's rounding alone 1.7e-3), and
    float32 ones for float16 and float32: tokens of those types choose them, at half the rate.  expert_p is taken to x's type.  A slot whose id lies outside [0, E) (padding) adds nothing, whatever its gate, and has no gradient.  A step that asks for the gradient of expert_p keeps the experts' rows in float32.  Weights, scales and biases are constants.  The gradient of x needs the transposed weights w1_t (E, d, 2F
    rounded up to 16) and w2_t (E, F, d rounded up to 16); the step then keeps the pre-activation in 8 bits, and nothing else of its
    width, and the gradients that its products read are taken to 8 bits too."""
    what = "glu_mlp_8bit"
    if x.dim() < 1 or w1.dim() != 3 or w2.dim() != 3 or expert_idxs.dim() != 2 or expert_p.shape != expert_idxs.shape:
        raise ValueError("%s: x (..., d), expert_p and expert_idxs (tokens, k), w1 (E, 2F, d) and w2 (E, d, F)" % what)
    d, E, F = x.size(-1), w1.size(0), w1.size(1) // 2
    T, k = expert_idxs.shape
    if d == 0 or F == 0 or E == 0 or k == 0 or w1.size(1) != 2 * F or x.numel() != T * d:
        raise ValueError("%s: sizes of x %s, expert_idxs %s, w1 %s do not fit" % (what, tuple(x.shape), tuple(expert_idxs.shape), tuple(w1.shape)))
    _rows_and_bias(what, x, b1, "b1", (E, 2 * F))
    _rows_and_bias(what, x, b2, "b2", (E, d))
    w1, s1, w1_t = _weight(what, "w1", w1, s1, x.device, E, 2 * F, d, w1_t)
    w2, s2, w2_t = _weight(what, "w2", w2, s2, x.device, E, d, F, w2_t)
    if expert_p.device != x.device or expert_idxs.device != x.device:
        raise RuntimeError("%s: all tensors on the device of the rows (%s)" % (what, x.device))
    if x.requires_grad and torch.is_grad_enabled() and (w1_t is None or w2_t is None):
        raise ValueError("%s: the gradient of x needs w1_t and w2_t, the transposed weights" % what)
    act = ops.ACT_SILU_GATE_FIRST if gate_first else ops.ACT_SILU
    tokens = x if x.dim() == 2 else x.reshape(T, d)                  # (a view would be a node of the backward pass)
    trained = ((x.requires_grad or expert_p.requires_grad) and torch.is_grad_enabled()) or ops.has_tangents(x, expert_p, b1, b2)
    # (by the ids an expert's weights are read once for every 8 of its rows: 64 rows of 8 experts, 4096 / 14336, 368 us, in the experts' order 265.
    # The ids are on the device: of few experts, 64 rows of one of 16, 4096 / 4096, it is 151 us for 56 and the routing, of all 16 161 for 155)
    experts = ops._as_i64(expert_idxs).contiguous()
    if not trained and T * k <= min(ops.FEW_ROWS_8BIT, 4 * E):
        out = ops.glu_mlp_8bit(tokens, expert_p.to(x.dtype), w1, s1, b1, w2, s2, b2, experts=experts, act=act)[0]
        return out if x.dim() == 2 else out.view(x.shape)
    _, idx, off = flatten_sort_count(expert_idxs, num_experts=E)
    if trained:
        out = _GluMLP8bit.apply(tokens, expert_p, experts, w1, s1, w1_t, b1, w2, s2, w2_t, b2, idx, off, act)
    else:
        out = ops.glu_mlp_8bit(tokens, expert_p.to(x.dtype), w1, s1, b1, w2, s2, b2, experts=experts, order=(idx, off), act=act)[0]
    return out if x.dim() == 2 else out.view(x.shape)


class _CheckpointedGLU(torch.autograd.Function):
    """h = lin silu(gate) from pre itself; the backward pass has pre in 8 bits."""

    @staticmethod
    def forward(ctx, pre, act):
        h, p8, ps = ops.glu_8bit_fwd(pre, act)
        ctx.save_for_backward(p8, ps)
        ctx.act = act
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        p8, ps = ctx.saved_tensors
        return ops.glu_8bit_bwd(p8, ps, dh, ctx.act)[0], None


def checkpointed_glu(pre, gate_first=False):
    """The gated unit lin * silu(gate) of pre (..., 2F), halves (lin, gate), (gate, lin) when `gate_first`, that keeps for the backward
    pass pre in 8 bits, a scale for every 128 columns of each half: half the memory of a 16-bit pre, and an input gradient whose
    error is that of four significant bits of pre (2^-4 of lin or gate).  Values are those of the plain unit."""
    if pre.dim() < 1 or pre.size(-1) % 2 != 0:
        raise ValueError("checkpointed_glu: pre (..., 2F), got %s" % (tuple(pre.shape),))
    if pre.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("checkpointed_glu: float32, bfloat16 or float16, got %s" % pre.dtype)
    F = pre.size(-1) // 2
    act = ops.ACT_SILU_GATE_FIRST if gate_first else ops.ACT_SILU
    rows = pre                                                       # (a view would be a node of the backward pass)
    if pre.dim() != 2:
        rows = pre.reshape(-1, 2 * F) if F else pre.reshape(pre.shape[:-1].numel(), 0)
    if (pre.requires_grad and torch.is_grad_enabled()) or ops.has_tangents(pre):
        h = _CheckpointedGLU.apply(rows, act)
    else:
        h = ops.glu_fwd(rows, act)
    return h if pre.dim() == 2 else h.view(*pre.shape[:-1], F)


class GLUMLP8bit(nn.Module):
    """`GLUMLP` with its weights in 8 bits, held constant: buffers `w1`, `s1`, `w2`, `s2` (and `w1_t`, `w2_t` with `input_gradients`, twice
    the memory), biases `b1`, `b2` or None.  Made from a `GLUMLP` by `from_module`."""

    _held = ("w1", "s1", "w1_t", "w2", "s2", "w2_t")

    def __init__(self, input_size, hidden_size, num_experts, top_k, bias=False, dtype=torch.bfloat16, input_gradients=False,
                 scale_type=torch.float8_e8m0fnu):
        super().__init__()
        if scale_type not in (ops.SCALE_8BIT, torch.float32):
            raise TypeError("GLUMLP8bit: scales of float8_e8m0fnu or float32, got %s" % scale_type)
        self.input_size, self.hidden_size, self.num_experts, self.top_k = input_size, hidden_size, num_experts, min(top_k, num_experts)
        d, f, E = input_size, hidden_size, num_experts
        for i, (n, k) in ((1, (2 * f, d)), (2, (d, f))):
            self.register_buffer("w%d" % i, torch.zeros((E, n, ops.row_8bit(k)), dtype=ops.TYPE_8BIT))
            self.register_buffer("s%d" % i, torch.ones((E, ops.blocks_8bit(n), ops.blocks_8bit(k)), dtype=scale_type))
            self.register_buffer("w%d_t" % i, torch.zeros((E, k, ops.row_8bit(n)), dtype=ops.TYPE_8BIT) if input_gradients else None)
            self.register_buffer("b%d" % i, torch.zeros((E, n), dtype=dtype) if bias else None)

    @classmethod
    def from_module(cls, module, input_gradients=False):
        """The 8-bit copy of a `GLUMLP` on a GPU."""
        if type(getattr(module, "activation", None)) is not nn.SiLU:
            raise ValueError("GLUMLP8bit: the activation has to be SiLU")
        w1, w2 = module.experts.weight, module.output_experts.weight
        E, d, f = module.num_experts, module.input_size, module.hidden_size
        if w1.shape != (E, 2 * f, d) or w2.shape != (E, d, f):
            raise ValueError("GLUMLP8bit: a gated layer of %d experts has weights (E, 2F, d) = %s and (E, d, F) = %s, got %s, %s"
                             % (E, (E, 2 * f, d), (E, d, f), tuple(w1.shape), tuple(w2.shape)))
        m = cls(module.input_size, module.hidden_size, module.num_experts, module.top_k, bias=module.experts.bias is not None,
                dtype=w1.dtype, input_gradients=input_gradients)
        m.w1, m.s1, m.w1_t = ops.quantize_weights(w1.detach(), input_gradients)
        m.w2, m.s2, m.w2_t = ops.quantize_weights(w2.detach(), input_gradients)
        if m.b1 is not None:
            m.b1, m.b2 = module.experts.bias.detach().clone(), module.output_experts.bias.detach().clone()
        return m

    def _apply(self, fn, recurse=True):
        held = {name: self._buffers[name] for name in self._held}
        self._buffers.update(dict.fromkeys(self._held))              # (a cast to another type is for the biases only)
        try:
            super()._apply(fn, recurse)
            for name, t in held.items():
                if t is not None:
                    like = fn(t.new_empty(0))                        # where it goes, and whether as what it is
                    held[name] = fn(t) if like.dtype == t.dtype else t.to(device=like.device)
        finally:
            self._buffers.update(held)
        return self

    def extra_repr(self):
        return "input_size={}, hidden_size={}, num_experts={}, k={}, bias={}".format(
            self.input_size, self.hidden_size, self.num_experts, self.top_k, self.b1 is not None)

    def forward(self, x, expert_p, expert_idxs):
        return glu_mlp_8bit(x, expert_p, expert_idxs, self.w1, self.s1, self.w2, self.s2, b1=self.b1, b2=self.b2, w1_t=self.w1_t,
                            w2_t=self.w2_t)
