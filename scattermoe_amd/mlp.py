"""Sparse MoE MLP modules with the constructor / forward signatures of scattermoe/mlp.py
(`MLP` :6-49, `GLUMLP` :51-95) and the same state-dict keys
(`experts.weight`, `experts.bias`, `output_experts.weight`, `output_experts.bias`)."""
import torch
from torch import nn

from .kernels import ops
from .parallel_experts import ParallelExperts, flatten_sort_count


class _FusedGLU(torch.autograd.Function):
    """act(second half) * first half in one pass each way (saves the pre-activation, recomputes act)."""

    @staticmethod
    def forward(ctx, pre, act):
        ctx.save_for_backward(pre)
        ctx.act = act
        return ops.glu_fwd(pre, act)

    @staticmethod
    def backward(ctx, dh):
        (pre,) = ctx.saved_tensors
        return ops.glu_bwd(pre, dh, ctx.act), None


class _GatedMLP(torch.autograd.Function):
    """The whole gated expert MLP as one autograd node, so that the gated linear unit can ride in the epilogues
    of the GEMMs around it: forward = layer 1 + GLU (one launch), layer 2, gate-weighted combine; backward =
    the dataflow of two chained ParallelLinear nodes (reference parallel_experts.py:64-134) with the layer-2
    input gradient and the GLU gradient in one launch.  Same numerics as the unfused chain (intermediates are
    rounded to the storage type at the same points).

    w1 (E, d, 2F) and w2 (E, F, d) are the (E, in, out) views the kernels take, in either memory layout: the
    permuted ParallelExperts parameters, or weights stored that way (gpt-oss); their gradients come back in the
    layout of the weight they belong to.  `act`: ops.ACT_SILU / ACT_SILU_GATE_FIRST / ACT_GPT_OSS (+ alpha, limit).

    `checkpoint_8bit` (SiLU): between the passes the pre-activation is held in 8 bits and the hidden rows not at all; the
    backward pass takes the unit's gradient, and the hidden rows for w2's, from those bits."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, gates, eid, idx, off, k, act, alpha=1.702, limit=7.0, checkpoint_8bit=False):
        T = x.size(0)
        need_grad = any(ctx.needs_input_grad[:6])
        p8 = ps = None
        if checkpoint_8bit and need_grad:
            pre = ops.scatter2scatter(x, w1, eid, idx, k, b=b1, y_grouped=True, expert_offsets=off)
            h, p8, ps = ops.glu_8bit_fwd(pre, act)
        else:
            pre, h = ops.scatter2scatter_glu(x, w1, eid, idx, k, b=b1, act=act, expert_offsets=off,
                                             need_pre=need_grad, alpha=alpha, limit=limit)
        expanded = ops.scatter2scatter(h, w2, eid, idx, 1, b=b2, x_grouped=True, y_grouped=False,
                                       expert_offsets=off)
        kept = expanded.view(T, k, expanded.size(-1))
        out = ops.combine(kept, gates)
        if need_grad:
            if p8 is not None:
                pre = h = None
            ctx.save_for_backward(x, w1, b1, w2, b2, gates, eid, idx, off, pre, h, kept, p8, ps)
        ctx.k, ctx.act, ctx.alpha, ctx.limit = k, act, alpha, limit
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x, w1, b1, w2, b2, gates, eid, idx, off, pre, h, kept, p8, ps = ctx.saved_tensors
        k, act = ctx.k, ctx.act
        need_x, need_w1, need_b1, need_w2, need_b2, need_g = ctx.needs_input_grad[:6]
        need_b1 = need_b1 and b1 is not None
        need_b2 = need_b2 and b2 is not None
        E = w1.size(0)
        if not grad_out.is_contiguous():
            grad_out = grad_out.contiguous()
        if need_g:
            # gate gradient and dY of layer 2 (expert-sorted, scaled by each row's gate) in one pass over the
            # expert outputs
            d_gates, dy = ops.gate_grad_group(kept, grad_out, gates, idx)
        else:
            # dY alone reuses the expert-output buffer
            d_gates = None
            dy = ops.group(grad_out, idx, coeff=gates.reshape(-1).to(grad_out.dtype), fan_out=k, permutation=True,
                           out=kept.view(-1, kept.size(-1)))
        dpre = None
        need_pre = need_x or need_w1 or need_b1
        if p8 is not None and need_pre:
            dh = ops.scatter2scatter(dy, w2.permute(0, 2, 1), eid, idx, 1, x_grouped=True, y_grouped=True, expert_offsets=off)
            dpre, h = ops.glu_8bit_bwd(p8, ps, dh, act, need_h=need_w2 or need_b2)
        elif p8 is not None and (need_w2 or need_b2):
            h = ops.glu_fwd(ops.dequantize(p8, ps, 1, w2.size(1), dy.dtype).flatten(1), ops.ACT_SILU)
        d_w2 = d_b2 = None
        if need_w2 or need_b2:
            d_w2, d_b2 = ops.group_bwd_W(DY=dy, X=h, expert_offsets=off, E=E, has_bias=b2 is not None, like=w2)
            d_w2 = d_w2 if need_w2 else None
        d_x = d_w1 = d_b1 = None
        if need_pre:
            if dpre is None:
                dpre = ops.scatter2scatter_glu_bwd(dy, w2.permute(0, 2, 1), pre, eid, idx, act=act, expert_offsets=off,
                                                   alpha=ctx.alpha, limit=ctx.limit)
            if need_w1 or need_b1:
                # rows of x by idx: looked up inside the launch, or copied ahead of it where that is faster
                d_w1, d_b1 = ops.group_bwd_W(DY=dpre, X=x, expert_offsets=off, E=E, has_bias=b1 is not None, like=w1,
                                             gather=(idx, k))
                d_w1 = d_w1 if need_w1 else None
            if need_x:
                d_exp = ops.scatter2scatter(dpre, w1.permute(0, 2, 1), eid, idx, 1, x_grouped=True, y_grouped=False,
                                            expert_offsets=off)
                d_x = ops.slot_sum(d_exp, x.size(0), k)
        return d_x, d_w1, (d_b1 if need_b1 else None), d_w2, (d_b2 if need_b2 else None), d_gates, \
            None, None, None, None, None, None, None, None


class _SparseMLP(nn.Module):
    """Shared body: route once, expert layer 1 (grouped output), activation, expert layer 2 (+gates)."""

    _hidden_mult = 1

    def __init__(self, input_size, hidden_size, num_experts, top_k, bias, activation):
        super().__init__()
        self.num_experts = num_experts
        self.input_size = input_size
        self.hidden_size = hidden_size
        self.experts = ParallelExperts(num_experts, input_size, self._hidden_mult * hidden_size, bias=bias)
        self.output_experts = ParallelExperts(num_experts, hidden_size, input_size, bias=bias)
        self.top_k = min(top_k, self.num_experts)
        self.activation = activation

    def extra_repr(self):
        return "k={}".format(self.top_k)

    def _hidden(self, pre):
        raise NotImplementedError

    def forward(self, x: torch.Tensor, expert_p: torch.Tensor, expert_idxs: torch.Tensor):
        lead = x.shape[:-1]
        tokens = x.view(-1, x.size(-1))
        eid, idx, off = flatten_sort_count(expert_idxs, num_experts=self.num_experts)
        pre = self.experts(tokens, self.top_k, eid, idx, off, grouped_out=True)
        hid = self._hidden(pre)
        out = self.output_experts(hid, 1, eid, idx, off, grouped_in=True, gates=expert_p)
        return out.view(*lead, out.size(-1))


class MLP(_SparseMLP):
    """y = sum_j p_j * W2[e_j] act(W1[e_j] x)."""

    def __init__(self, input_size, hidden_size, num_experts, top_k, bias=False, activation=None):
        super().__init__(input_size, hidden_size, num_experts, top_k, bias, activation)

    def _hidden(self, pre):
        return self.activation(pre)


class GLUMLP(_SparseMLP):
    """Gated variant: layer 1 produces 2*hidden columns; the FIRST half is the linear branch and the
    SECOND half goes through the activation (reference mlp.py:81-87).

    `checkpoint_8bit` (SiLU only): a training step keeps layer 1's rows in 8 bits, a scale for every 128 columns of each half, and not
    the hidden rows: 2 bytes per hidden value instead of 6 of a 16-bit type.  The output is the same; gradients of x, the first
    layer and the second layer's weights carry the 8 bits' error (up to 2^-4 of a linear or gate value)."""

    _hidden_mult = 2
    checkpoint_8bit = False

    def __init__(self, input_size, hidden_size, num_experts, top_k, bias=False, activation=nn.SiLU(), checkpoint_8bit=False):
        if checkpoint_8bit and type(activation) is not nn.SiLU:
            raise ValueError("GLUMLP: checkpoint_8bit goes with SiLU")
        super().__init__(input_size, hidden_size, num_experts, top_k, bias, activation)
        self.checkpoint_8bit = checkpoint_8bit

    def _hidden(self, pre):
        if type(self.activation) is nn.SiLU and pre.dim() == 2:
            return _FusedGLU.apply(pre, ops.ACT_SILU)
        lin, gate = pre.chunk(2, dim=-1)
        return self.activation(gate) * lin

    def forward(self, x: torch.Tensor, expert_p: torch.Tensor, expert_idxs: torch.Tensor):
        if type(self.activation) is not nn.SiLU:
            if self.checkpoint_8bit and torch.is_grad_enabled():       # (an activation that was put in later)
                raise ValueError("GLUMLP: checkpoint_8bit goes with SiLU")
            return super().forward(x, expert_p, expert_idxs)
        lead = x.shape[:-1]
        tokens = x.view(-1, x.size(-1))
        if (expert_idxs.numel() <= ops.DECODE_MAX_ROWS and not torch.is_grad_enabled() and expert_idxs.dim() == 2
                and not ops.in_dual_level()):
            out = ops.decode_glu_mlp(tokens, expert_p, expert_idxs, self.experts.weight, self.experts.bias,
                                     self.output_experts.weight, self.output_experts.bias, ops.ACT_SILU)
            if out is not None:
                return out.view(*lead, out.size(-1))
        eid, idx, off = flatten_sort_count(expert_idxs, num_experts=self.num_experts)
        out = _GatedMLP.apply(tokens, self.experts.weight.permute(0, 2, 1), self.experts.bias,
                              self.output_experts.weight.permute(0, 2, 1), self.output_experts.bias, expert_p,
                              eid, idx, off, self.top_k, ops.ACT_SILU, 1.702, 7.0, self.checkpoint_8bit)
        return out.view(*lead, out.size(-1))


def routed_glu_mlp(x, router_weight, w1, w2, k, b1=None, b2=None, renormalize=True, gate_first=False):
    """A gated MoE layer from its tokens: (output of x's shape, router logits (tokens, E) float32).

    x (..., d); router_weight (E, d); w1 (E, 2F, d) and w2 (E, d, F) in the ParallelExperts parameter layout, biases
    (E, 2F) / (E, d) or None, all of one type.  Every token goes to the k experts with the largest logits, weighted by its
    softmax over all logits, divided by their sum when `renormalize`; SiLU on the second half of layer 1's columns, on the first
    when `gate_first` (the routing of scattermoe/utils/replace_moe.py:67-71 in front of GLUMLP.forward, mlp.py:74-95).

    Where nothing asks for a gradient and for few tokens (`ops.few_tokens_pay`) the layer is one call of the library (`ops.routed_glu_mlp`); otherwise
    router product, `topk_softmax`, `flatten_sort_count` and the gated MLP's launches, differentiable in all float
    arguments (forward-mode derivatives are refused).  Both keep the logits in float32; the general path stores gates, hidden and expert rows in x's type, the
    other hidden values in two parts of it (float16: infinite above 65504 in both) and rounds the output."""
    if x.dim() < 1 or router_weight.dim() != 2 or w1.dim() != 3 or w2.dim() != 3:
        raise ValueError("routed_glu_mlp: x (..., d), router_weight (E, d), w1 (E, 2F, d) and w2 (E, d, F)")
    E, d = router_weight.shape
    F = w2.size(2)
    if x.size(-1) != d or w1.shape != (E, 2 * F, d) or w2.shape != (E, d, F) or d == 0 or F == 0:
        raise ValueError("routed_glu_mlp: sizes of x %s, router_weight %s, w1 %s, w2 %s do not fit"
                         % (tuple(x.shape), tuple(router_weight.shape), tuple(w1.shape), tuple(w2.shape)))
    if (b1 is not None and b1.shape != (E, 2 * F)) or (b2 is not None and b2.shape != (E, d)):
        raise ValueError("routed_glu_mlp: biases are (E, 2F) and (E, d)")
    if not 0 < k <= min(E, 64) or E > 512:
        raise ValueError("routed_glu_mlp: k must be in 1..min(num_experts, 64), and there are at most 512 experts")
    trained = x.requires_grad
    for t in (router_weight, w1, w2, b1, b2):
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError("routed_glu_mlp: dtype mismatch (%s vs %s)" % (x.dtype, t.dtype))
        if t.device != x.device:
            raise RuntimeError("routed_glu_mlp: all tensors on the device of x (%s)" % x.device)
        trained = trained or t.requires_grad
    tokens = x.reshape(-1, d)
    T = tokens.size(0)
    trained = trained and torch.is_grad_enabled()
    if T == 0 and not trained:
        return x.new_empty(x.shape), x.new_empty((0, E), dtype=torch.float32)
    act = ops.ACT_SILU_GATE_FIRST if gate_first else ops.ACT_SILU
    streams = w1.stride(2) == 1 and w2.stride(2) == 1
    if (ops.few_tokens_pay(T, k, E, d, F, x.dtype, streams) and not trained
            and not ops.has_tangents(x, router_weight, w1, w2, b1, b2)):
        out, logits = ops.routed_glu_mlp(tokens, router_weight, w1, b1, w2, b2, k, act, renormalize)
        return out.view(x.shape), logits
    with torch.autocast(x.device.type, enabled=False):               # (it would take this product, and no other here, to 16 bits)
        logits = nn.functional.linear(tokens.float(), router_weight.float())
    gates, experts = ops.topk_softmax(logits, k, renormalize)
    eid, idx, off = flatten_sort_count(experts, num_experts=E)
    out = _GatedMLP.apply(tokens, w1.permute(0, 2, 1), b1, w2.permute(0, 2, 1), b2, gates.to(x.dtype), eid, idx, off, k, act)
    return out.view(x.shape), logits


class RoutedGLUMLP(GLUMLP):
    """GLUMLP with its router: forward(x) -> (output, router logits).  State-dict keys of GLUMLP and `router.weight`."""

    def __init__(self, input_size, hidden_size, num_experts, top_k, bias=False, renormalize=True):
        super().__init__(input_size, hidden_size, num_experts, top_k, bias=bias)
        self.router = nn.Linear(input_size, num_experts, bias=False)
        self.renormalize = renormalize

    def forward(self, x: torch.Tensor):
        if self.checkpoint_8bit and torch.is_grad_enabled():
            raise ValueError("RoutedGLUMLP: checkpoint_8bit goes with GLUMLP")
        return routed_glu_mlp(x, self.router.weight, self.experts.weight, self.output_experts.weight, self.top_k,
                              b1=self.experts.bias, b2=self.output_experts.bias, renormalize=self.renormalize)
