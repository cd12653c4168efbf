"""`GLUMLP8bit` and `GLUMLP` with its checkpoint in 8 bits: what their construction and their use refuse (no GPU)."""
import pytest
import torch

from scattermoe_amd import eight_bit
from scattermoe_amd.kernels import ops
from scattermoe_amd.mlp import GLUMLP, MLP, RoutedGLUMLP


@pytest.mark.parametrize("hidden", [8, 16, 64])
def test_an_ungated_layer_is_no_gated_one(hidden):
    """Its first weights have half the rows, and where both widths round up to the same 16 bytes its copy would run as a gated layer."""
    with pytest.raises(ValueError, match="gated"):
        eight_bit.GLUMLP8bit.from_module(MLP(32, hidden, 2, 1, activation=torch.nn.SiLU()))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        eight_bit.GLUMLP8bit.from_module(GLUMLP(32, hidden, 2, 1))


def test_a_checkpoint_that_a_layer_cannot_keep_is_refused_where_it_would_be():
    m = GLUMLP(8, 16, 2, 1, checkpoint_8bit=True)
    x, p, ids = torch.zeros(3, 8), torch.ones(3, 1), torch.zeros(3, 1, dtype=torch.int64)
    m.activation = torch.nn.GELU()
    with pytest.raises(ValueError, match="SiLU"):
        m(x, p, ids)
    r = RoutedGLUMLP(8, 16, 2, 1)
    r.checkpoint_8bit = True
    with pytest.raises(ValueError, match="checkpoint_8bit"):
        r(x)
    with torch.no_grad():                                             # (nothing is kept: on to the kernels)
        for call in (lambda: m(x, p, ids), lambda: r(x)):
            with pytest.raises(RuntimeError, match="ROCm GPU"):
                call()


def test_weights_whose_experts_lie_apart_are_taken_where_they_are():
    """Every second expert of a checkpoint's, one expert for all, the last ones, one alone; a weight whose rows lie apart is copied."""
    E, N, K = 6, 40, 32
    full = torch.zeros(2 * E, N, K, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(E, 1, 1)
    for q in (full[::2], full[:1].expand(E, N, K), full[E:], full.view(torch.uint8).as_strided((E, N, K), (N * K + 48, K, 1)).view(full.dtype)):
        got, _, t = eight_bit._weight("call", "w", q, s, q.device, E, N, K)
        assert got.data_ptr() == q.data_ptr() and got.stride() == q.stride() and t is None
    one = full.view(torch.uint8).as_strided((1, N, K), (7, K, 1)).view(full.dtype)
    held = ops._weight_8bit(eight_bit._weight("call", "w", one, s[:1], one.device, 1, N, K)[0], s[:1])
    assert held.q == one.data_ptr() and held.q_expert % 16 == 0
    for q in (full[:E].transpose(1, 2).contiguous().transpose(1, 2), full.view(torch.uint8).as_strided((E, N, K), (N * K + 8, K, 1)).view(full.dtype),
              full.view(torch.uint8).as_strided((E, N, K), (N * 2 * K, 2 * K, 1)).view(full.dtype)):
        assert eight_bit._weight("call", "w", q, s, q.device, E, N, K)[0].stride() == (N * K, K, 1)


def test_casting_a_module_does_not_cast_its_weights_on_the_way():
    m = eight_bit.GLUMLP8bit(64, 48, 3, 2, bias=True, input_gradients=True)
    keys, seen = list(m.state_dict()), []

    def cast(t):
        seen.append((t.dtype, t.numel()))
        return t.to(torch.float16)

    held = {n: getattr(m, n) for n in m._held}
    m._apply(cast)
    assert all(n == 0 for dtype, n in seen if dtype not in (torch.bfloat16,))
    assert m.b1.dtype == torch.float16 and all(getattr(m, n) is t for n, t in held.items()) and list(m.state_dict()) == keys
    # what is no cast reaches them: another device, memory of their own
    m = m.to("meta")
    assert all(getattr(m, n).device.type == "meta" and getattr(m, n).dtype == t.dtype for n, t in held.items())
    m = m.to_empty(device="cpu")
    assert all(getattr(m, n).shape == t.shape and getattr(m, n).device.type == "cpu" for n, t in held.items())
    n = eight_bit.GLUMLP8bit(64, 48, 3, 2, scale_type=torch.float32).to("meta", torch.float16)
    assert n.w1.device.type == n.s1.device.type == "meta" and n.s1.dtype == torch.float32 and n.w1.dtype == m.w1.dtype and n.w1_t is None
