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
