"""`GLUMLP8bit` and `GLUMLP` with its checkpoint in 8 bits: what their construction and their use refuse (no GPU)."""
import pytest
import torch

from scattermoe_amd import eight_bit
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
