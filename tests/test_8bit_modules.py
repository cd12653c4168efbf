"""`GLUMLP8bit` and `GLUMLP` with its checkpoint in 8 bits: what their construction and their use refuse (no GPU)."""
import pytest
import torch

from scattermoe_amd import eight_bit
from scattermoe_amd.mlp import GLUMLP, MLP


@pytest.mark.parametrize("hidden", [8, 16, 64])
def test_an_ungated_layer_is_no_gated_one(hidden):
    """Its first weights have half the rows, and where both widths round up to the same 16 bytes its copy would run as a gated layer."""
    with pytest.raises(ValueError, match="gated"):
        eight_bit.GLUMLP8bit.from_module(MLP(32, hidden, 2, 1, activation=torch.nn.SiLU()))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        eight_bit.GLUMLP8bit.from_module(GLUMLP(32, hidden, 2, 1))
