"""What the passes over a token's float32 rows refuse before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

from scattermoe_amd import _C
from scattermoe_amd.kernels import ops


def test_c_entry_points_name_bad_calls():
    lib = _C.load()
    one, zero = ctypes.c_void_p(256), None

    def combine(y=one, experts=zero, E=0, T=4, k=2, N=8, dtype=_C.BF16):
        return lib.smoe_combine_f32(y, 8, one, 2, 1, experts, E, one, 8, T, k, N, dtype, None)

    def gate_grad(y=one, T=4, k=2, N=8, dtype=_C.BF16):
        return lib.smoe_gate_grad_f32(y, 8, one, 8, one, 2, 1, T, k, N, dtype, None)

    for call in (combine, gate_grad):
        assert call(dtype=5) == -3 and call(T=-1) == -2 and call(k=0) == -2 and call(N=-1) == -2 and call(T=1 << 31) == -5 and call(N=1 << 31) == -5
        assert call(y=zero) == -1 and b"NULL" in lib.smoe_last_error() and call(T=0) == 0
    assert combine(experts=one) == -2 and combine(N=0) == 0 and gate_grad(T=1 << 30, k=4) == -5


def test_rows_of_another_type_are_float32():
    rows = torch.zeros(3, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="mismatch"):
        ops.combine(rows, dtype=torch.float16)
    with pytest.raises(TypeError, match="mismatch"):
        ops.gate_grad(rows, torch.zeros(3, 8, dtype=torch.float16))
    for call in (lambda: ops.combine(rows.float(), dtype=torch.float16), lambda: ops.gate_grad(rows.float(), torch.zeros(3, 8, dtype=torch.float16))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_workspace_of_float32_rows():
    """The same bytes whether or not the product's rows come out in float32, however the caller asks for them."""
    lib = _C.load()
    for dtype in (_C.F32, _C.BF16, _C.F16):
        for L, K, N, E in ((8, 64, 64, 2), (300, 16384, 256, 2), (300, 9000, 9000, 4)):
            plain, floats = (lib.smoe_linear_8bit_workspace_bytes(L, K, N, E, 1, 0, 0, d) for d in (dtype, dtype | _C.Y_FLOAT32_8BIT))
            assert plain == floats > 0
