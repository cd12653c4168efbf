"""What the 8-bit entry points refuse, before anything reaches a GPU, and what the C entry points say of bad calls."""
import ctypes

import pytest
import torch

from scattermoe_amd import _C, eight_bit
from scattermoe_amd.mlp import GLUMLP, MLP

Q8, S8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _w(E, N, K, scales=S8):
    return torch.zeros(E, N, -(-K // 16) * 16).to(Q8), torch.ones(E, -(-N // 128), -(-K // 128)).to(scales)


def _linear(x=None, w=None, s=None, k=2, idx=None, off=None, **kw):
    a, b = _w(3, 40, 20)
    x = torch.zeros(4, 20) if x is None else x
    idx = torch.arange(8) if idx is None else idx
    return eight_bit.parallel_linear_8bit(x, a if w is None else w, b if s is None else s, k, idx, idx,
                                          torch.tensor([2, 4, 8]) if off is None else off, **kw)


def test_linear_refuses():
    for kw in (dict(x=torch.zeros(4, 33)), dict(x=torch.zeros(4, 16)), dict(x=torch.zeros(20)), dict(k=3), dict(off=torch.zeros(2, dtype=torch.int64)),
               dict(w=_w(3, 40, 33)[0]), dict(s=torch.ones(3, 2, 1).to(S8)), dict(grouped_in=True), dict(expert_biases=torch.zeros(3, 41)),
               dict(gates=torch.zeros(4, 3)), dict(gates=torch.zeros(4, 2), grouped_out=True), dict(weight_t=_w(3, 20, 41)[0].new_zeros(3, 20, 64))):
        with pytest.raises(ValueError):
            _linear(**kw)
    for kw in (dict(x=torch.zeros(4, 20, dtype=torch.float64)), dict(w=torch.zeros(3, 40, 32)), dict(s=torch.ones(3, 1, 1, dtype=torch.bfloat16)),
               dict(w=torch.zeros(3, 40, 32).to(torch.float8_e5m2)), dict(expert_biases=torch.zeros(3, 40, dtype=torch.bfloat16)),
               dict(weight_t=torch.zeros(3, 20, 48))):
        with pytest.raises(TypeError):
            _linear(**kw)
    with pytest.raises(ValueError, match="weight_t"):
        _linear(x=torch.zeros(4, 20, requires_grad=True))
    with pytest.raises(ValueError, match="constant"):
        _linear(expert_biases=torch.zeros(3, 40, requires_grad=True))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        _linear()
    with pytest.raises(RuntimeError, match="device"):
        _linear(x=torch.zeros(4, 20, device="meta"))


def _layer(x=None, p=None, ids=None, w1=None, w2=None, **kw):
    a, sa = _w(3, 24, 20)
    b, sb = _w(3, 20, 12)
    return eight_bit.glu_mlp_8bit(torch.zeros(4, 20) if x is None else x, torch.zeros(4, 2) if p is None else p,
                                  torch.zeros(4, 2, dtype=torch.int64) if ids is None else ids, a if w1 is None else w1, sa, b if w2 is None else w2,
                                  sb, **kw)


def test_layer_refuses():
    for kw in (dict(x=torch.zeros(5, 20)), dict(x=torch.zeros(4, 19, 2)), dict(p=torch.zeros(4, 3)), dict(ids=torch.zeros(8, dtype=torch.int64)),
               dict(w1=_w(3, 40, 20)[0]), dict(w1=_w(3, 23, 20)[0]), dict(w2=_w(3, 20, 33)[0]), dict(b1=torch.zeros(3, 12)), dict(b2=torch.zeros(2, 20)),
               dict(ids=torch.zeros(4, 0, dtype=torch.int64), p=torch.zeros(4, 0))):
        with pytest.raises(ValueError):
            _layer(**kw)
    with pytest.raises(TypeError):
        _layer(x=torch.zeros(4, 20, dtype=torch.float64))
    with pytest.raises(TypeError):
        _layer(b1=torch.zeros(3, 24, dtype=torch.float16))
    with pytest.raises(ValueError, match="w1_t"):
        _layer(x=torch.zeros(4, 20, requires_grad=True))
    with pytest.raises(ValueError, match="constant"):
        _layer(b2=torch.zeros(3, 20, requires_grad=True))


def test_blocks_and_units_refuse():
    with pytest.raises(ValueError):
        eight_bit.quantize_blocks(torch.zeros(3, 4), 64)
    with pytest.raises(ValueError):
        eight_bit.quantize_blocks(torch.zeros(3, 4), 128)
    with pytest.raises(ValueError):
        eight_bit.quantize_blocks(torch.zeros(3, 4), transposed=True)
    q, s = torch.zeros(3, 32).to(Q8), torch.ones(3, 1).to(S8)
    for kw in (dict(size=33), dict(size=-1), dict(block_rows=2), dict(block_rows=128)):
        with pytest.raises(ValueError):
            eight_bit.dequantize_blocks(q, s, **kw)
    with pytest.raises(ValueError):
        eight_bit.dequantize_blocks(q, torch.ones(3, 2).to(S8))
    with pytest.raises(TypeError):
        eight_bit.dequantize_blocks(q, torch.ones(3, 1, dtype=torch.float16))
    with pytest.raises(ValueError):
        eight_bit.checkpointed_glu(torch.zeros(4, 5))
    with pytest.raises(TypeError):
        eight_bit.checkpointed_glu(torch.zeros(4, 6, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        eight_bit.checkpointed_glu(torch.zeros(4, 6, requires_grad=True))
    with pytest.raises(ValueError, match="SiLU"):
        eight_bit.GLUMLP8bit.from_module(MLP(8, 8, 2, 1, activation=torch.nn.GELU()))
    with pytest.raises(TypeError):
        eight_bit.GLUMLP8bit(8, 8, 2, 1, scale_type=torch.float16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        eight_bit.GLUMLP8bit.from_module(GLUMLP(8, 8, 2, 1))


def test_module_keeps_its_weights_whatever_type_it_is_taken_to():
    m = eight_bit.GLUMLP8bit(40, 24, 3, 2, bias=True, input_gradients=True).to(torch.float16)
    assert m.w1.dtype == m.w2_t.dtype == Q8 and m.s1.dtype == S8 and m.b1.dtype == torch.float16
    assert m.w1.shape == (3, 48, 48) and m.w2.shape == (3, 40, 32) and m.w1_t.shape == (3, 40, 48) and m.w2_t.shape == (3, 24, 48)
    m = eight_bit.GLUMLP8bit(40, 24, 3, 2, scale_type=torch.float32).half()
    assert m.s1.dtype == torch.float32 and m.w1_t is None and m.b1 is None
    other = eight_bit.GLUMLP8bit(40, 24, 3, 2, scale_type=torch.float32)
    m.s1.fill_(2.0)
    other.load_state_dict(m.state_dict())
    assert float(other.s1.sum()) == 2.0 * other.s1.numel()
    assert not list(m.parameters())


def test_linear_of_no_columns_is_refused():
    with pytest.raises(ValueError):
        _linear(w=torch.zeros(3, 0, 32, dtype=torch.uint8).view(Q8), s=torch.zeros(3, 0, 1, dtype=torch.uint8).view(S8))


def test_gated_layer_with_its_checkpoint_is_a_silu_one():
    with pytest.raises(ValueError, match="SiLU"):
        GLUMLP(8, 8, 2, 1, activation=torch.nn.GELU(), checkpoint_8bit=True)
    assert GLUMLP(8, 8, 2, 1, checkpoint_8bit=True).checkpoint_8bit and not GLUMLP(8, 8, 2, 1).checkpoint_8bit


def test_c_entry_points_name_bad_calls():
    lib = _C.load()
    one, zero = ctypes.c_void_p(256), None
    w = _C.Weight8bit(256, 4096, 256, 1, 1, 1, 0)
    bad = _C.Weight8bit(256, 4088, 256, 1, 1, 1, 0)
    none = _C.Weight8bit(256, 4096, None, 1, 1, 1, 0)
    assert lib.smoe_row_8bit_bytes(17) == 32 and lib.smoe_row_8bit_scales(129) == 4 and lib.smoe_row_8bit_scales(513) == 8
    assert lib.smoe_quantize_rows(zero, 0, 4, 4, one, one, _C.BF16, None) == -1
    assert lib.smoe_quantize_rows(one, 0, -1, 4, one, one, _C.BF16, None) == -2
    assert lib.smoe_quantize_rows(one, 0, 4, 4, one, one, 7, None) == -3
    assert lib.smoe_quantize_rows(one, 0, 4, 1 << 31, one, one, 0, None) == -5
    assert lib.smoe_quantize_rows(one, 0, 4, 4, ctypes.c_void_p(264), one, 0, None) == -2
    assert lib.smoe_quantize_rows(zero, 0, 0, 4, zero, zero, _C.BF16, None) == 0
    assert lib.smoe_quantize_weights(zero, 0, 0, 1, 1, 1, one, zero, one, 0, None) == -1
    assert lib.smoe_dequantize_8bit(one, 0, 0, one, 0, 0, 0, 0, 64, 1, 1, 1, one, 0, None) == -2
    assert lib.smoe_glu_8bit_fwd(one, 8, one, zero, one, 4, 4, 0, 0, None) == -1
    assert lib.smoe_glu_8bit_fwd(one, 8, one, one, one, 4, 4, 5, 0, None) == -2
    assert lib.smoe_glu_8bit_bwd(one, one, zero, 4, one, zero, 4, 4, 0, 0, None) == -1

    def linear(weight=w, L=8, k=2, ws=one, size=1 << 20, coeff=zero, grouped=0, dtype=_C.BF16, x=one):
        return lib.smoe_linear_8bit(x, 64, coeff, weight, 0, zero, 0, 0, one, 64, one, one, L, 64, 64, 2, k, grouped, 0, dtype, ws, size, None)

    assert linear(x=zero) == -1 and linear(L=7) == -2 and linear(k=0) == -2 and linear(dtype=9) == -3
    assert linear(weight=bad) == -2 and b"16 bytes" in lib.smoe_last_error()
    assert linear(weight=none) == -1 and linear(coeff=one, grouped=1) == -2
    need = lib.smoe_linear_8bit_workspace_bytes(8, 64, 64, 2, 2, 0, 0, _C.BF16)
    assert need == 1024 and lib.smoe_linear_8bit_workspace_bytes(8, 64, 64, 2, 2, 0, 1, _C.BF16) == 1536
    assert linear(size=need - 1) == -4 and linear(ws=zero) == -4 and linear(ws=ctypes.c_void_p(264)) == -4
    assert linear(L=1 << 32) == -5 and linear(L=0) == 0
    assert linear(weight=_C.Weight8bit(256, 4096, 256, 1, 1 << 28, 1, 0)) == -5 and linear(weight=_C.Weight8bit(256, 4096, 256, 1, 1, -1, 0)) == -5
    for K, N in (((1 << 21) + 1, 64), (64, (1 << 21) + 1)):
        assert lib.smoe_linear_8bit(one, K, zero, w, 0, zero, 0, 0, one, N, one, one, 8, K, N, 2, 2, 0, 0, _C.BF16, one, 1 << 40, None) == -5

    def layer(T=4, k=2, p8=zero, ps=zero, ws=one, size=1 << 24, act=0, idx=one):
        return lib.smoe_glu_mlp_8bit(one, 64, one, one, w, zero, 0, 0, w, zero, 0, 0, one, one, p8, ps, idx, one, T, k, 64, 64, 2, act, _C.BF16, ws, size, None)

    assert layer(k=0) == -2 and layer(act=9) == -2 and layer(p8=one) == -1 and layer(idx=zero, T=33) == -1 and layer(T=1 << 32) == -5 and layer(T=0) == 0
    assert layer(size=lib.smoe_glu_mlp_8bit_workspace_bytes(4, 2, 64, 64, 2, 1, 0, _C.BF16) - 1) == -4

    def back(T=4, k=2, ws=one, size=1 << 24, p8=one):
        return lib.smoe_glu_mlp_8bit_bwd(one, 64, one, w, w, p8, one, one, one, one, one, T, k, 64, 32, 2, 0, _C.BF16, ws, size, None)

    assert back(k=0) == -2 and back(p8=zero) == -1 and back(T=0) == 0
    assert back(size=lib.smoe_glu_mlp_8bit_bwd_workspace_bytes(4, 2, 64, 32, 2, _C.BF16) - 1) == -4
