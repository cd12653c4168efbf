"""How calls on 8 bits go about their rows, asked of the C entry points themselves: a host-only build of their source (no GPU, no device code) in
which the launching functions note what they are asked for instead of launching it."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from scattermoe_amd import _C, _build

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")

# A line per launch: what it is, and of the rows in 8 bits how many there are (quantize), whether they are copied in the experts'
# order (copies), whether the product takes them as they lie (grouped) and what a row number is divided by on a look-up (fan).
SOURCE = """
#include <hip/hip_runtime.h>
#include <string>
static std::string noted;
static void note(const char* what, int64_t a, int64_t b) {
  noted += std::string(what) + " " + std::to_string(a) + " " + std::to_string(b) + "\\n";
}
#include "%(csrc)s/capi_8bit.hip"
namespace smoe {
int launch_status(const char*) { return 0; }
void set_error(const char*, ...) {}
int launch_quantize_rows(const QuantRowsArgs& a, int, hipStream_t) { note("quantize", a.slots, a.idx != nullptr); return 0; }
int launch_quantize_weights(const QuantWeightsArgs&, int, hipStream_t) { return 0; }
int launch_dequantize(const DequantArgs&, int, hipStream_t) { return 0; }
int launch_unit_fwd(const UnitArgs&, int, hipStream_t) { note("unit", 0, 0); return 0; }
int launch_unit_bwd(const UnitBackArgs&, int, hipStream_t) { note("unit", 0, 0); return 0; }
int64_t product_8bit_floats(int64_t, int64_t, int64_t, int, bool) { return 0; }
bool unit_rides(int64_t, int64_t F) { return F %% 32 == 0; }
bool unit_grad_rides(int64_t F) { return F %% 128 == 0; }
int launch_product_8bit(const Product8Args& a, bool exact, int, int, hipStream_t, int) {
  note(exact ? "exact" : "product", a.x_grouped, a.fan);
  return 0;
}
int launch_few_rows_8bit(const Few8Args& a, int, int, int, hipStream_t) { note("stream", a.x_grouped, a.fan); return 0; }
int launch_few_combine(const float*, const void*, const int64_t*, void*, int, int, int, int, int, hipStream_t) { return 0; }
int launch_slots_combine(const float*, int64_t, const void*, int64_t, int64_t, const int64_t*, int, void*, int64_t, int64_t, int, int, int, hipStream_t) {
  return 0;
}
int launch_slots_gate_grad(const float*, int64_t, const void*, int64_t, void*, int64_t, int64_t, int64_t, int, int, int, hipStream_t) { return 0; }
}
extern "C" const char* noted_launches() { return noted.c_str(); }
extern "C" void forget_launches() { noted.clear(); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("eight_bit")
    src, so = d / "calls.hip", d / "calls.so"
    src.write_text(SOURCE % {"csrc": _build.CSRC})
    subprocess.run([_build._hipcc(), "--cuda-host-only", "-x", "hip", "-std=c++17", "-O1", "-fPIC", "-shared",
                    "-Wno-unused-command-line-argument", "-o", str(so), str(src)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.noted_launches.restype = ctypes.c_char_p
    for name, (restype, argtypes) in _C._SIGNATURES.items():
        if "8bit" in name:
            getattr(lib, name).restype, getattr(lib, name).argtypes = restype, argtypes
    return lib


ONE, WS, SIZE = ctypes.c_void_p(256), ctypes.c_void_p(1 << 20), 1 << 46
WEIGHT = _C.Weight8bit(256, 4096, 256, 1, 1, 1, 0)


def _noted(lib, rc):
    assert rc == 0
    found = [(w, int(a), int(b)) for w, a, b in re.findall(r"(\w+) (\d+) (\d+)", lib.noted_launches().decode())]
    lib.forget_launches()
    return found


def _forward(lib, T, k, d, F, E, dtype=_C.BF16):
    return _noted(lib, lib.smoe_glu_mlp_8bit(ONE, d, ONE, None, WEIGHT, None, 0, 0, WEIGHT, None, 0, 0, ONE, ONE, None, None, ONE, ONE, T, k, d, F, E, 0,
                                             dtype, WS, SIZE, None))


def _backward(lib, T, k, d, F, E, dtype=_C.BF16):
    return _noted(lib, lib.smoe_glu_mlp_8bit_bwd(ONE, d, ONE, WEIGHT, WEIGHT, ONE, ONE, ONE, ONE, ONE, ONE, T, k, d, F, E, 0, dtype, WS, SIZE, None))


def _linear(lib, T, k, K, N, E, scaled=False, dtype=_C.BF16):
    return _noted(lib, lib.smoe_linear_8bit(ONE, K, ONE if scaled else None, WEIGHT, 0, None, 0, 0, ONE, N, ONE, ONE, T * k, K, N, E, k, 0, 0, dtype,
                                            WS, SIZE, None))


def _rows_and_product(found, looked_up, copied):
    """The first pair of launches, as rows that are looked up want them, or as rows that were copied in the experts' order do."""
    (_, rows, copies), (what, grouped, fan) = found[:2]
    assert [f[0] for f in found[:2]] == ["quantize", what] and what in ("product", "stream")
    if grouped:
        assert copies and rows == copied
    else:
        assert not copies and rows == looked_up[0] and fan == looked_up[1]
    return bool(grouped)


# Rows of 4096 bytes pass what a look-up's 32-bit offsets hold at 2^20 of them.
@pytest.mark.parametrize("T,k,copied", [(1 << 19, 1, False), ((1 << 20) - 1, 1, False), (1 << 20, 1, True), ((1 << 20) + 64, 1, True),
                                        (1 << 19, 2, False), ((1 << 20) - 1, 2, False), (1 << 20, 2, True), (1 << 18, 8, False)])
def test_tokens_are_copied_where_a_look_up_would_not_reach_them(lib, T, k, copied):
    for d in (4096, 4000):                                            # (rows in a workspace are whole blocks of 128)
        d_copied = copied and (T * (-(-d // 128) * 128) >= 1 << 32)
        assert _rows_and_product(_forward(lib, T, k, d, 128, 8), (T, k), T * k) == d_copied
        assert _rows_and_product(_linear(lib, T, k, d, 64, 8), (T, k), T * k) == d_copied


@pytest.mark.parametrize("T,k,copied", [((1 << 20) - 1, 1, False), (1 << 20, 1, True), ((1 << 19) - 1, 2, False), (1 << 19, 2, True), (1 << 17, 8, True)])
def test_scaled_rows_are_copied_where_a_look_up_would_not_reach_them(lib, T, k, copied):
    assert _rows_and_product(_backward(lib, T, k, 4096, 128, 8), (T * k, 1), T * k) == copied
    assert _rows_and_product(_linear(lib, T, k, 4096, 64, 8, scaled=True), (T * k, 1), T * k) == copied


def test_streams_over_the_weights_look_tokens_up_too(lib):
    found = _forward(lib, 40, 1, 128, 128, 64)
    assert found[1][0] == "stream" and not _rows_and_product(found, (40, 1), 40)


def _kinds(found):
    return [f[0] for f in found if f[0] in ("stream", "exact", "product")]


def test_products_whose_results_go_to_8_bits_again_are_exact_of_more_bits_than_bfloat16(lib):
    """The first of a layer and the first of its backward pass; streams, which are exact, take up to 16 rows per expert then."""
    for dtype, first, other in ((_C.BF16, "product", "product"), (_C.F16, "exact", "product"), (_C.F32, "exact", "exact")):
        for F in (128, 96, 72):                                         # with the unit behind the product, and its gradient, or without
            assert _kinds(_forward(lib, 4096, 2, 128, F, 8, dtype)) == [first, other]
            assert _kinds(_backward(lib, 4096, 2, 128, F, 8, dtype)) == [first, other]
        for E, k in ((8, 2), (32, 4)):
            for per, few in ((4, True), (5, first == "exact"), (16, first == "exact"), (17, False)):
                assert _kinds(_forward(lib, per * E // k, k, 128, 128, E, dtype)) == (["stream"] * 2 if few else [first, other])
        # a product's own result is rounded to the rows' type: float16 costs 16 times the instruction's sums
        assert _kinds(_linear(lib, 4096, 2, 128, 128, 8, dtype=dtype)) == [other]
