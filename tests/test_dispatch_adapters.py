"""Which launches a call of the adapters makes, asked of the launchers' own rules: a host-only build of their sources (no GPU, no
device code) that notes launches instead of making them."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from scattermoe_amd import _build

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")

SOURCE = """
#include <hip/hip_runtime.h>
#include <string>
static std::string launched;
static void note(const char* from, const char* kernel, unsigned x, unsigned y) {
  launched += std::string(from) + " / " + kernel + " / " + std::to_string(x) + " / " + std::to_string(y) + "\\n";
}
#undef __global__
#define __global__ static __device__ __attribute__((unused))
#undef __launch_bounds__
#define __launch_bounds__(...)
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kernel, grid, ...) note(__PRETTY_FUNCTION__, #kernel, dim3(grid).x, dim3(grid).y)
%(includes)s
namespace smoe {
int launch_status(const char*) { return 0; }
void set_error(const char*, ...) {}
int launch_route_adapters(const int64_t*, int64_t, int, int64_t*, int64_t*, int64_t*, void*, hipStream_t) { return 0; }
size_t route_workspace_bytes(int64_t, int) { return 256; }
}
using namespace smoe;
static char* at(int64_t offset) { return (char*)0x10000 + offset; }
extern "C" const char* call(int64_t T, int64_t K, int64_t N, int64_t r, int64_t R, int dtype, int back) {
  launched.clear();
  AdapterCall c{};
  c.X = at(0), c.sxm = K, c.W = at(0), c.A = at(0), c.B = at(0);
  c.ids = (int64_t*)at(0), c.idx = (int64_t*)at(0), c.off = (int64_t*)at(0);
  c.U = (float*)at(0), c.Y = at(0), c.DY = at(0);
  if (back) c.DX = at(0);
  c.T = T, c.K = K, c.N = N, c.r = (int)r, c.R = (int)R, c.dtype = dtype;
  if (launch_adapter_call(c, back != 0, at(0), 0)) launched += "refused";
  return launched.c_str();
}
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    d = tmp_path_factory.mktemp("adapters")
    src, lib = d / "rules.hip", d / "rules.so"
    names = [n for n in _build.SOURCES if n.startswith("adapters")]
    src.write_text(SOURCE % {"includes": "\n".join('#include "%s/%s"' % (_build.CSRC, n) for n in names)})
    subprocess.run([_build._hipcc(), "--cuda-host-only", "-x", "hip", "-std=c++17", "-O1", "-fPIC", "-shared",
                    "-Wno-unused-command-line-argument", "-o", str(lib), str(src)], check=True)
    lib = ctypes.CDLL(str(lib))
    lib.call.restype = ctypes.c_char_p

    def ask(T, K, N, r, R, dtype=1, back=False):
        text = lib.call(*(ctypes.c_int64(v) for v in (T, K, N, r, R)), dtype, int(back)).decode()
        return [tuple(line.rsplit(" / ", 3)) for line in text.splitlines()]
    return ask


def _tiles(found):
    """(class, workgroups) of the launches of tiles."""
    return [(int(re.search(r"CLASS = (\d+)", who).group(1)), int(x)) for who, kernel, x, _ in found if "adapter_tiles_kernel" in kernel]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("T", [1, 4, 64, 65, 100, 160, 240, 300, 512, 700, 1024, 4099])
def test_no_launch_is_empty(launches, T, dtype):
    """Widths up to that of a vocabulary, where a row of tiles is more than a round of workgroups."""
    for K in (64, 520, 1024, 4096):
        for N in (64, 1000, 4096, 65536, 65544, 76800, 98304, 128256, 151936, 256000):
            for r, R in ((8, 1), (16, 4), (64, 64)):
                for back in (False, True):
                    found = launches(T, N, K, r, R, dtype, True) if back else launches(T, K, N, r, R, dtype)
                    assert found and "refused" not in found[-1][0]
                    for who, kernel, x, y in found:
                        assert int(x) > 0 and int(y) > 0, (K, N, r, R, back, who, kernel)


def test_one_row_of_tiles_beyond_a_round(launches):
    """A prompt's rows and the columns of a vocabulary: 594 tiles in one row, in one launch."""
    (which,) = _tiles(launches(100, 4096, 151936, 16, 8))
    assert which[0] == 0 and which[1] >= 594
    (which,) = _tiles(launches(100, 1024, 65800, 16, 8))
    assert which[0] == 1 and which[1] >= 258


def _f32(found):
    """The side of the float32 tiles of a call, 0 for the rows' kernel, and whether a weight or factor is copied."""
    side = [int(re.search(r"SIDE = (\d+)", who).group(1)) for who, kernel, _, _ in found if "adapter_tiles_f32_kernel" in kernel]
    return (side or [0])[0], any("pack" in kernel for _, kernel, _, _ in found)


@pytest.mark.parametrize("T,K,N,want,want_back", [
    (64, 4096, 4096, 0, 0), (65, 4096, 4096, 0, 0), (128, 1024, 1024, 0, 0), (128, 4096, 4096, 0, 64), (256, 4096, 4096, 64, 64),
    (512, 2048, 2048, 64, 64), (1024, 512, 512, 0, 0), (203, 1003, 1517, 0, 0), (1024, 1003, 1517, 64, 64), (1024, 2048, 2048, 64, 64),
    (1024, 4096, 4096, 128, 128), (1300, 4096, 4096, 64, 64), (4096, 4096, 4096, 128, 128), (2048, 1536, 2000, 128, 64)])
def test_float32_tiles(launches, T, K, N, want, want_back):
    """The rows' kernel read all weights per 32 rows (1024 rows, 4096 -> 4096 513 us where an elementary product takes 281)."""
    assert _f32(launches(T, K, N, 16, 8, 0)) == (want, False)
    side, copied = _f32(launches(T, K, N, 16, 8, 0, True))
    assert side == want_back and copied
