"""Which launches a call of the adapters makes, asked of the launchers' own rules: a host-only build of their sources (no GPU, no
device code) that notes launches instead of making them."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from scattermoe_amd import _C, _build

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
    """How a float32 product goes, and whether a weight or factor is copied."""
    names = [who + kernel for who, kernel, _, _ in found]
    if any("adapter_runs_f32_kernel" in n for n in names):
        assert "adapter_runs_join_f32_kernel" in names[-1]
        how = "runs"
    else:
        how = ([int(re.search(r"SIDE = (\d+)", n).group(1)) for n in names if "adapter_tiles_f32_kernel" in n] or ["rows"])[0]
    return how, any("pack" in n for n in names)


@pytest.mark.parametrize("T,K,N,want,want_back", [
    (64, 4096, 4096, "rows", "rows"), (65, 4096, 4096, "runs", "runs"), (128, 1024, 1024, "rows", "rows"), (128, 2048, 2048, "rows", "runs"),
    (256, 4096, 4096, 64, 64), (320, 4096, 4096, "runs", "runs"), (512, 2048, 2048, 64, 64), (1024, 512, 512, "rows", "rows"),
    (203, 1003, 1517, "rows", "rows"), (1024, 1472, 2064, "runs", "runs"), (1024, 4096, 4096, 128, 128), (4096, 4096, 4096, 128, 128),
    (2048, 1536, 2000, 128, 64), (300, 4, 4, "rows", 64)])
def test_float32_products(launches, T, K, N, want, want_back):
    """The rows' kernel reads all weights per 32 rows (1024 rows, 4096 -> 4096 509 us where an elementary product takes 281), and a few tiles more than
    whole rounds of them took a round more."""
    assert _f32(launches(T, K, N, 16, 8, 0)) == (want, False)
    how, copied = _f32(launches(T, K, N, 16, 8, 0, True))
    assert how == want_back and copied


def test_float32_runs_have_their_parts_in_the_workspace(launches):
    """512 runs of slices of 64 x 64 tiles leave at most two parts each."""
    lib = _C.load()
    size = lambda T, back: lib.smoe_adapter_workspace_bytes(T, 4096, 4096, 16, 8, back, 0)
    assert min(size(320, 0) - size(1024, 0), size(320, 1) - size(1024, 1)) > 0 and min(size(320, 0), size(320, 1)) >= 2 * 512 * 64 * 64 * 4
