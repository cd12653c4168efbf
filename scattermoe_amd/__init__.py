"""scattermoe_amd — ScatterMoE for MI355X (gfx950): the Python surface of shawntan/scattermoe over
hand-written HIP kernels (reference package root: scattermoe/__init__.py:1-15)."""
import os

from .parallel_experts import flatten_sort_count, flatten_and_sort, parallel_linear, ParallelExperts
from . import parallel_experts
from . import kernels
from . import mlp
from . import adapters
from .adapters import parallel_adapters, ParallelAdapters
from . import eight_bit
from .eight_bit import parallel_linear_8bit, GLUMLP8bit

if os.environ.get("SCATTERMOE_NO_HF_PATCH", "0") != "1":
    from . import utils
else:  # the submodule stays importable on demand; only the import-time Hugging Face patching is skipped
    utils = None

__all__ = [
    "flatten_sort_count",
    "flatten_and_sort",
    "parallel_linear",
    "ParallelExperts",
    "parallel_experts",
    "kernels",
    "mlp",
    "adapters",
    "parallel_adapters",
    "ParallelAdapters",
    "eight_bit",
    "parallel_linear_8bit",
    "GLUMLP8bit",
    "utils",
]
