"""vectors_b200: the integrallis/vectors batch distance + top-k scan on NVIDIA B200 (sm_100a).

The scans (FLAT exact search, the SQ8 / FP16 / sign-bit BQ quantized scans and the IVF-PQ ADC
list scan) run as hand-written CUDA kernels in ``libvx.so``; this package is the host-side
mirror of the reference's index SPI over that library's C ABI (include/vx.h).
"""
import sys as _sys

from ._native import VxError, device_count, kernel_launches, lib  # noqa: F401
from .index_spi import (  # noqa: F401
    FlatScanAdapter,
    GpuUnavailableException,
    IOException,
    IllegalArgumentException,
    IndexSpi,
    IvfFlatAdapter,
    IvfPqAdapter,
    NullPointerException,
    QuantizedFlatScanAdapter,
    SearchOutcome,
    SimilarityFunction,
    UnsupportedOperationException,
    ivf_graph_info,
    merge_shards_device,
    quantized_bin_info,
    shard_offsets,
)

__all__ = [
    "FlatScanAdapter",
    "QuantizedFlatScanAdapter",
    "IvfPqAdapter",
    "IvfFlatAdapter",
    "IndexSpi",
    "SearchOutcome",
    "SimilarityFunction",
    "IllegalArgumentException",
    "NullPointerException",
    "GpuUnavailableException",
    "UnsupportedOperationException",
    "IOException",
    "quantized_bin_info",
    "ivf_graph_info",
    "merge_shards_device",
    "shard_offsets",
    "fp8_check",
    "fp8_empty",
    "fp8_pitch",
    "fp8_read_device",
    "fp8_scores_device",
    "fp8_scores_grouped_device",
    "fp8_write_device",
    "device_count",
    "kernel_launches",
    "lib",
    "VxError",
]

_FP8 = frozenset(n for n in __all__ if n.startswith("fp8_"))


def __getattr__(name):
    """The 8-bit row functions (fp8.py) work on torch tensors.  Where torch is not imported yet, each is a
    stand-in that imports it when called: a star import needs no torch and loads none."""
    if name not in _FP8:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    if _sys.modules.get("torch") is None:

        def call(*args, **kwargs):
            from . import fp8

            return getattr(fp8, name)(*args, **kwargs)

        call.__name__ = call.__qualname__ = name
        call.__doc__ = f"``{__name__}.fp8.{name}``, which imports torch."
        return call
    from . import fp8

    globals().update({n: getattr(fp8, n) for n in _FP8})
    return globals()[name]
