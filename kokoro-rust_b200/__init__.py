"""kokoro-b200: B200-native batched ragged Kokoro-82M forward behind a C ABI.

The compute lives in ``libkokoro_b200.so`` (CUDA for sm_100a, built from ``csrc/``); this package
holds the host-side mirror of the reference engine API (``engine``), WAV output (``wav``), the
checkpoint manifest and seeded random-init generator (``weights``) and the build step (``build``).
``fp8`` (the 8-bit operators on torch tensors) is imported when it is first named, since it alone
needs torch.
"""
from . import multi, pth, shard, wav, weights  # noqa: F401
from .engine import (BatchItem, BatchPolicy, Engine, GpuKokoro, ItemNoise, KokoroError, Output, Synth, Voice,
                     load_library, mix_seed, plan_batches)

__all__ = ["BatchItem", "BatchPolicy", "Engine", "GpuKokoro", "ItemNoise", "KokoroError", "Output", "Synth",
           "Voice", "load_library", "mix_seed", "plan_batches"]


def __getattr__(name):
    if name == "fp8":
        import importlib

        return importlib.import_module(".fp8", __name__)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
