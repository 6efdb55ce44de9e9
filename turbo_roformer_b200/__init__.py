"""Blackwell (sm_100a) CUDA backend for the BS-RoFormer forward of turbo-roformer.

Public surface (mirrors the reference package): ``Separator`` (backend="cuda"; ``submit`` for queued
songs, ``stream`` for live input), ``CudaBSRoformer`` (the FastBSRoformer-compatible forward), the
chunking helpers, the device channel fold / resampler (``remix_device``, ``resample_device``), and the frame cache
of live input (``cache_plan``, ``cache_append``, ``cache_attention``).
"""

from .chunking import chunk_starts, hamming, overlap_add, step_for
from .config import RESURRECTION, TINY, ModelConfig

__all__ = ["Separator", "SeparationJob", "SeparationStream", "CudaBSRoformer", "ModelConfig", "RESURRECTION", "TINY",
           "chunk_starts", "hamming", "overlap_add", "step_for", "remix_device", "resample_device",
           "CachePlan", "cache_plan", "cache_append", "cache_attention"]


def __getattr__(name):
    if name in ("Separator", "SeparationJob", "SeparationStream"):
        from . import separator

        return getattr(separator, name)
    if name in ("remix_device", "resample_device"):
        from . import resample

        return getattr(resample, name)
    if name in ("CachePlan", "cache_plan", "cache_append", "cache_attention"):
        from . import frame_cache

        value = globals()[name] = getattr(frame_cache, name)  # found at once from now on: a push's calls are short
        return value
    if name == "CudaBSRoformer":
        from .backend import CudaBSRoformer

        return CudaBSRoformer
    raise AttributeError(name)
