"""cq35: MI355X-native Qwen3.5/3.6 token loop (hand-written gfx950 HIP
kernels behind a C ABI) with a host API mirroring catena-models' Model /
Session (src/model.rs)."""
import importlib.util
import sys

from .config import PRESETS, bytes_per_token, derived, is_full, preset
from .model import (Model, Session, SessionCheckpoint, decode_batch, gguf_config, gguf_tensor_name, gguf_validate,
                    kernel_classes, read_logits, weight_count, weight_info)
from ._lib import CQ35Error, LIBRARY, load

# decode attention over more cached keys than this runs split-K by default
# (include/cq35.h CQ35_SPLIT_KEYS_DEFAULT)
SPLIT_KEYS_DEFAULT = 8192

__all__ = [
    "PRESETS", "bytes_per_token", "derived", "is_full", "preset", "Model", "Session",
    "SessionCheckpoint", "decode_batch", "gguf_config", "gguf_tensor_name", "gguf_validate", "kernel_classes",
    "read_logits", "weight_count", "weight_info",
    "CQ35Error", "LIBRARY", "load", "SPLIT_KEYS_DEFAULT",
]

# the operators over torch tensors (paged.py), loaded on first use: the rest of
# the package runs without torch, and a star import takes them where torch is
_PAGED = ("PLAN_STATUS", "PagePlan", "page_plan", "paged_prepare", "paged_attention", "paged_attention_workspace")
if sys.modules["torch"] is not None if "torch" in sys.modules else importlib.util.find_spec("torch") is not None:
    __all__ += _PAGED


def __dir__():
    return sorted({*globals(), *_PAGED})


def __getattr__(name):
    if name in _PAGED:
        from . import paged
        globals().update((n, getattr(paged, n)) for n in _PAGED)
        return globals()[name]
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
