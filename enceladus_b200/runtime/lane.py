"""The short way from torch tensors to the decoding step's entry points (csrc/torch_lane.cpp).

`get()` is the extension module, or None where it is not built or torch is not in use; the wrappers in ops.py then go
through `kernel[grid](...)`, with the same results.  Its functions answer NotImplemented for every call that is not a plain
valid one on device tensors.
"""

from __future__ import annotations

import ctypes
import importlib.util
import sys
import threading
import warnings
from importlib.machinery import ExtensionFileLoader
from typing import Any

from enceladus_b200 import _native as N

LANE_PATH = N.LIB_PATH.parent / "enc_torch_lane.so"

_lock = threading.Lock()
_lane: Any = None
_tried = False


def get() -> Any:
    if _tried or "torch" not in sys.modules:
        return _lane
    return _load()


def _load() -> Any:
    global _lane, _tried
    with _lock:
        if _tried:
            return _lane
        lane = None
        if LANE_PATH.exists():
            lib = N.load()
            try:
                loader = ExtensionFileLoader("enc_torch_lane", str(LANE_PATH))
                lane = importlib.util.module_from_spec(importlib.util.spec_from_loader("enc_torch_lane", loader))
                loader.exec_module(lane)
                lane.init(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value
                            for f in ("enc_append_kv", "enc_paged_attention", "enc_paged_attention_work_bytes", "enc_penalize_logits")))
            except ImportError as e:  # built against another torch
                warnings.warn(f"{LANE_PATH.name} cannot be loaded ({e}); rebuild it with `python -m enceladus_b200.build`", RuntimeWarning, stacklevel=3)
                lane = None
        _lane, _tried = lane, True
        return _lane
