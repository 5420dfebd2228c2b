"""``ext``: the autograd module ``lib/cpmk_torch.*.so`` (csrc/torch/ffn.cpp: autograd of the row layer norm and the gated block in C++) with
the entry points of the C library that the ctypes layer has loaded.  Loaded on first use, so that a module that is missing or does not fit
the installed PyTorch concerns these operators only."""
import ctypes
import importlib.machinery
import importlib.util
import os
import threading

import torch  # noqa: F401  (its libraries are what the module links to)

from ..build import EXT_PATH
from ..library import cpmk

_ENTRY_POINTS = ("cpmk_last_error", "cpmk_layernorm_rows_forward", "cpmk_layernorm_rows_backward_scratch", "cpmk_layernorm_rows_backward",
                 "cpmk_gated_scratch", "cpmk_gated_backward_scratch", "cpmk_gated_linear_forward", "cpmk_gated_linear_backward",
                 "cpmk_gated_feed_forward_forward", "cpmk_gated_feed_forward_backward")      # in the order of its table


def _load():
    if not os.path.exists(EXT_PATH):
        raise RuntimeError("cpm_kernels_b200: autograd module not found at %s. Build it with `python -m cpm_kernels_b200.build`. "
                           "There is no fallback." % EXT_PATH)
    loader = importlib.machinery.ExtensionFileLoader("cpmk_torch", EXT_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("cpmk_torch", loader))
    loader.exec_module(module)
    module.bind([ctypes.cast(getattr(cpmk.lib, name), ctypes.c_void_p).value for name in _ENTRY_POINTS])
    return module


_lock = threading.Lock()


def __getattr__(name: str):
    if name != "ext":
        raise AttributeError("module %r has no attribute %r" % (__name__, name))
    with _lock:
        if "ext" not in globals():
            globals()["ext"] = _load()
    return globals()["ext"]
