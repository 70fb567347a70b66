"""Loads lib/_vsv_torch.so, the torch side (checks, allocation, autograd functions) of vsv.ssm and vsv.optim, and hands it the C
entries of the library that vsv.lib has loaded."""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os

from . import lib as _lib

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib", "_vsv_torch.so")
ENTRIES = ("vsv_last_error", "vsv_short_conv", "vsv_short_conv_backward_ws_bytes", "vsv_short_conv_backward", "vsv_short_conv_step",
           "vsv_ssm_saved_floats", "vsv_ssm_scan_ws_bytes", "vsv_ssm_scan", "vsv_ssm_scan_backward_ws_bytes", "vsv_ssm_scan_backward",
           "vsv_ssm_step", "vsv_adamw_multi", "vsv_adamw_read8")
_module = None


def load():
    global _module
    if _module is None:
        lib = _lib.load()                                                  # (torch first, then the kernels)
        if not os.path.exists(PATH):
            raise RuntimeError(f"{PATH} is missing: build it with `make -C vol-surface-vae-pub_amd/csrc` (there is no fallback)")
        loader = importlib.machinery.ExtensionFileLoader("_vsv_torch", PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_vsv_torch", PATH, loader=loader))
        loader.exec_module(module)
        module.bind({name: C.cast(getattr(lib, name), C.c_void_p).value for name in ENTRIES})
        _module = module
    return _module
