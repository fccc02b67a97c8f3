"""The compiled autograd nodes (csrc/autograd.cpp) bound to the library ugpg._C loaded.

As with libugpg there is no fallback: a missing or stale module raises.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from pathlib import Path

from ._C import lib

PATH = Path(__file__).resolve().parent / "_autograd.so"
ENTRIES = ("ugpg_last_error", "ugpg_group_norm_workspace", "ugpg_group_norm_fwd", "ugpg_group_norm_bwd",
           "ugpg_distill_workspace", "ugpg_distill_fwd", "ugpg_distill_bwd", "ugpg_top_logits")
_module = None


def _check_fresh(build_id):
    """Refuse nodes built from another source, header or torch than the ones beside them."""
    bpy = Path(__file__).resolve().parent.parent / "build.py"
    if not bpy.exists():
        return
    spec = importlib.util.spec_from_file_location("_ugpg_build", bpy)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    want = mod.autograd_id()
    if build_id != want:
        raise ImportError(f"ugpg: {PATH} is stale (built from {build_id}, tree has {want}) -- rebuild it "
                          "with `python ug-pg-unet_amd/build.py`. There is no fallback.")


def nodes():
    global _module
    if _module is None:
        if not PATH.exists():
            raise ImportError(f"ugpg: {PATH} not found -- build it with `python ug-pg-unet_amd/build.py`. "
                              "There is no fallback.")
        import torch  # noqa: F401  (its libraries, before the module that needs them)
        loader = importlib.machinery.ExtensionFileLoader("_autograd", str(PATH))
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_autograd", loader))
        loader.exec_module(mod)
        _check_fresh(mod.build_id)
        mod.bind([C.cast(getattr(lib, n), C.c_void_p).value for n in ENTRIES])
        _module = mod
    return _module
