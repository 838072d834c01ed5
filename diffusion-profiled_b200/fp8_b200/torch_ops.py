"""Loads ``libfp8torch.so``, the text-conditioning operators registered with torch in C++ (csrc/torch_ops.cpp).

The package loads the library where it is there and fits; the modules that call its
operators demand it.  So the FP8 operators, which do not need it, run without it.
"""

from __future__ import annotations

import torch

from . import _lib
from .build import TORCH_LIB_PATH, torch_library_fits

_loaded = False


def load(required: bool) -> bool:
    """Loads the library once; if it is missing or was built for another torch, raises (``required``) or returns False."""
    global _loaded
    if _loaded:
        return True
    if not torch_library_fits(torch.__version__):
        if not required:
            return False
        why = "was built for another torch than " + torch.__version__ if TORCH_LIB_PATH.exists() else "is missing"
        raise RuntimeError(f"{TORCH_LIB_PATH} {why}: build it with fp8_b200.build.build_library() "
                           "(or __graft_entry__.build()); there is no fallback implementation")
    _lib.load()  # libfp8ops.so, which the operators call
    torch.ops.load_library(str(TORCH_LIB_PATH))
    _loaded = True
    return True
