"""Loads ``lib/_row_ops.so``, the torch binding of the row-wise operators (built by
``llm720_b200.build`` from ``csrc/torch/row_ops.cpp``).  A missing library is an
error, there is no other code path."""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (the binding links against its libraries)

from . import _lib

EXT_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "_row_ops.so")

_ext = None


def load():
    """The extension module, loaded once."""
    global _ext
    if _ext is None:
        if not os.path.exists(EXT_PATH):
            raise RuntimeError(f"{EXT_PATH} is missing: build it with `python -m llm720_b200.build` (needs nvcc and g++).  "
                               "There is no fallback path.")
        _lib.load()                                   # checks the ABI version of the library the binding calls
        loader = importlib.machinery.ExtensionFileLoader("_row_ops", EXT_PATH)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_row_ops", loader))
        loader.exec_module(mod)
        if mod.abi_version != _lib.ABI_VERSION:
            raise RuntimeError("_row_ops.so was built from a different ABI version; rebuild it")
        _ext = mod
    return _ext
