"""The torch-side module of the library (csrc/fp4t_torch.cpp, built by csrc/build.sh into
lib/fp4t_torch.so): argument checks, outputs and autograd nodes of the operators between and behind the
quantized layers.  Like the library itself it has no fallback."""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (its libraries have to be loaded before the module's)

_HERE = os.path.dirname(os.path.abspath(__file__))
EXT_PATH = os.path.abspath(os.path.join(_HERE, "..", "lib", "fp4t_torch.so"))

_module = None


def ext():
    global _module
    if _module is None:
        if not os.path.isfile(EXT_PATH):
            raise RuntimeError(f"fp4t torch module not found at {EXT_PATH}; build it with fp4-training_b200/csrc/build.sh")
        loader = importlib.machinery.ExtensionFileLoader("fp4t_torch", EXT_PATH)
        spec = importlib.util.spec_from_file_location("fp4t_torch", EXT_PATH, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _module = module
    return _module


def launches():
    """(rotary, linear cross entropy) kernels that the module has enqueued, its backward passes' included."""
    return (0, 0) if _module is None else _module.launches()
