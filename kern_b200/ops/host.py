"""The C++ host side of the short operators (``kern_b200/_ops_host*.so``): brought in at the first call that needs it, so that nothing
else hangs on a library that is built against one PyTorch."""
from __future__ import annotations

import importlib

import torch

_ops = None


def ops():
    """The module, with the kernels of this process's GPUs at hand."""
    return _ops if _ops is not None else _load()


def loaded():
    """The module if something has called for it, or None."""
    return _ops


def _load():
    global _ops
    again = "build it again: python -m kern_b200._build"
    try:
        m = importlib.import_module("kern_b200._ops_host")
    except ImportError as e:
        raise RuntimeError(f"the operators over 8-bit caches and drafted trees need kern_b200/_ops_host, which does not load ({e}); {again}") from e
    if m.torch_version != torch.__version__:
        raise RuntimeError(f"kern_b200/_ops_host was built for PyTorch {m.torch_version}, and this is {torch.__version__}; {again}")
    m.on_missing(_provide)
    _ops = m
    return m


def _provide(gpu: int) -> None:
    """What the module needs of a GPU, at its first call there."""
    from .launcher import Kernels

    k = Kernels.get(gpu)
    _ops.provide(gpu, k.sm_count, k.err_word().data_ptr(), lambda module, entry: k.function(module, entry).handle)
