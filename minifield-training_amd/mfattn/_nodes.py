"""The autograd nodes of ``csrc/nodes`` (``_mfnodes.so``), bound to the loaded C ABI.

Outputs, workspaces and what a backward pass needs are made there, without the
interpreter.  Like the library it is loaded at import, and there is no fallback; modules
that have no nodes do not import this one.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import pathlib

import torch  # noqa: F401  (its libraries are loaded before the module that uses them)

from . import _lib

PATH = pathlib.Path(__file__).resolve().parent / "_mfnodes.so"

_FUNCTIONS = ("mf_norm", "mf_norm_bwd", "mf_norm_bwd_workspace_bytes", "mf_embed", "mf_embed_bwd",
              "mf_embed_bwd_workspace_bytes", "mf_distill", "mf_distill_bwd",
              "mf_distill_stats_bytes", "mf_last_error")


def _load():
    if not PATH.exists():
        raise ImportError(f"mfattn autograd nodes missing: {PATH} (build them with "
                          "`python minifield-training_amd/mfattn/build.py`)")
    loader = importlib.machinery.ExtensionFileLoader("_mfnodes", str(PATH))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_mfnodes", loader))
    loader.exec_module(module)
    module.init({name: ctypes.cast(getattr(_lib.LIB, name), ctypes.c_void_p).value
                 for name in _FUNCTIONS}, _lib.MfValueError, _lib.MfError)
    return module


_module = _load()
norm, embed, distill, rows_even = _module.norm, _module.embed, _module.distill, _module.rows_even
# the same with the checks of ordinary operands: None to a call that has others
usual_norm, usual_embed, usual_distill = (_module.usual_norm, _module.usual_embed,
                                          _module.usual_distill)


def even_rows(x: torch.Tensor) -> torch.Tensor:
    """``x [..., D]``, copied only where its last dimension is not dense, its rows are not evenly
    spaced or overlap, or its sign stands beside its memory (``torch.Tensor.is_neg``)."""
    x = x.resolve_neg()
    return x if x.is_contiguous() or rows_even(x) else x.contiguous()
