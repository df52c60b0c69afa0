"""The C++ binding of the training and serving operators (``lib/_torch_binding.so``).

It checks tensors, fills the C ABI's parameter blocks and calls
``libavey_b200.so`` (loaded by ``_native``) with a few microseconds of host work.
Loading fails loudly: there is no fallback when the binding is missing.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading
from pathlib import Path

import torch  # noqa: F401  (the binding links against its libraries)

from . import _native

BINDING_PATH = Path(__file__).resolve().parent / 'lib' / '_torch_binding.so'
_FUNCTIONS = ('avey_adamw_v1', 'avey_linear_fwd_v1', 'avey_linear_bwd_v1',
              'avey_linear_workspace_size', 'avey_loss_fwd_v1', 'avey_loss_bwd_v1',
              'avey_loss_workspace_size', 'avey_route_fwd_v1', 'avey_route_bwd_v1', 'avey_arrange_v1',
              'avey_arrange_workspace_size', 'avey_dispatch_v1', 'avey_combine_v1',
              'avey_combine_bwd_v1', 'avey_rows_workspace_size', 'avey_embedding_fwd_v1',
              'avey_embedding_bwd_v1', 'avey_embedding_workspace_size', 'avey_last_error')

_lock = threading.Lock()
_module = None


def module():
    """The loaded binding; raises if it has not been built."""
    global _module
    if _module is not None:
        return _module
    with _lock:
        if _module is None:
            if not BINDING_PATH.exists():
                raise RuntimeError(
                    f'avey_kernel_b200: binding not found at {BINDING_PATH}. Build it with '
                    '`python -m avey_kernel_b200.csrc.build` (there is no fallback).')
            dll = _native.lib()
            name = '_torch_binding'
            loader = importlib.machinery.ExtensionFileLoader(name, str(BINDING_PATH))
            mod = importlib.util.module_from_spec(importlib.util.spec_from_loader(name, loader))
            loader.exec_module(mod)
            mod.bind({f: ctypes.cast(getattr(dll, f), ctypes.c_void_p).value for f in _FUNCTIONS})
            _module = mod
    return _module
