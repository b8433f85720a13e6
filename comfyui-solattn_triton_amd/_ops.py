"""The host extension behind the operators around attention (``csrc/bind.cpp``): loaded
at import and given libsolattn's entry points; if it is missing or fails to load,
importing this module raises ImportError, as ``_capi`` does for the library."""

from __future__ import annotations

import ctypes

import torch  # noqa: F401  (the extension binds to its libraries)

from . import _capi

try:
    from . import _native
except ImportError as exc:
    raise ImportError(f"the host extension _native.so cannot be loaded ({exc}); build it with "
                      f"`python {_capi._HERE}/build.py`") from exc

_native.init({name: ctypes.cast(getattr(_capi.LIB, name), ctypes.c_void_p).value
              for name in _capi.SIGNATURES}, _capi.SolAttnError)

native = _native
