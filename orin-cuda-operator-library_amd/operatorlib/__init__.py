"""operatorlib for MI355X — Python entry points.

* ``load_operatorlib()`` registers ``torch.ops.operatorlib.{reduce_sum,
  softmax, transpose, rmsnorm, gemm, attention}`` and the language-model
  operators ``{rope_append, paged_attention, masked_attention}`` from the
  in-tree extension. Like the reference's ``python/load_extension.py:17-36``, which
  compiles its CUDA sources on first use, it builds the HIP library and the
  binding with hipcc for gfx950 when they are not built yet
  (``OPERATORLIB_NO_BUILD=1`` turns that off); a build that exists is loaded
  as it is.
* ``clib()`` returns the ``ctypes`` handle of ``liboperatorlib.so`` with the
  C ABI of ``include/operatorlib/operatorlib_c.h`` typed, for callers that
  want the library without the torch layer. It builds on first use in the
  same way.
* ``lm_clib()`` does the same for ``liboperatorlib_lm.so`` and the C ABI of
  ``include/operatorlib/lm_c.h``.

Both raise if the native library is missing and cannot be built: there is
no fallback implementation.
"""

from __future__ import annotations

import ctypes
import os
from pathlib import Path

from . import _build

LIB_DIR = _build.LIB_DIR
LIBRARY_PATH = _build.LIBRARY
LM_LIBRARY_PATH = _build.LM_LIBRARY
TORCH_EXT_PATH = _build.TORCH_EXT

__all__ = ["build", "load_operatorlib", "clib", "lm_clib", "LIBRARY_PATH", "LM_LIBRARY_PATH",
           "TORCH_EXT_PATH", "C_SYMBOLS", "LM_C_SYMBOLS", "Strides", "HIP_SUCCESS",
           "HIP_ERROR_INVALID_VALUE"]

HIP_SUCCESS = 0
HIP_ERROR_INVALID_VALUE = 1

_c = ctypes
# name -> (restype, argtypes); mirrors include/operatorlib/operatorlib_c.h
C_SYMBOLS = {
    "operatorlib_abi_version": (_c.c_int, []),
    "operatorlib_status_string": (_c.c_char_p, [_c.c_int]),
    "operatorlib_reduce_sum_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "operatorlib_reduce_sum_f32_noalloc": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_size_t,
                                                      _c.c_void_p]),
    "operatorlib_softmax_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int, _c.c_void_p]),
    "operatorlib_softmax_f16": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int, _c.c_void_p]),
    "operatorlib_rmsnorm_f16": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                           _c.c_float, _c.c_void_p]),
    "operatorlib_transpose_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int, _c.c_void_p]),
    "operatorlib_rmsnorm_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                           _c.c_float, _c.c_void_p]),
    "operatorlib_gemm_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                        _c.c_int, _c.c_void_p]),
    "operatorlib_gemm_f16": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                        _c.c_int, _c.c_void_p]),
    "operatorlib_attention_f32": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_void_p,
                                             _c.c_int, _c.c_int, _c.c_int, _c.c_int, _c.c_int,
                                             _c.c_void_p]),
    "operatorlib_attention_f16": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_void_p,
                                             _c.c_int, _c.c_int, _c.c_int, _c.c_int, _c.c_int,
                                             _c.c_void_p]),
    # workspace forms: the caller's device memory instead of the GPU's arena
    "operatorlib_reduce_sum_f32_workspace_size": (_c.c_size_t, [_c.c_void_p, _c.c_size_t]),
    "operatorlib_reduce_sum_f32_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_size_t,
                                                 _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "operatorlib_softmax_f32_workspace_size": (_c.c_size_t, [_c.c_int, _c.c_int]),
    "operatorlib_softmax_f32_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                              _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "operatorlib_softmax_f16_workspace_size": (_c.c_size_t, [_c.c_int, _c.c_int]),
    "operatorlib_softmax_f16_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_int, _c.c_int,
                                              _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "operatorlib_rmsnorm_f32_workspace_size": (_c.c_size_t, [_c.c_int, _c.c_int]),
    "operatorlib_rmsnorm_f32_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int,
                                              _c.c_int, _c.c_float, _c.c_void_p, _c.c_size_t,
                                              _c.c_void_p]),
    "operatorlib_rmsnorm_f16_workspace_size": (_c.c_size_t, [_c.c_int, _c.c_int]),
    "operatorlib_rmsnorm_f16_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int,
                                              _c.c_int, _c.c_float, _c.c_void_p, _c.c_size_t,
                                              _c.c_void_p]),
    "operatorlib_gemm_f32_workspace_size": (_c.c_size_t, [_c.c_void_p, _c.c_void_p, _c.c_int,
                                                          _c.c_int, _c.c_int]),
    "operatorlib_gemm_f32_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int,
                                           _c.c_int, _c.c_int, _c.c_void_p, _c.c_size_t,
                                           _c.c_void_p]),
    "operatorlib_gemm_f16_workspace_size": (_c.c_size_t, [_c.c_void_p, _c.c_void_p, _c.c_int,
                                                          _c.c_int, _c.c_int]),
    "operatorlib_gemm_f16_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_int,
                                           _c.c_int, _c.c_int, _c.c_void_p, _c.c_size_t,
                                           _c.c_void_p]),
    "operatorlib_attention_f32_workspace_size": (_c.c_size_t, [_c.c_void_p, _c.c_void_p,
                                                               _c.c_void_p, _c.c_void_p,
                                                               _c.c_int, _c.c_int, _c.c_int,
                                                               _c.c_int, _c.c_int]),
    "operatorlib_attention_f32_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p,
                                                _c.c_void_p, _c.c_int, _c.c_int, _c.c_int,
                                                _c.c_int, _c.c_int, _c.c_void_p, _c.c_size_t,
                                                _c.c_void_p]),
    "operatorlib_attention_f16_workspace_size": (_c.c_size_t, [_c.c_void_p, _c.c_void_p,
                                                               _c.c_void_p, _c.c_void_p,
                                                               _c.c_int, _c.c_int, _c.c_int,
                                                               _c.c_int, _c.c_int]),
    "operatorlib_attention_f16_ws": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p,
                                                _c.c_void_p, _c.c_int, _c.c_int, _c.c_int,
                                                _c.c_int, _c.c_int, _c.c_void_p, _c.c_size_t,
                                                _c.c_void_p]),
}


class Strides(_c.Structure):
    """operatorlib_strides_t: element strides of [batch, heads, sequence, head_dim]."""
    _fields_ = [("batch", _c.c_int64), ("head", _c.c_int64), ("token", _c.c_int64)]


_p, _i, _l, _f = _c.c_void_p, _c.c_int, _c.c_int64, _c.c_float
_ROPE = [_p, _l, _p, _l, _p, _l, _p, _i, *[_p] * 7, *[_i] * 8, _p]
_PAGED = [_p, _l, _p, _p, _p, _l, *[_p] * 3, *[_i] * 7, _f, _i, _f]
_MASKED = [_p, Strides, _p, Strides, _p, Strides, _p, _p, _p, _p, Strides, *[_i] * 5, _f, _i, _i,
           _f, _p]
# name -> (restype, argtypes); mirrors include/operatorlib/lm_c.h
LM_C_SYMBOLS = {"operatorlib_lm_abi_version": (_i, [])}
for _t in ("f16", "f32"):
    LM_C_SYMBOLS |= {
        f"operatorlib_rope_append_{_t}": (_i, _ROPE),
        f"operatorlib_paged_attention_{_t}_workspace_size": (_c.c_size_t, [_i] * 6),
        f"operatorlib_paged_attention_{_t}": (_i, [*_PAGED, _p]),
        f"operatorlib_paged_attention_{_t}_ws": (_i, [*_PAGED, _p, _c.c_size_t, _p]),
        f"operatorlib_masked_attention_{_t}": (_i, _MASKED),
    }

_clib = None
_lm_clib = None
_torch_loaded = False


def build(verbose: bool = False, torch_binding: bool = True) -> None:
    """Compile every native artefact for gfx950 (see ``_build``)."""
    _build.build(verbose=verbose, torch_binding=torch_binding)


def _require(path: Path, torch_binding: bool) -> None:
    """Build the native artefacts if `path` is missing; raise if that is not
    possible."""
    if path.exists():
        return
    if os.environ.get("OPERATORLIB_NO_BUILD", "0") == "1":
        raise RuntimeError(
            f"operatorlib native library missing: {path} (OPERATORLIB_NO_BUILD=1). "
            "Build it with python -c 'import __graft_entry__ as g; g.build()'.")
    try:
        if torch_binding:
            _build.build(torch_binding=True)
        else:
            _build.build_library()
    except Exception as exc:  # no silent fallback: report and stop
        raise RuntimeError(f"operatorlib native library missing: {path}, and building "
                           f"it failed: {exc}") from exc
    if not path.exists():
        raise RuntimeError(f"operatorlib build did not produce {path}")


def clib() -> ctypes.CDLL:
    """Load ``liboperatorlib.so`` and type its C ABI."""
    global _clib
    if _clib is None:
        _require(LIBRARY_PATH, torch_binding=False)
        try:
            # Share the HIP runtime torch already loaded (same SONAME) when
            # torch is importable, so both use one runtime instance.
            import torch  # noqa: F401
        except ImportError:
            pass
        _clib = _typed(LIBRARY_PATH, C_SYMBOLS)
    return _clib


def lm_clib() -> ctypes.CDLL:
    """Load ``liboperatorlib_lm.so`` and type its C ABI."""
    global _lm_clib
    if _lm_clib is None:
        _require(LM_LIBRARY_PATH, torch_binding=False)
        clib()  # liboperatorlib.so, which it links
        _lm_clib = _typed(LM_LIBRARY_PATH, LM_C_SYMBOLS)
    return _lm_clib


def _typed(path: Path, symbols: dict) -> ctypes.CDLL:
    lib = ctypes.CDLL(str(path), mode=ctypes.RTLD_GLOBAL)
    for name, (restype, argtypes) in symbols.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


def load_operatorlib(verbose: bool = False) -> None:
    """Register ``torch.ops.operatorlib.*`` (reference: load_extension.py:17)."""
    global _torch_loaded
    if _torch_loaded:
        return
    import torch
    _require(TORCH_EXT_PATH, torch_binding=True)
    lm_clib()  # the extension links both libraries; load them first, same runtime
    torch.ops.load_library(str(TORCH_EXT_PATH))
    if verbose:
        print(f"loaded {TORCH_EXT_PATH}")
    _torch_loaded = True
