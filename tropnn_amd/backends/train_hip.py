"""Binding of the operators that train a token model on its own answers
(include/tropnn_hip_train.h). The operators themselves are torch.ops.tropnn_hip's
token_log_probs, policy, preference and adam8 (csrc/train_op.cpp), which drive
the C ABI; tropnn_amd.policy and tropnn_amd.optim hold the public functions.
There is no CPU fallback."""
from __future__ import annotations

import ctypes
from typing import Any

import torch

from .logits_hip import load_logits_library
from .pairwise_hip import _LOCK, _pairwise_op, library_path

TRAIN_ABI_VERSION = 2
STATE_BLOCK = 32  # elements of an 8-bit state that share an exponent

TRAIN_SYMBOLS = (
    "tropnn_hip_train_abi_version",
    "tropnn_hip_capture_id",
    "tropnn_hip_token_log_probs",
    "tropnn_hip_token_gradient",
    "tropnn_hip_policy_grad_fits",
    "tropnn_hip_policy_workspace_size",
    "tropnn_hip_policy",
    "tropnn_hip_preference_workspace_size",
    "tropnn_hip_preference",
    "tropnn_hip_adam8_workspace_size",
    "tropnn_hip_adam8_step",
)
_LIB: ctypes.CDLL | None = None
_OPS: Any = None


def _declare(lib: ctypes.CDLL) -> None:
    i64, sz, p, i, d = ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    rows = [i64, i64, i64, p, i, p, d]  # rows, vocab, row stride, logits, type, tokens, temperature
    for name, args, result in (
        ("tropnn_hip_train_abi_version", [], i),
        ("tropnn_hip_capture_id", [p], ctypes.c_ulonglong),
        ("tropnn_hip_token_log_probs", [*rows, p, p, p, p], i),
        ("tropnn_hip_token_gradient", [*rows, p, p, i64, p, p, i, p, p], i),
        ("tropnn_hip_policy_grad_fits", [i64, i64, i], i),
        ("tropnn_hip_policy_workspace_size", [i64, i64, i, i], sz),
        ("tropnn_hip_policy", [*rows, p, p, p, p, d, d, d, d, i, p, p, p, p, p, p, p, sz, p], i),
        ("tropnn_hip_preference_workspace_size", [i64, i64], sz),
        ("tropnn_hip_preference", [i64, i64, p, p, p, p, d, d, d, i, d, i, p, p, p, p, p, sz, p], i),
        ("tropnn_hip_adam8_workspace_size", [i], sz),
        ("tropnn_hip_adam8_step", [i, p, p, p, p, p, p, p, p, d, d, d, d, d, i, p, sz, p], i),
    ):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, result


def load_train_library() -> ctypes.CDLL:
    """libtropnn_hip.so with the entry points of training declared. Raises
    RuntimeError if they are missing or of another version."""
    global _LIB
    if _LIB is not None:
        return _LIB
    lib = load_logits_library()
    with _LOCK:
        if _LIB is not None:
            return _LIB
        missing = [s for s in TRAIN_SYMBOLS if not hasattr(lib, s)]
        if missing:
            raise RuntimeError(f"{library_path()} lacks symbols {missing}")
        _declare(lib)
        version = lib.tropnn_hip_train_abi_version()
        if version != TRAIN_ABI_VERSION:
            raise RuntimeError(
                f"{library_path()} has training ABI version {version}, this package expects {TRAIN_ABI_VERSION}"
            )
        _LIB = lib
    return _LIB


def train_ops() -> Any:
    """torch.ops.tropnn_hip with the operators of training, loaded once and
    bound to the entry points of the library that load_train_library() checked."""
    global _OPS
    if _OPS is not None:
        return _OPS
    lib = load_train_library()
    _pairwise_op()  # loads the operator library
    with _LOCK:
        if _OPS is None:
            names = (*(s for s in TRAIN_SYMBOLS if s != "tropnn_hip_train_abi_version"), "tropnn_hip_last_error")
            torch.ops.tropnn_hip.bind_train_abi([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names],
                                                TRAIN_ABI_VERSION)
            _OPS = torch.ops.tropnn_hip
    return _OPS
