"""ctypes binding of the operators on rows of logits
(include/tropnn_hip_logits.h): top logits, distillation, sampling.

The functions here take checked tensors, allocate outputs and workspace and
launch on the current stream of the logits' device; tropnn_amd.logits holds the
public operators. There is no CPU fallback."""
from __future__ import annotations

import ctypes
import functools
from typing import Any

import torch
from torch import Tensor

from .pairwise_hip import _LOCK, _check, _pairwise_op, _ptr, _stream, library_path, load_library

LOGITS_ABI_VERSION = 1
LOGITS_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_VOCAB, MAX_TOP = 1 << 20, 1024

LOGITS_SYMBOLS = (
    "tropnn_hip_logits_abi_version",
    "tropnn_hip_top_logits_workspace_size",
    "tropnn_hip_top_logits",
    "tropnn_hip_distill_workspace_size",
    "tropnn_hip_distill",
    "tropnn_hip_distill_grad",
    "tropnn_hip_scale_in_place",
    "tropnn_hip_sample_workspace_size",
    "tropnn_hip_sample",
)
_LIB: ctypes.CDLL | None = None
_DISTILL_OP: Any = None


def _declare(lib: ctypes.CDLL) -> None:
    i64, sz, p, f, i = ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float, ctypes.c_int
    i32 = ctypes.c_int32
    for name, args, result in (
        ("tropnn_hip_logits_abi_version", [], i),
        ("tropnn_hip_top_logits_workspace_size", [i64, i64, i, i64], sz),
        ("tropnn_hip_top_logits", [i64, i64, i64, p, i, i64, f, p, p, p, p, sz, p], i),
        ("tropnn_hip_distill_workspace_size", [i64, i64, i, i64, i], sz),
        ("tropnn_hip_distill", [i64, i64, i64, p, i, i64, p, i, p, p, p, f, f, i, p, p, p, sz, p], i),
        ("tropnn_hip_distill_grad", [i64, i64, i64, p, i, i64, p, i, p, p, p, f, f, i, p, i, p, p, sz, p], i),
        ("tropnn_hip_scale_in_place", [i64, p, i, p, p], i),
        ("tropnn_hip_sample_workspace_size", [i64, i64, i], sz),
        ("tropnn_hip_sample", [i64, i64, i64, p, i, p, p, f, p, i32, p, f, p, f, p, p, p, sz, p], i),
    ):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, result


def load_logits_library() -> ctypes.CDLL:
    """libtropnn_hip.so with the logits entry points declared. Raises
    RuntimeError if they are missing or of another version."""
    global _LIB
    if _LIB is not None:
        return _LIB
    lib = load_library()
    with _LOCK:
        if _LIB is not None:
            return _LIB
        missing = [s for s in LOGITS_SYMBOLS if not hasattr(lib, s)]
        if missing:
            raise RuntimeError(f"{library_path()} lacks symbols {missing}")
        _declare(lib)
        version = lib.tropnn_hip_logits_abi_version()
        if version != LOGITS_ABI_VERSION:
            raise RuntimeError(
                f"{library_path()} has logits ABI version {version}, this package expects {LOGITS_ABI_VERSION}"
            )
        _LIB = lib
    return _LIB


def distill_op() -> Any:
    """torch.ops.tropnn_hip.distill (csrc/logits_op.cpp), loaded once and bound
    to the entry points of the library that load_logits_library() checked."""
    global _DISTILL_OP
    if _DISTILL_OP is not None:
        return _DISTILL_OP
    lib = load_logits_library()
    _pairwise_op()  # loads the operator library
    with _LOCK:
        if _DISTILL_OP is None:
            names = ("tropnn_hip_distill", "tropnn_hip_distill_workspace_size", "tropnn_hip_distill_grad",
                     "tropnn_hip_scale_in_place", "tropnn_hip_capture_id", "tropnn_hip_last_error")
            torch.ops.tropnn_hip.bind_logits_abi(
                *(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names), LOGITS_ABI_VERSION)
            _DISTILL_OP = torch.ops.tropnn_hip.distill.default
    return _DISTILL_OP


def on_device_of(fn):
    """Runs fn with its first argument's GPU as the current one: kernels are
    launched on that GPU's current stream."""

    @functools.wraps(fn)
    def call(logits: Tensor, *args, **kwargs):
        if logits.device.index == torch.cuda.current_device():
            return fn(logits, *args, **kwargs)
        with torch.cuda.device(logits.device):
            return fn(logits, *args, **kwargs)

    return call


def as_rows(logits: Tensor) -> tuple[Tensor, int, int, int]:
    """(tensor, rows, vocab, row stride in elements) of logits [..., vocab].
    Rows may lie apart (a slice of a wider tensor); any other layout than
    evenly spaced contiguous rows is copied."""
    vocab = logits.shape[-1]
    rows = logits.numel() // vocab
    if logits.is_contiguous():
        return logits, rows, vocab, vocab
    if logits.stride(-1) == 1 or vocab == 1:
        try:
            flat = logits.view(-1, vocab)
        except RuntimeError:  # the leading dimensions have no common stride
            flat = None
        if flat is not None and flat.stride(-1) == 1 and flat.stride(0) >= vocab:
            return flat, rows, vocab, flat.stride(0)
    return logits.contiguous(), rows, vocab, vocab


def _workspace(size: int, device: torch.device) -> Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


@on_device_of
def top_logits_hip(logits: Tensor, k: int, temperature: float) -> tuple[Tensor, Tensor, Tensor]:
    lib, device, lead = load_logits_library(), logits.device, logits.shape[:-1]
    x, rows, vocab, stride = as_rows(logits)
    dtype = LOGITS_DTYPES[x.dtype]
    values = torch.empty((*lead, k), dtype=x.dtype, device=device)
    indices = torch.empty((*lead, k), dtype=torch.int64, device=device)
    log_rest = torch.empty(lead, dtype=torch.float32, device=device)
    size = lib.tropnn_hip_top_logits_workspace_size(rows, vocab, dtype, k)
    ws = _workspace(size, device)
    rc = lib.tropnn_hip_top_logits(rows, vocab, stride, x.data_ptr(), dtype, k, temperature, values.data_ptr(),
                                   indices.data_ptr(), log_rest.data_ptr(), _ptr(ws), size, _stream(device))
    _check(rc, "tropnn_hip_top_logits")
    return values, indices, log_rest


@on_device_of
def scale_in_place(x: Tensor, factor: Tensor) -> Tensor:
    """x (contiguous) times the 0-dim f32 `factor`, in place; x is not touched
    where the factor is one."""
    rc = load_logits_library().tropnn_hip_scale_in_place(x.numel(), x.data_ptr(), LOGITS_DTYPES[x.dtype],
                                                        factor.data_ptr(), _stream(x.device))
    _check(rc, "tropnn_hip_scale_in_place")
    return x


@on_device_of
def sample_hip(logits: Tensor, uniforms: Tensor, temperature: float | Tensor, top_k: int | Tensor,
               top_p: float | Tensor, min_p: float | Tensor) -> tuple[Tensor, Tensor]:
    lib, device, lead = load_logits_library(), logits.device, logits.shape[:-1]
    x, rows, vocab, stride = as_rows(logits)
    dtype = LOGITS_DTYPES[x.dtype]
    uniforms = uniforms.contiguous()
    parameters, kept = [], []
    for value in (temperature, top_k, top_p, min_p):
        if isinstance(value, Tensor):
            kept.append(value.contiguous())
            parameters += [kept[-1].data_ptr(), 0]
        else:
            parameters += [None, value]
    tokens = torch.empty(lead, dtype=torch.int64, device=device)
    log_probs = torch.empty(lead, dtype=torch.float32, device=device)
    size = lib.tropnn_hip_sample_workspace_size(rows, vocab, dtype)
    ws = _workspace(size, device)
    rc = lib.tropnn_hip_sample(rows, vocab, stride, x.data_ptr(), dtype, uniforms.data_ptr(), *parameters,
                               tokens.data_ptr(), log_probs.data_ptr(), _ptr(ws), size, _stream(device))
    _check(rc, "tropnn_hip_sample")
    return tokens, log_probs
