"""The operators on rows of logits without a GPU: no CPU fallback, argument
checks before any launch, and the C ABI's own checks."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from tropnn_amd import distillation_loss, sample_tokens, top_logits
from tropnn_amd.backends import logits_hip as lh

HEADER = Path(__file__).resolve().parent.parent / "include" / "tropnn_hip_logits.h"
F32, F16, BF16 = (lh.LOGITS_DTYPES[t] for t in (torch.float32, torch.float16, torch.bfloat16))


@pytest.fixture(scope="module")
def lib():
    if not lh.library_path().exists():
        pytest.skip("libtropnn_hip.so not built (run __graft_entry__.build())")
    return lh.load_logits_library()


def define(name: str) -> int:
    m = re.search(rf"#define {name} (\d+)", HEADER.read_text())
    assert m, name
    return int(m.group(1))


def error(lib) -> str:
    lib.tropnn_hip_last_error.restype = ctypes.c_char_p
    return lib.tropnn_hip_last_error().decode()


def test_binding_matches_header(lib):
    text = re.sub(r"/\*.*?\*/", " ", HEADER.read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(tropnn_hip_\w+)\s*\(", text)))
    assert declared == sorted(lh.LOGITS_SYMBOLS)
    assert lib.tropnn_hip_logits_abi_version() == define("TROPNN_HIP_LOGITS_ABI_VERSION") == lh.LOGITS_ABI_VERSION
    assert (F32, F16, BF16) == tuple(define(f"TROPNN_LOGITS_{n}") for n in ("F32", "F16", "BF16"))
    assert lh.MAX_VOCAB == define("TROPNN_MAX_VOCAB") and lh.MAX_TOP == define("TROPNN_MAX_TOP")


def test_cpu_tensors_raise():
    x = torch.zeros(3, 9)
    with pytest.raises(ValueError, match="GPU"):
        top_logits(x, 2)
    with pytest.raises(ValueError, match="GPU"):
        distillation_loss(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        sample_tokens(x, torch.zeros(3))


class Fake:
    """A tensor's outside, as if it were on a GPU."""

    def __init__(self, shape, dtype=torch.float32):
        self.shape, self.dtype, self.ndim = torch.Size(shape), dtype, len(shape)
        self.device = torch.device("cuda:0")


def test_shapes_and_types_raise_before_launch():
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        top_logits(Fake((4, 3), torch.float64), 1)
    with pytest.raises(ValueError, match="at least one class"):
        top_logits(Fake((4, 0)), 1)
    with pytest.raises(ValueError, match="at least one class"):
        sample_tokens(Fake(()), Fake(()))
    with pytest.raises(NotImplementedError, match="classes"):
        sample_tokens(Fake((1, (1 << 20) + 1)), Fake((1,)))
    with pytest.raises(ValueError, match="k <="):
        top_logits(Fake((4, 3)), 0)
    with pytest.raises(TypeError, match="indices"):
        distillation_loss(Fake((4, 9)), WithDetach((4, 2)), Fake((4, 2), torch.int32))
    with pytest.raises(ValueError, match="list entry"):
        distillation_loss(Fake((4, 9)), Fake((4, 0)), Fake((4, 0), torch.int64))


class WithDetach(Fake):
    def detach(self):
        return self


def test_as_rows_reads_slices_where_they_are():
    x = torch.zeros(6, 40)
    assert lh.as_rows(x) == (x, 6, 40, 40) or lh.as_rows(x)[1:] == (6, 40, 40)
    t, rows, vocab, stride = lh.as_rows(x[:, 3:23])
    assert (rows, vocab, stride) == (6, 20, 40) and t.data_ptr() == x[:, 3:].data_ptr()
    t, rows, vocab, stride = lh.as_rows(x.view(2, 3, 40)[:, 1])
    assert (rows, vocab, stride) == (2, 40, 120) and t.data_ptr() == x[1].data_ptr()
    t, rows, vocab, stride = lh.as_rows(x.view(2, 3, 40)[:, :2, :5])  # no common stride: copied
    assert (rows, vocab, stride) == (4, 5, 5) and t.is_contiguous()
    t, rows, vocab, stride = lh.as_rows(x.t())  # classes apart: copied
    assert (rows, vocab, stride) == (40, 6, 6) and t.is_contiguous()
    t, rows, vocab, stride = lh.as_rows(x[:1].expand(6, 40))  # rows on top of each other: copied
    assert (rows, vocab, stride) == (6, 40, 40) and t.is_contiguous()
    assert lh.as_rows(x[0])[1:] == (1, 40, 40)
    assert lh.as_rows(torch.zeros(5, 1).expand(5, 1))[1:3] == (5, 1)
    assert lh.as_rows(torch.zeros(0, 7))[1:3] == (0, 7)


LAYOUTS = {
    "contiguous": lambda x: x,
    "one row": lambda x: x[0, 0],
    "slice of the classes": lambda x: x[..., 5:25],
    "one of the inner dimension": lambda x: x[:, 1],
    "every second row": lambda x: x[:, ::2, :],
    "every second of two": lambda x: x[:, :4:2, :],
    "no common stride": lambda x: x[:, :3, :20],
    "inner dimension broadcast": lambda x: x[:, :1].expand(4, 6, 40),
    "inner dimension broadcast, a slice": lambda x: x[:, 2:3, 3:23].expand(4, 6, 20),
    "outer dimension broadcast": lambda x: x[:1].expand(4, 6, 40),
    "both broadcast": lambda x: x[:1, :1].expand(4, 6, 40),
    "a new inner dimension": lambda x: x[:, 0][:, None].expand(4, 8, 40),
    "a new middle dimension": lambda x: x[:, None].expand(4, 3, 6, 40),
    "a new innermost of three": lambda x: x[:, :, None].expand(4, 6, 3, 40),
    "two new dimensions": lambda x: x[:, 0][:, None, None].expand(4, 2, 3, 40),
    "dimensions of one": lambda x: x[:, :1].unsqueeze(0),
    "dimensions exchanged": lambda x: x.transpose(0, 1),
    "classes apart": lambda x: x.transpose(1, 2),
    "classes broadcast": lambda x: x[..., :1].expand(4, 6, 40),
    "one class": lambda x: x[..., 7:8],
    "one class, broadcast": lambda x: x[:, :1, 7:8].expand(4, 6, 1),
    "no rows": lambda x: x[:0],
    "no rows, broadcast": lambda x: x[:, :0],
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rows_are_read_inside_the_tensor_and_in_order(lib, layout):
    """What the operators take as rows of logits, the Python functions' and the
    autograd operator's, is the tensor's rows, and inside its memory."""
    lh.distill_op()  # loads the operator library
    base = torch.arange(4 * 6 * 40, dtype=torch.float32)
    logits = LAYOUTS[layout](base.view(4, 6, 40))
    for as_rows in (lh.as_rows, torch.ops.tropnn_hip.logit_rows):
        t, rows, vocab, stride = as_rows(logits)
        assert (rows, vocab) == (logits.numel() // logits.shape[-1], logits.shape[-1])
        assert rows <= 1 or stride >= vocab
        if rows == 0:
            continue
        end = t.storage_offset() + (rows - 1) * stride + vocab
        assert end <= t.untyped_storage().nbytes() // 4, f"reads to element {end}"
        read = torch.as_strided(t, (rows, vocab), (stride, 1), t.storage_offset())
        assert torch.equal(read, logits.reshape(rows, vocab))


def test_abi_refuses_bad_arguments(lib):
    p = 4096  # an address that is never read: every call here ends before a launch
    top = [2, 10, 10, p, F32, 3, 1.0, p, p, p, p, 1 << 20, None]

    def bad(fn, args, at, value, word, code=1):
        args = list(args)
        args[at] = value
        assert fn(*args) == code and word in error(lib), (at, value, error(lib))

    fn = lib.tropnn_hip_top_logits
    bad(fn, top, 0, -1, "rows")
    bad(fn, top, 1, 0, "vocab")
    bad(fn, top, 1, (1 << 20) + 1, "vocab", 2)
    bad(fn, top, 2, 9, "row_stride")
    bad(fn, top, 3, None, "logits")
    bad(fn, top, 3, p + 2, "aligned")
    bad(fn, top, 4, 3, "dtype")
    bad(fn, top, 5, 0, "k must")
    bad(fn, top, 5, 1025, "k=", 2)
    bad(fn, top, 5, 11, "k must")
    bad(fn, top, 6, 0.0, "temperature")
    bad(fn, top, 6, float("nan"), "temperature")
    bad(fn, top, 7, None, "non-NULL")
    bad(fn, top, 8, p + 4, "aligned")
    assert fn(0, 10, 10, None, F32, 3, 1.0, None, None, None, None, 0, None) == 0

    distill = [2, 10, 10, p, BF16, 3, p, F16, p, p, p, 1.0, 1.0, 1, p, p, p, 1 << 20, None]
    fn = lib.tropnn_hip_distill
    bad(fn, distill, 0, 1 << 31, "rows")
    bad(fn, distill, 4, -1, "dtype")
    bad(fn, distill, 6, None, "non-NULL")
    bad(fn, distill, 7, 5, "values_dtype")
    bad(fn, distill, 8, p + 4, "aligned")
    bad(fn, distill, 9, p + 2, "aligned")
    bad(fn, distill, 11, -1.0, "temperature")
    bad(fn, distill, 14, None, "non-NULL")
    bad(fn, distill, 15, p + 1, "aligned")
    bad(fn, distill, 16, None, "workspace")
    bad(fn, distill, 16, p + 8, "workspace")
    bad(fn, distill, 17, 4, "workspace")

    sample = [2, 10, 10, p, F16, p, p, 1.0, p, 0, p, 1.0, p, 0.0, p, p, p, 1 << 20, None]
    fn = lib.tropnn_hip_sample
    bad(fn, sample, 2, 3, "row_stride")
    bad(fn, sample, 5, None, "non-NULL")
    bad(fn, sample, 6, p + 2, "aligned")
    bad(fn, sample, 14, p + 4, "aligned")
    assert fn(0, 10, 10, None, F16, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, 0, None) == 0

    scale = lib.tropnn_hip_scale_in_place
    assert scale(-1, p, F32, p, None) == 1 and scale(4, None, F32, p, None) == 1
    assert scale(4, p + 2, F32, p, None) == 1 and scale(4, p, 9, p, None) == 1 and scale(0, None, F32, None, None) == 0


def test_workspace_queries(lib):
    assert lib.tropnn_hip_distill_workspace_size(100, 1000, F32, 8, 1) >= 400
    assert lib.tropnn_hip_distill_workspace_size(100, 0, F32, 8, 1) == 0 and "vocab" in error(lib)
    assert lib.tropnn_hip_top_logits_workspace_size(-1, 10, F32, 8) == 0 and "rows" in error(lib)
    assert lib.tropnn_hip_sample_workspace_size(4, 10, 7) == 0 and "dtype" in error(lib)


def test_abi_refuses_bad_arguments_of_the_scaled_gradient(lib):
    p = 4096  # an address that is never read: every call here ends before a launch
    good = [2, 10, 10, p, BF16, 3, p, F16, p, p, p, 1.0, 1.0, 1, p, 1, p, p, 1 << 20, None]
    fn = lib.tropnn_hip_distill_grad
    for at, value, word, code in (
        (0, -1, "rows", 1), (1, (1 << 20) + 1, "vocab", 2), (2, 9, "row_stride", 1), (3, None, "logits", 1),
        (4, 3, "dtype", 1), (5, 0, "k must", 1), (5, 1025, "k=", 2), (6, None, "non-NULL", 1), (7, 5, "values_dtype", 1),
        (8, p + 4, "aligned", 1), (11, 0.0, "temperature", 1), (14, None, "non-NULL", 1), (14, p + 2, "aligned", 1),
        (16, None, "non-NULL", 1), (16, p + 1, "aligned", 1), (17, None, "workspace", 1), (18, 4, "workspace", 1),
    ):
        args = list(good)
        args[at] = value
        assert fn(*args) == code and word in error(lib), (at, value, error(lib))
    none = list(good)
    none[0], none[3] = 0, None
    assert fn(*none) == 0


def test_committed_profiles_match_the_kernel_sources():
    """profiles/logits_*.md name the digest of the kernel sources, comments
    aside, that they were made from."""
    import hashlib

    root = HEADER.parent.parent
    h = hashlib.sha256()
    for name in ("distill.hip", "select.hip", "logits.hpp"):
        text = re.sub(r"/\*.*?\*/", " ", (root / "tropnn_amd" / "csrc" / name).read_text(), flags=re.S)
        h.update(" ".join(re.sub(r"//[^\n]*", " ", text).split()).encode())
    profiles = sorted((root / "profiles").glob("logits_*.md"))
    assert [p.stem for p in profiles] == ["logits_counters", "logits_kernel_trace"]
    for p in profiles:
        assert h.hexdigest() in p.read_text(), f"{p.name} was made from other kernel sources"
