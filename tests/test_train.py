"""The operators that train a token model on its own answers without a GPU: no
CPU fallback, argument checks before any launch, the C ABI's own checks, and the
8-bit optimizer's host side."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from tropnn_amd import FusedAdam, FusedAdamW, policy_loss, preference_loss, token_log_probs
from tropnn_amd.backends import train_hip as th
from tropnn_amd.backends.logits_hip import LOGITS_DTYPES

HEADER = Path(__file__).resolve().parent.parent / "include" / "tropnn_hip_train.h"
F32, F16, BF16 = (LOGITS_DTYPES[t] for t in (torch.float32, torch.float16, torch.bfloat16))


@pytest.fixture(scope="module")
def lib():
    if not th.library_path().exists():
        pytest.skip("libtropnn_hip.so not built (run __graft_entry__.build())")
    return th.load_train_library()


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
    assert declared == sorted(th.TRAIN_SYMBOLS)
    assert lib.tropnn_hip_train_abi_version() == define("TROPNN_HIP_TRAIN_ABI_VERSION") == th.TRAIN_ABI_VERSION
    assert th.STATE_BLOCK == define("TROPNN_STATE_BLOCK")


def test_cpu_tensors_raise(lib):
    x, tokens, row = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(ValueError, match="GPU"):
        token_log_probs(x, tokens)
    with pytest.raises(ValueError, match="GPU"):
        policy_loss(x, tokens, row, row)
    with pytest.raises(ValueError, match="GPU"):
        preference_loss(torch.zeros(2, 3, 9), torch.zeros(2, 3, dtype=torch.int64))
    p = torch.nn.Parameter(torch.zeros(40))
    p.grad = torch.zeros(40)
    with pytest.raises(TypeError, match="GPU"):
        FusedAdamW([p], state_bits=8).step()
    codes, exponents = torch.zeros(40, dtype=torch.uint8), torch.zeros(2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        th.train_ops().adam8([p], [p.grad], [codes], [exponents], [codes], [exponents], [torch.zeros(())], 1e-3, 0.9, 0.999,
                             1e-8, 0.0, False)


class Fake:
    """A tensor's outside, as if it were on a GPU."""

    def __init__(self, shape, dtype=torch.float32):
        self.shape, self.dtype, self.ndim = torch.Size(shape), dtype, len(shape)
        self.device = torch.device("cuda:0")

    def detach(self):
        return self


def test_shapes_types_and_values_raise_before_launch():
    x, tokens, row = Fake((4, 9)), Fake((4,), torch.int64), Fake((4,))
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        token_log_probs(Fake((4, 9), torch.float64), tokens)
    with pytest.raises(TypeError, match="tokens"):
        token_log_probs(x, Fake((4,), torch.int32))
    with pytest.raises(ValueError, match="tokens"):
        token_log_probs(x, Fake((4, 1), torch.int64))
    with pytest.raises(ValueError, match="at least one class"):
        token_log_probs(Fake((4, 0)), tokens)
    with pytest.raises(NotImplementedError, match="classes"):
        token_log_probs(Fake((4, (1 << 20) + 1)), tokens)
    with pytest.raises(ValueError, match="temperature"):
        token_log_probs(x, tokens, temperature=0.0)
    for kw, word, kind in (
        (dict(old_log_probs=Fake((3,))), "old_log_probs", ValueError),
        (dict(old_log_probs=Fake((4,), torch.float16)), "old_log_probs", TypeError),
        (dict(advantages=Fake((1, 4))), "advantages", ValueError),
        (dict(ref_log_probs=Fake((4, 9))), "ref_log_probs", ValueError),
        (dict(weights=Fake((4,), torch.float64)), "weights", TypeError),
        (dict(clip=-0.1), "clip", ValueError),
        (dict(clip=(0.2, float("nan"))), "clip", ValueError),
        (dict(clip=(float("inf"), 0.2)), "clip", ValueError),
        (dict(kl_weight=float("inf")), "kl_weight", ValueError),
        (dict(temperature=-1.0), "temperature", ValueError),
        (dict(reduction="none"), "reduction", ValueError),
    ):
        with pytest.raises(kind, match=word):
            policy_loss(**{**dict(logits=x, tokens=tokens, old_log_probs=row, advantages=row), **kw})
    pairs, two = Fake((2, 3, 5, 9)), Fake((2, 3, 5), torch.int64)
    for kw, word, kind in (
        (dict(logits=Fake((2, 9)), tokens=Fake((2,), torch.int64)), "length", ValueError),
        (dict(logits=Fake((4, 5, 9)), tokens=Fake((4, 5), torch.int64)), "length", ValueError),
        (dict(tokens=Fake((2, 15), torch.int64)), "tokens", ValueError),
        (dict(reference=Fake((3,))), "reference", ValueError),
        (dict(reference=Fake((2, 3), torch.float64)), "reference", TypeError),
        (dict(weights=Fake((2, 3))), "weights", ValueError),
        (dict(beta=float("nan")), "beta", ValueError),
        (dict(margin=float("inf")), "margin", ValueError),
        (dict(label_smoothing=1.5), "label_smoothing", ValueError),
        (dict(label_smoothing=float("nan")), "label_smoothing", ValueError),
        (dict(reduction="none"), "reduction", ValueError),
    ):
        with pytest.raises(kind, match=word):
            preference_loss(**{**dict(logits=pairs, tokens=two), **kw})


P = 4096  # an address that is never read: every call below ends before a launch
ROWS = [2, 10, 10, P, F32, P, 1.0]
BAD_ROWS = ((0, -1, "rows", 1), (0, 1 << 31, "rows", 1), (1, 0, "vocab", 1), (1, (1 << 20) + 1, "vocab", 2),
            (2, 9, "row_stride", 1), (3, None, "logits", 1), (3, P + 2, "aligned", 1), (4, 3, "dtype", 1),
            (5, None, "tokens", 1), (5, P + 4, "aligned", 1), (6, 0.0, "temperature", 1), (6, float("nan"), "temperature", 1),
            (6, float("inf"), "temperature", 1), (6, 1e-39, "temperature", 1))


def refuses(lib, fn, good, cases):
    for at, value, word, code in cases:
        args = list(good)
        args[at] = value
        assert fn(*args) == code and word in error(lib), (at, value, error(lib))


def test_abi_refuses_bad_arguments_of_rows(lib):
    fn, good = lib.tropnn_hip_token_log_probs, [*ROWS, P, None, P, None]
    refuses(lib, fn, good, (*BAD_ROWS, (7, None, "log_probs", 1), (7, P + 2, "aligned", 1), (8, P + 4, "aligned", 1),
                            (9, P + 4, "aligned", 1)))
    assert fn(0, 10, 10, None, F32, None, 1.0, None, None, None, None) == 0

    fn, good = lib.tropnn_hip_token_gradient, [*ROWS, P, P, 1, P, P, 0, P, None]
    refuses(lib, fn, good, (*BAD_ROWS, (7, None, "non-NULL", 1), (7, P + 4, "aligned", 1), (8, None, "non-NULL", 1),
                            (8, P + 2, "aligned", 1), (9, 0, "rows_per_coef", 1), (10, P + 2, "aligned", 1),
                            (11, P + 2, "aligned", 1), (13, None, "non-NULL", 1), (13, P + 1, "aligned", 1)))
    assert fn(0, 10, 10, None, F32, None, 1.0, None, None, 1, None, None, 0, None, None) == 0


def test_abi_refuses_bad_arguments_of_the_losses(lib):
    fn = lib.tropnn_hip_policy
    good = [*ROWS, P, P, P, P, 0.2, 0.2, 0.1, 1.0, 1, P, P, P, P, P, None, P, 1 << 20, None]
    refuses(lib, fn, good, (*BAD_ROWS, (7, None, "non-NULL", 1), (7, P + 2, "aligned", 1), (8, None, "non-NULL", 1),
                            (9, P + 1, "aligned", 1), (10, P + 2, "aligned", 1), (11, -0.1, "low", 1),
                            (12, float("nan"), "low", 1), (16, None, "loss", 1), (17, None, "non-NULL", 1),
                            (18, None, "non-NULL", 1), (19, None, "norm", 1), (20, None, "non-NULL", 1),
                            (20, P + 4, "aligned", 1), (21, P + 1, "aligned", 1), (22, None, "workspace", 1),
                            (22, P + 8, "workspace", 1), (23, 4, "workspace", 1)))
    if not lib.tropnn_hip_policy_grad_fits(2, 1 << 20, F32):
        wide = list(good)
        wide[1] = wide[2] = 1 << 20
        wide[21] = P
        assert fn(*wide) == 2 and "gradient" in error(lib)

    fn = lib.tropnn_hip_preference
    good = [3, 5, P, P, P, P, 0.1, 0.0, 0.0, 0, 1.0, 1, P, P, P, P, P, 1 << 20, None]
    refuses(lib, fn, good, ((0, -1, "pairs", 1), (1, -1, "length", 1), (1, 1 << 31, "length", 1), (2, None, "non-NULL", 1),
                            (2, P + 4, "aligned", 1), (3, None, "non-NULL", 1), (3, P + 4, "aligned", 1), (4, P + 2, "aligned", 1),
                            (5, P + 2, "aligned", 1), (8, 1.5, "smoothing", 1), (8, float("nan"), "smoothing", 1),
                            (12, None, "loss", 1), (13, None, "non-NULL", 1), (14, None, "non-NULL", 1),
                            (14, P + 2, "aligned", 1), (15, None, "norm", 1), (16, None, "workspace", 1),
                            (17, 4, "workspace", 1)))


def test_abi_refuses_bad_arguments_of_the_step(lib):
    fn = lib.tropnn_hip_adam8_step

    def call(pointers=(P,) * 6, step=P, numel=40, n=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, ws=P, size=1 << 10):
        arrays = [(ctypes.c_void_p * 1)(p) for p in (*pointers, step)]
        return fn(n, *arrays[:6], (ctypes.c_int64 * 1)(numel), arrays[6], lr, b1, b2, eps, wd, 1, ws, size, None)

    for kw, word in ((dict(n=-1), "n_tensors"), (dict(lr=-1.0), "lr"), (dict(b1=1.0), "beta1"), (dict(b2=-0.1), "beta2"),
                     (dict(eps=float("nan")), "eps"), (dict(wd=-1.0), "weight_decay"), (dict(numel=-1), "numels"),
                     (dict(step=None), "steps"), (dict(step=P + 2), "steps"), (dict(ws=None), "workspace"),
                     (dict(size=4), "workspace"), (dict(pointers=(P + 2, P, P, P, P, P)), "aligned"),
                     *((dict(pointers=tuple(None if j == k else P for j in range(6))), "NULL") for k in range(6))):
        assert call(**kw) == 1 and word in error(lib), (kw, error(lib))
    assert fn(0, *([None] * 6), None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, None) == 0


def test_workspace_queries(lib):
    assert lib.tropnn_hip_policy_workspace_size(100, 1000, F32, 1) >= 400
    assert lib.tropnn_hip_policy_workspace_size(100, 0, F32, 1) == 0 and "vocab" in error(lib)
    assert lib.tropnn_hip_preference_workspace_size(10, 7) >= 40
    assert lib.tropnn_hip_preference_workspace_size(-1, 7) == 0 and "pairs" in error(lib)
    assert lib.tropnn_hip_adam8_workspace_size(7) >= 56 and lib.tropnn_hip_adam8_workspace_size(0) == 0
    assert lib.tropnn_hip_policy_grad_fits(4, -1, F32) == 0 and "vocab" in error(lib)


def test_state_bits_of_the_optimizers():
    p = torch.nn.Parameter(torch.zeros(5))
    for cls in (FusedAdam, FusedAdamW):
        assert cls([p]).param_groups[0]["state_bits"] == 32
        assert cls([p], state_bits=8).param_groups[0]["state_bits"] == 8
        for bits in (16, 0, "8"):
            with pytest.raises(ValueError, match="state_bits"):
                cls([p], state_bits=bits)
        with pytest.raises(ValueError, match="state_bits"):
            p.grad = torch.zeros(5)
            cls([{"params": [p], "state_bits": 16}]).step()


def with_state(bits: int, n: int = 70) -> FusedAdam:
    """An optimizer with a state, as a step leaves one."""
    p = torch.nn.Parameter(torch.zeros(n))
    opt = FusedAdam([p], state_bits=bits)
    state = opt._new_state(p, bits)
    gen = torch.Generator().manual_seed(n)
    for key, t in state.items():
        if t.dtype in (torch.uint8, torch.float8_e4m3fn):
            t.view(torch.uint8).copy_(torch.randint(0, 127, t.shape, generator=gen, dtype=torch.uint8))
    state["step"].fill_(3.0)
    opt.state[p] = state
    return opt


def test_a_saved_8_bit_state_keeps_its_bits():
    """torch's loader casts state to the parameter's type; a code's byte and an
    exponent's come back as they were."""
    opt = with_state(8)
    want = next(iter(opt.state.values()))
    assert want["exp_avg_8bit"].shape == (70,) and want["root_exponents"].shape == (3,)
    other = FusedAdam([torch.nn.Parameter(torch.zeros(70))])  # 32 bits until it loads
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["state_bits"] == 8
    got = next(iter(other.state.values()))
    assert set(got) == set(want)
    for key in want:
        assert got[key].dtype == want[key].dtype
        assert torch.equal(got[key].view(torch.uint8) if got[key].dim() else got[key],
                           want[key].view(torch.uint8) if want[key].dim() else want[key]), key


def test_a_torch_state_keeps_32_bits():
    p = torch.nn.Parameter(torch.ones(4))
    opt = torch.optim.Adam([p])
    p.grad = torch.ones(4)
    opt.step()
    ours = FusedAdam([torch.nn.Parameter(torch.ones(4))], state_bits=8)
    ours.load_state_dict(opt.state_dict())
    assert ours.param_groups[0]["state_bits"] == 32
    assert next(iter(ours.state.values()))["exp_avg"].dtype == torch.float32


def test_committed_profiles_match_the_kernel_sources():
    """profiles/train_*.md name the digest of the kernel sources, comments
    aside, that they were made from."""
    import hashlib

    root = HEADER.parent.parent
    h = hashlib.sha256()
    for name in ("policy.hip", "adam8.hip", "train.hpp", "logits.hpp"):
        text = re.sub(r"/\*.*?\*/", " ", (root / "tropnn_amd" / "csrc" / name).read_text(), flags=re.S)
        h.update(" ".join(re.sub(r"//[^\n]*", " ", text).split()).encode())
    profiles = sorted((root / "profiles").glob("train_*.md"))
    assert [p.stem for p in profiles] == ["train_counters", "train_kernel_trace"]
    for p in profiles:
        assert h.hexdigest() in p.read_text(), f"{p.name} was made from other kernel sources"


def test_loading_an_8_bit_state_leaves_its_types_alone():
    """Hooks around the loading see codes and exponents in their own types: they are
    never widened, which would take 8 bytes a parameter for a state of 2. What is
    loaded is the optimizer's own."""
    opt = with_state(8)
    saved = opt.state_dict()
    other = FusedAdam([torch.nn.Parameter(torch.zeros(70))])
    seen = []

    def note(states):
        seen.append({key: (t.dtype, t.shape) for s in states for key, t in s.items()})

    handles = (other.register_load_state_dict_pre_hook(lambda o, s: note(s["state"].values())),
               other.register_load_state_dict_post_hook(lambda o: note(o.state.values())))
    for _ in range(2):  # the second time over a state
        other.load_state_dict(saved)
    for handle in handles:
        handle.remove()
    want = next(iter(opt.state.values()))
    assert seen == [{key: (t.dtype, t.shape) for key, t in want.items()}] * 4
    got = next(iter(other.state.values()))
    for key in want:
        if key != "step":
            assert got[key].data_ptr() != want[key].data_ptr()
    # as a tool may have saved it: widened
    wide = {"param_groups": saved["param_groups"], "state": {0: {k: t.float() for k, t in want.items()}}}
    other.load_state_dict(wide)
    got = next(iter(other.state.values()))
    for key in want:
        assert got[key].dtype == want[key].dtype and torch.equal(got[key].float(), want[key].float())
    with pytest.raises(ValueError, match="parameter group"):
        other.load_state_dict({"param_groups": [], "state": {}})
    assert not other._optimizer_load_state_dict_pre_hooks and not other._optimizer_load_state_dict_post_hooks
