"""FusedAdam / FusedAdamW with 8-bit states against a 64-bit form of the same
step, from the states that the kernel itself left, one step at a time.

Tolerances (u = 2^-24): m and u are a few f32 operations from the codes, which are
exact, so they are within 4 u of the sum of their terms' sizes; a code is at least
8 of its steps, so the value in steps is within 64 u (|b1 m0| + |w1 g|) / |m| of
the 64-bit one, and a code may differ, by one step, where that reaches the random
number's threshold. p's step carries the relative errors of m, u and the division:
16 u of lr / (1 - b1^t) times the terms' size over the denominator, and u of p."""
from __future__ import annotations

import copy
import math

import pytest
import torch

from tropnn_amd import FusedAdam, FusedAdamW
from tropnn_amd.optim import adam8_step_hip

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0**-24
BLOCK = 32
E4M3 = torch.float8_e4m3fn


def random_of(n: int, t: int, first: int = 0) -> torch.Tensor:
    low = 0xFFFFFFFF
    x = ((torch.arange(first, first + n, dtype=torch.int64) & low) * 0x9E3779B9 + t * 0xBB67AE85) & low
    x = ((x ^ (x >> 16)) * 0x6A09E667) & low
    x = ((x ^ (x >> 15)) * 0x3C6EF373) & low
    return x ^ (x >> 16)


def value(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """What a state stands for, flat, in 64 bits."""
    flat = codes.detach().cpu().flatten().view(E4M3).double()
    units = torch.exp2(exponents.detach().cpu().double() - 127).repeat_interleave(BLOCK)[: len(flat)]
    return flat * units


def step_size_of(codes, exponents):
    """The distance from a held value to the next one up, flat."""
    flat = codes.detach().cpu().flatten().view(E4M3).double().abs()
    units = torch.exp2(exponents.detach().cpu().double() - 127).repeat_interleave(BLOCK)[: len(flat)]
    return torch.exp2(torch.floor(torch.log2(flat.clamp(min=2.0**-6))) - 3) * units


def check_held(codes, exponents, want, off, random16, what, *, root):
    """The state holds `want` (within `off`) rounded by the random numbers, in the
    least exponents that take every block."""
    n = len(want)
    pad = -n % BLOCK
    blocks = torch.nn.functional.pad(want.abs(), (0, pad)).view(-1, BLOCK)
    slack = torch.nn.functional.pad(off, (0, pad)).view(-1, BLOCK)
    fraction, k = torch.frexp(blocks.amax(1))
    exponent = (k - 9 + (fraction > 0.875).int()).clamp(min=-127) + 127
    exponent = torch.where(blocks.amax(1) > 0, exponent, 0)
    got = exponents.detach().cpu().int()
    near = ((blocks.amax(1) - 448 * torch.exp2(torch.floor(torch.log2(blocks.amax(1).clamp(min=1e-300) / 448)) + 0)).abs()
            <= slack.amax(1)) | ((got - exponent).abs() == 0)
    assert near.all(), (what, "exponents")
    unit = torch.exp2(got.double() - 127).repeat_interleave(BLOCK)[:n]
    x = want.abs() / unit
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0**-6))) - 3)
    r = (random16.double() + 0.5) / 65536
    lowest, highest = (torch.floor((x + s * off / unit).clamp(min=0) / step + r) * step for s in (-1.0, 1.0))
    if root:
        lowest, highest = (torch.where(want > 0, v.clamp(min=2.0**-9), v) for v in (lowest, highest))
    held = value(codes, exponents).abs() / unit
    assert ((held >= lowest) & (held <= highest)).all(), (what, held, lowest, highest)
    sign = value(codes, exponents).sign()
    assert ((sign == want.sign()) | (sign == 0)).all(), what
    # random bits below the 20 that are there move a threshold by 2^-20 of a step at most, far below `off` elsewhere
    assert (lowest == highest).double().mean() > 0.99, what


def reference_step(p, g, state, t, group):
    b1, b2 = group["betas"]
    lr, eps, wd = group["lr"], group["eps"], group["weight_decay"]
    p, g = p.detach().cpu().flatten().double(), g.detach().cpu().flatten().double()
    m0, u0 = value(state["exp_avg_8bit"], state["exp_avg_exponents"]), value(state["root_8bit"], state["root_exponents"])
    size = p.abs()
    if wd and group["decoupled_weight_decay"]:
        p = p * (1 - lr * wd)
    g_off = torch.zeros_like(g)
    if wd and not group["decoupled_weight_decay"]:
        g_off = 2 * U * (g.abs() + wd * p.abs())
        g = g + wd * p
    m = b1 * m0 + (1 - b1) * g
    u = torch.sqrt(b2 * u0 * u0 + (1 - b2) * g * g)
    m_off = 4 * U * (b1 * m0.abs() + (1 - b1) * g.abs()) + (1 - b1) * g_off + 1e-44
    u_off = 4 * U * u + math.sqrt(1 - b2) * g_off + 1e-22 * ((u > 0) & (u < 1e-17))  # squares below f32's smallest numbers
    denominator = u / math.sqrt(1 - b2**t) + eps
    lr_t = lr / (1 - b1**t)
    step = lr_t * m / denominator
    p_off = 4 * U * size + 8 * U * step.abs() + lr_t * (m_off / denominator + m.abs() / denominator**2 * u_off / math.sqrt(1 - b2**t))
    return p - step, p_off, m, m_off, u, u_off


def check_step(opt):
    """One step of the optimizer against the reference, for every parameter with a gradient."""
    before = []
    for group in opt.param_groups:
        for p in group["params"]:
            if p.grad is None:
                continue
            state = opt.state[p] if opt.state[p] else opt._new_state(p, 8)
            t = int(state["step"]) + 1
            before.append((p, group, t, reference_step(p, p.grad, state, t, group)))
    opt.step()
    torch.cuda.synchronize()
    for p, group, t, (want, off, m, m_off, u, u_off) in before:
        state = opt.state[p]
        assert float(state["step"]) == t
        assert state["exp_avg_8bit"].dtype == E4M3 and state["exp_avg_8bit"].shape == p.shape
        if p.numel() == 0:
            continue
        got = p.detach().cpu().flatten().double()
        assert ((got - want).abs() <= off).all(), float(((got - want).abs() - off).max())
        random = random_of(p.numel(), t)
        check_held(state["exp_avg_8bit"], state["exp_avg_exponents"], m, m_off, random & 0xFFFF, "exp_avg", root=False)
        check_held(state["root_8bit"], state["root_exponents"], u, u_off, random >> 16, "root", root=True)


def parameters(shapes, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(DEV)) for s in shapes]


def give_gradients(params, seed, scale=1.0):
    """Rows of very different sizes, some without a gradient."""
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        n = p.numel()
        rows = torch.exp(2 * torch.randn(-(-n // 50), 1, generator=gen)) * (torch.rand(-(-n // 50), 1, generator=gen) < 0.8)
        g = torch.randn(n, generator=gen) * rows.expand(-1, 50).flatten()[:n] * scale
        p.grad = g.view(p.shape).to(DEV)


SHAPES = [(136, 64, 128), (136, 6), (7,), (1,), (3, 5), (0,), (1025,), (31,), (32,), (33,), (4099,), ()]


@pytest.mark.parametrize("cls,kw,scale", [
    (FusedAdamW, dict(lr=1e-2, weight_decay=0.05), 1.0),
    (FusedAdam, dict(lr=1e-3), 1.0),
    (FusedAdam, dict(lr=3e-2, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.1), 1.0),
    (FusedAdamW, dict(lr=1e-3, betas=(0.0, 0.5)), 1e-6),
    (FusedAdam, dict(lr=1e-1, eps=1e-3), 1e3),
])
def test_steps(cls, kw, scale):
    params = parameters(SHAPES, 7)
    opt = cls(params, state_bits=8, **kw)
    for step in range(4):
        give_gradients(params, 100 + step, scale)
        if step == 1:
            params[3].grad = params[9].grad = None
        check_step(opt)
    assert float(opt.state[params[3]]["step"]) == 3 and float(opt.state[params[0]]["step"]) == 4


@pytest.mark.parametrize("count", [49, 50, 51, 257, 300])
def test_many_tensors(count):
    """More tensors than one launch takes, and than one launch counts."""
    params = parameters([(1 + (k * 37) % 90,) for k in range(count)], 3)
    opt = FusedAdamW(params, lr=1e-2, state_bits=8)
    for step in range(2):
        give_gradients(params, 5 + step)
        check_step(opt)


@pytest.mark.parametrize("shift", [1, 2, 3, 4])
def test_parameters_inside_a_buffer(shift):
    """Parameters and gradients off 16-byte boundaries; what lies around them stays."""
    n = 3001
    flat, grads = torch.full((n + 16,), 7.0, device=DEV), torch.full((n + 16,), 5.0, device=DEV)
    gen = torch.Generator().manual_seed(shift)
    p = torch.nn.Parameter(flat[shift:shift + n])
    with torch.no_grad():
        p.copy_(torch.randn(n, generator=gen))
    p.grad = grads[shift:shift + n].copy_(torch.randn(n, generator=gen))
    opt = FusedAdamW([p], lr=1e-2, state_bits=8)
    for _ in range(2):
        check_step(opt)
    assert (flat[:shift] == 7).all() and (flat[shift + n:] == 7).all()
    # states off 4-byte boundaries, as a loaded one may lie
    state = opt.state[p]
    for key in ("exp_avg_8bit", "root_8bit", "exp_avg_exponents", "root_exponents"):
        held = state[key].view(torch.uint8)
        wide = torch.full((held.numel() + 8,), 9, dtype=torch.uint8, device=DEV)
        wide[shift:shift + held.numel()] = held
        state[key] = wide[shift:shift + held.numel()].view(state[key].dtype)
        state[key + "_around"] = wide
    check_step(opt)
    for key in ("exp_avg_8bit", "root_8bit", "exp_avg_exponents", "root_exponents"):
        wide, held = state[key + "_around"], state[key].numel()
        assert (wide[:shift] == 9).all() and (wide[shift + held:] == 9).all()


def test_zero_gradients_and_zero_states():
    p = torch.nn.Parameter(torch.ones(100, device=DEV))
    opt = FusedAdam([p], lr=1e-2, state_bits=8)
    p.grad = torch.zeros_like(p)
    for _ in range(3):
        opt.step()
    assert (p == 1).all()
    for key, t in opt.state[p].items():
        assert key == "step" or int(t.view(torch.uint8).count_nonzero()) == 0
    p.grad[40] = 1.0  # one element of a block of zeros
    check_step(opt)
    assert int((p != 1).sum()) == 1
    check_step(opt)
    assert int((p != 1).sum()) == 1


def test_a_root_does_not_become_zero():
    """An element 1e9 below its block's largest keeps a root, so its first moment
    meets no denominator of eps alone."""
    p = torch.nn.Parameter(torch.zeros(64, device=DEV))
    opt = FusedAdam([p], lr=1e-3, eps=1e-30, state_bits=8)
    p.grad = torch.full_like(p, 1e-9)
    p.grad[::32] = 1.0
    for _ in range(20):
        before = p.detach().clone()
        opt.step()
        assert float((p.detach() - before).abs().max()) <= 2e-2
    assert (opt.state[p]["root_8bit"].float() > 0).all()


def test_very_small_and_very_large_gradients():
    """Exponents at both ends of their range: squares within f32's range are held,
    moments below 2^-127 too."""
    for size in (1e-37, 3e-30, 1e-18, 1e17):
        p = torch.nn.Parameter(torch.zeros(96, device=DEV))
        opt = FusedAdam([p], lr=1e-3, state_bits=8)
        p.grad = torch.randn(96, generator=torch.Generator().manual_seed(1)).to(DEV) * size
        opt.step()
        state = opt.state[p]
        m = value(state["exp_avg_8bit"], state["exp_avg_exponents"])
        want = 0.1 * p.grad.cpu().double()
        assert ((m - want).abs() <= step_size_of(state["exp_avg_8bit"], state["exp_avg_exponents"]) * 1.001 + 2.0**-136).all(), size
        assert torch.isfinite(p).all()
        # squares below f32's smallest numbers are in steps of 2^-149: roots in steps of 2^-74
        root = value(state["root_8bit"], state["root_exponents"])
        want = math.sqrt(1 - 0.999) * p.grad.cpu().double().abs()
        step = step_size_of(state["root_8bit"], state["root_exponents"])
        assert ((root - want).abs() <= step * 1.001 + 2.0**-73).all(), size


def test_no_eps():
    """A root of 0 stands in no denominator: its element has no first moment either."""
    p = torch.nn.Parameter(torch.ones(64, device=DEV))
    opt = FusedAdam([p], lr=1e-2, eps=0.0, state_bits=8)
    p.grad = torch.zeros_like(p)
    p.grad[3], p.grad[40] = 2.0, 1e-30
    opt.step()
    want = torch.ones(64)
    want[3] = 0.99
    assert torch.isfinite(p).all()
    keep = torch.arange(64) != 40
    assert torch.allclose(p.detach().cpu()[keep], want[keep], rtol=1e-6, atol=0)


def test_gradients_that_are_not_finite():
    """A NaN or an infinity stays with its element; its block's others are as without it."""
    def run(bad):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 200, device=DEV))
        opt = FusedAdamW([p], lr=1e-2, state_bits=8)
        for step in range(3):
            give_gradients([p], 50 + step)
            p.grad[7] = 0.0
            if step == 1 and bad is not None:
                p.grad[7] = bad
            opt.step()
        return p.detach(), opt.state[p]

    want, state = run(None)
    keep = torch.arange(200, device=DEV) != 7
    for bad in (math.nan, math.inf, -math.inf):
        p, other = run(bad)
        assert torch.isnan(p[7]) and torch.equal(p[keep], want[keep])
        for key in ("exp_avg_8bit", "root_8bit"):
            assert torch.isnan(other[key].float()[7])
            assert torch.equal(other[key].view(torch.uint8)[keep], state[key].view(torch.uint8)[keep])
        assert torch.equal(other["exp_avg_exponents"], state["exp_avg_exponents"])


def test_the_expected_value_is_kept():
    """2^16 elements with one gradient: their states' mean follows the 32-bit average
    over 300 steps. A step adds to an element's error one rounding of at most a code's
    step, variance step^2 / 4, forgotten at 1 - beta a step: the error of one element
    has a deviation below step / (2 sqrt(1 - beta^2)), the mean's is 256 times less, and
    six of those are allowed. The root's curvature adds its variance over twice the
    root."""
    n, b1, b2 = 1 << 16, 0.95, 0.99
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = FusedAdam([p], lr=0.0, betas=(b1, b2), state_bits=8)
    gen = torch.Generator().manual_seed(3)
    m = v = 0.0
    for step in range(300):
        g = 0.3 + 0.1 * float(torch.randn((), generator=gen))
        p.grad = torch.full_like(p, g)
        opt.step()
        g = float(torch.tensor(g))
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    state = opt.state[p]
    for codes, exponents, want, beta in (("exp_avg_8bit", "exp_avg_exponents", m, b1), ("root_8bit", "root_exponents", math.sqrt(v), b2)):
        held = value(state[codes], state[exponents])
        step = float(step_size_of(state[codes], state[exponents]).max())
        one = step / (2 * math.sqrt(1 - beta * beta))
        assert abs(float(held.mean()) - want) <= 6 * one / 256 + (one * one / want if "root" in codes else 0.0), codes
        assert float(held.std()) <= one


def twins(seed=11, bits=8):
    shapes = SHAPES[:7]
    out = []
    for _ in range(2):
        params = parameters(shapes, seed)
        out.append((params, FusedAdamW(params, lr=1e-2, weight_decay=0.01, state_bits=bits)))
    return out


def assert_same(a, b, what=""):
    (ps, opt), (qs, other) = a, b
    for p, q in zip(ps, qs):
        assert torch.equal(p.detach(), q.detach()), what
        for key, t in opt.state[p].items():
            o = other.state[q][key]
            assert torch.equal(t.view(torch.uint8) if t.dtype == E4M3 else t, o.view(torch.uint8) if o.dtype == E4M3 else o), (what, key)


def test_graph_replays_and_streams_match_eager():
    cap, eag = twins()
    give_gradients(cap[0], 1)
    give_gradients(eag[0], 1)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        cap[1].step()  # on another stream, and outside the graph: makes the states
    torch.cuda.current_stream(DEV).wait_stream(side)
    eag[1].step()
    assert_same(cap, eag, "stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap[1].step()
    for rep in range(4):
        give_gradients(eag[0], 10 + rep)
        for p, q in zip(cap[0], eag[0]):
            p.grad.copy_(q.grad)
        graph.replay()
        eag[1].step()
        _ = torch.ones(1024, device=DEV).sum().item()
        torch.cuda.synchronize()
        assert_same(cap, eag, rep)


@pytest.mark.parametrize("where", ["cpu", "cuda:0"])
def test_state_dict_resumes_bit_for_bit(where):
    a, b = twins()
    for step in range(3):
        give_gradients(a[0], step)
        a[1].step()
    saved = copy.deepcopy(a[1].state_dict())
    for s in saved["state"].values():
        for key in s:
            s[key] = s[key].to(where)
    with torch.no_grad():
        for p, q in zip(a[0], b[0]):
            q.copy_(p)
    b[1].load_state_dict(saved)
    assert_same(a, b, "loaded")
    for x in (a, b):
        give_gradients(x[0], 9)
        x[1].step()
    assert_same(a, b, "resumed")


def test_states_of_other_bits_are_refused():
    p = torch.nn.Parameter(torch.ones(40, device=DEV))
    p.grad = torch.ones_like(p)
    for bits in (8, 32):
        opt = FusedAdam([p], state_bits=bits)
        opt.step()
        opt.param_groups[0]["state_bits"] = 40 - bits
        with pytest.raises(ValueError, match="state_bits"):
            opt.step()
    # a torch state dict is of 32 bits and goes on with them
    twin = torch.optim.Adam([p])
    twin.step()
    opt = FusedAdam([p], state_bits=8)
    opt.load_state_dict(twin.state_dict())
    opt.step()
    assert opt.state[p]["exp_avg"].dtype == torch.float32


def test_versions_are_bumped():
    p = torch.nn.Parameter(torch.ones(40, device=DEV))
    p.grad = torch.ones_like(p)
    opt = FusedAdamW([p], state_bits=8)
    opt.step()
    before = {k: t._version for k, t in opt.state[p].items()}, p._version
    opt.step()
    assert p._version > before[1] and all(t._version > before[0][k] for k, t in opt.state[p].items())


def test_refusals():
    def lists(n=40):
        codes = lambda: [torch.zeros(n, dtype=torch.uint8, device=DEV)]  # noqa: E731
        exponents = lambda: [torch.zeros(-(-n // 32), dtype=torch.uint8, device=DEV)]  # noqa: E731
        floats = lambda: [torch.zeros(n, device=DEV)]  # noqa: E731
        return [floats(), floats(), codes(), exponents(), codes(), exponents(), [torch.zeros((), device=DEV)]]

    kw = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, decoupled_weight_decay=False)
    adam8_step_hip(*lists(), **kw)
    adam8_step_hip(*([[]] * 7), **kw)
    for at, bad, kind, word in (
        (0, torch.zeros(40, device=DEV, dtype=torch.float64), TypeError, "params"),
        (1, torch.zeros(40), ValueError, "grads"),
        (1, torch.zeros(80, device=DEV)[::2], ValueError, "contiguous"),
        (1, torch.zeros(39, device=DEV), ValueError, "grads"),
        (2, torch.zeros(40, device=DEV), TypeError, "exp_avgs"),
        (2, torch.zeros(41, device=DEV, dtype=torch.uint8), ValueError, "exp_avgs"),
        (3, torch.zeros(1, device=DEV, dtype=torch.uint8), ValueError, "exp_avg_exponents"),
        (5, torch.zeros(3, device=DEV, dtype=torch.uint8), ValueError, "root_exponents"),
        (6, torch.zeros(2, device=DEV), ValueError, "steps"),
    ):
        args = lists()
        args[at] = [bad]
        with pytest.raises(kind, match=word):
            adam8_step_hip(*args, **kw)
    args = lists()
    args[4] = []
    with pytest.raises(ValueError, match="roots"):
        adam8_step_hip(*args, **kw)
    for bad in (dict(lr=-1.0), dict(beta1=1.0), dict(eps=math.nan)):
        with pytest.raises(ValueError):
            adam8_step_hip(*lists(), **{**kw, **bad})
    twice = [a + b for a, b in zip(lists(), lists())]
    twice[6][1] = twice[6][0]  # one counter for two tensors
    with pytest.raises(ValueError, match="steps"):
        adam8_step_hip(*twice, **kw)
    twice = [a + b for a, b in zip(lists(), lists())]
    twice[0][1] = twice[0][0]
    with pytest.raises(ValueError, match="params"):
        adam8_step_hip(*twice, **kw)


def test_a_tensor_past_one_grid_and_32_bits():
    """2^33 + 5000 elements, launched in two grids: the ends and the elements around
    2^32 and the grids' border are as those of a short tensor in their place."""
    n = (1 << 33) + 5000
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = torch.zeros(n, device=DEV)
    windows = [0, (1 << 32) - 512, (1 << 33) - 512, n - 1000]
    gen = torch.Generator().manual_seed(1)
    gradients = [torch.randn(1000, generator=gen) for _ in windows]
    for at, g in zip(windows, gradients):
        p.grad[at:at + 1000] = g.to(DEV)
    opt = FusedAdamW([p], lr=1e-2, state_bits=8)
    opt.step()
    state = opt.state[p]
    assert float(state["step"]) == 1.0
    for at, g in zip(windows, gradients):
        got = p.detach()[at:at + 1000].cpu()
        want = -1e-2 * g.double() / (g.double().abs() + 1e-8)
        assert float((got - want).abs().max()) <= 1e-7
        lo, hi = -(-at // 32) * 32, (at + 1000) // 32 * 32  # whole blocks
        inside = g[lo - at:hi - at].double()
        random = random_of(hi - lo, 1, lo)
        for codes, exponents, size, r, root in (("exp_avg_8bit", "exp_avg_exponents", 1 - 0.9, random & 0xFFFF, False),
                                                ("root_8bit", "root_exponents", math.sqrt(1 - 0.999), random >> 16, True)):
            v = inside * size if not root else inside.abs() * size
            check_held(state[codes][lo:hi], state[exponents][lo // 32:hi // 32], v, 8 * U * v.abs(), r, codes, root=root)
    assert int(torch.count_nonzero(p.detach()[2000:1 << 20])) == 0
    del p, opt, state
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cls,decay", [(FusedAdamW, 0.05), (FusedAdamW, 0.0), (FusedAdam, 0.1)])
def test_gradients_whose_squares_leave_f32(cls, decay):
    """From 1.85e19 on a gradient's square is infinite, and so is the root: the
    element takes no step beyond its decay, neither then nor later, as with 32
    bits (whose squares go on to 5.8e20). Looked at after the very step. An
    infinite gradient has no quotient, and neither has a NaN."""
    sizes = [1e17, 1e18, 1e19, 1.8e19, 1.9e19, 2e19, 1e20, 1e21, 1e25, 3e38, math.inf, math.nan]
    lr, b1, b2, eps = 1e-2, 0.9, 0.999, 1e-8
    gradients = torch.randn(2 * len(sizes), BLOCK, generator=torch.Generator().manual_seed(1))
    gradients[:, 5] = torch.tensor([s * v for v in sizes for s in (1.0, -1.0)])  # one in a block
    gradients = gradients.flatten()
    before = torch.linspace(-2, 2, len(gradients))
    p, q = (torch.nn.Parameter(before.to(DEV)) for _ in range(2))
    p.grad, q.grad = gradients.to(DEV), gradients.to(DEV)
    opt = cls([p], lr=lr, weight_decay=decay, state_bits=8)
    twin = cls([q], lr=lr, weight_decay=decay)
    opt.step()
    twin.step()
    kept, g = before.double(), gradients
    if cls is FusedAdamW:
        kept = kept * (1 - lr * decay)
    else:
        g = gradients + decay * before
    root = torch.sqrt((g * g).double() * (1 - b2))
    want = kept - lr / (1 - b1) * ((1 - b1) * g.double()) / (root / math.sqrt(1 - b2) + eps)
    infinite = torch.isinf(root) & torch.isfinite(g)
    assert int(infinite.sum()) == 12 and torch.equal(want[infinite], kept[infinite])
    got = p.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(want).sum()) == 4
    # the decay and the step are roundings of p and of the step, which is lr at most
    off = (got - want).abs() - U * (4 * before.abs() + 32 * lr)
    assert (off.nan_to_num(0.0) <= 0).all(), off
    alike = (g.abs() < 1e19) | (g.abs() > 6e20) | torch.isnan(g)
    assert torch.allclose(p.detach().cpu()[alike], q.detach().cpu()[alike], rtol=8 * U, atol=U * 32 * lr, equal_nan=True)
    state = opt.state[p]
    assert torch.equal(torch.isnan(state["root_8bit"].float().cpu()), infinite | ~torch.isfinite(g))
    assert torch.equal(torch.isnan(state["exp_avg_8bit"].float().cpu()), ~torch.isfinite(g))
    for step in range(3):
        held = p.detach().cpu().double()
        give_gradients([p], 20 + step)
        opt.step()
        want = held * (1 - lr * decay) if cls is FusedAdamW else held
        got = p.detach().cpu().double()
        assert ((got - want).abs() <= 2 * U * held.abs())[infinite].all(), step
        assert torch.equal(torch.isnan(got), ~torch.isfinite(g)), step


def test_loading_takes_no_more_memory_than_the_state():
    n = 1 << 24
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    saved = FusedAdam([p], state_bits=8)
    saved.state[p] = saved._new_state(p, 8)
    opt = FusedAdam([p], state_bits=8)
    state = saved.state_dict()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(DEV)
    torch.cuda.reset_peak_memory_stats(DEV)
    opt.load_state_dict(state)
    # two codes and two sixteenths of a byte an element, and what the allocator rounds up
    assert torch.cuda.max_memory_allocated(DEV) - before <= n * (2 + 2 / 32) + 4096
    p.grad = torch.ones_like(p)
    opt.step()
    assert int(saved.state[p]["root_8bit"].view(torch.uint8).count_nonzero()) == 0
