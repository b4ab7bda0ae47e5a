"""The thresholds that 8-bit moments are rounded against: for element i at step t the upper 20 bits of i * phase + t * turn modulo
2^32, with phase = 2^32 times the fraction of the golden ratio (m) or of sqrt(2) (sqrt(v)) and turn = 2^32 / rho or 2^32 / rho^2
for the plastic number rho (rho^3 = rho + 1).  Codes, powers and weights are checked with the bounds of tests/test_adamw_gpu.py."""
import math

import pytest
import torch

from fsgs_amd.optim import FusedAdamW

from tests.test_adamw_gpu import DEV, DTYPES, E32, HALF, SIZES, TINY, check_codes, close, make, step64, values, wide

pytestmark = pytest.mark.gpu
GOLDEN, ROOT2 = 0x9E3779B9, 0x6A09E667
RHO_1, RHO_2 = 0xC13FA9A9, 0x91E10DA5


def test_the_constants_are_what_they_are_said_to_be():
    rho = 1.0
    for _ in range(60):
        rho = (1.0 + rho) ** (1.0 / 3.0)
    for word, x in ((GOLDEN, (math.sqrt(5) - 1) / 2), (ROOT2, math.sqrt(2) - 1), (RHO_1, 1 / rho), (RHO_2, 1 / rho ** 2)):
        assert abs(word - 2.0 ** 32 * x) <= 1.0


def thresholds(n, step, phase, turn, first=0):
    i = torch.arange(first, first + n, dtype=torch.int64)
    return (((i * phase + step * turn % 2 ** 32) % 2 ** 32) >> 12).double() / 2 ** 20


def check_step(opt, ps, before, grads, lr, wd, eps, b2, first=0):
    """every parameter, power and code after a step from the values in `before` = [(w, m, v)] in 64 bits"""
    for p, (w, m, v), g in zip(ps, before, grads):
        st = opt.state[p]
        t, n = st["step"], p.numel()
        w1, m1, v1, tw, tm, _ = step64(w, g, m, v, t, lr, 0.9, b2, eps, wd)
        if "master" in st:
            close(st["master"], w1, tw, "master")
            assert torch.equal(p.detach(), st["master"].to(p.dtype))
        else:
            close(p, w1, tw + HALF[p.dtype] * (w1.abs() + tw) + TINY[p.dtype], "w")
        check_codes(st["exp_avg_q"].view(torch.uint8), st["scales"][:, 0], m1, tm, thresholds(n, t, GOLDEN, RHO_1, first), False,
                    "m, %d elements, step %d" % (n, t))
        check_codes(st["exp_avg_sq_q"].view(torch.uint8), st["scales"][:, 1], v1.sqrt(), 5 * E32 * v1.sqrt(),
                    thresholds(n, t, ROOT2, RHO_2, first), True, "r, %d elements, step %d" % (n, t))


def held(opt, p):
    st, n = opt.state[p], p.numel()
    return (wide(st["master"] if "master" in st else p), values(st["exp_avg_q"], st["scales"][:, 0], n),
            values(st["exp_avg_sq_q"], st["scales"][:, 1], n) ** 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masters,wd", [(False, 0.1), (True, 0.0)])
def test_codes_of_every_type_and_size(dtype, masters, wd):
    ps, gs = make(SIZES, dtype, seed=3)
    zero = [torch.zeros(p.shape, dtype=torch.float64) for p in ps]
    opt = FusedAdamW(ps, lr=1e-3, eps=1e-8, weight_decay=wd, state_bits=8, master_weights=masters)
    for step in range(3):
        for p, g in zip(ps, gs):
            p.grad = (g.float() * (3 - step)).to(dtype)
        before = [held(opt, p) for p in ps] if step else [(wide(p), z, z) for p, z in zip(ps, zero)]
        opt.step()
        check_step(opt, ps, before, [wide(p.grad) for p in ps], 1e-3, wd, 1e-8, 0.999)


@pytest.mark.parametrize("start", [0, 3998, 2 ** 20 + 7, 2 ** 32 - 2, 2 ** 33 + 5])
def test_codes_over_many_steps(start):
    """thirty steps from any count on (a count times the turn passes 32 bits at once, a count itself in the last two), a part of
    the gradients zero"""
    (p,), (g,) = make([2500], torch.float32, seed=start % 97)
    opt = FusedAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8, betas=(0.9, 0.99))
    gen = torch.Generator().manual_seed(4)
    opt.set_moments(p, g * 0.1, g * g + 1e-6, start)
    for _ in range(30):
        p.grad = g * (torch.rand(2500, generator=gen) < 0.3).to(DEV)
        before = [held(opt, p)]
        opt.step()
        check_step(opt, [p], before, [wide(p.grad)], 1e-3, 0.0, 1e-8, 0.99)
    assert opt.state[p]["step"] == start + 30


def test_codes_of_a_captured_step():
    """the count on the device gives the same thresholds"""
    ps, gs = make([300, 4097], torch.float32, seed=9)
    opt = FusedAdamW(ps, lr=1e-3, weight_decay=0.0, state_bits=8, capturable=True)
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        torch.cuda.synchronize()
        before = [held(opt, p) for p in ps]
        graph.replay()
        torch.cuda.synchronize()
        for p, (w, m, v), g in zip(ps, before, gs):
            st, n, t = opt.state[p], p.numel(), k + 2
            assert float(st["step"]) == t
            _, m1, v1, _, tm, _ = step64(w, wide(g), m, v, t, 1e-3, 0.9, 0.999, 1e-8, 0.0)
            check_codes(st["exp_avg_q"].view(torch.uint8), st["scales"][:, 0], m1, tm, thresholds(n, t, GOLDEN, RHO_1), False, "m")
            check_codes(st["exp_avg_sq_q"].view(torch.uint8), st["scales"][:, 1], v1.sqrt(), 5 * E32 * v1.sqrt(),
                        thresholds(n, t, ROOT2, RHO_2), True, "r")


def without_gradients(r, d, first, steps):
    """sqrt(v) in 64 bits after `steps` steps of rounding r (1 - d)"""
    i = torch.arange(r.numel(), dtype=torch.int64)
    for t in range(first + 1, first + 1 + steps):
        r = r * (1 - d)
        _, ex = torch.frexp(r.view(-1, 128).amax(1) / 448)  # blocks' powers: 448 2^e is at least the largest value
        unit = (2.0 ** ex.double()).repeat_interleave(128)
        unit = torch.where((r.view(-1, 128).amax(1) / 448 == 2.0 ** (ex - 1.0)).repeat_interleave(128), unit / 2, unit)
        y = r / unit
        _, ex = torch.frexp(y.clamp(min=2.0 ** -6))
        grain = 2.0 ** (ex - 4.0)
        u = (((i * ROOT2 + t * RHO_2 % 2 ** 32) % 2 ** 32) >> 12).double() / 2 ** 20
        r = (torch.floor(y / grain + u) * grain).clamp(min=2.0 ** -9) * unit
    return r


def test_a_second_moment_without_gradients():
    """1500 steps against the definition in 64 bits.  A step's root is off by 3 roundings of up to 16 grains and the threshold by its
    last bit: 2 (48 / 2^24 + 1 / 2^20) = 8e-6 of the decisions may differ, 1.2 % of the elements over 1500 steps, each by
    about a code, 1/8 at most, from there on."""
    n, T, b2 = 8192, 1500, 0.999
    p = torch.zeros(n, device=DEV, requires_grad=True)
    opt = FusedAdamW([p], lr=0.0, betas=(0.9, b2), state_bits=8)
    opt.set_moments(p, torch.zeros(n, device=DEV), torch.exp(torch.randn(n, generator=torch.Generator().manual_seed(2))).to(DEV), 0)
    start = wide(opt.moments()[0][1]).sqrt()
    p.grad = torch.zeros(n, device=DEV)
    for _ in range(T):
        opt.step()
    got = wide(opt.moments()[0][1]).sqrt()
    want = without_gradients(start, 1 - math.sqrt(b2), 0, T)
    assert float((got != want).double().mean()) < 0.012
    assert float(((got - want).abs() / want).max()) < 0.3 and abs(float((got / want).mean()) - 1) < 0.012 / 8


def test_offsets_over_32_bits():
    """one bf16 tensor of 2^31 + 4099 elements (13 GB in all with 8-bit moments, 26 GB with 32-bit ones): gradients in its last
    elements alone"""
    n, tail = 2 ** 31 + 4099, 4099
    p = torch.zeros(n, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g = torch.randn(tail, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    p.grad[n - tail:] = g
    norm = math.sqrt(float((wide(g) ** 2).sum()))
    m1 = 0.1 * wide(g) / (norm + 1e-6)
    for bits in (8, 32):
        with torch.no_grad():
            p.zero_()
        opt = FusedAdamW([p], state_bits=bits, max_grad_norm=1.0, lr=1e-2)
        opt.step()
        assert abs(float(opt.last_grad_norm) - norm) <= 2 * E32 * norm
        st = opt.state[p]
        if bits == 8:
            check_codes(st["exp_avg_q"].view(torch.uint8)[n - tail:], st["scales"][(n - tail) // 128:, 0], m1, 12 * E32 * m1.abs(),
                        thresholds(tail, 1, GOLDEN, RHO_1, n - tail), False, "m")
            assert not bool(st["exp_avg_q"].view(torch.uint8)[:n - tail].any())
        else:
            close(st["exp_avg"][n - tail:], m1, 12 * E32 * m1.abs(), "m")
            assert not bool(st["exp_avg_sq"][:n - tail].any())
        assert bool((p.detach()[:100000] == 0).all())
        step = torch.where(g == 0, torch.zeros_like(g), -1e-2 * g.sign())
        assert float((p.detach()[n - tail:] - step).abs().max()) < 1e-4  # the first step is lr whatever the gradient's size
        del opt, st
