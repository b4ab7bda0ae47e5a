"""FusedAdamW, its 8-bit moments, grad_norm and clip_grad_norm_ (csrc/adamw.hip) against their definitions in 64 bits.

Tolerances, with e = 2^-24 (half a step of fp32) and S = |b1 m| + |(1 - b1) g|:
  m   beta1, 1 - beta1, the factor on g, the product and the sum are rounded once each: 5 e S
  v   beta2, 1 - beta2, g g, its product, the sum, and the factor on g twice: 7 e v
  w   w (1 - lr wd): the factor and the sum, 2 e |w|; the step u = a m / (sqrt(v) c + eps): half of v's 7, the root, c, the
      sum, the quotient, a and the product: 10 e |u| (and one for the step's own sum: 11), plus a / denominator times m's
      5 e S
A factor from a norm carries the norm's rounding, its sum's, the quotient's and its own: 4 e more for g (8 for g g).  A parameter of 16
bits is rounded once more: finfo.eps / 2 of the value, or half of the smallest subnormal.

8-bit codes: a value x of relative error d may land on either side of its threshold, so its code lies between
floor(k (1 - d) + u - 2^-20) and floor(k (1 + d) + u + 2^-20) for k = |x| / grain (2^-20: what adding 2^-6 rounds a
value below it to, and the threshold's last bit)."""
import copy
import math
import os

import pytest
import torch

from fsgs_amd.optim import FusedAdam, FusedAdamW, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
E32 = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
GOLDEN, ROOT2 = 0x9E3779B9, 0x6A09E667
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def make(sizes, dtype, seed=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for n in sizes:
        ps.append(torch.randn(n, generator=gen).to(DEV, dtype).requires_grad_(True))
        rows = torch.exp(2 * torch.randn(n, generator=gen)) * scale
        gs.append((torch.randn(n, generator=gen) * rows * (torch.rand(n, generator=gen) < 0.8)).to(DEV, dtype))
    return ps, gs


def wide(t):
    return t.detach().cpu().double()


def step64(w, g, m, v, t, lr, b1, b2, eps, wd, extra=0.0):
    """(w, m, v) after a step and how far each may be off; all float64 on the CPU"""
    s = (b1 * m).abs() + ((1 - b1) * g).abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    a, denom = lr / (1 - b1 ** t), v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    u = a * m / denom
    tol_m, tol_v = (5 + extra) * E32 * s, (7 + 2 * extra) * E32 * v + 2.0 ** -149
    tol_w = 2 * E32 * w.abs() + (11 + extra) * E32 * u.abs() + a / denom * tol_m + 2.0 ** -149
    return w * (1 - lr * wd) - u, m, v, tol_w, tol_m + 2.0 ** -149, tol_v


def close(got, want, tol, what):
    bad = (wide(got) - want).abs() > tol
    assert not bool(bad.any()), "%s: %d of %d off, first at %d: %r, %r +- %r" % (
        what, int(bad.sum()), bad.numel(), int(bad.nonzero()[0]), wide(got)[bad][0], want[bad][0], tol.expand_as(want)[bad][0])


SIZES = [1, 2, 3, 5, 63, 64, 65, 127, 128, 129, 255, 1000, 4095, 4096, 4097, 8192, 12345]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("maximize,wd,eps", [(False, 0.1, 1e-8), (True, 0.0, 1e-6)])
def test_steps_in_32_bits(dtype, masters, maximize, wd, eps):
    ps, gs = make(SIZES, dtype)
    lrs = [1e-3 * (1 + i % 11) for i in range(len(ps))]  # more sets of scalars than one launch holds
    opt = FusedAdamW([{"params": [p], "lr": lr} for p, lr in zip(ps, lrs)], eps=eps, weight_decay=wd, maximize=maximize,
                     master_weights=masters, betas=(0.9, 0.99))
    use = masters and dtype != torch.float32
    for step in range(3):
        before = []
        for p, g in zip(ps, gs):
            p.grad = (g.float() * (step + 1)).to(dtype)
            st = opt.state.get(p, {})
            zero = torch.zeros(p.shape, dtype=torch.float64)
            before.append((wide(st["master"]) if use and st else wide(p), wide(st["exp_avg"]) if st else zero,
                           wide(st["exp_avg_sq"]) if st else zero))
        versions = [p._version for p in ps]
        opt.step()
        for p, lr, (w, m, v), version in zip(ps, lrs, before, versions):
            st = opt.state[p]
            g = wide(p.grad) * (-1 if maximize else 1)
            w1, m1, v1, tw, tm, tv = step64(w, g, m, v, step + 1, lr, 0.9, 0.99, eps, wd)
            close(st["exp_avg"], m1, tm, "m"), close(st["exp_avg_sq"], v1, tv, "v")
            if use:
                close(st["master"], w1, tw, "master")
                assert torch.equal(p.detach(), st["master"].to(dtype))
            else:
                close(p, w1, tw + HALF[dtype] * (w1.abs() + tw) + TINY[dtype], "w")
            assert st["step"] == step + 1 and p._version > version


def thresholds(n, step, phase, which, first=0):
    x = 2 * step + which
    for shift, by in ((16, 0xBB67AE85), (15, 0x3C6EF373)):
        x = (x ^ x >> shift) * by & 0xFFFFFFFF
    i = torch.arange(first, first + n, dtype=torch.int64)
    return (((i * phase + (x ^ x >> 16)) & 0xFFFFFFFF) >> 12).double() / 2 ** 20


def check_codes(codes, exps, x, err, u, keep, what):
    """codes (uint8 [n]) and exponent bytes against x +- err (float64): see the module's first lines"""
    n = x.numel()
    fine = torch.isfinite(x)
    a = torch.where(fine, x.abs(), torch.zeros_like(x))
    top = lambda y: torch.cat((y, torch.zeros(-n % 128, dtype=torch.float64))).view(-1, 128).amax(1)  # noqa: E731
    e = exps.cpu().double() - 127
    assert bool((top(a - err) <= 448 * 2.0 ** e).all()), what + ": a block's largest value does not fit"
    assert bool(((top(a + err) > 448 * 2.0 ** (e - 1)) | (exps.cpu() == 1)).all()), what + ": a block's power is larger than it has to be"
    unit = (2.0 ** e).repeat_interleave(128)[:n]

    def code(y, slack):
        y = (y / unit).clamp(min=0.0, max=448.0)
        low = y.clamp(min=2.0 ** -6)  # below, the grain stays 2^-9
        ex = torch.floor(torch.log2(low))
        ex = torch.where(2.0 ** ex > low, ex - 1, ex)
        grains = y / 2.0 ** (ex - 3)  # 8 to 16 of them above 2^ex, whose code is 8 (ex + 7)
        return ((ex + 6) * 8 + torch.floor(grains + u + slack)).clamp(min=0, max=126)

    lo, hi = code(a - err, -(2.0 ** -20)), code(a + err, 2.0 ** -20)
    if keep:
        lo, hi = torch.where(x > 0, lo.clamp(min=1), lo), torch.where(x > 0, hi.clamp(min=1), hi)
    got = codes.cpu().to(torch.int64)
    mag = (got & 127).double()
    ok = (mag >= lo) & (mag <= hi) & ((got >> 7 == (x < 0).long()) | (mag == 0))
    ok = torch.where(fine, ok, mag == 127)
    assert bool(ok.all()), "%s: %d of %d codes wrong, first at %d: %d not in [%d, %d]" % (
        what, int((~ok).sum()), n, int((~ok).nonzero()[0]), int(mag[~ok][0]), int(lo[~ok][0]), int(hi[~ok][0]))
    assert n < 1000 or float((lo != hi).double().mean()) < 0.01  # the bounds say something


def values(codes, exps, n):
    return codes.cpu().float().double() * (2.0 ** (exps.cpu().double() - 127)).repeat_interleave(128)[:n]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masters,wd", [(False, 0.1), (True, 0.0)])
def test_steps_in_8_bits(dtype, masters, wd):
    ps, gs = make(SIZES, dtype, seed=3)
    opt = FusedAdamW([{"params": ps[::2], "lr": 1e-3}, {"params": ps[1::2], "lr": 3e-4, "maximize": True}], eps=1e-8, weight_decay=wd,
                     state_bits=8, master_weights=masters, betas=(0.9, 0.999))
    use = masters and dtype != torch.float32
    ascend = {id(p) for p in ps[1::2]}
    for step in range(3):
        before = []
        for p, g in zip(ps, gs):
            p.grad = (g.float() * (3 - step)).to(dtype)
            st = opt.state.get(p, {})
            zero = torch.zeros(p.shape, dtype=torch.float64)
            n = p.numel()
            before.append((wide(st["master"]) if use and st else wide(p),
                           values(st["exp_avg_q"], st["scales"][:, 0], n) if st else zero,
                           values(st["exp_avg_sq_q"], st["scales"][:, 1], n) ** 2 if st else zero))
        opt.step()
        for p, (w, m, v) in zip(ps, before):
            st, lr = opt.state[p], 3e-4 if id(p) in ascend else 1e-3
            g = wide(p.grad) * (-1 if id(p) in ascend else 1)
            w1, m1, v1, tw, tm, tv = step64(w, g, m, v, step + 1, lr, 0.9, 0.999, 1e-8, wd)
            if use:
                close(st["master"], w1, tw, "master")
                assert torch.equal(p.detach(), st["master"].to(dtype))
            else:
                close(p, w1, tw + HALF[dtype] * (w1.abs() + tw) + TINY[dtype], "w")
            n = p.numel()
            check_codes(st["exp_avg_q"].view(torch.uint8), st["scales"][:, 0], m1, tm, thresholds(n, step + 1, GOLDEN, 0),
                        False, "m, %d elements" % n)
            # r = sqrt(v): half of v's relative error, and the root's rounding
            check_codes(st["exp_avg_sq_q"].view(torch.uint8), st["scales"][:, 1], v1.sqrt(), 5 * E32 * v1.sqrt(),
                        thresholds(n, step + 1, ROOT2, 1), True, "r, %d elements" % n)


def test_moments_come_back_exactly_and_go_in_to_the_nearest():
    sizes = [1, 7, 128, 129, 4096, 5001]
    ps, gs = make(sizes, torch.float32, seed=5)
    opt = FusedAdamW(ps, state_bits=8)
    gen = torch.Generator().manual_seed(1)
    for p in ps:
        n = p.numel()
        m = torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen))
        v = torch.exp(4 * torch.randn(n, generator=gen)) * (torch.rand(n, generator=gen) < 0.9)
        opt.set_moments(p, m.to(DEV), v.to(DEV), 7)
        st = opt.state[p]
        half = torch.full((n,), 0.5, dtype=torch.float64)
        check_codes(st["exp_avg_q"].view(torch.uint8), st["scales"][:, 0], m.double(), torch.zeros(n, dtype=torch.float64), half, False, "m")
        check_codes(st["exp_avg_sq_q"].view(torch.uint8), st["scales"][:, 1], v.double().sqrt(), E32 * v.double().sqrt(), half, True, "r")
        assert st["step"] == 7
    for dtype in (torch.float32, torch.bfloat16):
        for p, (m, v) in zip(ps, opt.moments(dtype)):
            st = opt.state[p]
            assert m.dtype == v.dtype == dtype and m.shape == p.shape
            assert torch.equal(wide(m), values(st["exp_avg_q"], st["scales"][:, 0], p.numel()))
            assert torch.equal(wide(v), values(st["exp_avg_sq_q"], st["scales"][:, 1], p.numel()) ** 2)
    for p, (m, v) in zip(ps, opt.moments(torch.float32)):  # what codes stand for goes back to values of the same
        opt.set_moments(p, m, v, 7)
    for (m, v), (m2, v2) in zip(opt.moments(), opt.moments()):
        assert torch.equal(m, m2) and torch.equal(v, v2)
    pairs = opt.moments()  # cut from one buffer: apart from each other, and whole tensors in every other way
    spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for pair in pairs for t in pair)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(t.is_contiguous() for pair in pairs for t in pair)
    keep = pairs[5][1].clone()
    pairs[5][0].fill_(7.0), pairs[4][1].add_(1.0)
    assert torch.equal(pairs[5][1], keep) and torch.equal(pairs[5][0].cpu(), torch.full((sizes[5],), 7.0))
    last = opt.moments()[5][1]
    del pairs
    assert torch.equal(last, keep) and last.requires_grad is False and torch.equal(copy.deepcopy(last), keep)
    m16, v16 = opt.moments(torch.float16)[3]
    assert m16.dtype == v16.dtype == torch.float16


def test_the_rounding_is_unbiased_over_steps():
    """A second moment that decays by 5e-4 a step in its root, far under half a code, decays on in the mean: after T steps
    without gradients every element's v is beta2^T v0 within what the rounding's walk allows."""
    n, T, b2 = 20000, 1500, 0.999
    gen = torch.Generator().manual_seed(2)
    p = torch.zeros(n, device=DEV, requires_grad=True)
    opt = FusedAdamW([p], betas=(0.9, b2), lr=0.0, state_bits=8)
    v0 = torch.exp(torch.randn(n, generator=gen)).to(DEV)
    opt.set_moments(p, torch.zeros(n, device=DEV), v0, 0)
    v0 = opt.moments()[0][1]
    p.grad = torch.zeros(n, device=DEV)
    for _ in range(T):
        opt.step()
    ratio = (opt.moments()[0][1] / v0).double().sqrt() / b2 ** (T / 2)
    # a step down by q <= r / 8 is taken with the probability 5e-4 r / q: the variance of r / r0 grows by at most 5e-4 / 8 a
    # step, to 0.094 (a deviation of 0.31) for one element and 0.0022 for the mean of independent ones; those with nearly
    # equal codes and thresholds are not independent: some nine times that is allowed, 0.02
    assert abs(float(ratio.mean()) - 1) < 0.02 and float(ratio.std()) < 0.31


@pytest.mark.parametrize("bits", [32, 8])
def test_infinities_and_nan_stay_where_they_are(bits):
    n = 700
    p = torch.ones(n, device=DEV, requires_grad=True)
    opt = FusedAdamW([p], lr=1e-2, state_bits=bits, weight_decay=0.0)
    p.grad = torch.full((n,), 0.5, device=DEV)
    p.grad[3], p.grad[130], p.grad[699] = float("nan"), float("inf"), -float("inf")
    opt.step()
    opt.step()
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[3, 130, 699]] = True
    assert torch.equal(~torch.isfinite(p.detach()).cpu(), bad)
    # two steps of a constant gradient move by lr each, whatever its size; 8 bits: the second by at most 1/8 of m and of r away
    assert float((p.detach().cpu()[~bad] - 0.98).abs().max()) < (1e-6 if bits == 32 else 1e-2 * 0.3)
    m, v = opt.moments()[0]
    assert torch.equal(~torch.isfinite(m).cpu(), bad) and torch.equal(~torch.isfinite(v).cpu(), bad)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_zero_state_and_the_smallest_eps(bits):
    p = torch.randn(300, device=DEV).requires_grad_(True)
    before = p.detach().clone()
    opt = FusedAdamW([p], lr=0.1, eps=1e-15, state_bits=bits, weight_decay=0.0)
    p.grad = torch.zeros(300, device=DEV)
    opt.step()
    assert torch.equal(p.detach(), before)
    # a block that holds 1 and 1e-12: the small element's moments are under every code; it must not jump
    p.grad = torch.where(torch.arange(300, device=DEV) % 2 == 0, 1.0, 1e-12)
    for _ in range(5):
        opt.step()
    moved = (p.detach() - before).abs()
    # |m| <= 1, sqrt(v) / bias >= what g gave: a step is at most lr * (1 - b1) / sqrt(1 - b2) * sqrt(bc2) / bc1 <= 0.1 * 10
    assert float(moved.max()) < 5 * 1.0 and bool(torch.isfinite(p).all())
    if bits == 8:
        # after the first step the stored r is at least the smallest code of its block, 2^-9 / 448 of the largest value
        assert float(moved[1::2].max()) <= 0.1 * 1.0 + 1e-3


def test_tensors_that_are_cut_from_others_permuted_or_empty():
    base = torch.randn(4000, device=DEV)
    kept = base.clone()
    odd = base[1:1000].detach().requires_grad_(True)               # not 16-byte aligned
    odd16 = torch.randn(2000, device=DEV).bfloat16()[3:1500].detach().requires_grad_(True)
    perm = torch.randn(20, 30, 7, device=DEV).permute(2, 0, 1).detach().requires_grad_(True)
    empty = torch.zeros(0, 3, device=DEV, requires_grad=True)
    plain = [t.detach().clone().contiguous().requires_grad_(True) for t in (odd, odd16, perm, empty)]
    skipped = torch.ones(5, device=DEV, requires_grad=True)
    for bits in (32, 8):
        a, b = FusedAdamW([odd, odd16, perm, empty, skipped], state_bits=bits), FusedAdamW(plain, state_bits=bits)
        for step in range(2):
            for p, q in zip((odd, odd16, perm, empty), plain):
                g = torch.randn(p.shape, device=DEV).to(p.dtype)
                p.grad, q.grad = g, g.clone()       # the permuted parameter's gradient has another layout
            a.step(), b.step()
        for p, q in zip((odd, odd16, empty), (plain[0], plain[1], plain[3])):
            assert torch.equal(p, q)
        if bits == 32:  # in 8 bits the blocks follow memory, so a permuted tensor has blocks of its own
            assert torch.equal(perm, plain[2])
            assert torch.equal(a.state[perm]["exp_avg"], b.state[plain[2]]["exp_avg"])
        else:
            assert float((perm - plain[2]).detach().abs().max()) < 3e-3
            assert a.moments()[2][0].stride() == perm.stride()
        assert skipped not in a.state and bool((skipped == 1).all())
    assert torch.equal(base[:1], kept[:1]) and torch.equal(base[1000:], kept[1000:]) and not torch.equal(base, kept)


def test_nothing_beside_the_tensors_is_written():
    for bits in (32, 8):
        for n in (1, 5, 129, 4097):
            hold = torch.full((n + 32,), 7.0, device=DEV)
            p = hold[16:16 + n].detach().requires_grad_(True)
            p.grad = torch.ones(n, device=DEV)
            opt = FusedAdamW([p], state_bits=bits)
            opt.step()
            keys = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg_q", "exp_avg_sq_q")
            for k in keys:  # states cut from larger tensors too
                t = opt.state[p][k]
                room = torch.zeros(n + 32, device=DEV, dtype=torch.uint8 if bits == 8 else t.dtype).fill_(9)
                inside = room[16:16 + n]
                inside.copy_(t.view(torch.uint8) if bits == 8 else t)
                opt.state[p][k] = inside.view(t.dtype)
                opt.state[p][k + "_room"] = room
            p.grad = torch.ones(n, device=DEV)
            opt.step()
            assert bool((hold[:16] == 7).all()) and bool((hold[16 + n:] == 7).all()) and not bool((hold[16:16 + n] == 7).any())
            for k in keys:
                room = opt.state[p][k + "_room"]
                assert bool((room[:16] == 9).all()) and bool((room[16 + n:] == 9).all())


def test_wrong_state_is_refused_and_counts_stay():
    p, q = torch.ones(10, device=DEV, requires_grad=True), torch.ones(10, device=DEV, requires_grad=True)
    p.grad, q.grad = torch.ones(10, device=DEV), torch.ones(10, device=DEV)
    for bits, key, wrong in ((32, "exp_avg", torch.zeros(9, device=DEV)), (32, "exp_avg_sq", torch.zeros(10, device=DEV).half()),
                             (32, "exp_avg", torch.zeros(10)), (8, "scales", torch.zeros(1, 1, dtype=torch.uint8, device=DEV)),
                             (8, "exp_avg_q", torch.zeros(10, device=DEV))):
        opt = FusedAdamW([p, q], state_bits=bits)
        opt.step()
        opt.state[q][key] = wrong
        before = p.detach().clone()
        with pytest.raises(ValueError):
            opt.step()
        assert opt.state[p]["step"] == 1 and torch.equal(p.detach(), before)
    opt = FusedAdamW([p, q])
    opt.step()
    opt.state[q]["exp_avg"] = opt.state[p]["exp_avg"]
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    q.grad = torch.ones(10, device=DEV).to_sparse()
    with pytest.raises(RuntimeError):
        opt.step()
    bad = torch.zeros(10, 2, device=DEV)[:, 0].detach().requires_grad_(True)
    bad.grad = torch.ones(10, device=DEV)
    with pytest.raises(ValueError, match="dense"):
        FusedAdamW([bad]).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_counts_on_and_equals_eager_ones(bits):
    ps, gs = make([5, 300, 4097], torch.float32, seed=9)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    lr = torch.tensor(1e-3, device=DEV)
    # max_grad_norm: the norm's scratch and the scalars live in the graph's own pool
    a = FusedAdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": lr}], state_bits=bits, capturable=True, max_grad_norm=0.3)
    b = FusedAdamW([{"params": qs[:2]}, {"params": qs[2:], "lr": 1e-3}], state_bits=bits, max_grad_norm=0.3)
    for p, q, g in zip(ps, qs, gs):
        p.grad, q.grad = g.clone(), g.clone()
    a.step(), b.step()  # makes the states
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    norms = []
    for k in range(4):
        rate = 1e-3 / (k + 1)
        lr.fill_(rate)
        b.param_groups[1]["lr"] = float(lr)
        for p, q, g in zip(ps, qs, gs):
            p.grad.copy_(g * (k + 1)), q.grad.copy_(g * (k + 1))
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        norms.append(float(a.last_grad_norm))
        assert norms[-1] == float(b.last_grad_norm)
        for p, q in zip(ps, qs):
            assert float(a.state[p]["step"]) == b.state[q]["step"] == k + 2
            # the scalars come from pow() of the device there and of the host here: each within an ulp of 64 bits
            assert float((p - q).detach().abs().max()) <= 4 * E32 * float(q.detach().abs().max()), k
        for (m, v), (m2, v2) in zip(a.moments(), b.moments()):
            assert torch.equal(m, m2) and torch.equal(v, v2)
    assert norms == sorted(norms) and norms[0] > 0.3


def test_captures_that_would_freeze_or_reset_something_are_refused():
    p = torch.ones(100, device=DEV, requires_grad=True)
    p.grad = torch.ones(100, device=DEV)
    frozen, fresh = FusedAdamW([p]), FusedAdamW([p], capturable=True)
    frozen.step()
    torch.cuda.synchronize()
    for opt in (frozen, fresh):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(graph):
                opt.step()
    torch.cuda.synchronize()
    frozen.step()
    fresh.step()
    with pytest.raises(ValueError):
        FusedAdamW([p], lr=torch.tensor(1e-3, device=DEV))
    opt = FusedAdamW([p], lr=torch.tensor(1e-3))  # a number on the host is a number
    opt.step()
    assert opt.state[p]["step"] == 1


def test_two_graphs_with_norms_of_their_own():
    """two captured clips replayed on two streams at once share no scratch"""
    sets, graphs, streams = [], [], []
    for k in range(2):
        ps, gs = make([70001, 333], torch.float32, seed=20 + k)
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        out = {}
        clip_grad_norm_(ps, 1e9)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out["norm"] = clip_grad_norm_(ps, 0.25)
        sets.append((ps, gs, out)), graphs.append(graph), streams.append(stream)
    for _ in range(3):
        for ps, gs, _ in sets:
            for p, g in zip(ps, gs):
                p.grad.copy_(g)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for ps, gs, out in sets:
            want = math.sqrt(sum(float((wide(g) ** 2).sum()) for g in gs))
            assert abs(float(out["norm"]) - want) <= 2 * E32 * want
            c = 0.25 / (want + 1e-6)
            for p, g in zip(ps, gs):
                close(p.grad, wide(g) * c, 6 * E32 * (wide(g) * c).abs() + 2.0 ** -149, "g")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [3, 1, 4097], SIZES, [50] * 130, [300001, 2]])
def test_norm_and_clipping(dtype, sizes):
    ps, gs = make(sizes, dtype, seed=len(sizes))
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    want = math.sqrt(sum(float((wide(g) ** 2).sum()) for g in gs))
    norm = grad_norm([p.grad for p in ps])
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 2 * E32 * want
    assert float(norm) == float(grad_norm([p.grad for p in ps]))
    assert float(clip_grad_norm_(ps, 2 * want + 1)) == float(norm)
    for p, g in zip(ps, gs):
        assert torch.equal(p.grad, g)
    if want == 0:
        return
    versions = [p.grad._version for p in ps]
    assert float(clip_grad_norm_(ps, want / 3)) == float(norm)
    c = want / 3 / (want + 1e-6)
    for p, g, version in zip(ps, gs, versions):
        x = wide(g) * c
        close(p.grad, x, 6 * E32 * x.abs() + HALF[dtype] * x.abs() * (1 + 2.0 ** -20) + TINY[dtype], "g")
        assert p.grad._version > version


def test_norm_of_mixed_types_large_values_and_nan():
    a = torch.full((1000,), 1e30, device=DEV)                     # squares over fp32's range
    b = torch.full((777,), 3.0, device=DEV, dtype=torch.bfloat16)
    c = torch.full((10,), 2.0, device=DEV, dtype=torch.float16)
    assert abs(float(grad_norm([b, c])) - math.sqrt(777 * 9 + 40)) < 1e-4
    assert abs(float(grad_norm([a, b, c])) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert float(grad_norm([torch.zeros(5, device=DEV), torch.zeros(0, device=DEV)])) == 0.0
    assert float(grad_norm(torch.zeros(0, device=DEV))) == 0.0
    p = torch.ones(4, device=DEV, requires_grad=True)
    p.grad = torch.tensor([1.0, float("inf"), 2.0, 0.0], device=DEV)
    assert math.isinf(float(clip_grad_norm_(p, 1.0)))             # as torch: factor 0, so inf becomes NaN and the rest 0
    assert torch.isnan(p.grad[1]) and float(p.grad[0]) == 0.0
    assert math.isnan(float(clip_grad_norm_([p], 1.0))) and bool(torch.isnan(p.grad).all())
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    q = torch.ones(3, device=DEV, requires_grad=True)
    q.grad = torch.ones(3, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_([q, q], 0.1)
    r = torch.ones(2, device=DEV, requires_grad=True)
    r.grad = q.grad[1:]
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([q, r], 0.1)
    assert bool((q.grad == 1).all())
    s = torch.ones(6, device=DEV, requires_grad=True)
    s.grad = torch.full((6, 2), 2.0, device=DEV)[:, 0]            # a slice
    assert abs(float(grad_norm(s.grad)) - math.sqrt(24)) < 1e-5
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_([q, s], 1.0)
    assert bool((q.grad == 1).all())
    a, b = torch.ones(4, 5, device=DEV).t().requires_grad_(True), torch.ones(3, device=DEV, dtype=torch.float16, requires_grad=True)
    a.grad, b.grad = torch.full((4, 5), 3.0, device=DEV).t(), torch.full((3,), 2.0, device=DEV, dtype=torch.float16)
    for error in (True, False):  # a gradient of another order of dimensions, types side by side; both ways through
        want = math.sqrt(float((a.grad.double() ** 2).sum() + (b.grad.double() ** 2).sum()))
        g = a.grad.clone()
        assert abs(float(clip_grad_norm_([a, b], want / 2, error_if_nonfinite=error)) - want) <= 2 * E32 * want
        assert float((a.grad - g / 2).abs().max()) < 1e-6


def test_the_norm_bound_inside_a_step_is_the_clip_in_front_of_it():
    for dtype in (torch.float32, torch.bfloat16):
        ps, gs = make([700, 5000, 1], dtype, seed=31)
        opt = FusedAdamW(ps, max_grad_norm=0.05, lr=1e-2, weight_decay=0.0)
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        opt.step()
        want = math.sqrt(sum(float((wide(g) ** 2).sum()) for g in gs))
        assert abs(float(opt.last_grad_norm) - want) <= 2 * E32 * want and want > 0.05
        c = 0.05 / (want + 1e-6)
        for p, g in zip(ps, gs):
            assert torch.equal(p.grad, g)
            zero = torch.zeros(g.shape, dtype=torch.float64)
            _, m1, v1, _, tm, tv = step64(zero, wide(g) * c, zero, zero, 1, 1e-2, 0.9, 0.999, 1e-8, 0.0, extra=4)
            close(opt.state[p]["exp_avg"], m1, tm, "m"), close(opt.state[p]["exp_avg_sq"], v1, tv, "v")


@pytest.mark.parametrize("bits,masters", [(32, False), (8, True)])
def test_the_quick_walk_gives_what_the_general_one_gives(bits, masters, monkeypatch):
    """a step collected by the host extension against one collected tensor by tensor: groups of other options and types,
    parameters without gradients, more groups than a launch has scalars"""
    def build():
        ps = sum((make([5, 700, 4099, 1], dtype, seed=70)[0] for dtype in DTYPES), [])
        groups = [{"params": [p], "lr": 1e-3 * (1 + i % 9), "betas": (0.9, 0.99 if i % 4 else 0.9)} for i, p in enumerate(ps)]
        groups[3]["state_bits"], groups[5]["maximize"], groups[7]["weight_decay"] = 40 - bits, True, 0.3
        return ps, FusedAdamW(groups, state_bits=bits, master_weights=masters, max_grad_norm=0.2)

    (ps, a), (qs, b) = build(), build()
    quick = []
    ordinary = FusedAdamW._ordinary
    for k in range(4):
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * k + i)).to(DEV, p.dtype)
            p.grad, q.grad = (None, None) if (i + k) % 5 == 0 and k < 3 else (g, g.clone())
        monkeypatch.setattr(FusedAdamW, "_ordinary", lambda self: quick.append(ordinary(self)) or quick[-1])
        versions = [p._version for p in ps]
        a.step()
        assert all((p._version > v) == (p.grad is not None) for p, v in zip(ps, versions))
        monkeypatch.setattr(FusedAdamW, "_ordinary", lambda self: None)
        b.step()
    assert quick[0] is None and quick[-1] is not None
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and a.state[p]["step"] == b.state[q]["step"]
        for k, v in a.state[p].items():
            if torch.is_tensor(v):
                assert torch.equal(v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v,
                                   b.state[q][k].view(torch.uint8) if v.dtype == torch.float8_e4m3fn else b.state[q][k]), k
    for (m, v), (m2, v2) in zip(a.moments(), b.moments()):
        assert torch.equal(m, m2) and torch.equal(v, v2)


def test_streams_and_steps_behind_each_other():
    ps, gs = make([200000], torch.float32, seed=40)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    a, b = FusedAdamW(ps, state_bits=8), FusedAdamW(qs, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(5):
        qs[0].grad = gs[0] * (k + 1)
        b.step()
    with torch.cuda.stream(side):
        for k in range(5):
            ps[0].grad = gs[0] * (k + 1)
            a.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ps[0], qs[0])
    assert torch.equal(a.state[ps[0]]["exp_avg_q"].view(torch.uint8), b.state[qs[0]]["exp_avg_q"].view(torch.uint8))


def test_two_threads_step_at_once():
    """two optimizers in two threads, each on a stream of its own, against the same steps one after the other"""
    import threading

    def job(seed, out, stream):
        ps, gs = make([4097, 50, 300000], torch.bfloat16, seed=seed)
        opt = FusedAdamW(ps, state_bits=8, master_weights=True, max_grad_norm=0.1)
        if stream is not None:
            stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            for k in range(40):
                for p, g in zip(ps, gs):
                    p.grad = g * (k + 1)
                opt.step()
                clip_grad_norm_(ps, 0.5)
            torch.cuda.current_stream().synchronize()
        out[seed] = [p.detach() for p in ps] + [t for pair in opt.moments() for t in pair] + [p.grad for p in ps]

    alone, together = {}, {}
    for seed in (1, 2):
        job(seed, alone, None)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=job, args=(seed, together, torch.cuda.Stream())) for seed in (1, 2)]
    [t.start() for t in threads], [t.join() for t in threads]
    torch.cuda.synchronize()
    for seed in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[seed], together[seed]))


def test_steps_hold_on_to_nothing():
    import gc
    import sys

    ps, gs = make([100, 3000], torch.float32, seed=90)
    opt = FusedAdamW(ps, state_bits=8, max_grad_norm=1.0)
    for p, g in zip(ps, gs):
        p.grad = g.clone()

    def once():
        opt.step(), opt.moments(torch.bfloat16), clip_grad_norm_(ps, 0.5), grad_norm([p.grad for p in ps])

    def held():
        gc.collect()
        torch.cuda.synchronize()
        return ([sys.getrefcount(x) for x in ps + [opt.state, opt.param_groups] + [st for st in opt.state.values()]],
                [sys.getrefcount(v) for st in opt.state.values() for v in st.values() if torch.is_tensor(v)],
                torch.cuda.memory_allocated())

    once()
    before = held()
    for _ in range(50):
        once()
    assert held() == before


def test_changing_the_width_and_saving():
    ps, gs = make([1000, 130], torch.bfloat16, seed=50)
    opt = FusedAdamW(ps, state_bits=8, master_weights=True)
    step = lambda o, params: ([setattr(p, "grad", g.clone()) for p, g in zip(params, gs)], o.step())  # noqa: E731
    step(opt, ps)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    other = FusedAdamW(qs, state_bits=8, master_weights=True)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    step(opt, ps), step(other, qs)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["scales"], other.state[q]["scales"])
        assert torch.equal(opt.state[p]["master"], other.state[q]["master"])
    before = opt.moments()
    opt.param_groups[0]["state_bits"] = 32
    opt.param_groups[0]["betas"] = (0.0, 0.0)
    step(opt, ps)
    assert "exp_avg_q" not in opt.state[ps[0]] and opt.state[ps[0]]["step"] == 3
    other.widen(qs[0])
    assert torch.equal(other.state[qs[0]]["exp_avg"], before[0][0])
    step(other, qs)
    assert "exp_avg" not in other.state[qs[0]] and other.state[qs[0]]["step"] == 3


def test_masters_that_are_switched_off_and_on_start_from_the_parameter():
    p = torch.ones(50, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.ones(50, device=DEV, dtype=torch.bfloat16)
    opt = FusedAdamW([p], lr=1e-1, master_weights=True, weight_decay=0.0)
    opt.step()
    opt.param_groups[0]["master_weights"] = False
    for _ in range(3):
        opt.step()
    assert "master" not in opt.state[p]
    before = p.detach().float()
    opt.param_groups[0]["master_weights"] = True
    opt.step()
    assert float((opt.state[p]["master"] - (before - 0.1)).abs().max()) < 1e-5  # a constant gradient moves by lr a step


def test_moments_saved_in_another_layout_load():
    p = torch.randn(6, 5, device=DEV).requires_grad_(True)
    opt = FusedAdamW([p])
    p.grad = torch.randn(6, 5, device=DEV)
    opt.step()
    q = p.detach().t().contiguous().t().requires_grad_(True)
    other = FusedAdamW([q])
    other.load_state_dict(opt.state_dict())
    q.grad = p.grad
    opt.step(), other.step()
    assert other.state[q]["exp_avg"].stride() == q.stride() and torch.equal(p, q)


def test_saved_states_load_without_unpickling(tmp_path):
    ps, gs = make([300, 7], torch.float16, seed=8)
    opt = FusedAdamW(ps, state_bits=8, master_weights=True, eps=1e-6)
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    torch.save(opt.state_dict(), os.path.join(str(tmp_path), "opt.pth"))
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    other = FusedAdamW(qs, state_bits=8, master_weights=True, eps=1e-6)
    other.load_state_dict(torch.load(os.path.join(str(tmp_path), "opt.pth"), weights_only=True))
    for q, g in zip(qs, gs):
        q.grad = g
    opt.step(), other.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], other.state[q]["master"])


def test_a_norm_over_more_than_4_g_elements():
    n = 2 ** 32 + 4099
    g = torch.zeros(n, device=DEV, dtype=torch.float16)
    g[-3:], g[2 ** 31], g[0] = 2.0, 1.0, 4.0
    p = torch.zeros(n, device=DEV, dtype=torch.float16, requires_grad=True)
    p.grad = g
    want = math.sqrt(3 * 4 + 1 + 16)
    assert abs(float(clip_grad_norm_([p], want / 2)) - want) <= 2 * E32 * want
    for at, v in ((-1, 1.0), (-3, 1.0), (2 ** 31, 0.5), (0, 2.0), (1, 0.0), (-4, 0.0)):
        assert abs(float(g[at]) - v) < 1e-3


def test_offsets_over_32_bits():
    """one bf16 tensor of 2^31 + 4099 elements with 8-bit moments (13 GB in all), then with 32-bit ones (26 GB): gradients in its
    last elements alone"""
    n, tail = 2 ** 31 + 4099, 4099
    p = torch.zeros(n, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(1)
    g = torch.randn(tail, device=DEV, generator=gen).bfloat16()
    p.grad[n - tail:] = g
    opt = FusedAdamW([p], state_bits=8, max_grad_norm=1.0, lr=1e-2)
    opt.step()
    want = math.sqrt(float((wide(g) ** 2).sum()))
    assert abs(float(opt.last_grad_norm) - want) <= 2 * E32 * want
    st = opt.state[p]
    c = 1.0 / (want + 1e-6)
    m1 = 0.1 * wide(g) * c
    u = thresholds(tail, 1, GOLDEN, 0, n - tail)
    check_codes(st["exp_avg_q"].view(torch.uint8)[n - tail:], st["scales"][(n - tail) // 128:, 0], m1, 12 * E32 * m1.abs(), u, False, "m")
    assert bool((p.detach()[:100000] == 0).all()) and not bool(st["exp_avg_q"].view(torch.uint8)[:n - tail].any())
    del opt, st
    opt32 = FusedAdamW([p], state_bits=32, max_grad_norm=1.0, lr=1e-2)
    p.detach().zero_()
    opt32.step()
    close(opt32.state[p]["exp_avg"][n - tail:], m1, 12 * E32 * m1.abs(), "m")
    assert not bool(opt32.state[p]["exp_avg_sq"][:n - tail].any())
    step = torch.where(g == 0, torch.zeros_like(g), -1e-2 * g.sign())
    assert float((p.detach()[n - tail:] - step).abs().max()) < 1e-4  # the first step is lr whatever the gradient's size


def test_against_the_other_adam_of_the_package():
    """weight_decay = 0, fp32: FusedAdam's arithmetic"""
    ps, gs = make([3000, 7], torch.float32, seed=60)
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    a, b = FusedAdamW(ps, lr=1e-2, weight_decay=0.0, eps=1e-15), FusedAdam(qs, lr=1e-2, eps=1e-15)
    for k in range(10):
        for p, q, g in zip(ps, qs, gs):
            p.grad, q.grad = g * (k - 4.5), g * (k - 4.5)
        a.step(), b.step()
    for p, q in zip(ps, qs):
        # ten steps of at most 0.01 * 10 each, each off by some 30 e of itself on either side
        assert float((p - q).detach().abs().max()) <= 10 * 0.1 * 60 * E32 + 20 * E32 * float(q.detach().abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_cloud_trains_densifies_and_is_saved(bits, tmp_path):
    """the run together: mapping steps of the step driver with a bounded norm, densification, more steps, a checkpoint into
    another cloud, and the same next step from both"""
    from fsgs_amd import checkpoint, synth
    from fsgs_amd.fast_step import FastStepper
    from fsgs_amd.model import PARAM_NAMES, GaussianCloud
    from fsgs_amd.trainer import FrameData, PoseTrack, settings_from_cam

    W, H = 320, 256
    cam = synth.make_camera(W, H)
    sc = synth.init_scene(W, H, 3000, seed=0)

    def cloud():
        pc = GaussianCloud(sc, sh_degree=3, device=DEV, scene_radius=1.0)
        pc.cam = settings_from_cam(cam, DEV)
        pc.training_setup(adamw=dict(state_bits=bits, max_grad_norm=10.0))
        return pc

    pc, poses = cloud(), PoseTrack(2, DEV)
    img, dep = torch.tensor(sc["image"], device=DEV), torch.tensor(sc["depth_map"], device=DEV)
    frames = FrameData([img, img], [dep, dep], flows_fw=[torch.zeros(2, H, W, device=DEV)], K=cam["K"])
    fs = FastStepper(pc, poses, frames)
    for _ in range(3):
        loss = fs.mapping_step([0])
    assert math.isfinite(float(loss)) and math.isfinite(float(pc.optimizer.last_grad_norm))
    st = pc.optimizer.state[pc.params["_xyz"]]
    assert st["step"] == 3 and ("exp_avg_q" in st) == (bits == 8)
    with pytest.raises(RuntimeError, match="grad_sync"):
        fs.mapping_step([0], reduce_compact=lambda t: t)
    grown = torch.arange(pc.num_points, device=DEV) % 3 == 0
    pc.variables["xyz_gradient_accum"].copy_(grown.float()[:, None])
    pc.variables["denom"].fill_(1.0)
    wanted = dict(zip(PARAM_NAMES, pc.optimizer.moments()))
    info = pc.densify_and_prune_device(0.5, 0.0, None)
    assert info["cloned"] + info["split"] > 0
    kept = info["kept"]
    for name, (m, v) in zip(PARAM_NAMES, pc.optimizer.moments()):
        assert m.shape == pc.params[name].shape and not bool(m[kept:].any()) and not bool(v[kept:].any())
        if info["split"] == 0 and kept == wanted[name][0].shape[0]:
            assert torch.equal(m[:kept], wanted[name][0]) and torch.equal(v[:kept], wanted[name][1])
    pc.reset_opacity()
    fs = FastStepper(pc, poses, frames)
    fs.mapping_step([0])
    assert ("exp_avg_q" in pc.optimizer.state[pc.params["_xyz"]]) == (bits == 8)
    path = os.path.join(str(tmp_path), "cloud.pth")
    torch.save(checkpoint.capture_gaussians(pc), path)
    saved = torch.load(path, weights_only=True)
    assert all("exp_avg" in s and torch.is_tensor(s["step"]) for s in saved[10]["state"].values())
    other = checkpoint.restore_gaussians(cloud(), saved)
    other.cam = pc.cam
    for name in PARAM_NAMES:
        g = torch.randn(pc.params[name].shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
        pc.params[name].grad, other.params[name].grad = g, g.clone()
    pc.optimizer.step(), other.optimizer.step()
    for name in PARAM_NAMES:
        a, b = pc.optimizer.state[pc.params[name]], other.optimizer.state[other.params[name]]
        assert int(a["step"]) == int(b["step"]) and torch.equal(pc.params[name], other.params[name]), name
        if bits == 8:
            assert torch.equal(a["exp_avg_q"].view(torch.uint8), b["exp_avg_q"].view(torch.uint8))
    # and the file opens as one of torch's Adam
    plain = torch.optim.Adam([{"params": [pc.params[n].detach().clone().requires_grad_(True)]} for n in PARAM_NAMES], lr=0.0)
    plain.load_state_dict(saved[10])
    # and back: a cloud with the other width reads it
    third = cloud()
    third.adamw = dict(state_bits=40 - bits)
    third = checkpoint.restore_gaussians(third, saved)
    third.params["_xyz"].grad = torch.zeros_like(third.params["_xyz"])
    third.optimizer.step()
