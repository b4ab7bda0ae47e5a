"""What FusedAdamW's state goes through on the GPU: row operations, restored checkpoints, loaded states and captures."""
import math
import os

import pytest
import torch

from fsgs_amd import checkpoint, synth
from fsgs_amd.model import PARAM_NAMES, GaussianCloud
from fsgs_amd.optim import FusedAdamW
from tests.test_adamw_gpu import DEV, make

pytestmark = pytest.mark.gpu


def cloud(**adamw):
    pc = GaussianCloud(synth.init_scene(64, 48, 500, seed=0), sh_degree=3, device=DEV, scene_radius=1.0)
    pc.training_setup(adamw=adamw)
    return pc


def stepped(pc, steps=2, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for _ in range(steps):
        for p in pc.params.values():
            p.grad = torch.randn(p.shape, device=DEV, generator=gen)
        pc.optimizer.step()
    return pc


@pytest.mark.parametrize("before,after", [(8, 32), (32, 8), (8, 8)])
@pytest.mark.parametrize("op", ["prune", "densify", "opacity"])
def test_a_width_changed_in_front_of_a_row_operation(before, after, op):
    pc = stepped(cloud(state_bits=before))
    want = dict(zip(PARAM_NAMES, pc.optimizer.moments()))
    for g in pc.optimizer.param_groups:
        g["state_bits"] = after
    kept = torch.arange(pc.num_points, device=DEV)
    if op == "prune":
        kept = kept[kept % 3 != 0]
        pc.prune_points(torch.arange(pc.num_points, device=DEV) % 3 == 0)
    elif op == "densify":  # every third is cloned or split: the rows that stay come first, in order
        P = pc.num_points
        pc.variables["xyz_gradient_accum"].copy_((kept % 3 == 0).float()[:, None])
        pc.variables["denom"].fill_(1.0)
        big = pc.get_scaling.max(dim=1).values > pc.variables["scene_radius"] * 0.01
        info = pc.densify_and_prune_device(0.5, 0.0, None)
        kept = kept[~((kept % 3 == 0) & big)]
        assert info["kept"] == len(kept) and info["cloned"] + info["split"] == -(-P // 3)
    else:
        pc.reset_opacity()
    for name, (m, v) in zip(PARAM_NAMES, pc.optimizer.moments()):
        assert pc.optimizer.state[pc.params[name]]["step"] == 2 and m.shape == pc.params[name].shape
        if op == "opacity" and name == "_opacity":
            assert not bool(m.any()) and not bool(v.any())
            continue
        assert torch.equal(m[:len(kept)], want[name][0][kept]) and torch.equal(v[:len(kept)], want[name][1][kept])
        assert not bool(m[len(kept):].any()) and not bool(v[len(kept):].any())
    stepped(pc, 1)
    for p in pc.params.values():
        st = pc.optimizer.state[p]
        assert st["step"] == 3 and ("exp_avg_q" in st) == (after == 8) and ("exp_avg" in st) == (after == 32)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_cloud_of_the_other_width_and_decay_restores(bits, tmp_path):
    pc = stepped(cloud(state_bits=bits, weight_decay=0.1))
    torch.save(checkpoint.capture_gaussians(pc), os.path.join(str(tmp_path), "cloud.pth"))
    saved = torch.load(os.path.join(str(tmp_path), "cloud.pth"), weights_only=True)
    other = checkpoint.restore_gaussians(cloud(state_bits=40 - bits, weight_decay=0.0, max_grad_norm=5.0), saved)
    wide = dict(zip(PARAM_NAMES, other.optimizer.moments()))
    for (m, v), (m2, v2) in zip(pc.optimizer.moments(), wide.values()):
        assert torch.equal(m, m2) and torch.equal(v, v2)
    before = {k: p.detach().clone() for k, p in other.params.items()}
    for p in other.params.values():
        p.grad = torch.zeros_like(p)
    other.optimizer.step()
    for g in other.optimizer.param_groups:
        p, name = g["params"][0], g["name"]
        st = other.optimizer.state[p]
        assert g["state_bits"] == 40 - bits and st["step"] == 3 and ("exp_avg_q" in st) == (bits == 32) and ("exp_avg" in st) == (bits == 8)
        m, v = (0.9 * wide[name][0].double(), 0.999 * wide[name][1].double())
        if bits == 32:  # the moments went into codes before the step: 1/16 of a value, or half of the smallest code
            continue
        u = g["lr"] / (1 - 0.9 ** 3) * m / (v.sqrt() / math.sqrt(1 - 0.999 ** 3) + g["eps"])
        want = before[name].double() - u  # no decay: w and its sum 2 roundings, the step 16
        assert bool(((p.detach().double() - want).abs() <= 2.0 ** -24 * (2 * want.abs() + 16 * u.abs())).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [8, 32])
def test_states_of_torchs_adamw_go_on(dtype, bits):
    """the same gradients once more: 32-bit moments move as the formula says from the 16-bit ones that torch held"""
    ps, gs = make([300, 5], dtype, seed=8)
    theirs = torch.optim.AdamW(ps, lr=1e-2)
    for p, g in zip(ps, gs):
        p.grad = g
    theirs.step()
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    opt = FusedAdamW(qs, state_bits=bits)
    opt.load_state_dict(theirs.state_dict())
    for g in opt.param_groups:
        assert g["state_bits"] == bits and g["lr"] == 1e-2 and g["weight_decay"] == 1e-2
    for q, g in zip(qs, gs):
        q.grad = g
    opt.step()
    for p, q, g, (m, v) in zip(ps, qs, gs, opt.moments()):
        want = 0.9 * theirs.state[p]["exp_avg"].double() + 0.1 * g.double()
        size = 0.9 * theirs.state[p]["exp_avg"].double().abs() + 0.1 * g.double().abs()
        assert opt.state[q]["step"] == 2
        if bits == 32:
            assert bool(((m.double() - want).abs() <= 5 * 2.0 ** -24 * size + 2.0 ** -149).all())
        # torch's own fp16 step leaves infinities and NaN: eps = 1e-8 and 1e-3 g^2 for |g| < 5e-3 are under 2^-25, half of the
        # smallest fp16, so that it divides by zero.  They stay, and the step adds none.
        fine = torch.isfinite(p)
        assert bool(torch.isfinite(v).all()) and torch.equal(torch.isfinite(q), fine) and not torch.equal(p[fine], q[fine])


def test_two_optimizers_count_their_own_captured_steps():
    p = torch.ones(100, device=DEV, requires_grad=True)
    p.grad = torch.ones(100, device=DEV)
    opt = FusedAdamW([p], capturable=True)
    opt.step()
    q = p.detach().clone().requires_grad_(True)
    q.grad = p.grad.clone()
    other = FusedAdamW([q], capturable=True)
    other.load_state_dict(opt.state_dict())
    opt.step(), other.step(), other.step(), opt.step()
    assert float(opt.state[p]["step"]) == float(other.state[q]["step"]) == 3 and torch.equal(p, q)


@pytest.mark.parametrize("bits", [8, 32])
def test_set_moments_inside_a_capture_is_refused_and_changes_nothing(bits):
    p = torch.ones(100, device=DEV, requires_grad=True)
    p.grad = torch.ones(100, device=DEV)
    opt = FusedAdamW([p], state_bits=bits, capturable=True)
    opt.step()
    st, before = opt.state[p], opt.moments()[0]
    zero = torch.zeros(100, device=DEV)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.set_moments(p, zero, zero, 5)
    torch.cuda.synchronize()
    assert opt.state[p] is st and float(st["step"]) == 1
    assert all(torch.equal(a, b) for a, b in zip(opt.moments()[0], before))


@pytest.mark.parametrize("types", [(torch.float32,), (torch.float32, torch.bfloat16)])
def test_a_bound_that_is_set_later_is_checked(types):
    """with one launch sequence and with several"""
    ps = [torch.ones(10, device=DEV, dtype=t, requires_grad=True) for t in types]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = FusedAdamW(ps)
    opt.step()
    for bad in (-1.0, float("nan")):
        opt.max_grad_norm = bad
        before = [p.detach().clone() for p in ps]
        with pytest.raises(ValueError, match="max_norm"):
            opt.step()
        assert all(torch.equal(p, q) and opt.state[p]["step"] == 1 for p, q in zip(ps, before))
    opt.max_grad_norm = 1
    opt.step()
    assert abs(float(opt.last_grad_norm) - math.sqrt(10 * len(ps))) < 1e-5


@pytest.mark.parametrize("stepped_before", [False, True])
def test_codes_to_values_and_back_change_no_value(stepped_before):
    """what a densification and a checkpoint of an 8-bit run rely on.  A code is four bits times a power of two, its square eight
    bits: the values, and the root of v, are exact in fp32, and a value that is a code's is rounded to itself."""
    ps, gs = make([1, 7, 128, 129, 4096, 5001, 70003], torch.float32, seed=5)
    opt = FusedAdamW(ps, state_bits=8)
    gen = torch.Generator().manual_seed(1)
    for p, g in zip(ps, gs):
        n = p.numel()
        opt.set_moments(p, (torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen))).to(DEV),
                        (torch.exp(4 * torch.randn(n, generator=gen)) * (torch.rand(n, generator=gen) < 0.9)).to(DEV), 7)
        p.grad = g
    for _ in range(3 if stepped_before else 0):
        opt.step()
    before = opt.moments()
    for p, (m, v) in zip(ps, before):
        opt.set_moments(p, m, v, 7)
    for _ in range(2):  # the same again, by widening
        for p, (m, v), (m2, v2) in zip(ps, before, opt.moments()):
            assert torch.equal(m, m2) and torch.equal(v, v2) and bool(m.any()) and bool(v.any())
            opt.widen(p)
            st = opt.state[p]
            assert torch.equal(st["exp_avg"], m) and torch.equal(st["exp_avg_sq"], v)
            opt._ready(p, st, opt.param_groups[0])
            assert "exp_avg_q" in st and "exp_avg" not in st
