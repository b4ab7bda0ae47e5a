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
