"""What FusedAdamW's state goes through without a GPU: row operations of a cloud, checkpoints and state dicts of other optimizers,
what is refused."""
import pytest
import torch

from fsgs_amd import checkpoint, synth
from fsgs_amd.model import PARAM_NAMES, GaussianCloud
from fsgs_amd.optim import FusedAdamW, clip_grad_norm_


def cloud(**options):
    pc = GaussianCloud(synth.init_scene(16, 12, 20, seed=0), sh_degree=3, device="cpu", scene_radius=1.0)
    pc.training_setup(**options)
    return pc


def coded(p, step=5):
    """an 8-bit state: m = 1, sqrt(v) = 2 everywhere"""
    n = p.numel()
    return {"step": step, "exp_avg_q": torch.ones(p.shape).to(torch.float8_e4m3fn), "exp_avg_sq_q": torch.full(p.shape, 2.0).to(torch.float8_e4m3fn),
            "scales": torch.full((-(-n // 128), 2), 127, dtype=torch.uint8)}


@pytest.fixture
def decoded(monkeypatch):
    """the values of 8-bit moments without the kernel"""
    def read(self, items, dtype):
        out = []
        for p, st in items:
            unit = torch.exp2(st["scales"].float() - 127).repeat_interleave(128, 0)[:p.numel()]
            value = lambda k, j: (st[k].float().reshape(-1) * unit[:, j]).view(p.shape)  # noqa: E731
            out.append((value("exp_avg_q", 0).to(dtype), value("exp_avg_sq_q", 1).square().to(dtype)))
        return out

    monkeypatch.setattr(FusedAdamW, "_read", read)


@pytest.mark.parametrize("bits", [8, 32])
def test_row_operations_keep_moments_whatever_width_is_asked_for_next(decoded, bits):
    pc = cloud(adamw=dict(state_bits=8))
    for p in pc.params.values():
        pc.optimizer.state[p] = coded(p)
    for g in pc.optimizer.param_groups:
        g["state_bits"] = bits  # converted at the next step; until then the state holds codes
    mask = torch.zeros(pc.num_points, dtype=torch.bool)
    mask[::3] = True
    pc.prune_points(mask)
    for name in PARAM_NAMES:
        st = pc.optimizer.state[pc.params[name]]
        assert st["step"] == 5 and st["exp_avg"].shape == pc.params[name].shape
        assert bool((st["exp_avg"] == 1).all()) and bool((st["exp_avg_sq"] == 4).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_an_opacity_reset_keeps_the_count(decoded, bits):
    pc = cloud(adamw=dict(state_bits=8))
    pc.optimizer.state[pc.params["_opacity"]] = coded(pc.params["_opacity"])
    for g in pc.optimizer.param_groups:
        g["state_bits"] = bits
    pc.reset_opacity()
    st = pc.optimizer.state[pc.params["_opacity"]]
    assert st["step"] == 5 and not bool(st["exp_avg"].any()) and not bool(st["exp_avg_sq"].any())


@pytest.mark.parametrize("fused", [True, False])
def test_row_operations_after_an_8_bit_checkpoint_in_a_cloud_of_plain_adam(decoded, fused):
    pc = cloud(adamw=dict(state_bits=8))
    for p in pc.params.values():
        pc.optimizer.state[p] = coded(p)
    other = checkpoint.restore_gaussians(cloud(fused=fused), checkpoint.capture_gaussians(pc), fused=fused)
    other.reset_opacity()
    other.prune_points(torch.arange(other.num_points) % 2 == 0)
    st = other.optimizer.state[other.params["_xyz"]]
    assert int(st["step"]) == 5 and bool((st["exp_avg"] == 1).all()) and st["exp_avg"].shape == other.params["_xyz"].shape


def test_clipping_parameters_of_a_subclass_that_have_no_gradients():
    class Weight(torch.nn.Parameter):
        pass

    for params in (Weight(torch.ones(3)), [Weight(torch.ones(3)), torch.ones(2, requires_grad=True)], (p for p in [Weight(torch.ones(1))])):
        assert float(clip_grad_norm_(params, 1.0)) == 0.0
    w = Weight(torch.ones(3))
    w.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        clip_grad_norm_(w, 1.0)


def saved(**options):
    pc = cloud(**options)
    for i, g in enumerate(pc.optimizer.param_groups):
        g["lr"] = 1e-4 * (i + 1)
    for p in pc.params.values():
        if options.get("adamw", {}).get("state_bits") == 8:
            pc.optimizer.state[p] = coded(p)
        else:
            pc.optimizer.state[p] = {"step": 5, "exp_avg": torch.ones_like(p), "exp_avg_sq": torch.full_like(p, 4.0)}
    return checkpoint.capture_gaussians(pc)


@pytest.mark.parametrize("file,asked,want", [
    # the options that a cloud names go before the file's ...
    (dict(), dict(weight_decay=0.01, betas=(0.9, 0.99), eps=1e-8, state_bits=8),
     dict(weight_decay=0.01, betas=(0.9, 0.99), eps=1e-8, state_bits=8)),
    (dict(fused=False), dict(weight_decay=0.01, maximize=True), dict(weight_decay=0.01, maximize=True, state_bits=32)),
    (dict(adamw=dict(state_bits=8, weight_decay=0.1)), dict(state_bits=32, weight_decay=0.0), dict(state_bits=32, weight_decay=0.0)),
    # ... those that it does not name are the file's, but for how state is held
    (dict(adamw=dict(weight_decay=0.1, betas=(0.8, 0.99), eps=1e-6)), dict(state_bits=8),
     dict(weight_decay=0.1, betas=(0.8, 0.99), eps=1e-6, state_bits=8)),
    (dict(adamw=dict(state_bits=8, master_weights=True, capturable=True)), dict(),
     dict(state_bits=32, master_weights=False, capturable=False, eps=1e-15)),
])
def test_a_restored_cloud_has_the_options_that_it_names(decoded, file, asked, want):
    pc = cloud(adamw={**asked, "lr": 7.0, "max_grad_norm": 2.0})
    checkpoint.restore_gaussians(pc, saved(**file))
    assert isinstance(pc.optimizer, FusedAdamW) and pc.optimizer.max_grad_norm == 2.0
    for i, g in enumerate(pc.optimizer.param_groups):
        assert {k: g[k] for k in want} == want and g["lr"] == 1e-4 * (i + 1) and "max_grad_norm" not in g
    st = pc.optimizer.state[pc.params["_xyz"]]
    assert int(st["step"]) == 5 and bool((st["exp_avg"] == 1).all()) and bool((st["exp_avg_sq"] == 4).all())


def test_a_checkpoint_says_nothing_of_how_its_run_held_the_state(decoded):
    pc = cloud(adamw=dict(state_bits=8, master_weights=True, capturable=True))
    pc.optimizer.param_groups[0]["lr"] = torch.tensor(0.25)
    groups = checkpoint.capture_gaussians(pc)[10]["param_groups"]
    assert all("state_bits" not in g and "master_weights" not in g and g["capturable"] is False for g in groups)
    assert type(groups[0]["lr"]) is float and groups[0]["lr"] == 0.25
    assert all(g["state_bits"] == 8 and g["capturable"] for g in pc.optimizer.param_groups)  # the run's own stay


@pytest.mark.parametrize("options", [dict(weight_decay=0.1), dict(maximize=True)])
def test_a_checkpoint_whose_run_decayed_or_ascended_is_not_continued_without(options):
    file = saved(adamw=options)
    pc = cloud()
    before, optimizer = dict(pc.params), pc.optimizer
    with pytest.raises(ValueError, match=list(options)[0]):
        checkpoint.restore_gaussians(pc, file)
    assert all(pc.params[k] is before[k] for k in before) and pc.optimizer is optimizer
    for ready in (cloud(adamw={}), cloud(fused=False)):
        checkpoint.restore_gaussians(ready, file, fused=ready.adamw is not None)
        assert all({k: g[k] for k in options} == options for g in ready.optimizer.param_groups)
    assert ready.optimizer.param_groups[0]["decoupled_weight_decay"] is True
    checkpoint.restore_gaussians(cloud(), saved(adamw=dict(weight_decay=0.0)))  # nothing is lost


def adam_state(p, dtype=torch.float32, step=3):
    return {"step": step, "exp_avg": torch.full(p.shape, 2.0, dtype=dtype), "exp_avg_sq": torch.full(p.shape, 3.0, dtype=dtype)}


def test_hooks_of_a_load_have_the_last_word():
    p = torch.ones(2, 3, dtype=torch.bfloat16, requires_grad=True)
    opt = FusedAdamW([p])
    opt.state[p] = adam_state(p)
    other = FusedAdamW([p.detach().clone().requires_grad_(True)])
    q = other.param_groups[0]["params"][0]

    def another(_, sd):
        return {**sd, "state": {0: {"step": 9, "exp_avg": torch.full((2, 3), 1.001), "exp_avg_sq": torch.full((2, 3), 5.0)}}}

    def after(o):
        assert o.state[q]["exp_avg"].dtype == torch.float32  # a hook sees what has been loaded
        o.state[q]["exp_avg_sq"] = torch.full((2, 3), 7.0)

    other.register_load_state_dict_pre_hook(another)
    other.register_load_state_dict_post_hook(after)
    for _ in range(2):
        other.load_state_dict(opt.state_dict())
        st = other.state[q]
        assert st["step"] == 9 and bool((st["exp_avg"] == torch.tensor(1.001)).all()) and bool((st["exp_avg_sq"] == 7).all())
    with pytest.raises(ValueError):
        other.load_state_dict({"state": {}, "param_groups": []})
    assert len(other._optimizer_load_state_dict_pre_hooks) == len(other._optimizer_load_state_dict_post_hooks) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("bits", [8, 32])
def test_moments_of_any_floating_type_load_as_float32(dtype, bits):
    """torch's AdamW holds the moments of 16-bit parameters in 16 bits"""
    p = torch.ones(4, 3, dtype=dtype, requires_grad=True)
    p.grad = torch.full((4, 3), 0.25, dtype=dtype)
    theirs = torch.optim.AdamW([p])
    theirs.step()
    assert theirs.state[p]["exp_avg"].dtype == dtype
    q = torch.ones(3, 4, dtype=torch.bfloat16).t().requires_grad_(True)  # another order of dimensions
    opt = FusedAdamW([q], state_bits=bits, master_weights=True)
    sd = theirs.state_dict()
    sd["state"][0]["master"] = torch.full((4, 3), 1.5, dtype=dtype)
    opt.load_state_dict(sd)
    st = opt.state[q]
    for k, v in (("exp_avg", theirs.state[p]["exp_avg"]), ("exp_avg_sq", theirs.state[p]["exp_avg_sq"]), ("master", sd["state"][0]["master"])):
        assert st[k].dtype == torch.float32 and st[k].stride() == q.stride() and torch.equal(st[k], v.float()) and not st[k].requires_grad
    assert int(st["step"]) == 1 and opt._state_tensors(q, st, 32)[0] is st["exp_avg"]


def test_amsgrad_is_refused_and_changes_nothing():
    p, q = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    p.grad = torch.ones(3)
    theirs = torch.optim.AdamW([p], amsgrad=True, lr=0.5)
    theirs.step()
    opt = FusedAdamW([q], lr=0.25)
    opt.state[q] = adam_state(q)
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.state[q]["step"] == 3 and not opt._optimizer_load_state_dict_pre_hooks
    with pytest.raises(ValueError, match="amsgrad"):
        opt.add_param_group({"params": [torch.ones(2, requires_grad=True)], "amsgrad": True})
    assert len(opt.param_groups) == 1
    with pytest.raises(ValueError, match="amsgrad"):
        FusedAdamW([{"params": [q], "amsgrad": True}])
    theirs.param_groups[0]["amsgrad"] = False
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and int(opt.state[q]["step"]) == 1


@pytest.mark.parametrize("capturable", [True, False])
def test_a_loaded_state_shares_nothing_with_the_other_optimizer(capturable):
    p = torch.ones(3, requires_grad=True)
    opt = FusedAdamW([p], capturable=capturable)
    opt.state[p] = {**adam_state(p, step=torch.tensor(4.0)), **coded(p, step=torch.tensor(4.0)), "master": torch.ones(3)}
    other = FusedAdamW([p.detach().clone().requires_grad_(True)], capturable=capturable)
    other.load_state_dict(opt.state_dict())
    st = other.state[other.param_groups[0]["params"][0]]
    assert float(st["step"]) == 4.0 and all(st[k].data_ptr() != v.data_ptr() for k, v in opt.state[p].items())
    opt.state[p]["step"].add_(1.0)
    assert float(st["step"]) == 4.0


@pytest.mark.parametrize("n", [2 ** 63 - 1, 2 ** 63 - 2047, 2 ** 62, 2 ** 35])
def test_sizes_past_what_a_launch_takes_are_refused(n):
    """before anything is launched; the rounding up to whole workgroups passes 2^63 for the first"""
    from array import array

    from fsgs_amd import _lib

    lib, at = _lib.load(), [(k + 1) << 40 for k in range(6)]
    hyper = (_lib.FsgsAdamWHyper * 1)(_lib.FsgsAdamWHyper(1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None))
    for bits in (32, 8):
        row = array("q", (*at[:5], 0, n, 0))
        assert lib.fsgs_adamw_step(1, row.tobytes(), 1, hyper, 0, bits, 0, None, 0.0, None, None, 0, None, None) == _lib.FSGS_ERR_INVALID
    for write in (0, 1):
        assert lib.fsgs_adamw_moments(1, array("q", (*at[:5], n)).tobytes(), write, 0, None) == _lib.FSGS_ERR_INVALID
    grads = array("q", (at[0], n, 0)).tobytes()
    if n * 4 > 2 ** 40:
        assert lib.fsgs_grad_norm(1, grads, 1.0, at[1], 1 << 20, at[2], at[3], None) == _lib.FSGS_ERR_INVALID
        assert lib.fsgs_grad_scale(1, grads, at[1], None) == _lib.FSGS_ERR_INVALID


@pytest.mark.parametrize("step", [-1, 2.5, float("nan"), float("inf"), torch.tensor(-4.0)])
def test_set_moments_refuses_counts_that_are_none(step):
    p = torch.ones(3, requires_grad=True)
    opt = FusedAdamW([p])
    opt.state[p] = before = adam_state(p)
    with pytest.raises(ValueError, match="count"):
        opt.set_moments(p, torch.zeros(3), torch.zeros(3), step)
    assert opt.state[p] is before and before["step"] == 3
    opt.set_moments(p, torch.zeros(3), torch.zeros(3), torch.tensor(7.0))
    assert opt.state[p]["step"] == 7 and type(opt.state[p]["step"]) is int


def test_the_host_extension_is_loaded_for_its_own_torch_alone(monkeypatch):
    from fsgs_amd import _lib

    assert _lib.host().torch_version == torch.__version__
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    for _ in range(2):
        with pytest.raises(ImportError, match="built for torch"):
            _lib.host()
    monkeypatch.undo()
    assert _lib.host().grad_rows([], 16)[1] == -1
