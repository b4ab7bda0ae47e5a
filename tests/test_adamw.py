"""FusedAdamW, grad_norm and clip_grad_norm_ without a GPU: what is refused, and before anything is launched; layouts of the
C structures; state entries."""
import ctypes
from array import array

import pytest
import torch

from fsgs_amd import _lib
from fsgs_amd.optim import FusedAdamW, clip_grad_norm_, grad_norm

INVALID = _lib.FSGS_ERR_INVALID
A = 1 << 40  # addresses that nothing reads: every call below is refused, or has no elements


def hyper(step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step_dev=None):
    return _lib.FsgsAdamWHyper(lr, b1, b2, eps, wd, step, step_dev, None)


def step(rows, hypers=None, dtype=0, bits=32, scratch=None, limit=(None, 0.0, None, None, 0)):
    hypers = [hyper()] if hypers is None else hypers
    table = array("q", [w for r in rows for w in r])
    return _lib.load().fsgs_adamw_step(len(rows), table.buffer_info()[0] if rows else None, len(hypers),
                                       (_lib.FsgsAdamWHyper * len(hypers))(*hypers), dtype, bits, 0, *limit, scratch, None)


def row(k=0, n=100, p=0, g=1, m=2, v=3, scales=4, master=None, h=0):
    at = lambda i: A + (i << 20) + (k << 30)  # noqa: E731
    return (at(p), at(g), at(m), at(v), at(scales), 0 if master is None else at(master), n, h)


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(_lib.FsgsAdamWHyper) == 64
    assert (_lib.ADAMW_TENSOR_WORDS, _lib.ADAMW_MOMENTS_WORDS, _lib.GRAD_TENSOR_WORDS) == (8, 6, 3)


def test_step_without_tensors_or_elements_is_a_no_op():
    assert step([]) == 0
    assert step([(0, 0, 0, 0, 0, 0, 0, 0)]) == 0
    assert step([(0, 0, 0, 0, 0, 0, 0, 0)], bits=8) == 0


@pytest.mark.parametrize("bad", [
    dict(rows=[row(n=-1)]), dict(rows=[row(h=1)]), dict(rows=[row(h=-1)]), dict(rows=[row()], dtype=3), dict(rows=[row()], bits=16),
    dict(rows=[row()], hypers=[hyper(step=0)]), dict(rows=[row()], hypers=[hyper(lr=-1.0)]),
    dict(rows=[row()], hypers=[hyper(lr=float("nan"))]), dict(rows=[row()], hypers=[hyper(b1=1.0)]),
    dict(rows=[row()], hypers=[hyper(b2=-0.1)]), dict(rows=[row()], hypers=[hyper(eps=-1.0)]),
    dict(rows=[row()], hypers=[hyper(wd=-1.0)]),
    dict(rows=[row(master=5)]),                                       # masters of fp32 parameters
    dict(rows=[row(master=5), row(1)], dtype=1),                      # masters of some
    dict(rows=[(0,) + row()[1:]]), dict(rows=[row()[:1] + (0,) + row()[2:]]),
    dict(rows=[row()[:4] + (0,) + row()[5:]], bits=8),                # no scales
    dict(rows=[row(n=1 << 46)]),                                      # more workgroups than a launch has
    dict(rows=[row()], limit=(A, 1.0, A + 64, A + 128, 1 << 20)),     # a factor and a bound
    dict(rows=[row()], limit=(None, -1.0, A + 64, A + 128, 1 << 20)), dict(rows=[row()], limit=(None, float("nan"), A + 64, A + 128, 1 << 20)),
    dict(rows=[row()], limit=(None, 1.0, A + 64, None, 1 << 20)), dict(rows=[row()], limit=(None, 1.0, A + 64, A + 128, 8)),
    dict(rows=[row()], hypers=[hyper(step_dev=A)]),                   # a step on the device without scratch
    dict(rows=[row(), row(1, h=1)], hypers=[hyper(step_dev=A), hyper()], scratch=A + 64),
    dict(rows=[row(), row(1)], hypers=[hyper(step_dev=A + 8)], scratch=A + 64),  # two tensors on one count
])
def test_step_refuses(bad):
    assert step(**bad) == INVALID


@pytest.mark.parametrize("rows", [
    [row(), row()],                                   # the same tensor twice
    [row(m=3)],                                       # both moments in one place
    [row(g=0)],                                       # the gradient is the parameter
    [row(), (A + 396,) + row(1)[1:]],                 # the last element of one is the first of the next
    [row(), row(1)[:1] + (A + (2 << 20) + 8,) + row(1)[2:]],  # a gradient inside another tensor's moment
])
def test_step_refuses_memory_that_would_race(rows):
    assert step(rows) == INVALID
    assert step(list(reversed(rows))) == INVALID


def test_moments_norm_and_scale_refuse():
    lib = _lib.load()
    good = (A, A + (1 << 20), A + (2 << 20), A + (3 << 20), A + (4 << 20), 100)

    def call(r, write=0, dtype=0):
        table = array("q", r)
        return lib.fsgs_adamw_moments(1, table.buffer_info()[0], write, dtype, None)

    assert call((0, 0, 0, 0, 0, 0)) == 0
    for k in range(5):
        assert call(good[:k] + (0,) + good[k + 1:]) == INVALID
    assert call(good[:5] + (-1,)) == INVALID and call(good, 1, 1) == INVALID and call(good, 0, 7) == INVALID
    assert call(good[:4] + (good[3], 100)) == INVALID

    def norm(r, bound=1.0, out=A, scratch=A, nbytes=1 << 20):
        table = array("q", r)
        return lib.fsgs_grad_norm(1, table.buffer_info()[0], bound, scratch, nbytes, out, A + 128, None)

    assert norm((A, -1, 0)) == norm((0, 4, 0)) == norm((A, 4, 9)) == norm((A, 1 << 50, 0)) == INVALID
    assert norm((A, 4, 0), -1.0) == norm((A, 4, 0), float("nan")) == norm((A, 4, 0), out=None) == norm((A, 4, 0), scratch=None) == INVALID
    assert norm((A, 4, 0), nbytes=0) == _lib.FSGS_ERR_CAPACITY
    twice = array("q", (A, 4, 0, A + 12, 4, 0))
    assert lib.fsgs_grad_scale(2, twice.buffer_info()[0], A + 64, None) == INVALID
    assert lib.fsgs_grad_clip(2, twice.buffer_info()[0], 1.0, A, 1 << 20, A + 64, A + 128, None) == INVALID
    assert lib.fsgs_grad_clip(1, twice.buffer_info()[0], 1.0, A, 1 << 20, A + 64, None, None) == INVALID
    assert lib.fsgs_grad_scale(1, twice.buffer_info()[0], None, None) == INVALID
    assert lib.fsgs_grad_scale(0, None, None, None) == 0


def leaf(*shape, dtype=torch.float32):
    p = torch.ones(shape, dtype=dtype, requires_grad=True)
    p.grad = torch.ones(shape, dtype=dtype)
    return p


@pytest.mark.parametrize("kw", [dict(lr=-1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1),
                                dict(state_bits=4), dict(lr=float("nan")), dict(max_grad_norm=-1.0),
                                dict(max_grad_norm=float("nan")), dict(lr=torch.ones(2))])
def test_options_out_of_range_raise(kw):
    with pytest.raises(ValueError):
        FusedAdamW([leaf(3)], **kw)


def test_parameters_of_other_types_and_given_twice_raise():
    with pytest.raises(TypeError):
        FusedAdamW([leaf(3, dtype=torch.float64)])
    p = leaf(3)
    with pytest.raises(ValueError):
        FusedAdamW([p, p])
    opt = FusedAdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [leaf(2)], "lr": -1.0})
    assert len(opt.param_groups) == 1
    opt.param_groups[0]["lr"] = -1.0  # a schedule gone wrong
    with pytest.raises(ValueError):
        opt.step()


def test_tensors_on_the_cpu_raise():
    opt = FusedAdamW([leaf(3)])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()
    assert len(opt.state) == 0 or "step" not in opt.state[opt.param_groups[0]["params"][0]]
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        grad_norm([torch.ones(3)])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        clip_grad_norm_([leaf(3)], 1.0)
    opt8 = FusedAdamW([leaf(3)], state_bits=8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt8.set_moments(opt8.param_groups[0]["params"][0], torch.zeros(3), torch.zeros(3), 1)


def test_nothing_to_do():
    p = torch.ones(3, requires_grad=True)
    assert FusedAdamW([p]).step() is None and FusedAdamW([p]).step(lambda: 7) == 7
    assert FusedAdamW([p]).moments() == []
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    with pytest.raises(ValueError):
        clip_grad_norm_([p], 1.0, norm_type=1)
    with pytest.raises(ValueError):
        clip_grad_norm_([p], -1.0)
    with pytest.raises(TypeError):
        FusedAdamW([p]).moments(torch.float64)
    with pytest.raises(ValueError):
        FusedAdamW([p]).set_moments(torch.ones(3), p, p, 1)
    with pytest.raises(ValueError):
        FusedAdamW([p]).set_moments(p, torch.zeros(2), p, 1)


def test_set_moments_and_groups_of_another_adam():
    p = torch.ones(2, 3, requires_grad=True)
    opt = FusedAdamW([p])
    opt.set_moments(p, torch.full((2, 3), 2.0), torch.full((2, 3), 3.0), 5)
    (m, v), = opt.moments(torch.bfloat16)
    assert m.dtype == torch.bfloat16 and float(m.sum()) == 12.0 and float(v.sum()) == 18.0 and opt.state[p]["step"] == 5
    q = torch.ones(2, 3, requires_grad=True)
    other = torch.optim.Adam([q], lr=0.5)
    q.grad = torch.ones(2, 3)
    other.step()
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["state_bits"] == 32
    assert torch.equal(opt.state[p]["exp_avg"], other.state[q]["exp_avg"])


def test_state_dict_keeps_every_entrys_type():
    p = torch.ones(2, 3, dtype=torch.bfloat16, requires_grad=True)
    opt = FusedAdamW([p], state_bits=8, master_weights=True)
    codes = torch.arange(6, dtype=torch.uint8).view(2, 3).view(torch.float8_e4m3fn)
    opt.state[p] = {"step": 4, "exp_avg_q": codes, "exp_avg_sq_q": codes.clone(), "scales": torch.full((1, 2), 9, dtype=torch.uint8),
                    "master": torch.full((2, 3), 1.0001)}
    fresh = FusedAdamW([p.detach().clone().requires_grad_(True)], state_bits=8, master_weights=True)
    fresh.load_state_dict(opt.state_dict())
    st = fresh.state[fresh.param_groups[0]["params"][0]]
    assert st["step"] == 4 and st["exp_avg_q"].dtype == torch.float8_e4m3fn and st["scales"].dtype == torch.uint8
    assert torch.equal(st["exp_avg_q"].view(torch.uint8), codes.view(torch.uint8)) and st["exp_avg_q"] is not codes
    assert torch.equal(st["master"], opt.state[p]["master"])


def test_copies_and_pickles_keep_the_bound():
    import copy
    import pickle

    opt = FusedAdamW([leaf(3)], max_grad_norm=0.5, state_bits=8)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_grad_norm == 0.5 and other.last_grad_norm is None and other.param_groups[0]["state_bits"] == 8
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            other.param_groups[0]["params"][0].grad = torch.ones(3)
            other.step()


def test_the_cloud_takes_adamw_and_keeps_it():
    from fsgs_amd import synth
    from fsgs_amd.model import GaussianCloud

    pc = GaussianCloud(synth.init_scene(16, 12, 20, seed=0), sh_degree=3, device="cpu")
    pc.training_setup(adamw=dict(state_bits=8, max_grad_norm=1.0))
    opt = pc.optimizer
    assert isinstance(opt, FusedAdamW) and opt.max_grad_norm == 1.0
    assert all(g["weight_decay"] == 0.0 and g["state_bits"] == 8 for g in opt.param_groups)
    pc.initialize_optimizer()
    assert isinstance(pc.optimizer, FusedAdamW) and pc.optimizer is not opt and pc.optimizer.param_groups[0]["state_bits"] == 8
    pc.training_setup()
    assert not isinstance(pc.optimizer, FusedAdamW)
