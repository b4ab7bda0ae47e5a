"""Fused optimiser pieces: `FusedAdam` (drop-in for the torch.optim.Adam instances the reference
builds at scene/gaussian_model.py:372-378,408 and scene/pose_optimizer.py:489-493 -- same param_groups
and state layout, so densification's state surgery keeps working), `FusedAdamW` (decoupled weight decay, any number of
tensors, 16-bit parameters, moments in 32 or 8 bits), `grad_norm` / `clip_grad_norm_`, and the densification statistics."""
import ctypes as C
from array import array

import torch

from . import _lib


def mark_updated(tensors):
    """The HIP kernels write parameters behind autograd's back; bump the version counters like an in-place torch op
    would (no kernel is launched), so version-keyed caches and autograd's saved-tensor checks stay truthful."""
    for t in tensors:
        torch.autograd.graph.increment_version(t)


class FusedAdam(torch.optim.Optimizer):
    """torch.optim.Adam semantics (betas, eps, no weight decay / amsgrad / maximize) with every group
    updated by ONE HIP kernel launch.  state[p] = {'step' (python int), 'exp_avg', 'exp_avg_sq'}."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))

    @torch.no_grad()
    def step(self, closure=None):
        lib = _lib.load()
        by_hyper = {}
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("FusedAdam needs CUDA/HIP tensors; there is no CPU fallback")
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] = int(st["step"]) + 1
                g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                key = (group["betas"][0], group["betas"][1], group["eps"], p.device)
                by_hyper.setdefault(key, []).append((p, g, st, float(group["lr"])))
        for (b1, b2, eps, dev), items in by_hyper.items():
            with torch.cuda.device(dev):
                stream = _lib.current_stream()
                for i in range(0, len(items), 8):
                    chunk = items[i:i + 8]
                    arr = (_lib.FsgsAdamGroup * len(chunk))()
                    for k, (p, g, st, lr) in enumerate(chunk):
                        arr[k].param, arr[k].grad = p.data_ptr(), g.data_ptr()
                        arr[k].exp_avg, arr[k].exp_avg_sq = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
                        arr[k].n, arr[k].lr, arr[k].step = p.numel(), lr, st["step"]
                    _lib.check(lib.fsgs_adam_step(len(chunk), arr, b1, b2, eps, stream), "fsgs_adam_step")
                mark_updated([it[0] for it in items])
        return None


_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_F32, _Q = torch.float32, torch.float8_e4m3fn


def _dense(t):
    """every element of t's span of memory belongs to t exactly once (contiguous up to the order of the dimensions)"""
    if t.is_contiguous():
        return True
    want = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda ns: ns[1]):
        if stride != want:
            return False
        want *= size
    return True


def _same_layout(a, b):
    return a.shape == b.shape and ((a.is_contiguous() and b.is_contiguous()) or a.stride() == b.stride())


def _address(buf):
    return buf.buffer_info()[0]


class _on:
    """the device of a bucket of tensors made current (nothing to do where it is already)"""

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_grad(g, name="gradient"):
    if g.layout != torch.strided:
        raise RuntimeError("%s: sparse gradients are not supported" % name)
    if not g.is_cuda:
        raise RuntimeError("%s: needs CUDA/HIP tensors; there is no CPU fallback" % name)
    if g.dtype not in _DTYPES:
        raise TypeError("%s: float32, bfloat16 or float16, got %s" % (name, g.dtype))


class _Grads:
    """what a norm's launches need: rows of FsgsGradTensor as bytes, on one device (None: no gradients), the tensor for the norm,
    scratch whose first float is the factor; `dense`: whether all are; `slow`: what to keep until the launch, None where all
    were as one expects"""

    def __init__(self, device, table, norm, scratch, dense=True, slow=None):
        self.device, self.table, self.norm, self.scratch, self.dense, self.slow = device, table, norm, scratch, dense, slow

    def __len__(self):
        return len(self.table) // (8 * _lib.GRAD_TENSOR_WORDS)

    def launch(self, entry, max_norm):
        """the return code of fsgs_grad_norm / _clip, on the device's current stream (the device has been made current)"""
        at = self.factor = self.scratch.data_ptr()
        return entry(len(self), self.table, max_norm, at + 16, self.scratch.numel() - 16, self.norm.data_ptr(), at,
                     _lib.current_stream())


def _scratch_bytes(n):
    return 16 + _lib.load().fsgs_grad_norm_scratch_bytes(n)


def _grads_of(params, who):
    fast = _lib.host().grad_rows(params, _scratch_bytes(len(params)))
    if fast is not None:
        table, index, norm, scratch = fast
        return _Grads(torch.device("cuda", index) if index >= 0 else None, table, norm, scratch)
    grads = [p.grad for p in params if p.grad is not None]
    return _grads_from(grads, who) if grads else _Grads(None, b"", None, None)


@torch.no_grad()
def _grads_from(grads, who):
    dev, table, keep, dense = _one_device(grads, who), array("q"), [], True
    for g in grads:
        if g.is_neg():
            raise RuntimeError("%s: a gradient is a negated view (resolve_neg)" % who)
        if not _dense(g):
            dense, g = False, g.contiguous()
            keep.append(g)
        table.extend((g.data_ptr(), g.numel(), _DTYPES[g.dtype]))
    return _Grads(dev, table.tobytes(), torch.empty((), dtype=_F32, device=dev),
                  torch.empty(_scratch_bytes(len(grads)), dtype=torch.uint8, device=dev), dense, keep)


def _one_device(grads, who):
    dev = grads[0].device
    for g in grads:
        _check_grad(g, who)
        if g.device != dev:
            raise RuntimeError("%s: gradients on %s and on %s; call it once for each device" % (who, dev, g.device))
    return dev


def _max_norm(v):
    v = float(v)
    if not v >= 0.0:
        raise ValueError("max_norm is a number that is not negative, got %r" % v)
    return v


def grad_norm(tensors):
    """Global 2-norm of any number of float32 / bfloat16 / float16 tensors on one device: a 0-d float32 tensor there, without a
    gradient and without a host synchronisation.  Squares are summed in 64 bits and in a fixed order."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    found = _grads_from(tensors, "grad_norm")
    with _on(found.device):
        _lib.check(found.launch(_lib.load().fsgs_grad_norm, float("inf")), "fsgs_grad_norm")
    return found.norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ in two launches for every 192 tensors (norm, scaling), and one between them where all
    gradients make more than 256 pieces of 16 KB: the gradients' global 2-norm, and every gradient
    (dense, on one device, float32 / bfloat16 / float16 side by side) scaled in place by min(1, max_norm / (norm + 1e-6));
    where that factor is 1 no gradient is read again.  Returns the norm (0-d float32) without a host synchronisation, unless
    error_if_nonfinite asks for one."""
    if float(norm_type) != 2.0:
        raise ValueError("clip_grad_norm_: the 2-norm only, got norm_type=%r" % (norm_type,))
    max_norm = _max_norm(max_norm)
    parameters = [parameters] if torch.is_tensor(parameters) else list(parameters)
    lib = _lib.load()
    found = _grads_of(parameters, "clip_grad_norm_")
    if found.device is None:
        return torch.tensor(0.0)
    if not found.dense:
        raise ValueError("clip_grad_norm_: gradients are dense in memory; scale slices of other tensors by hand")
    with _on(found.device):
        rc = found.launch(lib.fsgs_grad_norm if error_if_nonfinite else lib.fsgs_grad_clip, max_norm)
        if error_if_nonfinite and rc == _lib.FSGS_OK:
            if not bool(torch.isfinite(found.norm)):
                raise RuntimeError("clip_grad_norm_: the gradients' norm is %s" % float(found.norm))
            rc = lib.fsgs_grad_scale(len(found), found.table, found.factor, _lib.current_stream())
        if rc == _lib.FSGS_ERR_INVALID:
            raise ValueError("clip_grad_norm_: two of the gradients share memory, or a parameter is given twice")
        _lib.check(rc, "fsgs_grad_clip")
    if found.slow is None:
        _lib.host().grads_written(parameters)
    else:
        mark_updated([p.grad for p in parameters if p.grad is not None])
    return found.norm


class FusedAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW semantics (decoupled weight decay; no amsgrad) over any number of tensors, 48 a kernel launch.

    Parameters may be float32, bfloat16 or float16 (gradients of the same type), dense in memory, on one or several devices.
    Options, each also per param_group except max_grad_norm:

    state_bits      32: state[p] = {'step', 'exp_avg', 'exp_avg_sq'} in float32, whatever the parameter's type.
                    8: {'step', 'exp_avg_q', 'exp_avg_sq_q', 'scales'}: e4m3 codes of m and of sqrt(v) under one power of two
                    per 128 elements (include/fsgs.h, fsgs_adamw_step); 2.02 bytes an element instead of 8.  `moments()`
                    and `set_moments()` convert.  Changing a group's state_bits converts its moments at the next step.
    master_weights  float32 copies of 16-bit parameters in state[p]['master'], which the step updates; the parameter is the
                    copy rounded to nearest.  Made from the parameter at its first step: after writing to a parameter by
                    hand, delete its 'master'.
    maximize        ascend.
    capturable      'step' is a 0-d float32 tensor on the parameter's device and lr may be one too, so that a step captured
                    into a graph counts on at every replay.  A step of any other group inside a capture is refused.  Run one
                    eager step before the capture: it makes the state.
    max_grad_norm   bound on the 2-norm over the gradients of ALL groups (one device then): the step uses the gradients times
                    min(1, max_grad_norm / (norm + 1e-6)) and leaves .grad as it is (a NaN among them makes every parameter
                    NaN, as clip_grad_norm_ in front of a step does); `last_grad_norm` is that norm, 0-d on the device.
                    Not part of state_dict()."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, state_bits=32,
                 master_weights=False, capturable=False, max_grad_norm=None):
        self.max_grad_norm = None if max_grad_norm is None else _max_norm(max_grad_norm)
        self.last_grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize,
                                      state_bits=state_bits, master_weights=master_weights, capturable=capturable))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._scalars(group)
            self._no_amsgrad(group)
            if len({id(p) for p in group["params"]}) != len(group["params"]):
                raise ValueError("FusedAdamW: a parameter is given twice in one group")
            for p in group["params"]:
                if p.dtype not in _DTYPES:
                    raise TypeError("FusedAdamW: float32, bfloat16 or float16 parameters, got %s" % p.dtype)
        except Exception:
            self.param_groups.pop()
            raise

    def __getstate__(self):
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("max_grad_norm", None)
        self.__dict__.setdefault("last_grad_norm", None)
        for group in self.param_groups:  # groups saved by another Adam
            for k, v in self.defaults.items():
                group.setdefault(k, v)

    @staticmethod
    def _no_amsgrad(group):
        if group.get("amsgrad"):
            raise ValueError("FusedAdamW: amsgrad is not supported")

    @staticmethod
    def _scalars(group):
        """(lr, beta1, beta2, eps, weight_decay, lr tensor or None) of a group, checked"""
        lr, lr_dev = group["lr"], None
        if torch.is_tensor(lr):
            if lr.numel() != 1:
                raise ValueError("FusedAdamW: lr is a number or a tensor of one element")
            if lr.is_cuda:
                if not group["capturable"]:
                    raise ValueError("FusedAdamW: lr as a tensor on the device needs capturable=True")
                lr_dev, lr = lr, 0.0
        lr, (b1, b2), eps, wd = float(lr), group["betas"], float(group["eps"]), float(group["weight_decay"])
        b1, b2 = float(b1), float(b2)
        for name, v, ok in (("lr", lr, lr >= 0), ("beta1", b1, 0 <= b1 < 1), ("beta2", b2, 0 <= b2 < 1), ("eps", eps, eps >= 0),
                            ("weight_decay", wd, wd >= 0)):
            if not ok:
                raise ValueError("FusedAdamW: invalid %s: %r" % (name, v))
        if group["state_bits"] not in (8, 32):
            raise ValueError("FusedAdamW: state_bits is 8 or 32, got %r" % (group["state_bits"],))
        return lr, b1, b2, eps, wd, lr_dev

    # ---- state ------------------------------------------------------------------------------------------------------
    @staticmethod
    def _blocks(p):
        return -(-p.numel() // _lib.ADAMW_BLOCK)

    @staticmethod
    def _no_capture(p):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: a parameter's state would be made inside a graph capture; run one eager step first")

    def _ready(self, p, st, group):
        """the entries that the group's options ask for: made on the first step, converted where the options changed"""
        self._no_capture(p)
        like = dict(memory_format=torch.preserve_format)
        if group["state_bits"] == 32 and "exp_avg" not in st:
            if "exp_avg_q" in st:
                self.widen(p)
                st = self.state[p]
            else:
                st["exp_avg"], st["exp_avg_sq"] = torch.zeros_like(p, dtype=_F32, **like), torch.zeros_like(p, dtype=_F32, **like)
        elif group["state_bits"] == 8 and "exp_avg_q" not in st:
            if "exp_avg" in st:
                self._write(p, st, st.pop("exp_avg"), st.pop("exp_avg_sq"))
            else:
                st["exp_avg_q"], st["exp_avg_sq_q"], st["scales"] = self._codes(p)
        if group["master_weights"] and p.dtype != _F32 and "master" not in st:
            st["master"] = p.detach().to(_F32, **like)
        step = st.get("step", 0)
        if group["capturable"]:
            if not (torch.is_tensor(step) and step.device == p.device and step.dtype == _F32):
                st["step"] = torch.full((), float(step), dtype=_F32, device=p.device)
        else:
            st["step"] = int(step)
        return st

    def _codes(self, p):
        q = lambda: torch.empty_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).zero_().view(_Q)  # noqa: E731
        return q(), q(), torch.zeros((self._blocks(p), 2), dtype=torch.uint8, device=p.device)

    def _state_tensors(self, p, st, bits):
        """(m, v, scales or None), checked: raw pointers cross the C ABI"""
        if bits == 32:
            m, v, scales, want = st["exp_avg"], st["exp_avg_sq"], None, _F32
        else:
            m, v, scales, want = st["exp_avg_q"], st["exp_avg_sq_q"], st["scales"], _Q
            if scales.dtype != torch.uint8 or scales.numel() != 2 * self._blocks(p) or not scales.is_contiguous() or \
                    scales.device != p.device:
                raise ValueError("FusedAdamW: state['scales'] is a contiguous uint8 [%d, 2] on %s" % (self._blocks(p), p.device))
        if m.dtype != want or v.dtype != want or m.device != p.device or v.device != p.device or \
                not _same_layout(m, p) or not _same_layout(v, p):
            raise ValueError("FusedAdamW: the moments of a parameter are %s tensors of its shape and strides on its device; got "
                             "%s %s and %s %s for %s" % (want, tuple(m.shape), m.dtype, tuple(v.shape), v.dtype, tuple(p.shape)))
        return m, v, scales

    def _read(self, items, dtype):
        """values of 8-bit moments: one launch per 48 tensors of a device"""
        lib, out, by_device = _lib.load(), [], {}
        for p, st in items:
            mq, vq, scales = self._state_tensors(p, st, 8)
            if not p.is_cuda:
                raise RuntimeError("FusedAdamW needs CUDA/HIP tensors; there is no CPU fallback")
            m = torch.empty_like(mq, dtype=dtype, memory_format=torch.preserve_format)
            v = torch.empty_like(mq, dtype=dtype, memory_format=torch.preserve_format)
            out.append((m, v))
            by_device.setdefault(p.device, array("q")).extend(
                (mq.data_ptr(), vq.data_ptr(), scales.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel()))
        for dev, table in by_device.items():
            with _on(dev):
                _lib.check(lib.fsgs_adamw_moments(len(table) // _lib.ADAMW_MOMENTS_WORDS, _address(table), 0, _DTYPES[dtype],
                                                  _lib.current_stream()), "fsgs_adamw_moments")
        return out

    def _write(self, p, st, m, v):
        lib = _lib.load()
        if not p.is_cuda:
            raise RuntimeError("FusedAdamW needs CUDA/HIP tensors; there is no CPU fallback")
        if not _dense(p):
            raise ValueError("FusedAdamW: parameters are dense in memory")
        st["exp_avg_q"], st["exp_avg_sq_q"], st["scales"] = self._codes(p)
        m, v = (torch.empty_like(p, dtype=_F32, memory_format=torch.preserve_format).copy_(x.detach()) for x in (m, v))
        table = array("q", (st["exp_avg_q"].data_ptr(), st["exp_avg_sq_q"].data_ptr(), st["scales"].data_ptr(), m.data_ptr(),
                            v.data_ptr(), p.numel()))
        with _on(p.device):
            _lib.check(lib.fsgs_adamw_moments(1, _address(table), 1, _lib.DTYPE_F32, _lib.current_stream()), "fsgs_adamw_moments")

    @torch.no_grad()
    def moments(self, dtype=torch.float32):
        """[(m, v)] of every parameter that has a state, in the order of the groups: copies of the parameter's shape in `dtype`.
        float32 and bfloat16 hold what 8-bit moments stand for exactly.  Those of packed 8-bit states are cut from one new
        buffer, which lives (and is saved by torch.save) as long as any of them: clone what is to be kept alone."""
        if dtype not in _DTYPES:
            raise TypeError("moments: float32, bfloat16 or float16, got %s" % dtype)
        fast = _lib.host().moment_rows(self.param_groups, self.state, dtype)
        if fast is not None:  # all of them in 8 bits, packed, on one device
            pairs, rows, index = fast
            with _on(torch.device("cuda", index)):
                _lib.check(_lib.load().fsgs_adamw_moments(len(pairs), rows, 0, _DTYPES[dtype], _lib.current_stream()),
                           "fsgs_adamw_moments")
            return pairs
        items = [(p, self.state[p]) for group in self.param_groups for p in group["params"]
                 if p in self.state and ("exp_avg" in self.state[p] or "exp_avg_q" in self.state[p])]
        read = iter(self._read([it for it in items if "exp_avg_q" in it[1]], dtype))
        return [next(read) if "exp_avg_q" in st else tuple(st[k].to(dtype, copy=True) for k in ("exp_avg", "exp_avg_sq"))
                for _, st in items]

    @torch.no_grad()
    def widen(self, p):
        """8-bit moments of parameter p as float32 'exp_avg' / 'exp_avg_sq' in its state (nothing to do where they are, or
        where p has no state), for code that cuts or joins their rows; p's next step brings them back to the group's
        state_bits"""
        if "exp_avg_q" in self.state.get(p, {}):
            self.state[p] = self.wide_state(p)

    @torch.no_grad()
    def wide_state(self, p):
        """a copy of p's state entry (tensors shared) with float32 'exp_avg' / 'exp_avg_sq' whatever the moments' width, and
        'step' as a number"""
        st = dict(self.state[p])
        if "step" in st and torch.is_tensor(st["step"]):
            st["step"] = int(st["step"])
        if "exp_avg_q" in st:
            st["exp_avg"], st["exp_avg_sq"] = self._read([(p, st)], _F32)[0]
            for k in ("exp_avg_q", "exp_avg_sq_q", "scales"):
                del st[k]
        return st

    @torch.no_grad()
    def set_moments(self, p, m, v, step):
        """install values as the moments of parameter p (8-bit groups: rounded to the nearest codes) and its count of steps;
        a 'master' that the state held is dropped and made again from p"""
        group = next((g for g in self.param_groups if any(q is p for q in g["params"])), None)
        if group is None:
            raise ValueError("set_moments: not a parameter of this optimizer")
        if m.shape != p.shape or v.shape != p.shape:
            raise ValueError("set_moments: moments of shape %s and %s for a parameter of shape %s" % (
                tuple(m.shape), tuple(v.shape), tuple(p.shape)))
        self._no_capture(p)
        if not (0 <= float(step) < 2 ** 53 and float(step) == int(step)):
            raise ValueError("set_moments: a count of steps is a whole number that is not negative, got %r" % (step,))
        st = {"step": step}
        if group["state_bits"] == 8:
            self._write(p, st, m, v)
        else:
            st["exp_avg"], st["exp_avg_sq"] = (
                torch.empty_like(p, dtype=_F32, memory_format=torch.preserve_format).copy_(x.detach()) for x in (m, v))
        self.state[p] = st
        self._ready(p, st, group)

    def load_state_dict(self, state_dict):
        """as torch's, but every entry keeps its own type (torch casts floating state to the parameter's), and moments and masters
        become float32 in the parameter's layout, whatever floating type another optimizer held them in"""
        taken = []

        def take(_, sd):  # the last of these hooks: what the others made of it
            for group in sd["param_groups"]:
                self._no_amsgrad(group)
            taken.append(sd)

        hooks = (self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self._keep_types(taken[-1]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _keep_types(self, state_dict):
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, mine):
            for k, v in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(v) and k == "step":  # torch has moved it where it belongs, and may have kept the very tensor
                    self.state[p][k] = self.state[p][k].clone()
                elif torch.is_tensor(v):
                    if k in ("exp_avg", "exp_avg_sq", "master") and v.is_floating_point() and v.shape == p.shape:
                        self.state[p][k] = torch.empty_like(p, dtype=_F32, memory_format=torch.preserve_format,
                                                            requires_grad=False).copy_(v.detach())
                    else:
                        self.state[p][k] = v.detach().to(p.device, copy=True)

    # ---- the step -----------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        work = self._ordinary()
        if work is None:
            work = self._general()
        if not work:
            return loss
        # (factor, bound, norm, scratch, its bytes): nothing, the bound that a single bucket applies by itself, or the factor
        # from the norm over several
        limit = (None, 0.0, None, None, 0)
        max_norm = None if self.max_grad_norm is None else _max_norm(self.max_grad_norm)  # it may have been set since
        if max_norm is not None and len(work) == 1:
            nbytes = _scratch_bytes(len(work[0].params))
            norm, hold = _lib.host().norm_buffers(work[0].device.index, nbytes)
            limit, self.last_grad_norm = (None, max_norm, norm.data_ptr(), hold.data_ptr(), nbytes), norm
        elif max_norm is not None:
            found = hold = _grads_of([p for b in work for p in b.params], "FusedAdamW(max_grad_norm)")
            with _on(found.device):
                _lib.check(found.launch(lib.fsgs_grad_norm, max_norm), "fsgs_grad_norm")
            limit, self.last_grad_norm = (found.factor, 0.0, None, None, 0), found.norm
        for b in work:
            n = len(b.params)
            rows, hypers = b.arrays()
            with _on(b.device):
                scratch = torch.empty(lib.fsgs_adamw_scratch_bytes(n), dtype=torch.uint8, device=b.device) if b.capturable else None
                rc = lib.fsgs_adamw_step(n, rows, len(hypers) // _lib.ADAMW_HYPER_BYTES, hypers, b.dtype, b.bits, b.maximize, *limit,
                                         _lib.ptr(scratch), _lib.current_stream())
                if rc == _lib.FSGS_ERR_INVALID:
                    raise ValueError("FusedAdamW: two of the tensors of a step share memory (or one has 2^35 elements or more)")
                _lib.check(rc, "fsgs_adamw_step")
            _lib.host().stepped(b.params, b.states)
        return loss

    def _ordinary(self):
        """The buckets of a step whose tensors and options are all as one expects them -- packed tensors with their states in
        place, options that are plain numbers in range -- collected by the host extension; None where anything is not."""
        found = _lib.host().step_rows(self.param_groups, self.state)
        if found is None or (found and torch.cuda.is_current_stream_capturing()):
            return None
        return [_Bucket(torch.device("cuda", index), dtype, bits, maximize, False, rows, hypers, params, states)
                for index, dtype, bits, maximize, rows, hypers, params, states in found]

    @torch.no_grad()
    def _general(self):
        """The buckets of any step that can be made: every tensor looked at in turn; states made or converted."""
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        buckets = {}
        for group in self.param_groups:
            lr, b1, b2, eps, wd, lr_dev = self._scalars(group)
            bits, masters, capturable = group["state_bits"], group["master_weights"], bool(group["capturable"])
            moment = "exp_avg" if bits == 32 else "exp_avg_q"
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                dt, dev = p.dtype, p.device
                if not p.is_cuda:
                    raise RuntimeError("FusedAdamW needs CUDA/HIP tensors; there is no CPU fallback")
                if g.layout != torch.strided:
                    raise RuntimeError("FusedAdamW: sparse gradients are not supported")
                if dt not in _DTYPES or g.dtype != dt or g.device != dev:
                    raise TypeError("FusedAdamW: a gradient has its parameter's type and device; got %s on %s for %s on %s" % (
                        g.dtype, g.device, dt, dev))
                if p.is_neg() or g.is_neg():
                    raise RuntimeError("FusedAdamW: a parameter or gradient is a negated view (resolve_neg)")
                if capturing and not capturable:
                    raise RuntimeError("FusedAdamW: a step inside a graph capture needs capturable=True (its count and "
                                       "learning rate would be frozen at every replay)")
                keep = None
                if not (p.is_contiguous() and g.is_contiguous()):
                    if not _dense(p):
                        raise ValueError("FusedAdamW: parameters are dense in memory; got strides %s for %s" % (
                            tuple(p.stride()), tuple(p.shape)))
                    if not _same_layout(g, p):
                        g = keep = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
                st = self.state[p]
                use_master = bool(masters) and dt != _F32
                step = st.get("step")
                if moment not in st or step is None or (use_master and "master" not in st) or capturable != torch.is_tensor(step) or \
                        (capturable and (step.device != dev or step.dtype != _F32)):
                    st = self._ready(p, st, group)
                m, v, scales = self._state_tensors(p, st, bits)
                master = 0
                if use_master:
                    w = st["master"]
                    if w.dtype != _F32 or w.device != dev or not _same_layout(w, p):
                        raise ValueError("FusedAdamW: state['master'] is a float32 tensor of the parameter's shape and strides")
                    master = w.data_ptr()
                else:
                    st.pop("master", None)  # it would be out of date from this step on
                key = (dev, dt, bits, use_master, bool(group["maximize"]), capturable)
                b = buckets.get(key)
                if b is None:
                    b = buckets[key] = _Bucket(dev, _DTYPES[dt], bits, key[4], capturable, array("q"), [], [], [])
                if capturable:
                    if lr_dev is not None and (lr_dev.device != dev or lr_dev.dtype != _F32):
                        raise ValueError("FusedAdamW: lr as a tensor is float32 on the parameters' device")
                    hyper = (lr, b1, b2, eps, wd, 1, st["step"].data_ptr(), None if lr_dev is None else lr_dev.data_ptr())
                else:
                    hyper = (lr, b1, b2, eps, wd, st["step"] + 1, None, None)
                at = b.index.setdefault(hyper, len(b.hypers))
                if at == len(b.hypers):
                    b.hypers.append(hyper)
                b.table.extend((p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(),
                                0 if scales is None else scales.data_ptr(), master, p.numel(), at))
                b.keep.append(keep)
                b.params.append(p)
                b.states.append(st)
        return list(buckets.values())


class _Bucket:
    """tensors of one launch sequence: one device, type, width of the moments and direction"""

    def __init__(self, device, dtype, bits, maximize, capturable, table, hypers, params, states):
        self.device, self.dtype, self.bits, self.maximize, self.capturable = device, dtype, bits, maximize, capturable
        self.table, self.hypers, self.params, self.states = table, hypers, params, states
        self.index, self.keep = {}, []

    def arrays(self):
        """(tensors, hypers) as the bytes that the C entry reads"""
        if isinstance(self.table, bytes):
            return self.table, self.hypers
        return self.table.tobytes(), bytes((_lib.FsgsAdamWHyper * len(self.hypers))(*self.hypers))


def densify_stats(radii, viewspace_grad, max_radii2D, xyz_gradient_accum, denom):
    """add_densification_stats + max_radii2D update in one launch (scene/gaussian_model.py:678-681)."""
    lib = _lib.load()
    P = int(radii.shape[0])
    g = viewspace_grad.detach().contiguous()
    # raw pointers cross the C ABI: the kernel reads int32 radii and fp32 [P,3] / [P,1] / [P] rows, nothing else
    assert radii.dtype == torch.int32 and radii.is_contiguous() and radii.is_cuda, "radii: contiguous int32 on the GPU"
    for name, t, n in (("viewspace_grad", g, 3 * P), ("max_radii2D", max_radii2D, P),
                       ("xyz_gradient_accum", xyz_gradient_accum, P), ("denom", denom, P)):
        assert t.dtype == torch.float32 and t.is_contiguous() and t.numel() == n and t.device == radii.device, \
            "%s: contiguous fp32 with %d elements on %s" % (name, n, radii.device)
    with torch.cuda.device(radii.device):
        rc = lib.fsgs_densify_stats(P, _lib.ptr(radii), _lib.ptr(g), _lib.ptr(max_radii2D),
                                    _lib.ptr(xyz_gradient_accum), _lib.ptr(denom), _lib.current_stream())
    _lib.check(rc, "fsgs_densify_stats")
