"""Gradient norm, gradient clipping and the Adam step on the GPU (include/cista_optim.h).

The tail of a training step (reference train_e2v.py:63-65,120-121 trains with Adam and a StepLR
schedule): what happens between ``loss.backward()`` and the next forward.  Each operator runs over
all of its tensors in a few launches, whatever their number, sizes and places in memory.

* ``grad_norm(tensors)`` -- the norm of all elements of all tensors;
* ``clip_grad_norm_(parameters, max_norm)``, ``clip_grads_with_norm_(parameters, max_norm, norm)``
  -- gradients scaled in place by min(1, max_norm / (norm + 1e-6));
* ``Adam``, ``AdamW`` -- the optimizers, with clipping folded into the step (``max_norm``).

Types: float32, bfloat16, float16.  Norms are float32, from sums in float64; products are float32,
rounded once to the gradient's type; moments are float32, and a 16-bit parameter is updated on a
float32 master copy.  The order of a sum follows from the tensors' sizes and their places
within a 128-byte line alone, so equal gradients in equal buffers give equal bits: data-parallel
replicas stay alike.  Everything runs on the tensors' device, on its current stream, and nothing
waits for the GPU unless ``error_if_nonfinite`` asks for it, so the calls can be captured into a
graph.  CPU tensors raise: there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib

NORMS = {1.0: 1, 2.0: 2, math.inf: 3}                     # CISTA_NORM_*
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # CISTA_F32, ...


class CistaTensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("numel", ctypes.c_longlong), ("type", ctypes.c_longlong)]


class CistaAdamTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "master", "step")] + [
        ("numel", ctypes.c_longlong), ("type", ctypes.c_longlong)]


class CistaAdamGroup(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [
        ("lr_device", ctypes.c_void_p)] + [(n, ctypes.c_int) for n in ("n", "decoupled", "maximize", "reserved")]


def _norm_kind(norm_type) -> int:
    kind = NORMS.get(float(norm_type))
    if kind is None:
        raise _lib.CistaError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise _lib.CistaError(f"max_norm must be at least 0, got {max_norm}")
    return max_norm


def _check_tensor(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected torch.Tensor, got {type(t).__name__}")
    if t.layout != torch.strided:
        raise _lib.CistaError(f"{what}: only strided tensors are supported, got {t.layout}")
    if not t.is_cuda:
        raise _lib.CistaError(f"{what} is on {t.device}: the training operators run on a ROCm GPU only (no CPU fallback)")
    if t.dtype not in TYPES:
        raise _lib.CistaError(f"{what} has type {t.dtype}: float32, bfloat16 and float16 are supported")


def _same_device(tensors, what):
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev:
            raise _lib.CistaError(f"{what} are on {dev} and {t.device}: one call takes the tensors of one device")
    return dev


class _on:
    """Makes `device` the current one, if it is not."""

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _table(tensors):
    return (CistaTensor * len(tensors))(*[(t.data_ptr(), t.numel(), TYPES[t.dtype]) for t in tensors])


def _workspace(n, device):
    return torch.empty(_lib.lib().cista_optim_workspace_bytes(n), dtype=torch.uint8, device=device)


def _as_list(tensors):
    return tensors if type(tensors) is list else [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _short(name, *args):
    """A call of csrc/cista_torch.cpp: its result, or NotImplemented where it leaves the call to Python."""
    got = getattr(_lib.torch_lib(), name)(*args)
    if type(got) is int:
        _lib.check(got, name.replace("_torch", ""))
    return got


def _dense(t) -> bool:
    """Whether the elements fill one run of memory, in whatever order of the dimensions."""
    return (t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)) and not t.is_neg()


def _grads(parameters):
    return [p.grad for p in _as_list(parameters) if p.grad is not None]


def _raise_if_nonfinite(norm, norm_type):
    if not math.isfinite(norm.item()):
        raise RuntimeError(f"the total norm of order {norm_type} is not finite ({norm.item()}): the gradients are left "
                           "as they are")


def grad_norm(tensors, norm_type=2.0, error_if_nonfinite=False):
    """The norm of all elements of `tensors` (one, or an iterable) together, as a float32 scalar
    on their device: norm_type 2, 1 (sum of magnitudes) or inf (largest magnitude; NaN if any
    element is).  Tensors of any strides; the same one may come twice and then counts twice."""
    kind = _norm_kind(norm_type)
    tensors = _as_list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    norm = _short("cista_torch_grad_norm", tensors, kind)
    if norm is not NotImplemented:
        if error_if_nonfinite:
            _raise_if_nonfinite(norm, norm_type)
        return norm
    for t in tensors:
        _check_tensor(t, "tensor")
    dev = _same_device(tensors, "tensors")
    with _on(dev), torch.no_grad():
        tensors = [t if _dense(t) else t.resolve_neg().contiguous() for t in tensors]
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ws = _workspace(len(tensors), dev)
        _lib.check(_lib.lib().cista_grad_norm(_table(tensors), len(tensors), kind, norm.data_ptr(), ws.data_ptr(),
                                              ws.numel(), _lib.stream_handle(dev)), "cista_grad_norm")
    if error_if_nonfinite:
        _raise_if_nonfinite(norm, norm_type)
    return norm


class _Memory:
    """A tensor's elements as numpy describes an array's; their memory is never touched."""

    def __init__(self, t):
        size, at = t.element_size(), t.data_ptr()
        self.dense, self.begin, self.end = _dense(t), at, at
        if t.numel():
            self.end += size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
        self.__array_interface__ = dict(version=3, data=(at, False), typestr=f"|V{size}", shape=tuple(t.shape),
                                        strides=tuple(s * size for s in t.stride()))


def _refuse_shared(grads):
    """Raises if an element of one gradient is another's too, where a copy would stand for one of them (the
    library checks the others).  Views may lie between each other: columns of a matrix, real and imaginary parts."""
    if all(_dense(g) for g in grads):
        return
    open_ = []                                               # those that reach past the next one's begin
    for m in sorted((_Memory(g) for g in grads if g.numel()), key=lambda m: m.begin):
        open_ = [o for o in open_ if o.end > m.begin]
        for o in open_:
            if not (o.dense and m.dense) and np.shares_memory(np.asarray(o), np.asarray(m)):
                raise _lib.CistaError("a gradient overlaps another one: those that share memory cannot be written")
        open_.append(m)


def _written(grads, call):
    """Runs `call` on dense stand-ins of the gradients, and writes those that are copies back."""
    _refuse_shared(grads)
    torch.autograd.graph.increment_version(grads)        # raises for what may not be written
    dense = [g if _dense(g) else g.resolve_neg().contiguous() for g in grads]
    call(dense)
    for g, d in zip(grads, dense):
        if d is not g:
            g.copy_(d)


def _check_grads(grads):
    for g in grads:
        _check_tensor(g, "gradient")
        if any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise _lib.CistaError(f"a gradient of strides {g.stride()} overlaps itself and cannot be written")
    return _same_device(grads, "gradients")


def clip_grads_with_norm_(parameters, max_norm, total_norm):
    """Scales the gradients of `parameters` in place by min(1, max_norm / (total_norm + 1e-6)), 1
    for max_norm = inf.  total_norm: a scalar tensor on their device, for instance grad_norm's,
    or one that ranks have put together.  Gradients that share memory are refused."""
    max_norm = _max_norm(max_norm)
    grads = _grads(parameters)
    if not grads:
        return
    dev = _check_grads(grads)
    if not isinstance(total_norm, torch.Tensor) or total_norm.numel() != 1 or total_norm.device != dev:
        raise _lib.CistaError(f"total_norm must be a scalar tensor on {dev}")
    with _on(dev), torch.no_grad():
        total = total_norm.detach().to(torch.float32).resolve_neg()
        _written(grads, lambda dense: _lib.check(
            _lib.lib().cista_scale_grads(_table(dense), len(dense), max_norm, total.data_ptr(), _lib.stream_handle(dev)),
            "cista_scale_grads"))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clips the gradients of `parameters` (one, or an iterable; those without are left out) to a
    joint norm of max_norm, in place, and returns the norm that they had (grad_norm's).  An infinite
    norm turns the finite gradients to 0 and a NaN norm all of them to NaN, unless
    error_if_nonfinite asks for a RuntimeError before anything is written (which waits for the GPU)."""
    max_norm, kind = _max_norm(max_norm), _norm_kind(norm_type)
    parameters = _as_list(parameters)
    if not error_if_nonfinite:
        norm = _short("cista_torch_clip_grads", parameters, kind, max_norm)
        if norm is not NotImplemented:
            return norm
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    dev = _check_grads(grads)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type, True)
        clip_grads_with_norm_(parameters, max_norm, norm)
        return norm
    with _on(dev), torch.no_grad():
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ws = _workspace(len(grads), dev)
        _written(grads, lambda dense: _lib.check(
            _lib.lib().cista_clip_grads(_table(dense), len(dense), kind, max_norm, norm.data_ptr(), ws.data_ptr(),
                                        ws.numel(), _lib.stream_handle(dev)), "cista_clip_grads"))
    return norm


class Adam(torch.optim.Optimizer):
    """Adam with the constructor arguments of the training script's optimizer (train_e2v.py:63:
    ``Adam(model.parameters(), lr)``), and

    * ``decoupled_weight_decay`` -- decay on the parameter instead of in the gradient (``AdamW``);
    * ``max_norm``, ``norm_type`` -- the gradients of all groups are clipped to this joint norm
      within the step: the update uses them scaled, ``.grad`` stays as it is, and the norm they had
      is in ``optimizer.grad_norm``.

    ``lr`` is a number, or a float32 scalar tensor on the parameters' device, which a captured step
    reads at each replay.  State of each parameter: ``step`` (float32 scalar on the device),
    ``exp_avg``, ``exp_avg_sq`` (float32, the parameter's shape) and, for a 16-bit parameter,
    ``master`` (float32; made from the parameter when first needed, so from then on a parameter
    is changed through it; dropped by a step, or a state_dict loaded, while the parameter is float32).
    A state_dict keeps those types when it is loaded; one without ``master`` loads too.  A captured step replays the update; weights that the network has packed are then
    repacked after ``model.invalidate_packed()``.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, *,
                 decoupled_weight_decay=False, maximize=False, max_norm=None, norm_type=2.0):
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError("lr as a tensor must have one element")
        elif not 0.0 <= lr:
            raise ValueError(f"invalid learning rate {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"invalid eps {eps}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"invalid betas {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"invalid weight_decay {weight_decay}")
        self.max_norm = None if max_norm is None else _max_norm(max_norm)
        self.norm_type = norm_type
        _norm_kind(norm_type)
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      decoupled_weight_decay=decoupled_weight_decay, maximize=maximize))

    def _slot(self, p):
        """The parameter's state as the kernels take it; made or put right where it is not."""
        st = self.state[p]

        def made():
            if torch.cuda.is_current_stream_capturing():
                raise _lib.CistaError("the first step makes the optimizer's state and cannot be captured: take one step "
                                      "(or load a state_dict and take one) before")

        def moment(name):
            t = st.get(name)
            if t is None:
                made()
                t = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
            elif (t.dtype != torch.float32 or t.device != p.device or t.shape != p.shape or t.stride() != p.stride()
                  or t.is_neg()):
                if t.shape != p.shape:
                    raise _lib.CistaError(f"state {name} has shape {tuple(t.shape)}, its parameter {tuple(p.shape)}")
                made()
                t = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(t)
            st[name] = t

        step = st.get("step", 0.0)
        if isinstance(step, torch.Tensor) and step.numel() != 1:
            raise _lib.CistaError(f"state step has {step.numel()} elements")
        if not isinstance(step, torch.Tensor) or step.dtype != torch.float32 or step.device != p.device or step.is_neg():
            made()
            st["step"] = torch.full((), float(step), dtype=torch.float32, device=p.device)
        moment("exp_avg")
        moment("exp_avg_sq")
        if p.dtype == torch.float32:
            st.pop("master", None)                            # of 16-bit steps before: older than the parameter from here on
        else:
            if st.get("master") is None:
                made()
                st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
            moment("master")
        return st

    def __getstate__(self):
        return dict(super().__getstate__(), max_norm=self.max_norm, norm_type=self.norm_type, grad_norm=None)

    @staticmethod
    def _refuse_amsgrad(state):
        if any(g.get("amsgrad") for g in state["param_groups"]):
            raise _lib.CistaError("amsgrad is not built")

    def __setstate__(self, state):
        self._refuse_amsgrad(state)                           # before anything is taken over
        super().__setstate__(state)
        for g in self.param_groups:
            for k, v in self.defaults.items():
                g.setdefault(k, v)

    def load_state_dict(self, state_dict):
        """The state keeps its float32 values (the base class casts it to the parameter's type), in memory of
        its own: step counts and moments are advanced in place, and the state_dict may be a live optimizer's.
        What is loaded is what pre-hooks make of the state_dict; post-hooks see the state as it stays."""
        loaded = []

        def last(_, given):
            self._refuse_amsgrad(given)
            loaded.append(given)

        hooks = [self.register_load_state_dict_pre_hook(last),
                 self.register_load_state_dict_post_hook(lambda _: self._take_over(loaded[-1]), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _take_over(self, state_dict):
        params = [p for g in self.param_groups for p in g["params"]]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, params):
            if p not in self.state:
                continue
            given, mine = state_dict["state"].get(i, {}), self.state[p]
            for name, t in mine.items():
                if name in ("exp_avg", "exp_avg_sq", "master") and p.dtype != torch.float32 and given.get(name) is not None:
                    mine[name] = given[name].to(device=p.device, dtype=torch.float32, copy=True)
                elif isinstance(t, torch.Tensor) and t is given.get(name):      # taken over as it is
                    mine[name] = t.clone()
            if p.dtype == torch.float32:
                mine.pop("master", None)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        kind = 0 if self.max_norm is None else _norm_kind(self.norm_type)
        norm = _short("cista_torch_adam_step", self.param_groups, self.state, kind, self.max_norm or 0.0)
        if norm is not NotImplemented:
            self.grad_norm = norm
            return loss
        self._step(kind)
        return loss

    @torch.no_grad()
    def _step(self, kind):
        """The step where it is not plain: makes or converts state, copies layouts, refuses."""
        rows, groups, keep, changed = [], [], [], []
        for g in self.param_groups:
            params = [p for p in g["params"] if p.grad is not None]
            for p in params:
                _check_tensor(p, "parameter")
                grad = p.grad
                _check_tensor(grad, "gradient")
                if not _dense(p):                         # a negated view is none
                    raise _lib.CistaError(f"a parameter of strides {p.stride()} does not fill its memory")
                if grad.shape != p.shape or grad.dtype != p.dtype or grad.device != p.device:
                    raise _lib.CistaError(f"a gradient ({tuple(grad.shape)}, {grad.dtype}, {grad.device}) is not like its "
                                          f"parameter ({tuple(p.shape)}, {p.dtype}, {p.device})")
                if grad.is_neg() or (
                        grad.stride() != p.stride() and not (grad.is_contiguous() and p.is_contiguous())):
                    grad = torch.empty_like(p, requires_grad=False).copy_(grad)
                    keep.append(grad)
                st = self._slot(p)
                master = st["master"].data_ptr() if p.dtype != torch.float32 else None
                rows.append((p.data_ptr(), grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(),
                             master, st["step"].data_ptr(), p.numel(), TYPES[p.dtype]))
                changed.append(p)
            lr, lr_device = g["lr"], None
            if isinstance(lr, torch.Tensor):
                if lr.is_cuda:
                    if lr.dtype != torch.float32 or lr.numel() != 1 or (params and lr.device != params[0].device):
                        raise _lib.CistaError("lr as a tensor must be one float32, on the parameters' device")
                    keep.append(lr.resolve_neg())
                    lr, lr_device = 0.0, keep[-1].data_ptr()
                else:
                    lr = float(lr)
            groups.append((lr, g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"], lr_device, len(params),
                           int(g["decoupled_weight_decay"]), int(g["maximize"]), 0))
        if not rows:
            self.grad_norm = None
            return
        dev = _same_device(changed, "parameters")
        torch.autograd.graph.increment_version(changed)      # the network repacks changed weights
        with _on(dev):
            norm = torch.empty((), dtype=torch.float32, device=dev) if kind else None
            ws = _workspace(len(rows), dev)
            _lib.check(_lib.lib().cista_adam_step(
                (CistaAdamTensor * len(rows))(*rows), (CistaAdamGroup * len(groups))(*groups), len(groups), kind,
                self.max_norm or 0.0, _lib.ptr(norm), ws.data_ptr(), ws.numel(), _lib.stream_handle(dev)),
                "cista_adam_step")
        self.grad_norm = norm


class AdamW(Adam):
    """Adam with decoupled weight decay, 0.01 unless given."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, maximize=False,
                 max_norm=None, norm_type=2.0):
        super().__init__(params, lr, betas, eps, weight_decay, decoupled_weight_decay=True, maximize=maximize,
                         max_norm=max_norm, norm_type=norm_type)
