"""The optimizer of large language models on libsegmi: orthogonalised updates for matrices, AdamW for everything else.

`orthogonalize`  replaces matrices by their nearest (semi-)orthogonal ones, by Newton-Schulz products.
`Muon`           momentum -> orthogonalize -> update for every parameter that is a matrix (convolution filters [K, C, R, S] are
                 K x C*R*S), AdamW for the rest (norms, biases, depthwise filters).  One optimizer for a whole network.
`FusedAdamW`     AdamW alone.

All three are reached through `segmi.optim`, and the two optimizers by name from config.json (`"optimizer": {"type": "Muon", ...}`), the
way the reference resolves its optimizers (`base/base_trainer.py:57`).  `AdamW` in a config stays torch.optim.AdamW.
Pointers travel as kernel arguments: no table is uploaded, gradients may move between steps (the host then makes the descriptors anew), nothing
waits for the GPU.
"""
import contextlib
import ctypes as C
import math
from itertools import chain
from operator import is_, itemgetter

import numpy as np
import torch

from ._lib import SegmiError, check, lib

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_NS_DTYPE = np.dtype([("src", "<u8"), ("dst", "<u8"), ("src_rs", "<i8"), ("src_cs", "<i8"), ("dst_rs", "<i8"), ("dst_cs", "<i8"),
                      ("rows", "<i4"), ("cols", "<i4"), ("dtype", "<i4"), ("reserved", "<i4")])
_NS_CODES = {torch.float32: 0, torch.bfloat16: 1}
_MUON_DTYPE = np.dtype([("param", "<u8"), ("grad", "<u8"), ("momentum", "<u8"), ("rows", "<i4"), ("cols", "<i4"), ("factor", "<f4"), ("group", "<i4")])
_ADAMW_DTYPE = np.dtype([("param", "<u8"), ("grad", "<u8"), ("exp_avg", "<u8"), ("exp_avg_sq", "<u8"), ("step_dev", "<u8"), ("step", "<f8"),
                         ("count", "<i8"), ("group", "<i4"), ("reserved", "<i4")])
_MAX_GROUPS = 8
_ADAMW_HYPER = 5                              # lr, weight decay, beta 1, beta 2, eps


def _check_iteration(steps, coefficients, eps, what):
    if isinstance(steps, bool) or int(steps) != steps or not 1 <= steps <= 32:
        raise ValueError("%s: the number of Newton-Schulz steps must be an integer in 1..32, got %r" % (what, steps))
    coefficients = tuple(float(c) for c in coefficients)
    if len(coefficients) != 3:
        raise ValueError("%s: three Newton-Schulz coefficients (a, b, c) are needed, got %d" % (what, len(coefficients)))
    if not (float(eps) > 0.0 and math.isfinite(eps)):
        raise ValueError("%s: eps must be positive and finite, got %r" % (what, eps))
    arr = (C.c_double * 3)(*coefficients)
    if not all(math.isfinite(c) for c in coefficients) or not lib.segmi_ns_coefficients_ok(arr, int(steps)):
        raise ValueError("%s: with coefficients %r the singular values do not stay bounded over %d steps" % (what, coefficients, steps))
    return arr


def _unit_of(sizes, strides):
    """The stride u of the densely packed run these dimensions form (in any order), or None."""
    dims = sorted((st, n) for n, st in zip(sizes, strides) if n > 1)
    if not dims:
        return 1
    unit = expect = dims[0][0]
    for st, n in dims:
        if st != expect:
            return None
        expect = st * n
    return unit if unit > 0 else None


def _matrix_strides(t):
    """(row stride, column stride) of t, of three or more dimensions, seen as shape[0] x rest, columns in the order of memory; None if it has none."""
    cs = _unit_of(t.shape[1:], t.stride()[1:])
    return None if cs is None else (t.stride(0), cs)


@torch.no_grad()
def orthogonalize(matrices, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """X = M / max(|M|_F, eps), then `steps` times X <- (a I + b X X^T + c (X X^T)^2) X on the shorter side: all singular values
    of M go to about 1.

    `matrices`: a float32 or bfloat16 CUDA tensor of two or more dimensions (seen as shape[0] x the rest), or a list of them, any sizes
    and strides; all of them share the launches.  Returns new tensors of the same shapes, types and (where dense) strides.  Computed
    in both types to the accuracy of an fp32 iteration over a matrix.  Values are held to 2^-22 of themselves and 2^-39 of the matrix's norm: a row or
    column that is 1e-6 of the matrix comes out to 4e-5 (64 x 576) - 3e-4 (300 x 5000) of its own size, in fp32 to 1e-5.  The last bits may depend on what else is in the list.  No gradient is recorded.  A matrix that holds NaN or infinity comes back as NaN, a zero one as zero.
    Runs on the current stream of the tensors' device; may be captured into a hipGraph."""
    single = isinstance(matrices, torch.Tensor)
    mats = [matrices] if single else list(matrices)
    coef = _check_iteration(steps, coefficients, eps, "segmi.optim.orthogonalize")
    outs, rows = [], []
    keep = []                                     # copies of inputs without a matrix order live until the launches are queued
    device, index = None, -1
    for t in mats:
        if not isinstance(t, torch.Tensor) or t.dim() < 2:
            raise ValueError("segmi.optim.orthogonalize: a tensor of two or more dimensions is needed, got %s" %
                             (tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__,))
        if not t.is_cuda:
            raise SegmiError("segmi.optim.orthogonalize: tensor is on %s — the kernels only run on the MI355X (there is deliberately no "
                             "CPU / eager fallback)" % t.device)
        code = _NS_CODES.get(t.dtype)
        if code is None:
            raise SegmiError("segmi.optim.orthogonalize: expected float32 or bfloat16, got %s" % t.dtype)
        if device is None:
            device, index = t.device, t.get_device()
        elif t.get_device() != index:
            raise SegmiError("segmi.optim.orthogonalize: all matrices must be on one device, got %s and %s" % (device, t.device))
        if t.is_neg():                            # memory holds the opposite sign (the imaginary part of a conjugate)
            t = t.resolve_neg()
            keep.append(t)
        out = torch.empty_like(t)
        n = t.numel()
        if n and t.dim() == 2:
            st, so = t.stride(), out.stride()
        elif n:
            st = _matrix_strides(t)
            if st is None or out.stride() != t.stride():
                t = t.contiguous()
                keep.append(t)
                out = torch.empty_like(t)
                st = _matrix_strides(t)
            so = _matrix_strides(out)
        outs.append(out)
        if n:
            r = t.shape[0]
            rows.append((t.data_ptr(), out.data_ptr(), *st, *so, r, n // r, code, 0))
    if rows:
        desc = np.array(rows, dtype=_NS_DTYPE)
        with torch.cuda.device(device):
            nbytes = lib.segmi_ns_workspace(desc.ctypes.data, len(rows))
            if not nbytes:
                raise SegmiError("segmi.optim.orthogonalize: a matrix is too large (4 GiB of float32 after padding its sides to 64)")
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            check(lib.segmi_ns_orthogonalize(desc.ctypes.data, len(rows), coef, int(steps), float(eps), ws.data_ptr(), nbytes,
                                             torch.cuda.current_stream().cuda_stream), "ns_orthogonalize")
    return outs[0] if single else outs


def _same_layout(a, b):
    return a.shape == b.shape and all(sa == sb or n == 1 for sa, sb, n in zip(a.stride(), b.stride(), a.shape))


_ptr, _numel = torch.Tensor.data_ptr, torch.Tensor.numel
_params = itemgetter("params")


class _Hyper:
    """Per-group numbers in device memory (graphs): a ring of pinned slots and stream-ordered copies, as segmi.optim.SGD's."""
    RING = 8

    def __init__(self, nbytes, device):
        self.slots = torch.zeros(self.RING, nbytes, dtype=torch.uint8).pin_memory()
        self.events = [None] * self.RING
        self.dev = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self.at = 0

    def push(self, values):
        i, self.at = self.at, (self.at + 1) % self.RING
        if self.events[i] is not None:
            self.events[i].synchronize()             # the copy that last read this slot has executed
        self.slots[i].copy_(torch.from_numpy(values))
        self.dev.copy_(self.slots[i], non_blocking=True)
        self.events[i] = torch.cuda.Event()
        self.events[i].record()


def _on(device):
    """The device as the current one (a context manager that costs nothing where it is already)."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


class _FusedOptimizer(torch.optim.Optimizer):
    """What both optimizers share: state buffers in the parameters' memory order, descriptors that are rebuilt only when a pointer
    moved, step numbers, capture."""

    def __init__(self, params, defaults, capturable):
        super().__init__(params, defaults)
        self.capturable = bool(capturable)
        self._hyper = None
        self._where = None                           # see _device
        self._captured = []                          # what the graphs that hold a step of this optimizer point at
        self._kept = None                            # what the last step saw and the descriptors made from it, see _plan
        self._steps, self._step_of, self._views = None, {}, []      # one flat host tensor of step numbers; state[p]["step"] are views of it

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            if len(self.param_groups) > _MAX_GROUPS:
                raise ValueError("%s supports up to %d parameter groups" % (self._name(), _MAX_GROUPS))
            self._check_group(self.param_groups[-1])         # completed from the defaults
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, group):
        """ValueError for settings that the kernels have no formula for."""
        raise NotImplementedError

    def _name(self):
        return "segmi.optim." + type(self).__name__

    def __getstate__(self):
        return dict(super().__getstate__(), capturable=self.capturable)

    def __setstate__(self, state):                   # (torch's load_state_dict comes here too, with everything in place)
        super().__setstate__(state)
        for name, value in (("capturable", False), ("_hyper", None), ("_where", None), ("_captured", []), ("_kept", None), ("_steps", None), ("_step_of", {}), ("_views", [])):
            self.__dict__.setdefault(name, value)

    def load_state_dict(self, state_dict):
        """As torch's, but the buffers are this optimizer's own: torch keeps the tensors of the dictionary where type and device fit,
        and the kernels here would advance those of the optimizer it came from as well.  Buffers that were there keep their place
        and take the values, so a captured step goes on with what was loaded; once a step was captured, those that the dictionary lacks
        are set to zero in their place.  Settings that the dictionary lacks (another class wrote it) are
        this optimizer's defaults; one that asks for a formula that is not here, or holds settings the constructor would refuse, is refused."""
        for g in state_dict["param_groups"]:
            for key in ("amsgrad", "maximize", "dampening"):
                if g.get(key):
                    raise ValueError("%s has no %s" % (self._name(), key))
            if g.get("decoupled_weight_decay") is False and g.get("weight_decay"):
                raise ValueError("%s has decoupled weight decay only" % self._name())
            self._check_group({**self.defaults, **g})
        scales = [self._momentum_scale(g) for g in state_dict["param_groups"]]
        before = {p: dict(st) for p, st in self.state.items()}
        super().load_state_dict(state_dict)
        scale_of = {p: s for g, s in zip(self.param_groups, scales) for p in g["params"]}
        for g in self.param_groups:
            for key, value in self.defaults.items():
                g.setdefault(key, value)
        with torch.no_grad():
            if self._captured:
                for p, st in before.items():
                    for key, own in st.items():
                        if isinstance(own, torch.Tensor) and self.state[p].get(key) is None:
                            self.state[p][key] = own.zero_()
            for p, st in self.state.items():
                for key, v in st.items():
                    if not isinstance(v, torch.Tensor):
                        continue
                    own = before.get(p, {}).get(key)
                    if own is v:
                        continue
                    if isinstance(own, torch.Tensor) and own.shape == v.shape and own.dtype == v.dtype and (own.device == v.device or key == "step"):
                        st[key] = own.copy_(v)
                    else:
                        st[key] = v.clone()
                    if key == "momentum_buffer" and scale_of.get(p, 1.0) != 1.0:
                        st[key].mul_(scale_of[p])
        self._kept = None

    def _momentum_scale(self, group):
        """Factor that makes the momentum buffers of a dictionary's group sums, as they are here."""
        return 1.0

    def _buffer(self, p, key):
        """state[p][key] in p's own memory order; created, or re-laid once if it arrived in another (a loaded state_dict)."""
        st = self.state[p]
        buf = st.get(key)
        if buf is None:
            buf = st[key] = torch.zeros_like(p, memory_format=torch.preserve_format)
        elif not (buf.shape == p.shape and _same_layout(buf, p) and buf.device == p.device and buf.dtype == p.dtype):
            if buf.shape != p.shape:
                raise RuntimeError("%s: %s has shape %s for a parameter of shape %s" % (self._name(), key, tuple(buf.shape), tuple(p.shape)))
            fixed = torch.empty_like(p, memory_format=torch.preserve_format)
            fixed.copy_(buf)
            buf = st[key] = fixed
        return buf

    def _checked(self, p):
        g = p.grad
        if not (p.is_cuda and p.dtype == torch.float32 and not g.is_sparse and g.dtype == torch.float32 and g.device == p.device and
                (g.shape == p.shape and g.stride() == p.stride() or _same_layout(g, p)) and (p.is_contiguous() or _unit_of(p.shape, p.stride()) == 1)):
            raise RuntimeError("%s: parameters and gradients must be float32 CUDA tensors on one device with identical (dense) strides" % self._name())
        if p.is_neg() or g.is_neg():
            raise RuntimeError("%s: a parameter or gradient is a negated view; resolve_neg() makes one the kernels can read" % self._name())
        if p.device != self._device():
            raise RuntimeError("%s: all parameters must be on one device, got %s and %s" % (self._name(), self._device(), p.device))
        return g

    def _device(self):
        """Where the step runs: the device of the last step's first parameter with a gradient (groups may be empty, and what is frozen may lie
        anywhere); before a step that of the first parameter on a GPU."""
        if self._where is not None:
            return self._where.device
        params = list(chain.from_iterable(map(_params, self.param_groups)))
        return next((p.device for p in params if p.is_cuda), params[0].device if params else None)

    def _is_matrix(self, group, p):
        return False

    def _plan(self):
        """The step's descriptors.  They are made anew when anything they were made from is another: the parameters, which of them have
        gradients, the groups' settings that enter them, a parameter's state dictionary or a tensor in it, any pointer or size.  (Addresses are
        compared, not objects alone: `p.data = ...` keeps the object.)  The comparison is the host's share of a small step, so it runs over whole lists."""
        flat = list(chain.from_iterable(map(_params, self.param_groups)))
        grads = [p.grad for p in flat]
        missing = [g is None for g in grads]
        live = [g for g in grads if g is not None] if True in missing else grads
        if live:
            self._where = flat[missing.index(False)]
        k = self._kept
        if (k is not None and len(flat) == len(k["flat"]) and all(map(is_, flat, k["flat"])) and missing == k["missing"] and
                list(map(_ptr, live)) == k["grad_ptrs"] and self._strides(flat, live, k["deep"], k["shallow"]) == k["strides"]):
            held = list(chain.from_iterable(map(dict.values, k["states"])))
            if (len(self.state) == len(k["owners"]) and all(map(is_, self.state.values(), k["dicts"])) and all(map(is_, self.state, k["owners"])) and
                    len(held) == len(k["held"]) and all(map(is_, held, k["held"])) and list(map(_ptr, k["tensors"])) == k["ptrs"] and
                    list(map(_numel, flat)) == k["numels"] and [p.shape for _, p in k["members"]] == k["shapes"] and
                    list(map(len, map(_params, self.param_groups))) == k["lengths"] and self._settings() == k["settings"]):
                return k
        self._kept = None
        k = dict(mats=None, rest=None)
        if not live:
            return k
        if self._device().type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("%s: a parameter, gradient or state buffer is new while a hipGraph is being captured.  Keep gradients persistent "
                               "(segmi.distributed.DistributedModel does) and run at least one eager step before capturing." % self._name())
        mats, rest = [], []
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                if p.grad is not None and p.numel():
                    (mats if self._is_matrix(g, p) else rest).append((gi, p))
        if mats:
            k["mats"] = self._matrix_descriptors(mats)
        if rest:
            k["rest"] = self._adamw_descriptors(rest)
            k["rows"] = None if self.capturable else np.array([self._step_of[p] for _, p in rest])
        self._check_apart(k["mats"][0] if mats else None, k["rest"])
        states = [self.state[p] for _, p in mats + rest]
        held = list(chain.from_iterable(map(dict.values, states)))
        tensors = flat + [t for st in states for key, t in st.items() if (key != "step" or self.capturable) and isinstance(t, torch.Tensor)]
        deep = [(i, j) for j, i in enumerate(i for i, g in enumerate(grads) if g is not None) if grads[i].dim() > 1]      # (among the parameters, among the gradients)
        shallow = [j for j, g in enumerate(live) if g.dim() == 1]
        k.update(flat=flat, missing=missing, grad_ptrs=list(map(_ptr, live)), deep=deep, shallow=shallow,
                 strides=self._strides(flat, live, deep, shallow), owners=list(self.state), dicts=list(self.state.values()), states=states, held=held,
                 tensors=tensors, ptrs=list(map(_ptr, tensors)), numels=list(map(_numel, flat)), members=mats, shapes=[p.shape for _, p in mats],
                 lengths=list(map(len, map(_params, self.param_groups))), settings=self._settings())
        self._kept = k
        return k

    def _check_apart(self, mats, rest):
        """Everything the kernels write lies in memory of its own: the updates of two tensors run at the same time."""
        at, size = [], []
        if mats is not None:
            at += [mats["param"], mats["momentum"]]
            size += [mats["rows"].astype(np.int64) * mats["cols"] * 4] * 2
        if rest is not None:
            at += [rest["param"], rest["exp_avg"], rest["exp_avg_sq"]]
            size += [rest["count"] * 4] * 3
            if self.capturable:
                at.append(rest["step_dev"])
                size.append(np.full(len(rest), 4))
        if not at:
            return
        at, size = np.concatenate(at).astype(np.int64), np.concatenate(size)
        order = np.argsort(at)
        if np.any(at[order][:-1] + size[order][:-1] > at[order][1:]):
            raise RuntimeError("%s: two of the parameters with gradients, or of their state buffers, share memory" % self._name())

    def _settings(self):
        return None

    @staticmethod
    def _strides(flat, live, deep, shallow):
        return [(flat[i].stride(), live[j].stride()) for i, j in deep] + [live[j].is_contiguous() for j in shallow]

    def _adamw_descriptors(self, members):
        rows = []
        for gi, p in members:
            g = self._checked(p)
            rows.append((p.data_ptr(), g.data_ptr(), self._buffer(p, "exp_avg").data_ptr(), self._buffer(p, "exp_avg_sq").data_ptr(),
                         0, 0.0, p.numel(), gi, 0))
        self._adopt_steps([p for _, p in members])
        desc = np.array(rows, dtype=_ADAMW_DTYPE)
        if self.capturable:
            desc["step_dev"] = [self.state[p]["step"].data_ptr() for _, p in members]
        return desc

    def _adopt_steps(self, params):
        """state[p]["step"] keeps its value and becomes a view of one flat host tensor; for graphs a float on the device, which stays
        where it is once it is there: captured steps advance it."""
        value = lambda p: float(self.state[p]["step"]) if self.state[p].get("step") is not None else 0.0
        if self.capturable:
            there = lambda t: isinstance(t, torch.Tensor) and t.device == self._device() and t.dtype == torch.float32 and t.numel() == 1
            fresh = [p for p in params if not there(self.state[p].get("step"))]
            if fresh:
                for p, t in zip(fresh, torch.tensor([value(p) for p in fresh], dtype=torch.float32, device=self._device())):
                    self.state[p]["step"] = t
            return
        mine = self._step_of
        if all(p in mine and self.state[p].get("step") is self._views[mine[p]] for p in params):
            return
        every = list(dict.fromkeys([p for p in mine if self.state.get(p, {}).get("step") is not None] + list(params)))
        self._steps = torch.tensor([value(p) for p in every], dtype=torch.float32)
        self._step_of = {p: i for i, p in enumerate(every)}
        self._views = [self._steps[i] for i in range(len(every))]
        for p, i in self._step_of.items():
            self.state[p]["step"] = self._views[i]

    def _hyper_values(self):
        raise NotImplementedError

    def push_hyper(self):
        """Stream-ordered refresh of the device-resident hyper-parameters from `param_groups` (capturable=True only): eager steps do it
        by themselves, a captured step needs it before each replay."""
        if not self.capturable:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("%s.push_hyper must stay outside the captured region (call it before graph replay)" % self._name())
        device = self._device()
        if device is None:
            return
        values = np.concatenate([v.reshape(-1).view(np.uint8) for v in self._hyper_values()])
        with _on(device):
            if self._hyper is None or self._hyper.dev.device != device:
                self._hyper = _Hyper(values.size, device)
            self._hyper.push(values)

    def _ready(self, k):
        if torch.cuda.is_current_stream_capturing():
            if not self.capturable:
                raise RuntimeError("%s: a step inside a hipGraph capture needs capturable=True (learning rates and step numbers would be "
                                   "frozen)" % self._name())
            if self._hyper is None or self._hyper.dev.device != self._device():
                raise RuntimeError("%s(capturable=True): run one eager step before capturing" % self._name())
            # the graph's addresses stay valid for as long as the optimizer lives, whatever becomes of the state and the gradients
            self._captured += [t.detach() for t in [*k["tensors"], *(p.grad for p in k["flat"] if p.grad is not None), self._hyper.dev]]
        else:
            self.push_hyper()

    def _adamw_hyper(self, betas, eps, lr_ratio):
        h = np.zeros((_MAX_GROUPS, _ADAMW_HYPER), dtype=np.float64)
        for i, g in enumerate(self.param_groups):
            h[i] = (float(g["lr"]), float(g["weight_decay"]), float(g[betas][0]), float(g[betas][1]), float(g[eps]))
            if lr_ratio is not None:
                h[i, 0] *= float(g[lr_ratio])
        return h

    def _adamw_launch(self, k, hyper, hyper_dev, stream):
        desc, ws, nbytes = k["rest"], None, 0
        if self.capturable:
            nbytes = 8 * len(desc)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self._device())
        else:
            steps = self._steps.numpy()
            steps[k["rows"]] += 1.0
            desc["step"] = steps[k["rows"]]
        check(lib.segmi_adamw_step(desc.ctypes.data, len(desc), hyper.ctypes.data, len(self.param_groups), hyper_dev,
                                   None if ws is None else ws.data_ptr(), nbytes, stream), "adamw_step")


def _check_common(name, lr, weight_decay, betas, eps):
    if not float(lr) >= 0.0:
        raise ValueError("%s: invalid learning rate %r" % (name, lr))
    if not float(weight_decay) >= 0.0:
        raise ValueError("%s: invalid weight_decay %r" % (name, weight_decay))
    if len(betas) != 2 or not all(0.0 <= float(b) < 1.0 for b in betas):
        raise ValueError("%s: betas must be two numbers in [0, 1), got %r" % (name, betas))
    if not float(eps) >= 0.0:
        raise ValueError("%s: invalid eps %r" % (name, eps))


class FusedAdamW(_FusedOptimizer):
    """AdamW (decoupled weight decay) with torch.optim.AdamW's formula, arguments and state layout (`step`, `exp_avg`, `exp_avg_sq`), every
    parameter in a launch per 56 tensors.  Parameters are float32 CUDA tensors, dense in any memory order.  capturable=True keeps the
    hyper-parameters and step numbers on the device, for a step captured into a hipGraph (`push_hyper()` before each replay)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, capturable=False):
        _check_common("segmi.optim.FusedAdamW", lr, weight_decay, betas, eps)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay), capturable)

    def _check_group(self, group):
        _check_common(self._name(), group["lr"], group["weight_decay"], group["betas"], group["eps"])

    def _hyper_values(self):
        return [self._adamw_hyper("betas", "eps", None)]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        k = self._plan()
        if k["rest"] is not None:
            with _on(self._device()):
                self._ready(k)
                self._adamw_launch(k, self._hyper_values()[0], self._hyper.dev.data_ptr() if self.capturable else None, torch.cuda.current_stream().cuda_stream)
        return loss


def _matrix_of(p):
    """(rows, cols) of the dense matrix in p's memory, or None where p is no matrix: vectors, single rows or columns, depthwise filters
    [C, 1, R, S].  shape[0] x rest, or its transpose where shape[0] runs fastest: the two are orthogonalised alike."""
    if p.dim() < 2 or (p.dim() == 4 and p.shape[1] == 1):
        return None
    r = p.shape[0]
    c = p.numel() // r if r else 0
    if min(r, c) < 2:
        return None
    if p.stride(0) == c:
        return r, c
    if p.stride(0) == 1:
        return c, r
    raise RuntimeError("segmi.optim.Muon: a matrix parameter must have its first dimension outermost or innermost in memory, got shape %s "
                       "strides %s" % (tuple(p.shape), tuple(p.stride())))


def _check_muon(g):
    name = "segmi.optim.Muon"
    _check_common(name, g["lr"], g["weight_decay"], g["adamw_betas"], g["adamw_eps"])
    if not 0.0 <= float(g["momentum"]) < 1.0:
        raise ValueError("%s: momentum must be in [0, 1), got %r" % (name, g["momentum"]))
    if not float(g["adamw_lr_ratio"]) >= 0.0:
        raise ValueError("%s: invalid adamw_lr_ratio %r" % (name, g["adamw_lr_ratio"]))
    _check_adjust(g["adjust_lr_fn"])
    _check_algorithm(g["algorithm"])
    _check_iteration(g["ns_steps"], g["ns_coefficients"], g["eps"], name)


def _check_adjust(adjust_lr_fn):
    if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
        raise ValueError("segmi.optim.Muon: adjust_lr_fn must be None, 'original' or 'match_rms_adamw', got %r" % (adjust_lr_fn,))


def _check_algorithm(algorithm):
    if algorithm not in ("auto", "adamw"):
        raise ValueError("segmi.optim.Muon: a group's algorithm is 'auto' or 'adamw', got %r" % (algorithm,))


class Muon(_FusedOptimizer):
    """Momentum orthogonalised by Newton-Schulz products, for every parameter that is a matrix:

        B <- momentum B + grad;   U = grad + momentum B (nesterov) or B
        p <- (1 - lr weight_decay) p - lr f orthogonalize(U)

    f = sqrt(max(1, rows / cols)) (adjust_lr_fn None or "original") or 0.2 sqrt(max(rows, cols)) ("match_rms_adamw": updates as
    large as AdamW's, so one learning rate suits both halves), rows = shape[0].  Argument names follow torch.optim.Muon, which takes 2-D parameters
    only; this one takes a whole network: vectors, single rows and columns, depthwise filters and the parameters of groups
    with `"algorithm": "adamw"` are updated by AdamW with learning rate lr * adamw_lr_ratio, adamw_betas, adamw_eps and the group's weight_decay.
    State: `momentum_buffer`, or `step`, `exp_avg`, `exp_avg_sq`.  torch.optim.Muon's buffer is a mean of the gradients, (1 - momentum) B: its
    dictionaries are rescaled when they are loaded here, one of this class has to be before torch's loads it.  Learning rate, weight decay, momentum and the AdamW
    numbers may differ between groups (up to 8); nesterov, eps, ns_coefficients and ns_steps are one for all.  A parameter without gradient is
    left alone.  capturable=True: as segmi.optim.SGD."""

    _SHARED = ("nesterov", "eps", "ns_coefficients", "ns_steps")

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=NS_COEFFICIENTS, eps=1e-7, ns_steps=5,
                 adjust_lr_fn=None, adamw_lr_ratio=1.0, adamw_betas=(0.9, 0.95), adamw_eps=1e-8, capturable=False):
        _check_muon(dict(lr=lr, weight_decay=weight_decay, momentum=momentum, ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                         adamw_lr_ratio=adamw_lr_ratio, adamw_betas=adamw_betas, adamw_eps=adamw_eps, algorithm="auto"))
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=bool(nesterov),
                                      ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                                      adamw_lr_ratio=adamw_lr_ratio, adamw_betas=tuple(adamw_betas), adamw_eps=adamw_eps, algorithm="auto"),
                         capturable)

    def _check_group(self, group):
        _check_muon(group)

    def _momentum_scale(self, group):
        # torch.optim.Muon keeps a mean, buf.lerp_(grad, 1 - momentum); its groups have the iteration's settings and none for vectors
        theirs = "ns_steps" in group and "adamw_lr_ratio" not in group
        return 1.0 / (1.0 - float(group["momentum"])) if theirs else 1.0

    def _hyper_values(self):
        h = np.zeros((3, _MAX_GROUPS), dtype=np.float32)
        for i, g in enumerate(self.param_groups):
            h[:, i] = float(g["lr"]), float(g["weight_decay"]), float(g["momentum"])
        return [h, self._adamw_hyper("adamw_betas", "adamw_eps", "adamw_lr_ratio")]

    def _is_matrix(self, group, p):
        algorithm = group.get("algorithm", "auto")
        _check_algorithm(algorithm)
        return algorithm == "auto" and _matrix_of(p) is not None

    def _settings(self):
        return [(g["adjust_lr_fn"], g.get("algorithm", "auto")) for g in self.param_groups]

    def _matrix_descriptors(self, members):
        for gi in {gi for gi, _ in members}:
            _check_adjust(self.param_groups[gi]["adjust_lr_fn"])
        rows = []
        for gi, p in members:
            g, (r, c) = self._checked(p), _matrix_of(p)
            k, rest = p.shape[0], p.numel() // p.shape[0]
            if self.param_groups[gi]["adjust_lr_fn"] == "match_rms_adamw":
                f = 0.2 * math.sqrt(max(k, rest))
            else:
                f = math.sqrt(max(1.0, k / rest))
            rows.append((p.data_ptr(), g.data_ptr(), self._buffer(p, "momentum_buffer").data_ptr(), r, c, f, gi))
        desc = np.array(rows, dtype=_MUON_DTYPE)
        nbytes = lib.segmi_muon_workspace(desc.ctypes.data, len(desc))
        if not nbytes:
            raise SegmiError("segmi.optim.Muon: a matrix is too large (4 GiB of float32 after padding its sides to 64)")
        return desc, nbytes

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = self.param_groups
        first = groups[0]
        for g in groups[1:]:
            if any(g[k] != first[k] for k in self._SHARED):
                raise ValueError("segmi.optim.Muon: %s must be the same in all parameter groups" % ", ".join(self._SHARED))
        k = self._plan()
        if k["mats"] is None and k["rest"] is None:
            return loss
        coef = _check_iteration(first["ns_steps"], first["ns_coefficients"], first["eps"], "segmi.optim.Muon")
        with _on(self._device()):
            self._ready(k)
            hd = self._hyper.dev.data_ptr() if self.capturable else None
            h, a = self._hyper_values()
            stream = torch.cuda.current_stream().cuda_stream
            if k["mats"] is not None:
                desc, nbytes = k["mats"]
                ws = torch.empty(nbytes, dtype=torch.uint8, device=self._device())
                check(lib.segmi_muon_step(desc.ctypes.data, len(desc), h[0].ctypes.data, h[1].ctypes.data, h[2].ctypes.data, len(groups), hd,
                                          1 if first["nesterov"] else 0, coef, int(first["ns_steps"]), float(first["eps"]), ws.data_ptr(), nbytes,
                                          stream), "muon_step")
            if k["rest"] is not None:
                self._adamw_launch(k, a, hd + 4 * 3 * _MAX_GROUPS if hd else None, stream)
        return loss
