"""The host's part of segmi.optim.Muon / FusedAdamW without a GPU: the launches are replaced by a recorder of their descriptors."""
import collections
import contextlib
import ctypes as C
import types

import numpy as np
import pytest
import torch

from segmi import muon, optim


class Recorder:
    """The library with the two steps' launches recorded: `calls` holds (name, descriptors)."""

    def __init__(self, lib):
        self._lib, self.calls = lib, []

    def __getattr__(self, name):
        return getattr(self._lib, name)

    def _record(self, name, dtype, at, count):
        raw = (C.c_char * (count * dtype.itemsize)).from_address(at)
        self.calls.append((name, np.frombuffer(raw, dtype).copy()))
        return 0

    def segmi_muon_step(self, at, count, *rest):
        return self._record("muon", muon._MUON_DTYPE, at, count)

    def segmi_adamw_step(self, at, count, *rest):
        return self._record("adamw", muon._ADAMW_DTYPE, at, count)

    def last(self, name):
        return [d for n, d in self.calls if n == name][-1]


@pytest.fixture
def host(monkeypatch):
    recorder = Recorder(muon.lib)
    monkeypatch.setattr(muon, "lib", recorder)
    monkeypatch.setattr(muon, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=0))
    monkeypatch.setattr(muon._FusedOptimizer, "_checked", lambda self, p: p.grad)
    return recorder


def parameters():
    ps = [torch.nn.Parameter(torch.zeros(80, 70)), torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(9))]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


OPTIMIZERS = [optim.Muon, optim.FusedAdamW]


# ------------------------------------------------------------------------------------------------ state that is taken away
def clear(opt):
    opt.state.clear()


def replace(opt):
    opt.state = collections.defaultdict(dict)


def empty_each(opt):
    for p in list(opt.state):
        opt.state[p] = {}


def empty_one(opt):
    opt.state[opt.param_groups[0]["params"][1]] = {}


@pytest.mark.parametrize("cls", OPTIMIZERS)
@pytest.mark.parametrize("reset", [clear, replace, empty_each, empty_one])
def test_a_reset_state_starts_anew(host, cls, reset):
    """As with torch's optimizers: momentum and moments of zero, step 1, and the state is the optimizer's again (a checkpoint has it)."""
    ps = parameters()
    opt = cls(ps)
    opt.step()
    opt.step()
    before = {p: dict(opt.state[p]) for p in ps}
    kept = {p for p in ps if reset is empty_one and p is not ps[1]}
    for p in ps:
        for v in before[p].values():
            v.fill_(7.0)
    reset(opt)
    opt.step()
    assert len(opt.state_dict()["state"]) == len(ps)
    steps = {int(r["param"]): float(r["step"]) for r in host.last("adamw")}
    for p in ps:
        st = opt.state[p]
        assert set(st) == set(before[p])
        for key, v in st.items():
            if p in kept:
                assert float(v.flatten()[0]) == (8.0 if key == "step" else 7.0), key
            elif key == "step":
                assert float(v) == 1.0
            else:
                assert v is not before[p][key] and not v.any(), key
        if "step" in st:
            assert steps[p.data_ptr()] == float(st["step"])
    pointers = {int(r["param"]): int(r["momentum"]) for r in host.last("muon")} if cls is optim.Muon else {int(r["param"]): int(r["exp_avg"]) for r in host.last("adamw")}
    for p in ps:
        key = "momentum_buffer" if "momentum_buffer" in opt.state[p] else "exp_avg"
        if p.data_ptr() in pointers:
            assert pointers[p.data_ptr()] == opt.state[p][key].data_ptr()


# ------------------------------------------------------------------------------------------------ groups
BAD_SETTINGS = [(optim.Muon, key, value) for key, value in
                (("adjust_lr_fn", "foo"), ("momentum", 1.5), ("momentum", -0.1), ("momentum", float("nan")), ("lr", -1.0), ("weight_decay", -0.1), ("adamw_betas", (0.9, 1.0)),
                 ("adamw_betas", (0.9,)), ("adamw_eps", -1e-8), ("adamw_lr_ratio", -1.0), ("algorithm", "sgd"), ("ns_steps", 0), ("eps", 0.0),
                 ("ns_coefficients", (9.0, 0.0, 0.0)))]
BAD_SETTINGS += [(optim.FusedAdamW, key, value) for key, value in
                 (("lr", -1.0), ("lr", float("nan")), ("weight_decay", -0.1), ("betas", (1.0, 0.9)), ("betas", (0.9, 0.9, 0.9)), ("eps", -1e-8))]


@pytest.mark.parametrize("cls,key,value", BAD_SETTINGS, ids=lambda v: getattr(v, "__name__", str(v)))
def test_a_groups_settings_are_checked(cls, key, value):
    """What the constructor refuses as a default is refused in a group, in a group added later and in a loaded dictionary, which then
    changes nothing."""
    ps = parameters()
    with pytest.raises(ValueError):
        cls([{"params": ps[:1], key: value}])
    opt = cls(ps[:2])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": ps[2:], key: value})
    assert len(opt.param_groups) == 1
    before = opt.state_dict()
    bad = opt.state_dict()
    bad["param_groups"] = [dict(g, lr=0.125) for g in bad["param_groups"]]
    bad["param_groups"][0][key] = value
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    assert opt.state_dict() == before
    opt.add_param_group({"params": ps[2:], "lr": 0.5})
    assert len(opt.param_groups) == 2


@pytest.mark.parametrize("key,value", [("adjust_lr_fn", "foo"), ("algorithm", "AdamW")])
def test_an_unknown_setting_made_later_is_refused(host, key, value):
    opt = optim.Muon(parameters())
    opt.step()
    opt.param_groups[0][key] = value
    with pytest.raises(ValueError, match=key):
        opt.step()


# ------------------------------------------------------------------------------------------------ dictionaries of other classes
@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_coupled_weight_decay_is_refused(cls):
    """torch.optim.Adam adds the decay to the gradient, the formula here takes it off the parameter.  Without decay they are the same."""
    ps = parameters()
    opt = cls(ps)
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(torch.optim.Adam(ps, weight_decay=0.1).state_dict())
    opt.load_state_dict(torch.optim.Adam(ps, lr=0.25, weight_decay=0.0).state_dict())
    opt.load_state_dict(torch.optim.AdamW(ps, lr=0.25, weight_decay=0.1).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["weight_decay"] == 0.1


def test_momentum_of_torchs_muon_is_rescaled(host):
    """torch.optim.Muon's buffer is a mean, buf.lerp_(grad, 1 - momentum); here it is a sum, 1 / (1 - momentum) times as large.  One
    multiplication in fp32: half a step."""
    p = torch.nn.Parameter(torch.zeros(80, 70))
    theirs = torch.optim.Muon([{"params": [p], "momentum": 0.9}, {"params": [torch.nn.Parameter(torch.zeros(4, 6))]}], lr=0.0, weight_decay=0.0)
    total = torch.zeros(80, 70, dtype=torch.float64)
    gen = torch.Generator().manual_seed(3)
    for _ in range(12):
        p.grad = torch.randn(80, 70, generator=gen)
        total = 0.9 * total + p.grad.double()
        theirs.step()
    sd = theirs.state_dict()
    buf = theirs.state[p]["momentum_buffer"]
    kept = buf.clone()
    for warm in (False, True):                        # into an optimizer without state, and over the state of one
        q = torch.nn.Parameter(torch.zeros(80, 70))
        q.grad = torch.ones(80, 70)
        opt = optim.Muon([{"params": [q]}, {"params": [torch.nn.Parameter(torch.zeros(4, 6))]}])
        if warm:
            opt.step()
        opt.load_state_dict(sd)
        got = opt.state[q]["momentum_buffer"]
        assert torch.equal(buf, kept) and opt.param_groups[0]["momentum"] == 0.9
        assert torch.allclose(got.double(), kept.double() / (1 - 0.9), rtol=2.0 ** -24 * 2, atol=0)
        # torch's twelve steps: each rounds (1 - momentum) g, the difference and the sum, and the scale gives each back ten times as large
        assert float((got.double() - total).abs().max()) <= 12 * 3 * 2.0 ** -24 * float(total.abs().max() + 10 * 5.0)
        again = opt.state_dict()                      # its own dictionary is not rescaled
        opt.load_state_dict(again)
        assert torch.equal(opt.state[q]["momentum_buffer"], got)
        other = optim.Muon([{"params": [torch.nn.Parameter(torch.zeros(80, 70))]}, {"params": [torch.nn.Parameter(torch.zeros(4, 6))]}])
        other.load_state_dict(again)
        assert torch.equal(other.state[other.param_groups[0]["params"][0]]["momentum_buffer"], got)


def test_momentum_of_sgd_is_taken_as_it_is_and_dampened_sums_are_refused(host):
    ps = parameters()
    sgd = torch.optim.SGD(ps, lr=0.1, momentum=0.9)
    for _ in range(2):
        sgd.step()
    opt = optim.Muon(ps)
    opt.load_state_dict(sgd.state_dict())
    assert torch.equal(opt.state[ps[0]]["momentum_buffer"], sgd.state[ps[0]]["momentum_buffer"])
    with pytest.raises(ValueError, match="dampening"):
        opt.load_state_dict(torch.optim.SGD(ps, lr=0.1, momentum=0.9, dampening=0.5).state_dict())


# ------------------------------------------------------------------------------------------------ which device
@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_groups_without_parameters_and_without_gradients(host, cls):
    """As torch.optim allows: an empty first group (everything in it frozen), no parameter at all, first parameters without a gradient."""
    ps = parameters()
    opt = cls([{"params": []}, {"params": ps}])
    opt.step()
    assert len(opt.state) == 3
    cls([{"params": []}]).step()
    held = torch.nn.Parameter(torch.zeros(3, device="meta"))              # elsewhere, and without a gradient
    opt = cls([{"params": [held]}, {"params": ps}])
    opt.step()
    assert len(opt.state) == 3 and opt._device() == ps[0].device
    empty = cls([{"params": []}], capturable=True)
    empty.push_hyper()
    empty.step()


# ------------------------------------------------------------------------------------------------ memory that two updates would write
@pytest.mark.parametrize("cls", OPTIMIZERS)
@pytest.mark.parametrize("shape", [(80, 70), (5600,)], ids=str)
def test_parameters_that_share_memory_are_refused(host, cls, shape):
    """One parameter twice, two parameters of one memory, overlapping views, one state buffer for two: their updates run at the same
    time."""
    def made(t):
        p = torch.nn.Parameter(t)
        p.grad = torch.ones_like(p)
        return p

    p = made(torch.zeros(shape))
    flat = torch.zeros(3 * 5600)
    near = made(flat[5600:11200].view(shape))
    for other in (made(p.data), made(p.data.view(-1)), made(p.data.view(-1)[5599:])):
        with pytest.raises(RuntimeError, match="share memory"):
            cls([p, other]).step()
        other.grad = None
        cls([p, other]).step()                        # tied to one that is trained: not an update of its own
    with pytest.raises(RuntimeError, match="share memory"):
        cls([near, made(flat[11199:16799].view(shape))]).step()
    cls([near, made(flat[:5600].view(shape)), made(flat[11200:].view(shape))]).step()           # neighbours
    with pytest.warns(UserWarning, match="duplicate"):
        twice = cls([p, p])
    with pytest.raises(RuntimeError, match="share memory"):
        twice.step()
    q = made(torch.zeros(shape))
    opt = cls([p, q])
    opt.step()
    key = next(k for k in opt.state[p] if k != "step")
    opt.state[q][key] = opt.state[p][key]
    with pytest.raises(RuntimeError, match="share memory"):
        opt.step()
    assert not host.calls or len(host.calls[-1][1])


def test_a_refused_step_changes_no_step_numbers(host):
    p = torch.nn.Parameter(torch.zeros(7))
    q = torch.nn.Parameter(torch.zeros(7))
    for t in (p, q):
        t.grad = torch.ones(7)
    opt = optim.FusedAdamW([p, q])
    opt.step()
    q.data = p.data
    with pytest.raises(RuntimeError, match="share memory"):
        opt.step()
    assert float(opt.state[p]["step"]) == 1.0


# ------------------------------------------------------------------------------------------------ what a captured step points at
@pytest.fixture
def capture(host, monkeypatch):
    """capture(opt): one step as if a graph were being captured."""
    class Hyper:
        def __init__(self, nbytes, device):
            self.dev = torch.zeros(nbytes, dtype=torch.uint8, device=device)

        def push(self, values):
            pass

    monkeypatch.setattr(muon, "_Hyper", Hyper)

    def run(opt):
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            opt.step()
    return run


@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_a_captured_steps_buffers_outlive_a_load_without_state(host, capture, cls):
    """A graph holds addresses: a dictionary without state (a new optimizer's) sets the buffers to zero where they are, and buffers that
    leave the state stay allocated."""
    ps = parameters()
    opt = cls(ps, lr=0.5, capturable=True)
    opt.step()
    capture(opt)
    captured = host.calls[-1][1].copy()
    buffers = {p: dict(opt.state[p]) for p in ps}
    for st in buffers.values():
        for v in st.values():
            v.fill_(3.0)
    opt.load_state_dict(cls(parameters(), lr=0.25).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25
    for p in ps:
        assert opt.state[p].keys() == buffers[p].keys()
        for key, v in opt.state[p].items():
            assert v is buffers[p][key] and not v.any(), key
    opt.step()
    assert all(np.array_equal(host.calls[-1][1][f], captured[f]) for f in captured.dtype.names)


@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_a_captured_steps_memory_is_kept(host, capture, cls):
    import gc
    import weakref
    ps = parameters()
    opt = cls(ps, capturable=True)
    opt.step()
    storages = lambda: [t.untyped_storage().data_ptr() for p in ps for t in [p, p.grad, *opt.state[p].values()]]
    before = storages()
    capture(opt)
    held = {t.untyped_storage().data_ptr() for t in opt._captured}
    assert held.issuperset(before)
    watched = [weakref.ref(t) for t in opt._captured]
    opt.state.clear()
    for p in ps:
        p.data = p.data.clone()
        p.grad = None
        p.grad = torch.ones_like(p)
    opt.step()
    gc.collect()
    assert all(w() is not None for w in watched)
    assert not set(storages()) & set(before)             # the eager step has buffers of its own
    import copy
    assert copy.deepcopy(opt)._captured == []


@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_a_load_without_state_and_without_a_graph_leaves_none(host, cls):
    ps = parameters()
    opt = cls(ps)
    opt.step()
    opt.load_state_dict(cls(parameters()).state_dict())
    assert not opt.state_dict()["state"]
    opt.step()
    assert all(float(st["step"]) == 1.0 for st in opt.state.values() if "step" in st)


@pytest.mark.parametrize("cls", OPTIMIZERS)
def test_state_dictionaries_that_change_places_are_seen(host, cls):
    a, b = (torch.nn.Parameter(torch.zeros(80, 70)) for _ in range(2))
    for p in (a, b):
        p.grad = torch.ones_like(p)
    opt = cls([a, b])
    opt.step()
    key = next(k for k in opt.state[a] if k != "step")
    opt.state[a], opt.state[b] = opt.state[b], opt.state[a]
    opt.step()
    name, field = ("muon", "momentum") if cls is optim.Muon else ("adamw", key)
    assert {int(r["param"]): int(r[field]) for r in host.last(name)} == {p.data_ptr(): opt.state[p][key].data_ptr() for p in (a, b)}
    opt.state[torch.nn.Parameter(torch.zeros(3))] = {}        # another's: nothing changes here
    opt.step()
    assert {int(r["param"]): int(r[field]) for r in host.last(name)} == {p.data_ptr(): opt.state[p][key].data_ptr() for p in (a, b)}
