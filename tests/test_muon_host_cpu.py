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
