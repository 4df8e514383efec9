"""Matrix optimizer (segmi.optim.orthogonalize / Muon / FusedAdamW): refusals and the host's part, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import segmi
from segmi import muon, optim
from segmi._lib import lib


def test_orthogonalize_refuses_what_it_cannot_run():
    with pytest.raises(segmi.SegmiError, match="only run on the MI355X"):
        optim.orthogonalize(torch.randn(4, 4))
    with pytest.raises(ValueError, match="two or more dimensions"):
        optim.orthogonalize(torch.randn(4))
    with pytest.raises(ValueError, match="two or more dimensions"):
        optim.orthogonalize([3.0])
    for steps in (0, -1, 33, 2.5, True):
        with pytest.raises(ValueError, match="Newton-Schulz steps"):
            optim.orthogonalize([], steps=steps)
    for eps in (0.0, -1e-7, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            optim.orthogonalize([], eps=eps)
    for coef in ((10.0, 0.0, 0.0), (0.0, 0.0, 0.0), (float("nan"), 1.0, 1.0), (3.4445, -4.7750, 20.0)):
        with pytest.raises(ValueError, match="bounded"):
            optim.orthogonalize([], coefficients=coef)
    with pytest.raises(ValueError, match="three"):
        optim.orthogonalize([], coefficients=(1.5, -0.5))
    assert optim.orthogonalize([]) == []


@pytest.mark.parametrize("coef", [muon.NS_COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (15 / 8, -10 / 8, 3 / 8)])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 12])
def test_usual_coefficients_are_accepted(coef, steps):
    assert lib.segmi_ns_coefficients_ok((C.c_double * 3)(*coef), steps) == 1
    # and their iterates do stay bounded
    s = np.linspace(0.0, 1.0, 2001)
    for _ in range(steps):
        s = coef[0] * s + coef[1] * s ** 3 + coef[2] * s ** 5
    assert np.abs(s).max() < 2.0


def test_optimizers_refuse_bad_arguments():
    p = [torch.nn.Parameter(torch.randn(3, 3))]
    for kw in (dict(lr=-1.0), dict(weight_decay=-0.1), dict(momentum=1.0), dict(momentum=-0.1), dict(adjust_lr_fn="x"), dict(adamw_betas=(0.9, 1.0)),
               dict(adamw_betas=(0.9,)), dict(adamw_eps=-1.0), dict(ns_steps=0), dict(eps=0.0), dict(ns_coefficients=(9.0, 0.0, 0.0)), dict(adamw_lr_ratio=-1.0)):
        with pytest.raises(ValueError):
            optim.Muon(p, **kw)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            optim.FusedAdamW(p, **kw)
    with pytest.raises(ValueError, match="algorithm"):
        optim.Muon([{"params": p, "algorithm": "sgd"}])
    for cls in (optim.Muon, optim.FusedAdamW):
        many = [{"params": [torch.nn.Parameter(torch.zeros(2))]} for _ in range(9)]
        with pytest.raises(ValueError, match="up to 8 parameter groups"):
            cls(many)
        opt = cls(many[:8])
        with pytest.raises(ValueError, match="up to 8 parameter groups"):
            opt.add_param_group(many[8])
        assert len(opt.param_groups) == 8


def test_cpu_parameters_are_refused_at_the_step():
    for cls, shape in ((optim.Muon, (4, 4)), (optim.Muon, (4,)), (optim.FusedAdamW, (4,))):
        p = torch.nn.Parameter(torch.zeros(shape))
        opt = cls([p])
        opt.step()                                   # nothing has a gradient: nothing happens
        p.grad = torch.ones(shape)
        with pytest.raises((RuntimeError, AssertionError, ValueError)):
            opt.step()


def test_which_parameters_are_matrices():
    cl = lambda *s: torch.zeros(s).contiguous(memory_format=torch.channels_last)
    assert muon._matrix_of(cl(8, 4, 3, 3)) == (8, 36)
    assert muon._matrix_of(torch.zeros(8, 4, 2, 2)) == (8, 16)
    assert muon._matrix_of(torch.zeros(8, 5)) == (8, 5)
    assert muon._matrix_of(torch.zeros(5, 8).t()) == (5, 8)
    for t in (torch.zeros(7), torch.zeros(()), torch.zeros(1, 9), torch.zeros(9, 1), cl(16, 1, 3, 3), cl(1, 8, 3, 3), torch.zeros(0, 3)):
        assert muon._matrix_of(t) is None
    with pytest.raises(RuntimeError, match="outermost or innermost"):
        muon._matrix_of(torch.zeros(3, 8, 5).transpose(0, 1))


def test_c_entries_refuse_before_anything_is_launched():
    coef = (C.c_double * 3)(*muon.NS_COEFFICIENTS)
    d = np.zeros(1, dtype=muon._NS_DTYPE)
    d["src"], d["dst"], d["rows"], d["cols"], d["src_rs"], d["src_cs"], d["dst_rs"], d["dst_cs"] = 256, 512, 4, 8, 8, 1, 8, 1
    need = lib.segmi_ns_workspace(d.ctypes.data, 1)
    assert need > 0
    call = lambda a, n=1, c=coef, steps=5, eps=1e-7, ws=4096, nb=need: lib.segmi_ns_orthogonalize(a.ctypes.data, n, c, steps, eps, ws, nb, None)
    assert call(d, n=0) == -1 and call(d, steps=0) == -1 and call(d, steps=33) == -1 and call(d, eps=0.0) == -1 and call(d, ws=None) == -1
    assert call(d, eps=float("nan")) == -1
    assert call(d, ws=4096 + 16) == -2
    assert call(d, nb=need - 1) == -3
    for field, bad in (("src", 0), ("dst", 0), ("rows", 0), ("cols", -3), ("dtype", 2)):
        e = d.copy()
        e[field] = bad
        assert call(e) == -1, field
    e = d.copy()
    e["rows"], e["cols"] = 1 << 15, 1 << 15
    assert lib.segmi_ns_workspace(e.ctypes.data, 1) == 0 and call(e) == -1
    m = np.zeros(1, dtype=muon._MUON_DTYPE)
    m["param"], m["grad"], m["momentum"], m["rows"], m["cols"] = 256, 512, 1024, 4, 8
    f = np.zeros(8, dtype=np.float32)
    need = lib.segmi_muon_workspace(m.ctypes.data, 1)
    call = lambda a, ng=1, hyper=f.ctypes.data, nb=need: lib.segmi_muon_step(a.ctypes.data, 1, hyper, hyper, hyper, ng, None, 1, coef, 5, 1e-7, 4096, nb, None)
    assert call(m, ng=0) == -1 and call(m, ng=9) == -1 and call(m, hyper=None) == -1 and call(m, nb=need - 1) == -3
    for field, bad in (("param", 0), ("grad", 0), ("momentum", 0), ("rows", 0), ("group", 1), ("group", -1)):
        e = m.copy()
        e[field] = bad
        assert call(e) == -1, field
    a = np.zeros(1, dtype=muon._ADAMW_DTYPE)
    a["param"], a["grad"], a["exp_avg"], a["exp_avg_sq"], a["count"], a["step"] = 256, 512, 1024, 2048, 7, 1.0
    h = np.zeros((8, muon._ADAMW_HYPER))
    call = lambda e, ng=1, hyper=h.ctypes.data, hd=None, ws=None, nb=0: lib.segmi_adamw_step(e.ctypes.data, 1, hyper, ng, hd, ws, nb, None)
    assert call(a, ng=0) == -1 and call(a, ng=9) == -1 and call(a, hyper=None) == -1
    assert call(a, hd=4096) == -3 and call(a, hd=4096, ws=4096, nb=8) == -1         # a graph's step needs a workspace and step numbers
    for field, bad in (("param", 0), ("grad", 0), ("exp_avg", 0), ("exp_avg_sq", 0), ("count", 0), ("group", 1), ("step", 0.0)):
        e = a.copy()
        e[field] = bad
        assert call(e) == -1, field


def test_descriptor_layouts_match_the_header(tmp_path):
    """The numpy records are the header's structs: sizes and offsets as the C compiler sees them."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    records = {"segmi_ns_matrix": muon._NS_DTYPE, "segmi_muon_matrix": muon._MUON_DTYPE, "segmi_adamw_tensor": muon._ADAMW_DTYPE}
    lines = ['#include <stdio.h>', '#include "segmi.h"', "int main(void){"]
    for name, dt in records.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f in dt.names]
    lines.append('printf("hyper %d\\n", SEGMI_ADAMW_HYPER); printf("steps %d\\n", SEGMI_NS_MAX_STEPS); return 0;}')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I" + os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, dt in records.items():
        assert int(got[name]) == dt.itemsize
        for f in dt.names:
            assert int(got[name + "." + f]) == dt.fields[f][1], (name, f)
    assert int(got["hyper"]) == muon._ADAMW_HYPER and int(got["steps"]) == 32


def test_trainer_resolves_the_optimizers_by_name():
    """config.json's optimizer.type: Muon and FusedAdamW come from segmi.optim, AdamW stays torch's."""
    import inspect
    from base import base_trainer
    src = inspect.getsource(base_trainer.BaseTrainer.__init__)
    assert "segmi_optim if fused else torch.optim" in src
    p = [torch.nn.Parameter(torch.zeros(3, 3))]
    get = base_trainer.get_instance
    for name in ("Muon", "FusedAdamW"):
        opt = get(optim, "optimizer", {"optimizer": {"type": name, "args": {"lr": 0.01, "weight_decay": 0.0}}}, p)
        assert type(opt).__name__ == name and type(opt).__module__.startswith("segmi")


def test_optimizers_copy_and_pickle():
    import copy
    import pickle
    for cls in (optim.Muon, optim.FusedAdamW):
        p = torch.nn.Parameter(torch.zeros(4, 4))
        for opt in (copy.deepcopy(cls([p], lr=0.5, capturable=True)), pickle.loads(pickle.dumps(cls([p], lr=0.5, capturable=True)))):
            assert opt.capturable and opt.param_groups[0]["lr"] == 0.5
            opt.step()                               # no gradient: nothing happens
            opt.param_groups[0]["params"][0].grad = torch.ones(4, 4)
            with pytest.raises((RuntimeError, AssertionError)):
                opt.step()
            opt.load_state_dict(opt.state_dict())


def test_loaded_settings():
    p = [torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(4))]
    opt = optim.Muon(p, lr=0.5, adamw_lr_ratio=0.25)
    sd = opt.state_dict()
    for g in sd["param_groups"]:                     # as written by a class that knows less
        for key in ("adamw_lr_ratio", "adamw_betas", "adamw_eps", "algorithm"):
            del g[key]
        g["lr"] = 0.125
    opt.load_state_dict(sd)
    g = opt.param_groups[0]
    assert (g["lr"], g["adamw_lr_ratio"], g["adamw_betas"], g["algorithm"]) == (0.125, 0.25, (0.9, 0.95), "auto")
    for key in ("amsgrad", "maximize"):
        other = torch.optim.AdamW(p, lr=0.1, **{key: True})
        with pytest.raises(ValueError, match=key):
            optim.FusedAdamW(p).load_state_dict(other.state_dict())
    mine = optim.FusedAdamW(p)
    mine.load_state_dict(torch.optim.AdamW(p, lr=0.1, betas=(0.5, 0.6)).state_dict())
    assert mine.param_groups[0]["lr"] == 0.1 and mine.param_groups[0]["betas"] == (0.5, 0.6)
