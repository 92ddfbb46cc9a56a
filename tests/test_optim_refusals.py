"""The training-step operators' checks of arguments (v2e2v_amd/optim.py, include/cista_optim.h): all
of them come before any device work, so they need no GPU."""
import copy
import ctypes
import math

import pytest
import torch

from v2e2v_amd import _lib, optim

FAKE = 1 << 20            # stands for device memory in calls that are refused before it is used


def table(*rows):
    return (optim.CistaTensor * max(len(rows), 1))(*rows)


def adam_row(param=FAKE, grad=2 * FAKE, m=3 * FAKE, v=4 * FAKE, master=None, step=5 * FAKE, numel=16, kind=0):
    return (param, grad, m, v, master, step, numel, kind)


def adam_call(rows, group=None, norm_kind=0, max_norm=0.0, norm=None, ws=FAKE, nbytes=1 << 30):
    t = (optim.CistaAdamTensor * max(len(rows), 1))(*rows)
    g = (optim.CistaAdamGroup * 1)(group or (1e-3, 0.9, 0.999, 1e-8, 0.0, None, len(rows), 0, 0, 0))
    return _lib.lib().cista_adam_step(t, g, 1, norm_kind, max_norm, norm, ws, nbytes, None)


def test_c_entries_refuse_bad_tables():
    L = _lib.lib()
    big = 1 << 30
    ok = (FAKE, 16, 0)
    for bad, status in [((FAKE, -1, 0), 1), ((None, 4, 0), 1), ((FAKE + 2, 4, 0), 1), ((FAKE + 1, 4, 1), 1),
                        ((FAKE, 4, 3), 1), ((FAKE, 4, -1), 1), ((FAKE, 1 << 41, 0), 2)]:
        assert L.cista_grad_norm(table(ok, bad), 2, 2, FAKE, FAKE, big, None) == status, bad
        assert L.cista_scale_grads(table(ok, bad), 2, 1.0, FAKE, None) == status, bad
        assert L.cista_clip_grads(table(ok, bad), 2, 2, 1.0, FAKE, FAKE, big, None) == status, bad
    assert L.cista_grad_norm(table(ok), -1, 2, FAKE, FAKE, big, None) == 1
    assert L.cista_grad_norm(None, 1, 2, FAKE, FAKE, big, None) == 1
    assert L.cista_grad_norm(table(ok), 1, 0, FAKE, FAKE, big, None) == 1
    assert L.cista_grad_norm(table(ok), 1, 4, FAKE, FAKE, big, None) == 1
    assert L.cista_grad_norm(table(ok), 1, 2, None, FAKE, big, None) == 1
    assert L.cista_grad_norm(table(ok), 1, 2, FAKE, None, big, None) == 1
    assert L.cista_grad_norm(table(ok), 1, 2, FAKE + 2, FAKE, big, None) == 1           # misaligned
    assert L.cista_grad_norm(table(ok), 1, 2, FAKE, FAKE + 8, big, None) == 1
    assert L.cista_scale_grads(table(ok), 1, 1.0, FAKE + 1, None) == 1
    assert L.cista_clip_grads(table(ok), 1, 2, 1.0, FAKE, FAKE + 4, big, None) == 1
    need = L.cista_optim_workspace_bytes(1)
    assert L.cista_grad_norm(table(ok), 1, 2, FAKE, FAKE, need - 1, None) == 4
    assert L.cista_clip_grads(table(ok), 1, 2, 1.0, FAKE, FAKE, need - 1, None) == 4
    for bound in (-1.0, math.nan):
        assert L.cista_scale_grads(table(ok), 1, bound, FAKE, None) == 1
        assert L.cista_clip_grads(table(ok), 1, 2, bound, FAKE, FAKE, big, None) == 1
    assert L.cista_optim_workspace_bytes(-1) == 0
    assert L.cista_optim_workspace_bytes(400) > L.cista_optim_workspace_bytes(0) > 0


@pytest.mark.parametrize("a,b", [
    ((FAKE, 16, 0), (FAKE, 16, 0)),                    # the same tensor twice
    ((FAKE, 16, 0), (FAKE + 60, 4, 0)),                # the last element of one is the other's first
    ((FAKE + 60, 4, 0), (FAKE, 16, 0)),
    ((FAKE, 8, 1), (FAKE + 14, 1, 2)),
])
def test_gradients_that_share_memory_are_refused(a, b):
    L = _lib.lib()
    far = (FAKE * 8, 3, 0)
    assert L.cista_scale_grads(table(a, far, b), 3, 1.0, FAKE, None) == 5
    assert L.cista_clip_grads(table(far, a, b), 3, 2, 1.0, FAKE, FAKE, 1 << 30, None) == 5


def test_adam_entry_refuses():
    L = _lib.lib()
    need = L.cista_optim_workspace_bytes(1)
    assert adam_call([adam_row(param=None)]) == 1
    assert adam_call([adam_row(grad=None)]) == 1
    assert adam_call([adam_row(m=None)]) == 1
    assert adam_call([adam_row(v=FAKE + 2)]) == 1
    assert adam_call([adam_row(step=None)]) == 1
    assert adam_call([adam_row(numel=-3)]) == 1
    assert adam_call([adam_row(numel=1 << 40)]) == 2
    assert adam_call([adam_row(kind=1)]) == 1           # 16 bits without a master copy
    assert adam_call([adam_row(), adam_row(param=FAKE + 60)]) == 5
    assert adam_call([adam_row()], ws=None) == 1
    assert adam_call([adam_row()], ws=FAKE + 8) == 1
    assert adam_call([adam_row(step=FAKE + 2)]) == 1
    assert adam_call([adam_row()], group=(1e-3, 0.9, 0.9, 1e-8, 0.0, FAKE + 2, 1, 0, 0, 0)) == 1
    twice = [adam_row(), adam_row(param=9 * FAKE, grad=9 * FAKE, m=10 * FAKE, v=11 * FAKE, step=12 * FAKE)]
    for k in (2, 3, 5):                                  # the same m, v or step for two parameters
        rows = [twice[0], tuple(twice[0][j] if j == k else x for j, x in enumerate(twice[1]))]
        assert adam_call(rows) == 5
    half = [adam_row(master=6 * FAKE, kind=1), adam_row(9 * FAKE, 9 * FAKE, 10 * FAKE, 11 * FAKE, 6 * FAKE + 4, 12 * FAKE, kind=1)]
    assert adam_call(half) == 5
    assert adam_call([adam_row()], nbytes=need - 1) == 4
    assert adam_call([adam_row()], norm_kind=4, norm=FAKE) == 1
    assert adam_call([adam_row()], norm_kind=2, norm=None) == 1
    assert adam_call([adam_row()], norm_kind=2, norm=FAKE, max_norm=-1.0) == 1
    for b1, b2 in ((1.0, 0.9), (-0.1, 0.9), (0.9, 1.0), (0.9, math.nan)):
        assert adam_call([adam_row()], group=(1e-3, b1, b2, 1e-8, 0.0, None, 1, 0, 0, 0)) == 1
    assert adam_call([adam_row()], group=(1e-3, 0.9, 0.9, 1e-8, 0.0, None, -1, 0, 0, 0)) == 1
    assert L.cista_adam_step(None, None, 1, 0, 0.0, None, FAKE, 1 << 30, None) == 1


def test_python_surface_refuses():
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(_lib.CistaError, match="ROCm GPU only"):
        optim.grad_norm([p.grad])
    with pytest.raises(_lib.CistaError, match="ROCm GPU only"):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(_lib.CistaError, match="ROCm GPU only"):
        optim.clip_grads_with_norm_(p, 1.0, torch.tensor(1.0))
    with pytest.raises(_lib.CistaError, match="ROCm GPU only"):
        optim.Adam([p]).step()
    for order in (0.0, 3.0, -math.inf, math.nan):
        with pytest.raises(_lib.CistaError, match="norm_type"):
            optim.grad_norm([p.grad], order)
        with pytest.raises(_lib.CistaError, match="norm_type"):
            optim.Adam([p], norm_type=order)
    for bound in (-1.0, math.nan):
        with pytest.raises(_lib.CistaError, match="max_norm"):
            optim.clip_grad_norm_([p], bound)
        with pytest.raises(_lib.CistaError, match="max_norm"):
            optim.clip_grads_with_norm_([p], bound, torch.tensor(1.0))
        with pytest.raises(_lib.CistaError, match="max_norm"):
            optim.Adam([p], max_norm=bound)
    with pytest.raises(TypeError):
        optim.grad_norm([3.0])
    with pytest.raises(_lib.CistaError, match="strided"):
        optim.grad_norm([torch.eye(2).to_sparse()])
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0),
                dict(lr=torch.ones(2))):
        with pytest.raises(ValueError):
            optim.Adam([p], **bad)
    assert torch.equal(p.grad, torch.ones(3)) and torch.equal(p.detach(), torch.ones(3))


def test_nothing_to_do():
    """No tensors, or no gradients: the norm is 0 and nothing else happens."""
    assert optim.grad_norm([]).item() == 0.0
    p = torch.nn.Parameter(torch.ones(3))
    assert optim.clip_grad_norm_([p], 1.0).item() == 0.0
    assert optim.clip_grad_norm_(iter([]), 1.0).item() == 0.0
    optim.clip_grads_with_norm_([p], 1.0, torch.tensor(1.0))
    opt = optim.Adam([p], max_norm=1.0)
    assert opt.step() is None and opt.step(lambda: 7.0) == 7.0 and not opt.state


def test_optimizer_object():
    """Defaults, schedulers, copies and state_dicts keep what the step needs."""
    p, q = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(2, dtype=torch.bfloat16))
    opt = optim.AdamW([dict(params=[p], lr=0.5), dict(params=[q], betas=(0.0, 0.5))], max_norm=2.0, norm_type=math.inf)
    assert [g["lr"] for g in opt.param_groups] == [0.5, 1e-3]
    assert all(g["decoupled_weight_decay"] and g["weight_decay"] == 0.01 for g in opt.param_groups)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    opt.step()
    sched.step()
    assert opt.param_groups[0]["lr"] == 0.25
    twin = copy.deepcopy(opt)
    assert twin.max_norm == 2.0 and twin.norm_type == math.inf and twin.grad_norm is None
    # a checkpoint without the newer group entries, of a run that kept its moments in float32
    moments = dict(step=torch.tensor(4.0), exp_avg=torch.full((2,), 1.0 + 2.0 ** -20), exp_avg_sq=torch.ones(2))
    opt.load_state_dict(dict(state={1: moments}, param_groups=[
        dict(lr=0.1, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, params=[0]),
        dict(lr=0.1, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, params=[1])]))
    assert opt.param_groups[0]["decoupled_weight_decay"] is True and opt.param_groups[1]["maximize"] is False
    assert opt.state[q]["exp_avg"].dtype == torch.float32 and opt.state[q]["exp_avg"][0].item() == 1.0 + 2.0 ** -20
    with pytest.raises(_lib.CistaError, match="amsgrad"):
        opt.load_state_dict(dict(state={}, param_groups=[dict(g, amsgrad=True, params=[k])
                                                         for k, g in enumerate(opt.param_groups)]))


def test_tables_match_the_header():
    assert ctypes.sizeof(optim.CistaTensor) == 24 and ctypes.sizeof(optim.CistaAdamTensor) == 64
    assert ctypes.sizeof(optim.CistaAdamGroup) == 64


def test_bench_flags(monkeypatch):
    """bench.py: --max_norm goes with --mode train --adam hip only."""
    import sys

    import bench
    monkeypatch.setattr(sys, "argv", ["bench.py", "--mode", "train", "--adam", "hip", "--max_norm", "0.5"])
    args = bench.parse()
    assert args.adam == "hip" and args.max_norm == 0.5
    for argv in (["--mode", "train", "--max_norm", "0.5"], ["--adam", "hip", "--max_norm", "0.5"]):
        monkeypatch.setattr(sys, "argv", ["bench.py"] + argv)
        with pytest.raises(SystemExit):
            bench.parse()


@pytest.mark.parametrize("norm", [FAKE, FAKE + 32, FAKE + 60, FAKE * 8 + 8])
def test_a_norm_within_the_tensors_is_refused(norm):
    """Some workgroups would read, or write, it while others write the tensor."""
    L = _lib.lib()
    t = table((FAKE, 16, 0), (FAKE * 8, 3, 0))
    assert L.cista_scale_grads(t, 2, 1.0, norm, None) == 5
    assert L.cista_clip_grads(t, 2, 2, 1.0, norm, FAKE * 16, 1 << 30, None) == 5
    assert L.cista_scale_grads(table((norm + 2, 0, 1)), 1, 1.0, norm, None) != 5        # an empty one holds nothing


@pytest.mark.parametrize("k", [0, 1, 2, 3, 4, 5])
def test_a_norm_within_the_state_is_refused(k):
    row = adam_row(master=6 * FAKE, kind=1)
    at = row[k] + (0 if k == 5 else 4)
    assert adam_call([adam_row(9 * FAKE, 10 * FAKE, 11 * FAKE, 12 * FAKE, step=13 * FAKE), row], norm_kind=2, max_norm=1.0,
                     norm=at, ws=16 * FAKE) == 5


def test_the_host_library_goes_with_its_torch(monkeypatch):
    """Another torch: `make` builds the host library anew, and one that was not built anew is refused."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
    version = os.path.join(os.path.dirname(torch.__file__), "version.py")
    plan = ["make", "-n", "-C", root, "v2e2v_amd/libcista_torch.so"]
    assert "cista_torch.cpp" in subprocess.run(plan + ["-W", version], capture_output=True, text=True, check=True).stdout
    _lib.torch_lib()
    monkeypatch.setattr(_lib, "_torch_lib", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0+rocm1.0")
    with pytest.raises(_lib.CistaError, match="built for torch"):
        optim.grad_norm([torch.ones(1)])
