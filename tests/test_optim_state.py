"""The optimizers' state (v2e2v_amd/optim.py) as it is loaded: what needs no GPU."""
import pytest
import torch

from v2e2v_amd import _lib, optim


def live(dtype, step=4.0):
    """An optimizer of two parameters as it is in the middle of a run."""
    ps = [torch.nn.Parameter(torch.ones(n, dtype=dtype)) for n in (3, 5)]
    opt = optim.Adam(ps)
    for p in ps:
        opt.state[p] = dict(step=torch.tensor(step), exp_avg=torch.full_like(p, 0.25, dtype=torch.float32, requires_grad=False),
                            exp_avg_sq=torch.full_like(p, 0.5, dtype=torch.float32, requires_grad=False))
        if dtype != torch.float32:
            opt.state[p]["master"] = p.detach().float() + 2.0 ** -12
    return ps, opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_master_copy_goes_with_a_16_bit_parameter_only(dtype):
    _, saved = live(torch.bfloat16)
    ps, opt = live(dtype)
    opt.load_state_dict(saved.state_dict())
    for p in ps:
        assert ("master" in opt.state[p]) == (dtype != torch.float32)
        if dtype != torch.float32:
            assert bool((opt.state[p]["master"] == 1 + 2.0 ** -12).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_loaded_state_is_a_copy(dtype):
    """The state_dict of a live optimizer: neither one's step counts or moments are the other's memory."""
    ps, saved = live(dtype)
    qs, opt = live(dtype, 9.0)
    opt.load_state_dict(saved.state_dict())
    for p, q in zip(ps, qs):
        assert set(opt.state[q]) == set(saved.state[p])
        for name, t in opt.state[q].items():
            assert torch.equal(t, saved.state[p][name]) and t.data_ptr() != saved.state[p][name].data_ptr(), name
    a = optim.Adam([torch.nn.Parameter(torch.ones(2))])
    a.load_state_dict(dict(state={0: dict(step=3)}, param_groups=a.state_dict()["param_groups"]))    # a plain number
    assert a.state[a.param_groups[0]["params"][0]]["step"] == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_hooks_of_load_state_dict(dtype):
    """What a pre-hook returns is what is loaded, and a post-hook sees the state that stays."""
    _, saved = live(dtype)
    qs, opt = live(dtype, 9.0)
    value = 0.125 + 2.0 ** -20                               # no 16-bit value
    seen = []

    def doubled(o, sd):
        return dict(sd, state={i: dict(s, exp_avg=torch.full_like(s["exp_avg"], value)) for i, s in sd["state"].items()})

    opt.register_load_state_dict_pre_hook(doubled)
    opt.register_load_state_dict_post_hook(lambda o: seen.extend(o.state[q]["exp_avg"] for q in qs))
    for _ in range(2):
        opt.load_state_dict(saved.state_dict())
        assert len(seen) == 2
        for q, t in zip(qs, seen):
            assert opt.state[q]["exp_avg"] is t and t.dtype == torch.float32 and bool((t == value).all())
        seen.clear()
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 1


def test_a_refused_state_dict_changes_nothing():
    """amsgrad is refused before the state or the hyperparameters are taken over."""
    _, saved = live(torch.float32)
    qs, opt = live(torch.float32, 9.0)
    sd = saved.state_dict()
    sd["param_groups"][0].update(amsgrad=True, lr=123.0)
    with pytest.raises(_lib.CistaError, match="amsgrad"):
        opt.load_state_dict(sd)
    assert "amsgrad" not in opt.param_groups[0] and opt.param_groups[0]["lr"] == 1e-3
    assert all(opt.state[q]["step"].item() == 9.0 for q in qs)
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks
