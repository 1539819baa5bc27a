"""CPU: what gs_localization_amd.map_optimizer refuses, and what its optimiser keeps in groups and states, before any GPU is touched."""
import ctypes as C

import pytest
import torch

from gs_localization_amd import _lib, map_optimizer as MO


def coded(origin, **kw):
    """gsr_adamw_step_coded of one 8-bit tensor on made-up addresses: refusals come before a pointer is used, and one that is not refused gets as far as
    looking for its device"""
    lib = _lib.load()
    buf, origins = bytearray(MO._OPT.size), bytearray(MO._ORIGIN.size)
    MO._OPT.pack_into(buf, 0, *dict(dict(param=0x1000, grad=0x20000, state0=0x30000, state1=0x40000, window=0x50000, clock=0x60000, lr_device=0, lr=0.1, decay=0.0,
                                         n=64, pt=0, gt=0), **kw).values())
    MO._ORIGIN.pack_into(origins, 0, *origin, 0)
    args = _lib.AdamwArgs(1, 8, MO._address(buf), 0.9, 0.999, 1e-8, None, 0, None)
    checked, said = lib.gsr_adamw_check(C.byref(args), MO._address(origins)), lib.gsr_last_error().decode()
    rc = lib.gsr_adamw_step_coded(C.byref(args), MO._address(origins))
    assert checked == (0 if rc == -4 else rc) and (rc == -4 or said == lib.gsr_last_error().decode())
    return rc, lib.gsr_last_error().decode()


def test_betas_of_the_codes_are_checked():
    for bad in ((0.99, 0.9), (1.0, 1.0), (-0.1, 0.9), (0.9, 1.0), (float("nan"), 0.9), (0.5, float("nan")), (0.0, 0.0)):
        rc, said = coded(bad)
        assert rc == -1 and "codes" in said, (bad, rc, said)
    assert coded((0.5, 0.3))[0] == -4
    assert _lib.load().gsr_adamw_step_coded(None, None) == -1


def test_one_cycle_schedule_on_8_bit_groups():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = MO.AdamW([p], lr=0.1, state_bits=8)
    torch.optim.lr_scheduler.OneCycleLR(opt, 0.1, total_steps=10)
    assert opt.param_groups[0]["betas"] == (0.95, 0.999) and opt.param_groups[0]["state_betas"] == (0.9, 0.999)
    again = MO.AdamW([torch.nn.Parameter(torch.zeros(4))], lr=0.1, state_bits=8)
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["betas"] == (0.95, 0.999) and again.param_groups[0]["state_betas"] == (0.9, 0.999)


def test_state_dict_without_the_betas_of_its_codes():
    """one that was saved before groups had "state_betas" was stored with the group's"""
    saved = MO.AdamW([torch.nn.Parameter(torch.zeros(4))], betas=(0.8, 0.95), state_bits=8).state_dict()
    saved = dict(saved, param_groups=[{k: v for k, v in g.items() if k != "state_betas"} for g in saved["param_groups"]])
    opt = MO.AdamW([torch.nn.Parameter(torch.zeros(4))], state_bits=8)
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["state_betas"] == (0.8, 0.95)


def trained(cls, old=False, **kw):
    """The state_dict of torch's optimiser after a step; old: as releases before "decoupled_weight_decay" wrote it."""
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    ref = cls([p], lr=0.1, **kw)
    ref.step()
    saved = ref.state_dict()
    for g in saved["param_groups"]:
        if old:
            del g["decoupled_weight_decay"]
    return saved


def test_decay_that_is_added_to_the_gradient_is_refused():
    """torch.optim.Adam's weight_decay is, AdamW's is not: the same number means another step"""
    opt = MO.AdamW([torch.nn.Parameter(torch.zeros(4))], lr=0.3)
    for saved in (trained(torch.optim.Adam, weight_decay=0.1), trained(torch.optim.Adam, old=True, weight_decay=0.1), trained(torch.optim.AdamW, old=True)):
        with pytest.raises(ValueError, match="decoupled"):
            opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] == 0.3 and opt.param_groups[0]["weight_decay"] == 0.0 and not opt.state
    for saved, decay in ((trained(torch.optim.Adam), 0.0), (trained(torch.optim.Adam, old=True), 0.0), (trained(torch.optim.AdamW, weight_decay=0.1), 0.1),
                         (trained(torch.optim.Adam, decoupled_weight_decay=True, weight_decay=0.2), 0.2), (opt.state_dict(), 0.0),
                         (MO.AdamW([torch.nn.Parameter(torch.zeros(4))], weight_decay=0.4).state_dict(), 0.4)):
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["weight_decay"] == decay and "decoupled_weight_decay" not in opt.param_groups[0]
    # which it is can be said where the file does not
    saved = trained(torch.optim.AdamW, old=True, weight_decay=0.1)
    saved["param_groups"][0]["decoupled_weight_decay"] = True
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["weight_decay"] == 0.1
