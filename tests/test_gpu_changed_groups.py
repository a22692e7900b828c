"""Fused optimizers whose groups change between steps, on the GPU: every step against a twin that forgets everything before it."""
import copy

import pytest
import torch

from rannc_amd.fused_optim import FusedAdam, FusedAdamW, FusedSGD

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MAKE = {"adam": lambda ps: FusedAdam(ps, lr=1e-2, weight_decay=0.1), "adamw8": lambda ps: FusedAdamW(ps, lr=1e-2, state_bits=8),
        "sgd": lambda ps: FusedSGD(ps, lr=0.05, momentum=0.9), "plain sgd": lambda ps: FusedSGD(ps, lr=0.05),
        "capturable8": lambda ps: FusedAdam(ps, lr=1e-2, state_bits=8, capturable=True)}


def same(a, b, what):
    for i, (p, q) in enumerate(zip(a.param_groups[0]["params"], b.param_groups[0]["params"])):
        assert torch.equal(p, q), (what, i)
    sa, sb = a.state_dict()["state"], b.state_dict()["state"]
    assert sa.keys() == sb.keys(), what
    for i in sa:
        assert sa[i].keys() == sb[i].keys() and all(torch.equal(v.cpu(), sb[i][k].cpu()) for k, v in sa[i].items()), (what, i)


@pytest.mark.parametrize("name", sorted(MAKE))
@pytest.mark.parametrize("place", [0, 1, 3])
@pytest.mark.parametrize("size", [3, 70001])
def test_entries_replaced_in_place(name, place, size):
    gen = torch.Generator().manual_seed(13)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in (700, 257, 5, 4096)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, twin = MAKE[name](ps), MAKE[name](qs)
    for step in range(7):
        if step == 3:
            data = torch.randn(size, generator=gen).to(DEV)
            for o in (opt, twin):
                group = o.param_groups[0]["params"]
                old, group[place] = group[place], torch.nn.Parameter(data.clone())
                st = {k: v for k, v in o.state.pop(old, {}).items() if k == "step"}
                if "capturable" in name:          # one count for the group: the new parameter's moments come along
                    o.state[group[place]] = st
                    o._make_moments(0, [group[place]])
        for o in (opt, twin):
            g = torch.Generator().manual_seed(step)
            for p in o.param_groups[0]["params"]:
                p.grad = torch.randn(p.shape, generator=g).to(DEV)
        twin.invalidate_tables()
        opt.step()
        twin.step()
        same(opt, twin, (name, step))


@pytest.mark.parametrize("name", sorted(MAKE))
def test_a_copy_goes_on_by_itself(name):
    gen = torch.Generator().manual_seed(14)
    model = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 3)).to(DEV)
    opt = MAKE[name](model.parameters())

    def step(m, o, seed):
        m.zero_grad(set_to_none=True)
        m(torch.randn(8, 33, generator=torch.Generator().manual_seed(seed)).to(DEV)).square().mean().backward()
        o.step()
    for k in range(3):
        step(model, opt, k)
    model2, opt2 = copy.deepcopy((model, opt))
    assert opt2.param_groups[0]["params"][0] is next(model2.parameters())
    for k in range(3, 6):
        step(model, opt, k)
    for k in range(3, 6):
        step(model2, opt2, k)
    same(opt, opt2, name)
    if getattr(opt, "state_bits", 32) == 8:
        assert all(b.numel() for b in opt2.state_buffers().values())


def test_refused_steps_of_a_real_table():
    """Hyper-parameters that the library refuses, before a full step and before a steady one, with the count on the host and on the device."""
    for capturable in (False, True):
        runs = []
        for refuse in (False, True):
            gen = torch.Generator().manual_seed(15)
            ps = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in (300, 41)]
            opt = FusedAdam(ps, lr=1e-2, state_bits=8, capturable=capturable)
            for step in range(4):
                for p in ps:
                    p.grad = torch.randn(p.shape, generator=gen).to(DEV)
                for bad in (dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=-1.0), dict(betas=(0.9, 1.0))) if refuse else ():
                    good = {k: opt.param_groups[0][k] for k in bad}
                    opt.param_groups[0].update(bad)
                    with pytest.raises(ValueError, match="hyper-parameters"):
                        opt.step()
                    opt.param_groups[0].update(good)
                opt.step()
            assert all(float(opt.state[p]["step"]) == 4 for p in ps)
            runs.append(opt)
        same(*runs, capturable)
