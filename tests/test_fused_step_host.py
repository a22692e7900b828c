"""The host side of the fused optimizers' steps without a GPU: which parameters, gradients and counts reach a table, with the
tables replaced by a record of what they are told.  Each test runs with the compiled module and without it."""
import copy
import io

import pytest
import torch

from rannc_amd import fused_optim
from rannc_amd.fused_optim import FusedAdam, FusedAdamW, FusedSGD


class Param(torch.nn.Parameter):
    """A CPU parameter that passes for one on the GPU."""
    is_cuda = True


class Table:
    """What ``_lib.OptimTable`` is told."""
    made = []
    refuse = None          # an exception that the next launches raise

    def __init__(self, device, params, grads, state1, state2, copies, numels, grad_dtypes, copy_dtypes=None, scales1=None, scales2=None):
        self.params, self.grads, self.state1, self.state2, self.scales2 = list(params), list(grads), state1, state2, scales2
        self.numels, self.grad_dtypes, self.steps = list(numels), grad_dtypes, []
        self.handle = id(self)
        Table.made.append(self)

    def update_pointers(self, params=None, grads=None, state1=None, state2=None, copies=None, stream=0):
        for name, given in (("params", params), ("grads", grads), ("state1", state1), ("state2", state2)):
            if given is not None:
                setattr(self, name, list(given))

    def adam_step(self, lr, beta1, beta2, eps, weight_decay, step, **kw):
        if Table.refuse is not None:
            raise Table.refuse
        self.steps.append((step, list(self.params), list(self.grads)))

    def sgd_step(self, *args, first_step=False, **kw):
        if Table.refuse is not None:
            raise Table.refuse
        self.steps.append((first_step, list(self.params), list(self.grads)))


@pytest.fixture(params=["compiled", "python"], autouse=True)
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(fused_optim, "_native", None)
    elif fused_optim._native is None:
        pytest.skip("the compiled module is not built")
    monkeypatch.setattr(fused_optim._lib, "OptimTable", Table)
    monkeypatch.setattr(fused_optim, "stream_handle", lambda device: 0)
    monkeypatch.setattr(Table, "made", [])
    monkeypatch.setattr(Table, "refuse", None)
    return request.param


MAKE = {"adam": lambda ps: FusedAdam(ps, lr=1e-2), "adamw8": lambda ps: FusedAdamW(ps, lr=1e-2, state_bits=8),
        "sgd": lambda ps: FusedSGD(ps, lr=0.05)}


@pytest.fixture(params=sorted(MAKE))
def make(request):
    return MAKE[request.param]


def parameters(sizes=(4, 6, 5)):
    return [Param(torch.zeros(n)) for n in sizes]


def give(params):
    for p in params:
        p.grad = torch.ones_like(p.detach())


# ---------------------------------------------------------------- entries of a group replaced in place

@pytest.mark.parametrize("place", [0, 1, 2])
@pytest.mark.parametrize("size", [4, 400000])
def test_replaced_parameters_bring_their_own_gradients(make, place, size):
    ps = parameters()
    opt = make(ps)
    for _ in range(3):
        give(ps)
        opt.step()
    group = opt.param_groups[0]["params"]
    old, new = group[place], Param(torch.zeros(size))
    group[place] = new
    if not isinstance(opt, FusedSGD):         # the count moves along, so that the group stays in step
        opt.state[new]["step"] = torch.tensor(float(opt.state[old]["step"]))
        opt._make_moments(0, [new])
    kept = old.grad                            # nothing clears it: it is no longer the optimizer's
    for _ in range(3):
        for p in group:
            p.grad = torch.ones_like(p.detach())
        opt.step()
        table = Table.made[-1]
        _, params, grads = table.steps[-1]
        assert params == [p.data_ptr() for p in group] and grads == [p.grad.data_ptr() for p in group]
        assert table.numels == [p.numel() for p in group] and kept.data_ptr() not in grads


def test_cleared_gradients_are_those_of_the_moment(make):
    ps = parameters()
    opt = make(ps)
    give(ps)
    opt.zero_grad()
    new = Param(torch.zeros(7))
    old, opt.param_groups[0]["params"][1] = ps[1], new
    give([old, new])
    opt.zero_grad()
    assert new.grad is None and old.grad is not None


def test_steps_stay_on_the_short_path(make, monkeypatch):
    """An unchanged group, also one whose list was replaced by an equal one, is not looked at parameter by parameter."""
    ps = parameters()
    opt = make(ps)
    for _ in range(2):
        give(ps)
        opt.step()
    monkeypatch.setattr(opt, "_table", None)
    for _ in range(2):
        give(ps)
        opt.step()
    opt.param_groups[0]["params"] = list(ps)
    give(ps)
    opt.step()
    assert len(Table.made) == 1 and len(Table.made[0].steps) == 5


@pytest.mark.parametrize("sources", [False, True])
def test_gradients_of_another_size_are_refused(make, sources):
    """A steady group whose parameter (and gradient source) changed size behind the optimizer's back."""
    ps = parameters()
    opt = make(ps)
    for _ in range(2):
        give(ps)
        opt.step()
    before = len(Table.made[0].steps)
    short = torch.ones(2)
    if sources:
        opt.set_grad_sources(ps, [ps[0].grad, short, ps[2].grad])
    else:
        class Short(Param):
            grad = short
        ps[1].__class__ = Short
        if fused_optim._native is not None:
            pytest.skip("the compiled module reads the real gradient, whose size torch checks")
    with pytest.raises(ValueError, match="size"):
        opt.step()
    assert len(Table.made[0].steps) == before


def test_feed_rows_have_to_be_the_groups_parameters(make):
    """A feed whose parameters have the group's ends but another one between them is not pushed into the group's table."""
    if fused_optim._native is None:
        pytest.skip("only the compiled module has feeds")
    ps = parameters()
    opt = make(ps)
    for _ in range(2):
        give(ps)
        opt.step()

    class Feed:
        pushed = 0

        def held(self):
            return 3

        def source_dtype(self):
            return fused_optim._lib.RG_F32

        def sources(self):
            return self.grads

        def forget_optim(self, handle):
            pass

        def push_sources_to_optim(self, handle, off, n):
            Feed.pushed += 1
            return True

    feed = Feed()
    other = Param(torch.zeros(6))
    feed.grads = [torch.ones_like(p.detach()) for p in ps]
    opt.set_grad_feed(feed, [ps[0], other, ps[2]])
    opt.step()
    assert Feed.pushed == 0 and Table.made[-1].steps[-1][2] == [feed.grads[0].data_ptr(), ps[1].grad.data_ptr(), feed.grads[2].data_ptr()]
    opt.set_grad_feed(feed, list(ps))
    opt.step()
    assert Feed.pushed == 1


def test_lists_know_their_objects():
    native = fused_optim._native
    if native is None:
        pytest.skip("the compiled module is switched off")
    ps = parameters()
    held = native.TensorList(ps)
    assert held.holds(ps) and held.holds(tuple(ps)) and held.holds([None] + ps + [None], 1) and not held.holds(ps, 1)
    assert not held.holds(ps[:2]) and not held.holds(ps[::-1]) and not held.holds(ps, 7) and not held.holds([])
    alias = ps[1].detach()                     # the same memory, another object
    assert not held.holds([ps[0], alias, ps[2]])
    assert native.TensorList([]).holds([])
    give(ps)
    grads = [p.grad for p in ps]
    assert held.addresses_of(grads, torch.float32) == held.grad_addresses(torch.float32)
    for bad in (grads[:2], [grads[0], None, grads[2]], [grads[0], torch.ones(5), grads[2]], [g.half() for g in grads],
                [grads[0], grads[1].to("meta"), grads[2]]):
        assert held.addresses_of(bad, torch.float32) is None


# ---------------------------------------------------------------- steps that are refused or fail

def _raise(error):
    def anything(*args, **kwargs):
        raise error
    return anything


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("earlier", [0, 1, 2])          # steps before: none, one (the next is a full one), two (a steady one)
@pytest.mark.parametrize("what", ["gradient type", "moments", "conversion", "table", "launch"])
def test_failed_steps_count_for_nothing(bits, earlier, what, monkeypatch):
    ps = parameters()
    opt = FusedAdam(ps, state_bits=bits)
    for _ in range(earlier):
        give(ps)
        opt.step()
    if earlier == 1:
        opt.invalidate_tables()
    give(ps)
    for _ in range(3):
        with monkeypatch.context() as m:
            if what == "gradient type":
                opt.set_grad_sources(ps, [p.grad.double() if i == 1 else p.grad for i, p in enumerate(ps)])
            elif what == "moments":
                if earlier:
                    pytest.skip("they are there")
                made = torch.zeros if bits == 8 else torch.zeros_like          # the second allocation fails
                calls = []
                m.setattr(torch, made.__name__, lambda *a, **k: made(*a, **k) if not calls.append(1) and len(calls) % 2 else _raise(MemoryError("none left"))())
            elif what == "conversion":
                opt.invalidate_tables()
                m.setattr(FusedAdam, "_settle_moments", _raise(MemoryError("none left")))
            elif what == "table":
                opt.invalidate_tables()
                m.setattr(fused_optim._lib, "OptimTable", _raise(MemoryError("none left")))
            else:
                m.setattr(Table, "refuse", ValueError("bad hyper-parameters"))
            with pytest.raises((MemoryError, ValueError, TypeError)):
                opt.step()
        opt.set_grad_sources([], [])
        assert sum(len(t.steps) for t in Table.made) == earlier
        for p in ps:
            state = opt.state.get(p, {})
            assert float(state.get("step", 0)) == earlier and ("exp_avg" in state) == ("exp_avg_sq" in state)
            assert what != "moments" or not state
    for step in range(earlier + 1, earlier + 4):
        give(ps)
        opt.step()
        assert Table.made[-1].steps[-1][0] == step and all(float(opt.state[p]["step"]) == step for p in ps)


def test_counts_of_parameters_that_join_late():
    ps = parameters()
    opt = FusedAdam(ps)
    for step in range(1, 6):
        give(ps if step > 2 else ps[:2])
        opt.step()
        assert [float(opt.state[p]["step"]) for p in ps[:2]] == [step] * 2
        assert step <= 2 or float(opt.state[ps[2]]["step"]) == step - 2
    counts = [s[0] for t in Table.made for s in t.steps]
    assert sorted(counts) == [1, 1, 2, 2, 3, 3, 4, 5]


def test_counts_given_as_numbers():
    ps = parameters()
    opt = FusedAdam(ps)
    for p in ps:
        opt.state[p].update(step=4, exp_avg=torch.zeros_like(p), exp_avg_sq=torch.zeros_like(p))
    give(ps)
    opt.step()
    assert Table.made[-1].steps[-1][0] == 5 and all(float(opt.state[p]["step"]) == 5 for p in ps)


@pytest.mark.parametrize("what", ["gradient type", "buffers", "table", "launch"])
def test_failed_first_step_leaves_no_momentum(what, monkeypatch):
    """Momentum starts as the gradient itself, not dampened: a first step that failed is still to come."""
    ps = parameters()
    opt = FusedSGD(ps, lr=0.1, momentum=0.9, dampening=0.5)
    give(ps)
    for _ in range(2):
        with monkeypatch.context() as m:
            if what == "gradient type":
                opt.set_grad_sources(ps, [p.grad.double() if i == 1 else p.grad for i, p in enumerate(ps)])
            elif what == "buffers":
                made, calls = torch.zeros_like, []
                m.setattr(torch, "zeros_like", lambda *a, **k: made(*a, **k) if not calls.append(1) and len(calls) < 2 else _raise(MemoryError("none left"))())
            elif what == "table":
                m.setattr(fused_optim._lib, "OptimTable", _raise(MemoryError("none left")))
            else:
                m.setattr(Table, "refuse", ValueError("bad hyper-parameters"))
            with pytest.raises((MemoryError, ValueError, TypeError)):
                opt.step()
        opt.set_grad_sources([], [])
        assert not any("momentum_buffer" in opt.state.get(p, {}) for p in ps)
    for first in (True, False, False):
        give(ps)
        opt.step()
        assert Table.made[-1].steps[-1][0] is first and len(Table.made[-1].steps[-1][1]) == 3
        assert list(Table.made[-1].state1) == [opt.state[p]["momentum_buffer"].data_ptr() for p in ps]


# ---------------------------------------------------------------- parameters whose memory changes

@pytest.mark.parametrize("size", [3, 4, 500])
def test_parameters_of_another_size_get_a_table_of_their_own(size):
    """``p.data`` replaced between steps: a table keeps the sizes that it was made with."""
    ps = parameters()
    opt = FusedSGD(ps, lr=0.1)
    for _ in range(2):
        give(ps)
        opt.step()
    ps[0].grad = None
    ps[0].data = torch.zeros(size)
    give(ps)
    opt.step()
    assert Table.made[-1].numels == [size, 6, 5] and Table.made[-1].steps[-1][1] == [p.data_ptr() for p in ps]
    assert len(Table.made) == (1 if size == 4 else 2)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("size", [3, 500])
def test_states_of_another_size_are_refused(bits, size):
    ps = parameters()
    opt = FusedAdam(ps, state_bits=bits)
    for _ in range(2):
        give(ps)
        opt.step()
    ps[0].grad = None
    ps[0].data = torch.zeros(size)
    give(ps)
    with pytest.raises(ValueError, match="elements"):
        opt.step()
    assert sum(len(t.steps) for t in Table.made) == 2 and float(opt.state[ps[0]]["step"]) == 2


@pytest.mark.parametrize("name,wrong", [("exp_avg", lambda t: t.double()), ("exp_avg", lambda t: t[:3]), ("exp_avg_sq", lambda t: t.to("meta")),
                                        ("exp_avg_sq", lambda t: t.repeat_interleave(2)[::2])])
def test_states_that_do_not_fit_are_refused(name, wrong):
    ps = parameters()
    opt = FusedAdam(ps)
    give(ps)
    opt.step()
    opt.state[ps[0]][name] = wrong(opt.state[ps[0]][name])
    opt.invalidate_tables()
    with pytest.raises(ValueError, match="elements"):
        opt.step()
    assert float(opt.state[ps[0]]["step"]) == 1


@pytest.mark.parametrize("make", [lambda ps: FusedAdam(ps), lambda ps: FusedSGD(ps, momentum=0.9)], ids=["adam", "sgd"])
def test_loaded_states_in_another_memory_order(make):
    ps = [Param(torch.zeros(2, 3, 4, 5))]
    opt = make(ps)
    for _ in range(2):
        give(ps)
        opt.step()
    sd = opt.state_dict()
    want = {}
    for name, value in sd["state"][0].items():
        if torch.is_tensor(value) and value.dim() == 4:
            want[name] = torch.arange(120.0).view(2, 3, 4, 5)
            sd["state"][0][name] = want[name].to(memory_format=torch.channels_last)
    assert want
    opt.load_state_dict(sd)
    for name, value in want.items():
        assert opt.state[ps[0]][name].is_contiguous() and torch.equal(opt.state[ps[0]][name], value)
    opt.step()
    assert list(Table.made[-1].state1) == [opt.state[ps[0]][list(want)[0]].data_ptr()]


# ---------------------------------------------------------------- the step count on the device

@pytest.fixture
def clock(monkeypatch):
    """Counts what the clock's kernel and the step that reads it are told."""
    ticks = []
    monkeypatch.setattr(fused_optim._lib, "adam_clock_advance", lambda *args: ticks.append(args))

    def adam_step_clocked(self, clock_ptr, lr, beta1, beta2, eps, weight_decay, **kw):
        if not (eps >= 0 and weight_decay >= 0):
            raise ValueError("bad hyper-parameters")
        self.steps.append((len(ticks), list(self.params), list(self.grads)))
    monkeypatch.setattr(Table, "adam_step_clocked", adam_step_clocked, raising=False)
    return ticks


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [dict(eps=-1.0), dict(weight_decay=-0.1), dict(eps=float("nan"))])
def test_refused_capturable_step_does_not_advance_the_clock(clock, bits, bad):
    ps = parameters()
    opt = FusedAdam(ps, capturable=True, state_bits=bits)
    give(ps)
    group = opt.param_groups[0]
    good = {k: group[k] for k in bad}
    for steps in (0, 1, 2):                         # before the first step, and before a steady one
        group.update(bad)
        with pytest.raises(ValueError, match="hyper-parameters"):
            opt.step()
        assert len(clock) == steps
        group.update(good)
        opt.step()


@pytest.mark.parametrize("bad,match", [(lambda g: g.repeat_interleave(2)[::2], "contiguous"), (lambda g: g[:1].expand(6), "contiguous"),
                                       (lambda g: g[:5], "size"), (lambda g: g.double(), "dtype")])
def test_capturable_steps_check_gradients_every_time(clock, bad, match):
    ps = parameters()
    opt = FusedAdam(ps, capturable=True)
    for _ in range(3):
        give(ps)
        opt.step()
    opt.set_grad_sources(ps, [bad(p.grad) if i == 1 else p.grad for i, p in enumerate(ps)])
    with pytest.raises(ValueError, match=match):
        opt.step()
    assert len(clock) == 3
    opt.set_grad_sources([], [])
    opt.step()
    assert len(clock) == 4 and Table.made[-1].steps[-1][0] == 4


@pytest.mark.parametrize("size", [3, 6, 500])
def test_capturable_group_with_another_parameter(clock, size):
    ps = parameters()
    opt = FusedAdam(ps, capturable=True)
    for _ in range(2):
        give(ps)
        opt.step()
    group = opt.param_groups[0]["params"]
    old, new = group[1], Param(torch.zeros(size))
    group[1] = new
    new.grad = torch.ones(size)
    with pytest.raises(RuntimeError, match="without moments"):
        opt.step()
    opt.state[new] = {"step": opt.state[old]["step"], "exp_avg": torch.zeros(size), "exp_avg_sq": torch.zeros(size)}
    opt.step()
    assert Table.made[-1].numels == [4, size, 5] and Table.made[-1].steps[-1][1] == [p.data_ptr() for p in group]
    assert Table.made[0].numels == [4, 6, 5]


def test_differing_counts_leave_the_state_alone(clock):
    ps = parameters()
    opt = FusedAdam(ps, capturable=True)
    opt.state[ps[0]] = {"step": torch.tensor(3.0), "exp_avg": torch.zeros(4), "exp_avg_sq": torch.zeros(4)}
    give(ps)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="counts differ"):
            opt.step()
        assert list(opt.state) == [ps[0]] and not Table.made


# ---------------------------------------------------------------- state dicts and copies

def _convert_on_the_host(held, entries, to_codes):
    """Stands for the conversion kernels: what it writes is recognised by the tests."""
    for st, entry in zip(held, entries):
        for name in ("exp_avg", "exp_avg_sq"):
            if to_codes:
                st[name + "_scale"].fill_(2.0)
            else:
                entry[name].fill_(0.25 if name == "exp_avg" else 0.5)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("prepend", [False, True])
def test_state_dict_hooks_see_float32_moments(bits, prepend, monkeypatch):
    monkeypatch.setattr(FusedAdam, "_convert_moments", staticmethod(_convert_on_the_host))
    ps = parameters()
    opt = FusedAdam(ps, state_bits=bits)
    give(ps)
    opt.step()
    seen = []

    def replace(optimizer, sd):
        assert optimizer is opt
        seen.append({i: sorted(st) for i, st in sd["state"].items()})
        assert all(st[k].dtype == torch.float32 for st in sd["state"].values() for k in ("exp_avg", "exp_avg_sq"))
        sd["state"][1] = dict(sd["state"][1], exp_avg=torch.full((6,), 7.0))

    handle = opt.register_state_dict_post_hook(replace, prepend=prepend)
    sd = opt.state_dict()
    assert seen == [{i: ["exp_avg", "exp_avg_sq", "step"] for i in range(3)}]
    assert sd["state"][1]["exp_avg"].tolist() == [7.0] * 6 and sorted(sd["state"][0]) == ["exp_avg", "exp_avg_sq", "step"]
    if bits == 8:
        assert sd["state"][0]["exp_avg"].tolist() == [0.25] * 4 and opt.state[ps[0]]["exp_avg"].dtype == torch.float8_e4m3fn
    handle.remove()
    assert opt.state_dict()["state"][1]["exp_avg"].tolist() == [0.25 if bits == 8 else 0.0] * 6


@pytest.mark.parametrize("make", [lambda ps: FusedAdam(ps, lr=0.5), lambda ps: FusedAdamW(ps, state_bits=8), lambda ps: FusedAdam(ps, capturable=True),
                                  lambda ps: FusedSGD(ps, momentum=0.9)], ids=["adam", "adamw8", "capturable", "sgd"])
@pytest.mark.parametrize("pickled", [False, True])
def test_copies_are_optimizers_of_their_own(make, pickled, clock, monkeypatch):
    monkeypatch.setattr(FusedAdam, "_convert_moments", staticmethod(_convert_on_the_host))
    ps = parameters()
    opt = make(ps)
    for _ in range(2):
        give(ps)
        opt.step()
    if pickled:
        file = io.BytesIO()
        torch.save(opt, file)
        file.seek(0)
        other = torch.load(file, weights_only=False)       # written here
    else:
        other = copy.deepcopy(opt)
    qs = other.param_groups[0]["params"]
    assert type(other) is type(opt) and all(q is not p for p, q in zip(ps, qs))
    a, b = opt.state_dict(), other.state_dict()
    assert a["param_groups"] == b["param_groups"] and a["state"].keys() == b["state"].keys()
    for i, st in a["state"].items():
        assert st.keys() == b["state"][i].keys() and all(torch.equal(v, b["state"][i][k]) for k, v in st.items())
    if getattr(opt, "state_bits", 32) == 8:
        assert other.state_bits == 8 and other.state_buffers()["exp_avg"].data_ptr() == other.state[qs[0]]["exp_avg"].data_ptr()
        assert len(other._optimizer_state_dict_post_hooks) == 1
    launches = sum(len(t.steps) for t in Table.made)
    qs = [Param(q.detach()) for q in qs] if pickled else qs       # (a saved parameter is a plain one, which is on the CPU)
    if pickled:
        for old, q in zip(other.param_groups[0]["params"], qs):
            other.state[q] = other.state.pop(old)
        other.param_groups[0]["params"] = qs
    give(qs)
    other.step()
    assert sum(len(t.steps) for t in Table.made) == launches + 1
    assert Table.made[-1].params == [q.data_ptr() for q in qs]
    if isinstance(opt, FusedAdam) and not opt.capturable:
        assert Table.made[-1].steps[-1][0] == 3 and float(opt.state[ps[0]]["step"]) == 2
    other.load_state_dict(opt.state_dict())


@pytest.mark.parametrize("name", ["exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"])
def test_state_buffers_are_where_the_states_lie(name):
    ps = parameters((4, 0, 300))
    opt = FusedAdam(ps, state_bits=8)
    give(ps)
    opt.step()
    assert opt.state_buffers()[name].data_ptr() == opt.state[ps[0]][name].data_ptr()
    opt.state[ps[2]][name] = opt.state[ps[2]][name].clone()
    with pytest.raises(RuntimeError, match=f"{name} has been given memory"):
        opt.state_buffers()


def test_moved_8_bit_states_get_another_table():
    """Without ``invalidate_tables``: the states' addresses are compared whenever a step looks at every parameter."""
    ps = parameters()
    opt = FusedAdam(ps, state_bits=8)
    for _ in range(2):
        give(ps)
        opt.step()
    opt.state[ps[1]]["exp_avg_sq_scale"] = opt.state[ps[1]]["exp_avg_sq_scale"].clone()
    opt._steady.clear()
    for _ in range(2):
        opt.step()
    assert len(Table.made) == 2 and [len(t.steps) for t in Table.made] == [2, 2]
    assert list(Table.made[1].scales2) == [opt.state[p]["exp_avg_sq_scale"].data_ptr() for p in ps]


@pytest.mark.parametrize("momentum", [0.0, 0.9])
def test_sgd_state_dict_names_every_stepped_parameter(momentum):
    ps = parameters()
    opt = FusedSGD(ps, lr=0.1, momentum=momentum)
    give(ps[:2])
    opt.step()
    assert [sorted(st) for st in opt.state_dict()["state"].values()] == [["momentum_buffer"] if momentum else []] * 2


def test_a_parameter_resized_between_the_ends_leaves_the_short_path():
    """Its gradient is then of another size than the table's row, whatever the parameter's size is by now."""
    ps = parameters()
    opt = FusedSGD(ps, lr=0.1)
    for _ in range(3):
        give(ps)
        opt.step()
    ps[1].grad = None
    ps[1].data = torch.zeros(9)
    for _ in range(3):
        give(ps)
        opt.step()
        assert Table.made[-1].numels == [4, 9, 5] and Table.made[-1].steps[-1][1:] == ([p.data_ptr() for p in ps], [p.grad.data_ptr() for p in ps])
    assert len(Table.made) == 2 and [len(t.steps) for t in Table.made] == [3, 3]


def test_addresses_of_the_very_list():
    native = fused_optim._native
    if native is None:
        pytest.skip("the compiled module is switched off")
    ps = parameters()
    held = native.TensorList(ps)
    give(ps)
    want = held.grad_addresses(torch.float32)
    assert want is not None and held.grad_addresses_in(ps, torch.float32) == want == held.grad_addresses_in(tuple(ps), torch.float32)
    for other in (ps + ps[:1], ps[:2], ps[::-1], [ps[0], ps[1].detach(), ps[2]], []):
        assert held.grad_addresses_in(other, torch.float32) is None
    assert held.grad_addresses_in(ps, torch.float16) is None
