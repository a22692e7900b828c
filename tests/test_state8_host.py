"""Optimizer states in 8 bits without a GPU: the oracle against torch's float8 conversion and hand-worked values, and the
library's refusals, none of which reaches a device."""
import numpy as np
import pytest
import torch

from oracle import state8 as oracle
from rannc_amd import _lib
from rannc_amd.fused_optim import FusedAdam, FusedAdamW
from rannc_amd.multi_tensor import State8Plan, allocate_state8


def test_grid_is_e4m3():
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(oracle.GRID, want)


def test_nearest_rounding_matches_torch():
    rng = np.random.default_rng(0)
    # every block's largest is 256, so that 256 x / s is x itself; midpoints between neighbours among the numbers
    x = np.clip(rng.standard_normal(256 * 40) * np.exp(rng.standard_normal(256 * 40) * 4), -256, 256).astype(np.float32)
    x[1:120] = (oracle.GRID[:119] + oracle.GRID[1:120]) / 2
    x[::256] = 256
    codes, scales, _ = oracle.quantize(x, root=False)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert scales.tolist() == [256.0] * 40 and np.array_equal(codes, want)


def test_hand_worked_block():
    # scale 2: y = 128 x.  0.5 -> 64 (code 0x68), 1/192 -> 0.6667 between 0.625 and 0.6875, -2 -> -256, 1e-9 -> 0
    x = np.array([0.5, 1 / 192, -2.0, 1e-9])
    codes, scales, _ = oracle.quantize(x, root=False)
    assert scales.tolist() == [2.0]
    assert oracle.values_of(codes).tolist() == [64.0, 0.6875, -256.0, 0.0]
    assert oracle.read_back(codes, scales).tolist() == [0.5, 0.6875 / 128, -2.0, 0.0]
    # the same as second moments: roots 0.7071, 0.0722, and a root that is small against the largest keeps e4m3's smallest
    codes, scales, _ = oracle.quantize(np.array([0.25, 0.0, 1e-30]), root=True)
    assert scales.tolist() == [0.5] and oracle.values_of(codes).tolist() == [256.0, 0.0, 2.0 ** -9]


def test_blocks_without_numbers():
    for x, want in ((np.full(3, 2.0 ** -101), 0.0), (np.array([1.0, np.inf]), np.nan), (np.array([np.nan, 1.0]), np.nan),
                    (np.zeros(5), 0.0)):
        codes, scales, _ = oracle.quantize(x, root=False)
        assert not (codes & 0x7F).any() and np.array_equal(scales, [want], equal_nan=True)


def test_dither_is_right_on_average():
    """Over the steps the dither's numbers fill the range evenly: rounding up happens as often as the part says."""
    steps = np.arange(1, 4097, dtype=np.uint64)
    for place in (0, 7, 12345):
        for factor in (oracle.FIRST, oracle.ROOT):
            u = ((np.uint64(place * oracle.PLACE) + steps * np.uint64(factor)) & np.uint64(0xFFFFFFFF)).astype(np.float64) / 2.0 ** 32
            for part in (0.01, 0.3, 0.9):
                # an additive recurrence with these fractions strays by less than a few counts in 4096
                assert abs((part + u >= 1).sum() - part * 4096) <= 12


def test_first_step_by_hand():
    """From zero states Adam's first step is lr in the gradient's direction, whatever its size."""
    g = np.array([3.0, -0.25, 0.0, 1e-3])
    zero, s = np.zeros(4, dtype=np.uint8), np.zeros(1)
    out = oracle.adam_step(np.ones(4), g, zero, s, zero, s, 1, 0.1, 0.9, 0.999, 0.0, 0.0)
    np.testing.assert_allclose(out["p"][[0, 1, 3]], [0.9, 1.1, 0.9], rtol=1e-12)
    assert np.isnan(out["p"][2])                     # 0 / 0 with eps = 0, as torch.optim.Adam has it
    np.testing.assert_allclose(out["scales1"], [0.3], rtol=1e-12)
    np.testing.assert_allclose(out["scales2"], [3.0 * 0.001 ** 0.5], rtol=1e-12)


# ---------------------------------------------------------------- refusals

def test_num_scales():
    assert [_lib.state8_num_scales(n) for n in (0, 1, 255, 256, 257, 2 ** 33 + 1)] == [0, 1, 1, 1, 2, 2 ** 25 + 1]
    with pytest.raises(ValueError):
        _lib.state8_num_scales(-1)


def test_table_refusals_come_before_the_device():
    ok = dict(device=0, codes=[0x1000], scales=[0x2000], values=[0x3000], numels=[10], roots=[False])
    for bad, match in ((dict(codes=[0x1001]), "aligned"), (dict(scales=[0x2002]), "aligned"), (dict(values=[0x3002]), "aligned"),
                       (dict(codes=[0]), "lacks"), (dict(scales=[0]), "lacks"), (dict(values=[0]), "lacks"),
                       (dict(numels=[-1]), "elements"), (dict(numels=[2 ** 45]), "elements"),
                       (dict(codes=[]), "length")):
        with pytest.raises(ValueError, match=match):
            _lib.State8Table(**{**ok, **bad})


def test_optim_table_refusals_come_before_the_device():
    def make(**bad):
        a = dict(device=0, params=[0x1000], grads=[0x2000], state1=[0x3000], state2=[0x4000], copies=None, numels=[10],
                 grad_dtypes=[_lib.RG_F32], scales1=[0x5000], scales2=[0x6000])
        a.update(bad)
        return _lib.OptimTable(**a)
    for bad, match in ((dict(state1=[0x3001]), "aligned"), (dict(state2=[0x4002]), "aligned"), (dict(scales1=[0x5002]), "aligned"),
                       (dict(scales2=[0]), "scales"), (dict(scales1=None), "bad arguments"), (dict(scales2=None), "bad arguments"),
                       (dict(state1=None), "bad arguments"), (dict(state2=[0]), "state pointer"), (dict(params=[0x1002]), "aligned"),
                       (dict(grads=[0]), "gradient"), (dict(numels=[-1]), "bad size"), (dict(numels=[2 ** 45]), "bad size"),
                       (dict(grad_dtypes=[7]), "dtype")):
        with pytest.raises(ValueError, match=match):
            make(**bad)


def test_empty_tables_work_without_a_device():
    t = _lib.State8Table(0, [], [], [], [], [])
    t.quantize()
    t.dequantize()
    t.close()
    assert not t.is_open()
    with pytest.raises(ValueError, match="null"):
        t.quantize()
    o = _lib.OptimTable(0, [], [], [], [], None, [], [], None, [], [])
    o.adam_step(1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    with pytest.raises(ValueError, match="8-bit"):
        o.sgd_step(1e-3)
    with pytest.raises(ValueError, match="stay where they are"):
        o.update_pointers(state1=[])
    with pytest.raises(ValueError, match="hyper-parameters"):
        o.adam_step(1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    o.close()


def test_plan_refuses_what_is_not_on_a_gpu():
    v = torch.zeros(10)
    with pytest.raises(ValueError, match="GPU"):
        State8Plan([v], [torch.zeros(10, dtype=torch.float8_e4m3fn)], [torch.zeros(1)])
    with pytest.raises(ValueError, match="length"):
        State8Plan([v], [], [torch.zeros(1)])
    with pytest.raises(ValueError, match="length"):
        State8Plan([v], [torch.zeros(10, dtype=torch.float8_e4m3fn)], [torch.zeros(1)], root=[True, False])


def test_allocation_layout():
    codes, scales, all_codes, all_scales = allocate_state8([torch.zeros(3, 100), torch.zeros(0), torch.zeros(256), torch.zeros(1)])
    assert [tuple(c.shape) for c in codes] == [(3, 100), (0,), (256,), (1,)] and [s.numel() for s in scales] == [2, 0, 1, 1]
    assert all_codes.numel() == 1024 and all_codes.dtype == torch.float8_e4m3fn and all_scales.numel() == 4
    assert [c.storage_offset() for c in codes] == [0, 512, 512, 768] and [s.storage_offset() for s in scales] == [0, 2, 2, 3]
    with pytest.raises(ValueError, match="no tensors"):
        allocate_state8([])


@pytest.mark.parametrize("cls", [FusedAdam, FusedAdamW])
def test_optimizer_arguments(cls):
    p = [torch.zeros(4)]
    for bits in (4, 16, "8", None):
        with pytest.raises(ValueError, match="state_bits"):
            cls(p, state_bits=bits)
    assert cls(p).state_bits == 32
    opt = cls(p, state_bits=8)
    with pytest.raises(RuntimeError, match="not there yet"):
        opt.state_buffers()
    with pytest.raises(RuntimeError, match="32 bits"):
        cls(p).state_buffers()
    assert opt.state_dict()["state"] == {}
    p[0].grad = torch.zeros(4)
    with pytest.raises(ValueError, match="GPU"):
        opt.step()


@pytest.mark.parametrize("bits", [8, 32])
def test_raw_codes_are_not_loaded(bits):
    p = [torch.zeros(4)]
    opt = FusedAdam(p, state_bits=bits)
    sd = opt.state_dict()
    codes, scales, _, _ = allocate_state8(p)
    sd["state"] = {0: {"step": torch.tensor(1.0), "exp_avg": codes[0], "exp_avg_scale": scales[0], "exp_avg_sq": codes[0], "exp_avg_sq_scale": scales[0]}}
    with pytest.raises(ValueError, match="8-bit codes"):
        opt.load_state_dict(sd)
    assert not opt.state
