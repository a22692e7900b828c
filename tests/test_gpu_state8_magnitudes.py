"""Adam steps with 8-bit states at the ends of fp32's range, against the float64 oracle (tolerances as in test_gpu_state8.py)."""
import numpy as np
import pytest
import torch

from oracle import state8 as oracle
from rannc_amd.multi_tensor import State8Plan, allocate_state8
from tests.test_gpu_state8 import KW, Step, launch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def small_state(rng, exponents, zero_gradients):
    """``special`` for ``Step``: block b of tensor 0 has its largest first moment and root at 2^exponents[b], the rest spread over the
    17 octaves below, and gradients of the roots' size or none."""
    def special(t, g):
        n = t.sizes[0]
        top = 2.0 ** np.repeat(np.asarray(exponents, dtype=np.float64), 256)[:n]
        spread = 2.0 ** -rng.uniform(0, 17, n)
        spread[::256] = 1.0
        c1, s1, _ = oracle.quantize(top * spread * np.where(rng.random(n) < 0.5, -1, 1) * 0.5, False)
        c2, s2, _ = oracle.quantize((top * spread) ** 2, True)
        t.state[0] = [c1, s1.astype(np.float32), c2, s2.astype(np.float32)]
        g[0][:] = torch.from_numpy((0.0 if zero_gradients else 10.0) * top * spread * rng.standard_normal(n))
    return special


@pytest.mark.parametrize("zero_gradients,beta2", [(True, 0.999), (True, 0.9), (False, 0.999), (False, 0.9), (False, 0.0)])
def test_roots_below_the_square_root_of_fp32s_smallest_number(zero_gradients, beta2):
    """Stored roots reach down to 2^-117, their squares to 2^-234.  Blocks whose largest is at 2^-99 (the square of every root is
    no fp32 number, times 2^50 or not) up to 2^-60 (some squares times 2^50 lie below the quick square root's range, some above).
    Exponents of the oracle have no such end, and its bounds of the error are relative ones; eps = 0 shows the root in the parameter."""
    exponents = list(range(-97, -58))
    rng = np.random.default_rng(11)
    kw = dict(lr=1.0, beta1=0.9, beta2=beta2, eps=0.0, weight_decay=0.0)
    t = Step([256 * len(exponents) - 100, 300], "f32", None, special=small_state(rng, exponents, zero_gradients))
    old = t.state[0][2] != 0
    launch(t, 3, kw)
    # sums that cancel in m leave fewer of the codes to the bounds; zeros' codes are as sure as can be
    t.compare(3, kw, sure_share=0.98)
    codes = t.dc2[0].cpu().numpy()
    if beta2 > 0:
        assert old.any() and (codes[old] != 0).all()      # a root that is not zero never gets the code of zero
    t.table.close()


def test_a_small_root_decays_without_vanishing():
    """Many steps without a gradient: the block's roots keep their places until its largest falls below 2^-100."""
    rng = np.random.default_rng(12)
    t = Step([256], "f32", None, special=small_state(rng, [-90], True))
    kw = dict(KW, beta2=0.5, weight_decay=0.0)
    assert (t.state[0][2] != 0).all()
    for step in range(1, 24):
        launch(t, step, kw)
        s = float(t.ds2[0].cpu()[0])
        want = 2.0 ** (-90 - step / 2)
        if want > 2.0 ** -100 * 1.01:
            # the largest is rounded (half a step of fp32) in the square and in the root at every step
            assert abs(s / want - 1) <= 4 * step * oracle.EPS and bool((t.dc2[0] != 0).all()), step
        elif want < 2.0 ** -100 * 0.99:
            assert s == 0.0 and not t.dc2[0].any(), step
    t.table.close()


@pytest.mark.parametrize("mantissa", [1.5, 1.75, 1.0 + 2.0 ** -23, 1.6180339887, 2.0 - 2.0 ** -23])
def test_codes_do_not_depend_on_the_power_of_two(mantissa):
    """The same block times 2^e, from 2^-100 up to fp32's largest numbers, with halfway numbers among its elements: the reciprocal of
    the scale has to keep its 24 bits everywhere."""
    grid = oracle.GRID[:oracle.GRID.searchsorted(256.0) + 1]
    y = np.concatenate([[256.0], (grid[1:] + grid[:-1]) / 2, grid, -grid[100:114]])[:256]
    mantissa = float(np.float32(mantissa))
    block = (y / 256 * mantissa).astype(np.float32)            # numbers from 2^-18 to 2: no exponent below makes them subnormal,
    exponents = [0, 127, 126, 125, 124, 60, -60, -99]          # but the last one's smallest
    x = np.concatenate([np.ldexp(block, e) for e in exponents])
    v = torch.from_numpy(x).to(DEV)
    codes, scales, _, _ = allocate_state8([v])
    plan = State8Plan([v], codes, scales)
    plan.quantize()
    assert scales[0].tolist() == [float(np.ldexp(mantissa, e)) for e in exponents]
    got = codes[0].view(torch.uint8).cpu().numpy().reshape(len(exponents), 256)
    assert y.size == 256 and (got == got[0]).all(), np.argwhere(got != got[0])
    if mantissa == 1.5:             # the reciprocal's rounding moves no halfway number here: ties to even, as the oracle has them
        assert np.array_equal(got[0], oracle.quantize(block.astype(np.float64), False)[0])
    plan.close()


def test_square_root_of_every_number():
    """All fp32 numbers from the smallest up to 2^78, one to a block of equal ones (the scale is then the root, and no zero sends the
    block another way): the quick square root is correctly rounded over its whole range, 2^-100 to infinity after the factor of
    2^50.  The root in float64 rounds to fp32 as the exact one does (53 >= 2 * 24 + 2)."""
    count = 1 << 20
    values = torch.empty(count * 256, device=DEV)
    codes, scales, _, _ = allocate_state8([values])
    plan = State8Plan([values], codes, scales, root=True)
    end = (127 + 78) << 23
    offsets = torch.arange(count, dtype=torch.int32, device=DEV)
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    for first in range(1, end, count):
        bits = torch.clamp(offsets + first, max=end - 1)
        x = bits.view(torch.float32)
        values.view(count, 256).copy_(x.unsqueeze(1).expand(count, 256))
        plan.quantize()
        # subnormal numbers by their bits: no conversion flushes them
        exact = torch.where(bits < 1 << 23, bits.double() * 2.0 ** -149, x.double())
        want = exact.sqrt().float()
        wrong += (scales[0].view(torch.int32) != want.view(torch.int32)).sum()
    assert int(wrong) == 0
    assert bool((codes[0].view(torch.uint8) == 0x78).all())          # 256: the largest of its block
    plan.close()
