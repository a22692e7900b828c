"""What rounding to 8 bits does to Adam's moments over a run, against the recurrences in float64, and conversions of the
largest tensors.

With q the distance of the two e4m3 numbers around a stored root r (q / r lies between 1/16 and 1/8) and D = E|g^2 / v - 1|, a step moves
the root by Delta = r (1 - beta2) / 2 * |g^2 / v - 1| on average, and the dither adds a variance of Delta q (for Delta much smaller than q; here
it is at most a few thousandths of r).  The next step squares the root, so v gains that variance in every step and forgets the share
1 - beta2 of it: v comes out too large by the factor 1 + q / (2 r) D.  The root's own error is forgotten at the same rate, so its
variance is Delta q / (1 - beta2^2), a relative error of sqrt(q / (4 r) D) rms.  For normal gradients D = 4 phi(1) = 0.968: v is 3.0 to
6.1 % too large and a root off by 12.3 to 17.4 %.  The bounds below leave 1 % for the sample (2^16 elements whose v is off by some
30 % each: 0.12 % if they were independent) and for what 4 horizons of beta2 have not reached yet (2 % of the figure)."""
import numpy as np
import pytest
import torch

from oracle import state8 as oracle
from rannc_amd.fused_optim import FusedAdam, FusedAdamW
from rannc_amd.multi_tensor import State8Plan, allocate_state8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_moments_over_four_horizons():
    """4,000 steps with other gradients in each, sizes of their own for every element (normal, their logarithm too)."""
    n, beta1, beta2 = 1 << 16, 0.9, 0.999
    gen = torch.Generator(device=DEV).manual_seed(3)
    size = torch.randn(n, generator=gen, device=DEV).exp()
    p = torch.zeros(n, device=DEV)
    opt = FusedAdam([p], lr=0.0, betas=(beta1, beta2), state_bits=8)
    p.grad = torch.empty(n, device=DEV)
    m, v = (torch.zeros(n, dtype=torch.float64, device=DEV) for _ in range(2))
    for _ in range(4000):
        torch.randn(n, generator=gen, device=DEV, out=p.grad)
        p.grad.mul_(size)
        opt.step()
        g = p.grad.double()
        m.mul_(beta1).add_(g, alpha=1 - beta1)
        v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    st = opt.state_dict()["state"][0]
    ratio = st["exp_avg_sq"].double() / v
    bias, rms = float(ratio.mean()) - 1, float((ratio.sqrt() - 1).square().mean().sqrt())
    print(f"second moment {bias:+.4f}, root rms {rms:.4f}")
    assert 0.030 - 0.01 <= bias <= 0.061 + 0.01, bias
    assert 0.123 - 0.01 <= rms <= 0.174 + 0.01, rms
    # the first moment enters linearly, so its error has no mean: two e4m3 numbers around it are at most 1/8 apart, which a step's
    # dither turns into at most 1/16 of |m| rms, times 1 / sqrt(1 - beta1^2) for the steps before, and |m| is 0.23 sqrt(v) rms here
    # (sqrt((1 - beta1) / (1 + beta1))): 0.033 sqrt(v) rms, 0.00013 for the mean of 2^16 - with five times that allowed
    off = (st["exp_avg"].double() - m) / v.sqrt()
    assert float(off.square().mean().sqrt()) <= 0.033 and abs(float(off.mean())) <= 5 * 0.00013


def test_parameters_move_as_with_32_bits():
    """2,000 steps with the same gradients (a mean of their own for every element, and noise) in 8 and in 32 bits: an element's steps
    differ by what its root is off, at most 17.4 % rms, so the two displacements form an angle of cosine 0.985 or more and their lengths
    agree within 3 % for the bias (half of v's) and 3 % (0.174^2) for the spread."""
    n = 1 << 14
    gen = torch.Generator(device=DEV).manual_seed(4)
    mean = torch.randn(n, generator=gen, device=DEV)
    ps = [torch.zeros(n, device=DEV) for _ in range(2)]
    opts = [FusedAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits) for p, bits in zip(ps, (8, 32))]
    for _ in range(2000):
        g = torch.randn(n, generator=gen, device=DEV) + mean
        for p, opt in zip(ps, opts):
            p.grad = g
            opt.step()
    a, b = (p.double() for p in ps)
    cosine, length = float(a @ b / (a.norm() * b.norm())), float(a.norm() / b.norm())
    print(f"cosine {cosine:.5f}, length {length:.4f}")
    assert cosine >= 0.985 and abs(length - 1) <= 0.061, (cosine, length)


def test_states_that_moved_without_a_word():
    """A state tensor replaced between steps, nothing invalidated, and the next step looks at every parameter: same bits as unmoved."""
    runs = []
    for move in (False, True):
        gen = torch.Generator().manual_seed(5)
        ps = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in (700, 3, 5000)]
        opt = FusedAdamW(ps, lr=1e-2, state_bits=8)
        for step in range(5):
            for p in ps:
                p.grad = torch.randn(p.shape, generator=gen).to(DEV)
            if step == 3:
                if move:
                    for name in ("exp_avg", "exp_avg_sq_scale"):
                        old = opt.state[ps[2]][name]
                        opt.state[ps[2]][name] = old.clone()
                        old.view(torch.uint8).fill_(0x33)
                    with pytest.raises(RuntimeError, match="memory of its own"):
                        opt.state_buffers()
                opt._steady.clear()
            opt.step()
        runs.append((ps, opt))
    for p, q in zip(runs[0][0], runs[1][0]):
        assert torch.equal(p, q)
        a, b = runs[0][1].state[p], runs[1][1].state[q]
        assert all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in a if k != "step")


def test_conversions_beyond_two_to_the_31_elements_are_lossless():
    """2^31 + 4099 numbers to codes, back, and to codes again over other bytes: the same codes and scales everywhere, and the oracle's
    around the places where 31 bits end; nothing is written behind the last element's."""
    n = 2 ** 31 + 4099
    gen = torch.Generator(device=DEV).manual_seed(9)
    values = torch.empty(n, device=DEV)
    part = 2 ** 28
    for a in range(0, n, part):
        values[a:a + part].normal_(generator=gen)
    like = [values]
    codes, scales, all_codes, all_scales = allocate_state8(like)
    tail = all_codes.view(torch.uint8)[n:]
    tail.fill_(0x5A)
    plan = State8Plan([values], codes, scales)
    plan.quantize()
    for a, b in [(0, 2048), (2 ** 30 - 256, 2 ** 30 + 512), (2 ** 31 - 1024, 2 ** 31 + 1024), (n - 4099 - 1024, n)]:
        a -= a % 256
        want, s, tie = oracle.quantize(values[a:b].double().cpu().numpy(), False)
        got = codes[0][a:b].view(torch.uint8).cpu().numpy()
        assert (got == want)[tie > 48 * oracle.EPS].all(), a
        assert np.array_equal(scales[0][a // 256:a // 256 + s.size].double().cpu().numpy(), s), a
    kept_codes, kept_scales = codes[0].view(torch.uint8).clone(), scales[0].clone()
    plan.dequantize()
    codes[0].view(torch.uint8).fill_(0x11)
    scales[0].fill_(-1.0)
    plan.quantize()
    assert torch.equal(scales[0], kept_scales)
    for a in range(0, n, part):
        assert torch.equal(codes[0][a:a + part].view(torch.uint8), kept_codes[a:a + part]), a
    assert bool((tail == 0x5A).all())
    plan.close()
