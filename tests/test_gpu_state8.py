"""Optimizer states in 8 bits on the GPU: the Adam step and the two conversions against the float64 oracle.

Tolerances.  The parameter must lie within the error bound that the oracle derives element by element from the fp32
operations of the step (half a step of fp32 each); scales within the bound of the element that sets them.  A code has
to be the oracle's wherever that bound cannot change which neighbour the dither picks, and one of its neighbours elsewhere."""
import math

import numpy as np
import pytest
import torch

from oracle import state8 as oracle
from rannc_amd import _lib
from rannc_amd.fused_optim import FusedAdam, FusedAdamW
from rannc_amd.multi_tensor import State8Plan, TensorPlan, allocate_state8, stream_handle
from tests.helpers import TORCH_DTYPE, assert_bits_equal, place_in_arena

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = [1, 3, 4, 5, 31, 255, 256, 257, 511, 768, 1023, 1024, 1025, 4095, 4096, 4097, 16383, 16384, 16385, 16384 + 255, 40961]
GUARD = 64           # bytes before and after every buffer that a kernel writes


def guarded(tensors, lead):
    """Copies of CPU tensors on the device, each ``lead`` elements into a buffer of its own whose other bytes are 0x5A;
    returns the views and a check that those bytes are still there."""
    views, buffers = [], []
    for t in tensors:
        size = t.element_size()
        raw = torch.full((2 * GUARD + (lead + t.numel()) * size,), 0x5A, dtype=torch.uint8, device=DEV)
        start = GUARD + lead * size
        v = raw[start:start + t.numel() * size].view(t.dtype).view(t.shape)
        v.copy_(t)
        views.append(v)
        buffers.append((raw, start, t.numel() * size))

    def check(what):
        for i, (raw, start, n) in enumerate(buffers):
            outside = torch.cat([raw[:start], raw[start + n:]])
            assert bool((outside == 0x5A).all()), f"{what}[{i}]: bytes outside the tensor were written"
    return views, check


class Step:
    """One table over ``sizes`` with known states, stepped on the device and by the oracle."""

    def __init__(self, sizes, grad="f32", copy=None, lead=0, seed=0, grad_std=1e-2, special=None):
        rng = np.random.default_rng(seed)
        self.sizes, self.copy_dt = sizes, copy
        self.p = [rng.standard_normal(n).astype(np.float32) for n in sizes]
        gdt = TORCH_DTYPE[grad]
        g = [torch.from_numpy((rng.standard_normal(n) * grad_std).astype(np.float32)).to(gdt) for n in sizes]
        self.state = []
        for n in sizes:
            row = np.repeat(np.exp(rng.standard_normal(-(-n // 256))), 256)[:n]
            m, r = rng.standard_normal(n) * grad_std * row * 0.3, np.exp(rng.standard_normal(n)) * grad_std * row
            if n > 600:
                m[256:512] = 0.0
                r[256:512] = 0.0
            c1, s1, _ = oracle.quantize(m, False)
            c2, s2, _ = oracle.quantize(r * r, True)
            self.state.append([c1, s1.astype(np.float32), c2, s2.astype(np.float32)])
        if special is not None:
            special(self, g)
        self.g = [t.double().numpy() for t in g]
        self.checks = []

        def put(ts, at, what):
            views, check = guarded(ts, at)
            self.checks.append((check, what))
            return views
        self.dp = put([torch.from_numpy(x) for x in self.p], lead, "param")
        self.dg = put(g, lead * 3, "grad")
        self.dc1 = put([torch.from_numpy(s[0]) for s in self.state], 4 * lead, "codes1")
        self.ds1 = put([torch.from_numpy(s[1]) for s in self.state], lead, "scales1")
        self.dc2 = put([torch.from_numpy(s[2]) for s in self.state], 8 * lead, "codes2")
        self.ds2 = put([torch.from_numpy(s[3]) for s in self.state], lead, "scales2")
        self.dcopy = put([torch.zeros(n, dtype=TORCH_DTYPE[copy]) for n in sizes], lead, "copy") if copy else None
        ptr = lambda ts: [t.data_ptr() for t in ts]  # noqa: E731
        self.table = _lib.OptimTable(0, ptr(self.dp), ptr(self.dg), ptr(self.dc1), ptr(self.dc2),
                                     ptr(self.dcopy) if copy else None, sizes, [_lib.DTYPE_CODES[grad]] * len(sizes),
                                     [_lib.DTYPE_CODES[copy]] * len(sizes) if copy else None, ptr(self.ds1), ptr(self.ds2))

    def snapshot(self):
        torch.cuda.synchronize()
        return [[t.cpu().clone() for t in ts] for ts in (self.dp, self.dc1, self.ds1, self.dc2, self.ds2)]

    def compare(self, step, kw, what="", sure_share=0.999):
        torch.cuda.synchronize()
        sure = total = 0
        for i, n in enumerate(self.sizes):
            c1, s1, c2, s2 = self.state[i]
            want = oracle.adam_step(self.p[i], self.g[i], c1, s1, c2, s2, step, **kw)
            got = self.dp[i].cpu().numpy().astype(np.float64)
            both_nan = np.isnan(got) & np.isnan(want["p"])
            bad = ~(both_nan | (np.abs(got - want["p"]) <= want["p_tol"]))
            assert not bad.any(), f"{what} param {i} ({n}): element {np.flatnonzero(bad)[0]} of {bad.sum()}: {got[bad][0]!r} {want['p'][bad][0]!r} tol {want['p_tol'][bad][0]!r}"
            for tag, dc, ds in (("1", self.dc1[i], self.ds1[i]), ("2", self.dc2[i], self.ds2[i])):
                gs, ws = ds.cpu().numpy().astype(np.float64), want["scales" + tag]
                ok = (np.isnan(gs) & np.isnan(ws)) | (np.abs(gs - ws) <= want["scale_tol" + tag])
                assert ok.all(), f"{what} scales{tag} {i} ({n}): {gs[~ok][0]!r} {ws[~ok][0]!r}"
                gc, wc = dc.cpu().numpy(), want["codes" + tag]
                signed = lambda c: np.where(c & 0x80, -1, 1) * (c & 0x7F).astype(int)  # noqa: E731
                apart = np.abs(signed(gc) - signed(wc))
                # a block whose scale lies near 2^-100 has no such block here; the rest as the docstring says
                assert (apart <= 1).all(), f"{what} codes{tag} {i} ({n}): {apart.max()} codes apart at {apart.argmax()}"
                wrong = (apart != 0) & want["sure" + tag]
                assert not wrong.any(), f"{what} codes{tag} {i} ({n}): {wrong.sum()} differ, first at {np.flatnonzero(wrong)[0]}"
                sure += want["sure" + tag].sum()
                total += n
            if self.dcopy is not None:
                assert_bits_equal(self.dcopy[i].cpu(), self.dp[i].cpu().to(self.dcopy[i].dtype), f"{what} copy {i}")
        assert sure >= sure_share * total, (sure, total)
        for check, name in self.checks:
            check(name)

    def carry_on(self):
        """The oracle continues from what the device holds."""
        for i in range(len(self.sizes)):
            self.p[i] = self.dp[i].cpu().numpy()
            self.state[i] = [self.dc1[i].cpu().numpy(), self.ds1[i].cpu().numpy(), self.dc2[i].cpu().numpy(), self.ds2[i].cpu().numpy()]


KW = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)


def launch(t, step, kw, **more):
    a = dict(kw)
    t.table.adam_step(a.pop("lr"), a.pop("beta1"), a.pop("beta2"), a.pop("eps"), a.pop("weight_decay"), step, **a,
                      stream=stream_handle(torch.device(DEV)), **more)


@pytest.mark.parametrize("grad,copy", [("f32", None), ("f32", "bf16"), ("f32", "f16"), ("f32", "f32"), ("bf16", None), ("bf16", "bf16"),
                                       ("bf16", "f16"), ("bf16", "f32"), ("f16", None), ("f16", "f16"), ("f16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("lead", [0, 1])
def test_step_matches_oracle(grad, copy, lead):
    t = Step(SIZES, grad, copy, lead, seed=lead)
    for step in (3, 4):
        launch(t, step, KW)
        t.compare(step, KW, f"step {step}")
        t.carry_on()
    t.table.close()


@pytest.mark.parametrize("kw", [
    dict(KW, decoupled=True), dict(KW, weight_decay=0.0), dict(KW, decoupled=True, weight_decay=0.5, lr=0.1),
    dict(KW, maximize=True), dict(KW, maximize=True, decoupled=True, grad_scale=0.125), dict(KW, grad_scale=2.0 ** -10),
    dict(KW, beta1=0.0, beta2=0.0), dict(KW, beta1=0.3, beta2=0.5, eps=1e-3), dict(KW, lr=0.0), dict(KW, beta2=0.99999),
])
def test_hyper_parameters(kw):
    t = Step([5, 700, 4096, 5000], "f32", "bf16", 0, seed=3)
    for step in (1, 2, 10 ** 6, 2 ** 32 + 5):
        launch(t, step, kw)
        t.compare(step, kw, f"step {step}")
        t.carry_on()
    t.table.close()


def test_zero_states_first_step_equals_the_32_bit_step():
    """Zero moments are exact in both forms, so the first step's parameters agree to rounding (of the division and of the
    product that replaces one: 4 units of the update), and so do the moments that it leaves, within a step of e4m3."""
    gen = torch.Generator().manual_seed(0)
    ps = [torch.randn(n, generator=gen) for n in SIZES]
    gs = [torch.randn(n, generator=gen) * 1e-3 for n in SIZES]
    a, b = [p.clone().to(DEV) for p in ps], [p.clone().to(DEV) for p in ps]
    oa, ob = FusedAdamW(a, lr=1e-2), FusedAdamW(b, lr=1e-2, state_bits=8)
    for params in (a, b):
        for p, g in zip(params, gs):
            p.grad = g.to(DEV)
    oa.step()
    ob.step()
    sa, sb = oa.state_dict()["state"], ob.state_dict()["state"]
    for i, (x, y) in enumerate(zip(a, b)):
        torch.testing.assert_close(y, x, rtol=2 * oracle.EPS, atol=8 * oracle.EPS * 1e-2)
        for key, part in (("exp_avg", 1 / 8), ("exp_avg_sq", 2 / 8 + 1 / 64)):       # neighbours are at most 1/8 apart
            full, short = sa[i][key].double(), sb[i][key].double()
            top = full.abs().max()
            floor = top * 2.0 ** -17 if key == "exp_avg" else top * 2.0 ** -34         # e4m3's smallest against 256
            assert ((short - full).abs() <= full.abs() * part * (1 + 1e-6) + floor).all(), (key, i)
        assert sb[i]["step"] == 1


# ---------------------------------------------------------------- where it can go wrong

def test_special_gradients_stay_in_their_block():
    def poison(t, g):
        g[0][300] = math.nan
        g[0][1000] = math.inf
        g[1][0] = -math.inf
    t = Step([5000, 300], "f32", "bf16", special=poison)
    launch(t, 5, KW)
    t.compare(5, KW, sure_share=0.85)
    s = t.ds1[0].cpu(), t.ds2[0].cpu()
    for x in s:
        assert torch.isnan(x).nonzero().flatten().tolist() == [1, 3]
    assert torch.isnan(t.dp[0]).nonzero().flatten().tolist() == [300, 1000]
    t.carry_on()
    t.g[0][:] = 0.0
    t.dg[0].zero_()
    launch(t, 6, KW)                                   # the poisoned blocks read back as NaN: all their parameters are
    assert torch.isnan(t.dp[0]).nonzero().flatten().tolist() == list(range(256, 512)) + list(range(768, 1024))
    t.table.close()


def test_blocks_of_zeros_and_of_tiny_and_huge_numbers():
    def scales(t, g):
        g[0][:256] = 0.0
        t.state[0][0][:256] = 0
        t.state[0][2][:256] = 0
        t.state[0][1][0] = t.state[0][3][0] = 0.0
        g[0][256:512] *= 2.0 ** -100                   # first moments under 2^-100: stored as zeros
        t.state[0][0][256:512] = 0
        t.state[0][2][256:512] = 0
        t.state[0][1][1] = t.state[0][3][1] = 0.0
        g[0][512:768] *= 2.0 ** 60
        g[0][768:1024] *= 2.0 ** -60                   # squares under the normal fp32 numbers
        t.state[0][0][768:1024] = 0
        t.state[0][2][768:1024] = 0
        t.state[0][1][3] = t.state[0][3][3] = 0.0
    kw = dict(KW, weight_decay=0.0)
    t = Step([1024, 2000], "f32", None, special=scales)
    before = t.snapshot()
    launch(t, 7, kw)
    torch.cuda.synchronize()
    s1, s2 = t.ds1[0].cpu(), t.ds2[0].cpu()
    assert s1[0] == 0 and s2[0] == 0 and not t.dc1[0][:512].any() and not t.dc2[0][:256].any()
    assert torch.equal(t.dp[0][:256].cpu(), before[0][0][:256])            # 0 / (0 + eps)
    assert s1[1] == 0 and s2[1] == 0
    # 2^60 times the gradients, and 2^-60 times: m and its scale follow by the same factor, which no rounding changes
    want = oracle.adam_step(t.p[0], t.g[0], *t.state[0], 7, **kw)
    np.testing.assert_allclose(s1[2:].double().numpy(), want["scales1"][2:], rtol=1e-6)
    np.testing.assert_allclose(s2[2].double().item(), want["scales2"][2], rtol=1e-6)
    # g^2 / 1000 near 2^-145: fp32 holds it to a few bits, the root to the nearest 1/8
    assert s2[3].item() == 0 or abs(s2[3].double().item() / want["scales2"][3] - 1) < 0.2
    assert not torch.isnan(t.dp[0]).any()
    t.table.close()


def test_a_root_never_becomes_zero():
    """Roots 2^-20 of their block's largest keep e4m3's smallest number; zeros stay zero."""
    sizes = [256]

    def state(t, g):
        g[0][:] = 0.0
        g[0][0] = 1.0
        g[0][1:100] = 2.0 ** -20
        for k in (0, 2):
            t.state[0][k][:] = 0
            t.state[0][k + 1][:] = 0
    t = Step(sizes, "f32", None, special=state)
    for step in range(1, 40):
        launch(t, step, dict(KW, weight_decay=0.0))
        c2 = t.dc2[0].cpu()
        assert (c2[1:100] >= 1).all() and not c2[100:].any(), step
        assert not torch.isnan(t.dp[0]).any()
    t.table.close()


def test_many_steps_follow_the_32_bit_moments():
    """Constant gradients for 400 steps: the root has to grow to them although each step moves it by less than e4m3 can
    show.  The dither's average is right, so the mean over many elements comes within a few percent (bound: one e4m3 step)."""
    n = 1 << 16
    p = torch.zeros(n, device=DEV)
    opt = FusedAdam([p], lr=0.0, state_bits=8)
    ref = torch.zeros(n, dtype=torch.float64)
    gen = torch.Generator().manual_seed(1)
    for step in range(400):
        g = torch.randn(n, generator=gen)
        p.grad = g.to(DEV)
        opt.step()
        ref = 0.999 * ref + 0.001 * g.double() ** 2
    got = opt.state_dict()["state"][0]["exp_avg_sq"].double().cpu()
    ratio = float(got.sqrt().mean() / ref.sqrt().mean())
    assert abs(ratio - 1) < 1 / 16, ratio


def test_same_inputs_same_bits_and_no_other_bytes():
    outs = []
    for _ in range(2):
        t = Step(SIZES, "bf16", "bf16", 1, seed=9)
        for step in (1, 2, 3):
            launch(t, step, KW)
        outs.append(t.snapshot())
        for check, name in t.checks:
            check(name)
        t.table.close()
    for a, b in zip(*outs):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_streaming_sizes():
    """Above the size where loads and stores bypass the caches; the result is that of the same tensor in small pieces."""
    n = (300 << 20) // 18 + 77
    gen = torch.Generator(device=DEV).manual_seed(4)
    p0 = torch.randn(n, generator=gen, device=DEV)
    g = torch.randn(n, generator=gen, device=DEV) * 1e-2
    piece = 1 << 22                      # a whole number of blocks; the dither goes by the place in the tensor
    results = []
    for cut in (False, True):
        p = p0.clone()
        spans = [(a, min(n, a + piece)) for a in range(0, n, piece)] if cut else [(0, n)]
        codes1, codes2 = (torch.zeros(n, dtype=torch.uint8, device=DEV) for _ in range(2))
        sc1, sc2 = (torch.zeros(-(-n // 256), device=DEV) for _ in range(2))
        for a, b in spans:
            table = _lib.OptimTable(0, [p[a:].data_ptr()], [g[a:].data_ptr()], [codes1[a:].data_ptr()], [codes2[a:].data_ptr()], None,
                                    [b - a], [_lib.RG_F32], None, [sc1[a // 256:].data_ptr()], [sc2[a // 256:].data_ptr()])
            table.adam_step(1e-3, 0.9, 0.999, 1e-8, 0.0, 1, stream=stream_handle(torch.device(DEV)))
            torch.cuda.synchronize()
            table.close()
        results.append((p, sc1, sc2, codes1, codes2, spans))
    (pa, sa1, sa2, ca1, ca2, _), (pb, sb1, sb2, cb1, cb2, spans) = results
    assert torch.equal(pa, pb) and torch.equal(sa1, sb1) and torch.equal(sa2, sb2)
    a, b = spans[0]
    assert torch.equal(ca1[a:b], cb1[a:b]) and torch.equal(ca2[a:b], cb2[a:b])
    # other pieces have another dither: at most one code apart
    assert int(((ca1 & 0x7F).int() - (cb1 & 0x7F).int()).abs().max()) <= 1
    assert int((ca2.int() - cb2.int()).abs().max()) <= 1


# ---------------------------------------------------------------- gate, clock, scale on the device

def test_gate_clips_and_skips():
    t = Step([4096, 300, 5000], "f16", "f16", 0, seed=5, grad_std=4.0)
    dst = [torch.zeros(n, device=DEV) for n in t.sizes]
    plan = TensorPlan(t.dg, dst)
    plan.step_begin(0.25)
    plan.step_decide(1.0)
    res = plan.result()
    assert res.clipped == 1 and 0 < res.coef < 1
    kw = dict(KW, grad_scale=0.25)
    launch(t, 3, kw, gate=plan.plan.result_device_ptr())
    t.compare(3, dict(kw, coef=res.coef))
    t.carry_on()
    t.dg[1][7] = math.inf
    plan.step_begin(0.25)
    plan.step_decide(1.0)
    assert plan.result().skipped == 1
    before = t.snapshot()
    launch(t, 4, kw, gate=plan.plan.result_device_ptr())
    for a, b in zip(before, t.snapshot()):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    plan.close()
    t.table.close()


def test_clock_and_scale_on_the_device_match_the_host():
    runs = []
    for clocked in (False, True):
        t = Step([4096, 300, 5000], "f32", "bf16", 0, seed=6)
        clock = torch.zeros(_lib.ADAM_CLOCK_BYTES // 4, device=DEV)
        scale = torch.full((1,), 0.5, device=DEV)
        for maximize in (False, True):
            for step in ((1, 2) if not maximize else (3, 4)):
                if clocked:
                    t.table.set_grad_scale_source(scale.data_ptr())
                    s = stream_handle(torch.device(DEV))
                    _lib.adam_clock_advance(clock.data_ptr(), KW["lr"], 0.9, 0.999, 0, 0, s)
                    t.table.adam_step_clocked(clock.data_ptr(), KW["lr"], 0.9, 0.999, 1e-8, 0.01, maximize=maximize, stream=s)
                else:
                    launch(t, step, dict(KW, grad_scale=0.5, maximize=maximize))
        runs.append(t.snapshot())
        t.table.close()
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---------------------------------------------------------------- conversions

def convert_case(sizes, root, lead, seed=0):
    rng = np.random.default_rng(seed)
    values = []
    for n in sizes:
        x = rng.standard_normal(n) * np.exp(rng.standard_normal(n) * 4) * np.repeat(np.exp(rng.standard_normal(-(-n // 256)) * 5), 256)[:n]
        x[rng.random(n) < 0.05] = 0.0
        values.append((x * x if root else x).astype(np.float32))
    return values


@pytest.mark.parametrize("root", [False, True])
@pytest.mark.parametrize("lead", [0, 1, 7])
def test_conversions_match_oracle(root, lead):
    sizes = SIZES + [0, 100003]
    values = convert_case(sizes, root, lead)
    dv, check_v = guarded([torch.from_numpy(v) for v in values], lead)
    dc, check_c = guarded([torch.zeros(n, dtype=torch.uint8) for n in sizes], 4 * lead)
    ds, check_s = guarded([torch.zeros(-(-n // 256)) for n in sizes], lead)
    codes = [c.view(torch.float8_e4m3fn) for c in dc]
    plan = State8Plan(dv, codes, ds, root)
    plan.quantize()
    for i, v in enumerate(values):
        wc, ws, tie = oracle.quantize(v, root)
        gs, gc = ds[i].cpu().numpy(), dc[i].cpu().numpy()
        # the root of an fp32 number rounds once; the largest of the block is one of the numbers themselves
        assert np.array_equal(gs, ws.astype(np.float32)), i
        apart = np.abs(np.where(gc & 0x80, -1, 1) * (gc & 0x7F).astype(int) - np.where(wc & 0x80, -1, 1) * (wc & 0x7F).astype(int))
        # three roundings (root, 256 / s, the product) move y by 3 eps, at most 16 * 3 eps of the neighbours' distance
        assert not (apart[tie > 48 * oracle.EPS]).any() and (apart <= 1).all(), i
        back = oracle.read_back(gc, gs)
        want = back * back if root else back
        dv[i].fill_(7.0)
        values[i] = want
    plan.dequantize()
    torch.cuda.synchronize()
    for i, want in enumerate(values):
        got = dv[i].cpu().double().numpy()
        # one rounding, and with roots the square's and twice the first one's; squares below the normal numbers lose to them
        assert (np.abs(got - want) <= np.abs(want) * 3.01 * oracle.EPS + 2.0 ** -149).all(), i
    kept = [c.clone() for c in dc], [s.clone() for s in ds]
    plan.quantize()                                     # what was read back gives the same codes and scales
    torch.cuda.synchronize()
    for i in range(len(sizes)):
        normal = bool((dv[i][dv[i] > 0] > 2.0 ** -120).all()) if root else True
        if normal:
            assert torch.equal(dc[i], kept[0][i]) and torch.equal(ds[i], kept[1][i]), i
    for check in (check_v, check_c, check_s):
        check("conversion")
    plan.close()


def test_conversion_of_special_values():
    v = torch.zeros(5 * 256 + 10, device=DEV)
    v[0] = math.nan
    v[256:300] = math.inf
    v[512:768] = 2.0 ** -101
    v[768:1024] = torch.finfo(torch.float32).max
    v[1024] = -0.0
    v[1025] = 1.0
    codes, scales, _, _ = allocate_state8([v])
    plan = State8Plan([v], codes, scales)
    plan.quantize()
    assert np.array_equal(scales[0].cpu().numpy(), np.array([np.nan, np.nan, 0.0, torch.finfo(torch.float32).max, 1.0, 0.0], dtype=np.float32), equal_nan=True)
    w = codes[0].view(torch.uint8).cpu()
    assert not w[:768].any() and (w[768:1024] == 0x78).all() and w[1024].item() == 0x80 and w[1025].item() == 0x78
    plan.dequantize()
    assert torch.isnan(v[:512]).all() and not v[512:768].any() and (v[768:1024] == torch.finfo(torch.float32).max).all()
    plan.close()
    v[:] = 1.0
    v[3] = -1e-30                                       # no second moment
    plan = State8Plan([v], codes, scales, root=True)
    plan.quantize()
    assert torch.isnan(scales[0]).cpu().tolist() == [True] + [False] * 5
    plan.close()


def test_conversion_refusals():
    v = torch.zeros(300, device=DEV)
    codes, scales, _, _ = allocate_state8([v])
    ok = ([v], codes, scales)
    for bad in (([v.half()], codes, scales), ([v[:299]], codes, scales), ([v], [codes[0].view(torch.uint8)], scales),
                ([v], codes, [scales[0][:1]]), ([torch.zeros(300, 2, device=DEV)[:, 0]], codes, scales), ([v], [codes[0].cpu()], scales)):
        with pytest.raises(ValueError):
            State8Plan(*bad)
    raw = torch.zeros(304, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="aligned"):
        State8Plan([v], [raw[1:301].view(torch.float8_e4m3fn)], scales)
    plan = State8Plan(*ok)
    plan.close()
    with pytest.raises(ValueError):
        plan.quantize()


def test_streaming_conversion_and_another_stream():
    n = (300 << 20) // 5 + 3
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        v = torch.randn(n, device=DEV)
        codes, scales, _, _ = allocate_state8([v])
        plan = State8Plan([v], codes, scales)
        plan.quantize()
        back = torch.empty_like(v)
        plan2 = State8Plan([back], codes, scales)
        plan2.dequantize()
    side.synchronize()
    s = torch.nn.functional.pad(v.abs(), (0, -n % 256)).view(-1, 256).amax(1)
    assert torch.equal(scales[0], s)
    # to nearest: half a step of e4m3 (1/16 of the number, 1/8 of its binade's start) or of its smallest numbers
    err = (back - v).abs()
    lim = v.abs() / 16 * (1 + 1e-5) + s.repeat_interleave(256)[:n] * 2.0 ** -18 * (1 + 1e-5)
    assert bool((err <= lim).all())
    plan.close()
    plan2.close()


# ---------------------------------------------------------------- the optimizers

def make_params(seed=0, sizes=((40, 64), (64,), (64, 64), (64,), (3, 64), (3,), (0,), (700,))):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(DEV)) for s in sizes]


def give_grads(params, seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(100 + seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=gen) * 1e-2).to(dtype).to(DEV)


def same_state(a, b, pa, pb):
    for x, y in zip(pa, pb):
        assert torch.equal(x, y)
        assert a.state[x].keys() == b.state[y].keys()
        for k, v in a.state[x].items():
            w = b.state[y][k]
            assert torch.equal(v.view(torch.uint8), w.view(torch.uint8)) if v.dtype == torch.float8_e4m3fn else torch.equal(v.cpu(), w.cpu()), k


@pytest.mark.parametrize("cls", [FusedAdam, FusedAdamW])
def test_checkpoint_round_trip_is_exact(cls):
    pa = make_params()
    a = cls(pa, lr=1e-3, weight_decay=0.01, state_bits=8)
    for step in range(5):
        give_grads(pa, step)
        a.step()
    sd = a.state_dict()
    assert all(e["exp_avg"].dtype == torch.float32 and "exp_avg_scale" not in e for e in sd["state"].values())
    assert a.state[pa[0]]["exp_avg"].dtype == torch.float8_e4m3fn             # the live states are untouched
    pb = [torch.nn.Parameter(p.detach().clone()) for p in pa]
    b = cls(pb, lr=1e-3, weight_decay=0.01, state_bits=8)
    host = {"param_groups": sd["param_groups"],
            "state": {i: {k: v.cpu() for k, v in e.items()} for i, e in sd["state"].items()}}
    b.load_state_dict(host)
    same_state(a, b, pa, pb)
    for step in range(5, 8):
        for params, opt in ((pa, a), (pb, b)):
            give_grads(params, step)
            opt.step()
    same_state(a, b, pa, pb)


def test_checkpoints_go_both_ways_with_torch_adam():
    ref_p = [torch.nn.Parameter(p.detach().cpu().clone()) for p in make_params()]
    ref = torch.optim.Adam(ref_p, lr=1e-3)
    for step in range(3):
        for p in ref_p:
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(step)) * 1e-2
        ref.step()
    params = [torch.nn.Parameter(p.detach().to(DEV)) for p in ref_p]
    opt = FusedAdam(params, lr=1e-3, state_bits=8)
    opt.load_state_dict(ref.state_dict())
    for p, q in zip(params, ref_p):
        if p.numel():
            codes, scales, _ = oracle.quantize(ref.state[q]["exp_avg_sq"].numpy().reshape(-1), True)
            assert torch.equal(opt.state[p]["exp_avg_sq_scale"].cpu(), torch.from_numpy(scales).float())
        assert opt.state[p]["exp_avg"].shape == p.shape and float(opt.state[p]["step"]) == 3
    ref.load_state_dict(opt.state_dict())
    give_grads(params, 9)
    opt.step()
    assert float(opt.state[params[0]]["step"]) == 4


def test_parameters_without_gradients_and_late_ones():
    params = make_params()
    opt = FusedAdam([{"params": params[:3]}, {"params": params[3:]}], lr=1e-3, state_bits=8)
    give_grads(params, 0)
    params[1].grad = None
    opt.step()
    assert "exp_avg" not in opt.state.get(params[1], {}) and set(opt.state_dict()["state"]) == {0, 2, 3, 4, 5, 6, 7}
    give_grads(params, 1)
    opt.step()
    assert float(opt.state[params[1]]["step"]) == 1 and float(opt.state[params[0]]["step"]) == 2
    with pytest.raises(RuntimeError, match="several buffers"):
        opt.state_buffers(0)
    flat = opt.state_buffers(1)
    assert flat["exp_avg"].dtype == torch.float8_e4m3fn and flat["exp_avg"].numel() == 256 * flat["exp_avg_scale"].numel()
    # each parameter with its own count, against the same states stepped one by one
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    one = FusedAdam(alone, lr=1e-3, state_bits=8)
    one.load_state_dict({"state": opt.state_dict()["state"], "param_groups": one.state_dict()["param_groups"]})
    for ps, o in ((params, opt), (alone, one)):
        give_grads(ps, 2)
        o.step()
    same_state(opt, one, params, alone)


def test_moved_gradients_and_moved_states_are_followed():
    runs = []
    for fresh in (False, True):
        params = make_params()
        opt = FusedAdamW(params, lr=1e-3, state_bits=8)
        keep = []
        for step in range(4):
            if fresh:
                keep.append([p.grad for p in params])
                give_grads(params, step)
                if step == 2:                             # as code that re-homes state tensors does
                    st = opt.state[params[0]]
                    st["exp_avg"] = st["exp_avg"].clone()
                    opt.invalidate_tables()
            else:
                old = [p.grad for p in params]
                give_grads(params, step)
                for p, g in zip(params, old):
                    if g is not None:
                        g.copy_(p.grad)
                        p.grad = g
            opt.step()
        runs.append((opt, params))
    same_state(runs[0][0], runs[1][0], runs[0][1], runs[1][1])


def test_captured_steps_replay_as_eager_ones():
    """The capturable optimizer recorded once and replayed, with eager work between the replays."""
    def build():
        params = make_params()
        opt = FusedAdamW(params, lr=1e-3, state_bits=8, capturable=True)
        give_grads(params, 0)
        opt.step()
        return params, opt
    pa, a = build()
    pb, b = build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        b.step()
    for step in range(1, 6):
        fresh = [torch.randn(p.shape, generator=torch.Generator().manual_seed(step)).to(DEV) for p in pa]
        for p, q, g in zip(pa, pb, fresh):
            p.grad.copy_(g)
            q.grad.copy_(g)
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(pa, pb):
            assert torch.equal(x, y), step
        for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
            assert torch.equal(a.state_buffers()[k].view(torch.uint8), b.state_buffers()[k].view(torch.uint8)), (k, step)
    assert float(b.state[pb[0]]["step"]) == 6


def test_conversions_in_a_graph():
    v = torch.randn(70001, device=DEV)
    codes, scales, flat_codes, _ = allocate_state8([v])
    back = torch.empty_like(v)
    write, read = State8Plan([v], codes, scales), State8Plan([back], codes, scales)
    write.quantize()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        write.quantize()
        read.dequantize()
    for step in range(4):
        v.normal_(generator=torch.Generator(device=DEV).manual_seed(step))
        graph.replay()
        torch.cuda.synchronize()
        got = back.clone()
        back.zero_()
        write.quantize()
        read.dequantize()
        torch.cuda.synchronize()
        assert torch.equal(got, back), step
    write.close()
    read.close()


def test_model_copies_and_gradient_sources():
    """Scaled bf16 gradients in and bf16 weights out, as the mixed-precision layer drives an optimizer."""
    params = [torch.nn.Parameter(p.detach()) for p in make_params()]
    models = [torch.zeros(p.shape, dtype=torch.bfloat16, device=DEV) for p in params]
    plain = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, ref = FusedAdamW(params, lr=1e-2, state_bits=8), FusedAdamW(plain, lr=1e-2, state_bits=8)
    opt.set_model_copies(params, models)
    opt.grad_scale = 2.0 ** -10
    for step in range(3):
        gen = torch.Generator().manual_seed(step)
        grads = [(torch.randn(p.shape, generator=gen) * 10).to(torch.bfloat16).to(DEV) for p in params]
        opt.set_grad_sources(params, grads)
        for p, g in zip(plain, grads):
            p.grad = g.float() * 2.0 ** -10
        opt.step()
        ref.step()
    same_state(opt, ref, params, plain)
    for p, m in zip(params, models):
        assert_bits_equal(m.cpu(), p.detach().cpu().to(torch.bfloat16))
