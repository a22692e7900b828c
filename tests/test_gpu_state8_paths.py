"""Optimizer states in 8 bits along the framework's own paths: the mixed-precision layer, checkpoints in the global numbering
with and without ZeRO, parameters kept on the host between steps, the loss scale on the device; and the sizes and alignments that
only large tables reach.  Where a 32-bit run is the yardstick, it is one step from zero states, which both forms hold exactly."""
import math

import numpy as np
import pytest
import torch

import rannc_amd
from oracle import state8 as oracle
from rannc_amd import _lib, _pyrannc, amp
from rannc_amd.fused_optim import FusedAdam, FusedAdamW
from rannc_amd.multi_tensor import State8Plan, allocate_state8, stream_handle
from tests.helpers import assert_bits_equal

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _base(seed=31):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(24, 37), torch.nn.Tanh(), torch.nn.Linear(37, 45)).to(DEV)   # odd sizes


def _inputs(n, dtype, seed=32):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(8, 24, generator=g).to(DEV).to(dtype) for _ in range(n)]


def _train(rm, opt, xs, use_amp):
    for x in xs:
        loss = rm(x).float().pow(2).mean()
        if use_amp:
            with amp.scale_loss(loss, opt) as scaled:
                scaled.backward()
        else:
            loss.backward()
        rm.clip_grad_norm(0.05)
        opt.step()
        opt.zero_grad()


def _same_moments(a, b):
    assert a.keys() == b.keys()
    for order in a:
        assert sorted(a[order]) == sorted(b[order])
        for k, v in a[order].items():
            assert_bits_equal(torch.as_tensor(v).float().cpu(), torch.as_tensor(b[order][k]).float().cpu(), f"{k} of {order}")


def test_fp32_checkpoint_resumes_with_identical_steps(tmp_path):
    _pyrannc.clear()
    xs = _inputs(6, torch.float32)
    model = _base()
    opt = FusedAdam(model.parameters(), lr=1e-2, state_bits=8)
    rm = rannc_amd.RaNNCModule(model, opt)
    _train(rm, opt, xs[:3], False)
    torch.save(rm.state_dict(), tmp_path / "model.pt")
    torch.save(opt.state_dict(from_global=True), tmp_path / "opt_state.pt")
    _train(rm, opt, xs[3:], False)
    want = [p.detach().cpu().clone() for p in model.parameters()]

    _pyrannc.clear()
    ld_model = _base(seed=99)
    ld_model.load_state_dict(torch.load(tmp_path / "model.pt", map_location="cpu"))
    ld_opt = FusedAdam(ld_model.parameters(), lr=1e-2, state_bits=8)
    ld_rm = rannc_amd.RaNNCModule(ld_model, ld_opt)
    ld_rm._deploy()
    global_sd = torch.load(tmp_path / "opt_state.pt")
    assert all(st["exp_avg"].dtype == torch.float32 for st in global_sd["state"].values())
    ld_opt.load_state_dict(global_sd, from_global=True)
    _train(ld_rm, ld_opt, xs[3:], False)
    for p, w in zip(ld_model.parameters(), want):
        assert_bits_equal(p.detach().cpu(), w, "resumed run")


@pytest.mark.parametrize("enable_zero", [False, True])
def test_amp_checkpoint_round_trip(tmp_path, enable_zero):
    """The moments come back in the global numbering, in the parameters' shapes, and load - cut to the local ranges under
    ZeRO - as the very same codes and scales."""
    _pyrannc.clear()
    xs = _inputs(4, torch.float16)
    model = _base()
    opt = FusedAdam(model.parameters(), lr=1e-2, state_bits=8)
    model, opt = amp.initialize(model, opt, opt_level="O2", max_loss_scale=2.0 ** 8)
    rm = rannc_amd.RaNNCModule(model, opt, enable_apex_amp=True, enable_zero=enable_zero)
    _train(rm, opt, xs[:3], True)
    opt_sd = opt.state_dict(from_global=True)
    torch.save(rm.state_dict(), tmp_path / "model.pt")
    torch.save(opt_sd, tmp_path / "opt_state.pt")
    loaded, global_sd = torch.load(tmp_path / "model.pt", map_location="cpu"), torch.load(tmp_path / "opt_state.pt")
    for (n, p), st in zip(model.named_parameters(), global_sd["state"].values()):
        assert sorted(st) == ["exp_avg", "exp_avg_sq", "step"] and st["exp_avg"].shape == p.shape and not st["exp_avg"].is_cuda

    ld_model = _base(seed=99)
    ld_model.load_state_dict(loaded)
    ld_opt = FusedAdam(ld_model.parameters(), lr=1e-2, state_bits=8)
    ld_model, ld_opt = amp.initialize(ld_model, ld_opt, opt_level="O2", max_loss_scale=2.0 ** 8)
    ld_rm = rannc_amd.RaNNCModule(ld_model, ld_opt, enable_apex_amp=True, enable_zero=enable_zero)
    ld_rm._deploy()
    ld_opt.load_state_dict(global_sd, from_global=True)
    for p, q in zip((p for g in ld_opt.param_groups for p in g["params"]), (p for g in opt.param_groups for p in g["params"])):
        for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"):
            a, b = ld_opt.state[p][k], opt.state[q][k]
            assert a.is_cuda and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8)), k
    _same_moments(ld_opt.state_dict(from_global=True)["state"], opt_sd["state"])
    _train(rm, opt, xs[3:], True)
    _train(ld_rm, ld_opt, xs[3:], True)
    for p, q in zip(ld_model.parameters(), model.parameters()):        # masters differ by the half rounding of the reload
        torch.testing.assert_close(p.detach().float().cpu().flatten()[:q.numel()], q.detach().float().cpu().flatten(),
                                   rtol=2e-2, atol=2e-3)


def test_zero_mode_and_plain_mode_train_alike():
    """At one rank ZeRO's segments are whole parameters, so blocks and dither are the same."""
    runs = []
    for enable_zero in (False, True):
        _pyrannc.clear()
        model = _base()
        opt = FusedAdamW(model.parameters(), lr=1e-2, state_bits=8)
        model, opt = amp.initialize(model, opt, opt_level="O2", max_loss_scale=2.0 ** 8)
        rm = rannc_amd.RaNNCModule(model, opt, enable_apex_amp=True, enable_zero=enable_zero)
        _train(rm, opt, _inputs(5, torch.float16), True)
        runs.append([p.detach().cpu().flatten() for p in model.parameters()])
    for a, b in zip(*runs):
        assert_bits_equal(a, b[:a.numel()], "zero against plain")


@pytest.mark.parametrize("fused", [True, False])
def test_amp_first_step_is_the_32_bit_step(fused):
    outs = []
    for bits in (32, 8):
        _pyrannc.clear()
        model = _base()
        opt = FusedAdam(model.parameters(), lr=1e-2, state_bits=bits)
        model, opt = amp.initialize(model, opt, opt_level="O2", max_loss_scale=2.0 ** 8, fused=fused)
        rm = rannc_amd.RaNNCModule(model, opt, enable_apex_amp=True)
        _train(rm, opt, _inputs(1, torch.float16), True)
        outs.append([m.detach().cpu().clone() for m in opt._amp_stash.all_fp32_from_fp16_params])
        for m, p in zip(opt._amp_stash.all_fp32_from_fp16_params, opt._amp_stash.all_fp16_params):
            assert_bits_equal(p.detach().cpu(), m.detach().cpu().half(), "model copy")
    for a, b in zip(*outs):
        torch.testing.assert_close(b, a, rtol=2 * oracle.EPS, atol=8 * oracle.EPS * 1e-2)


def test_overflow_skips_the_step():
    _pyrannc.clear()
    model = _base()
    opt = FusedAdam(model.parameters(), lr=1e-2, state_bits=8)
    model, opt = amp.initialize(model, opt, opt_level="O2", max_loss_scale=2.0 ** 8)
    rm = rannc_amd.RaNNCModule(model, opt, enable_apex_amp=True)
    _train(rm, opt, _inputs(2, torch.float16), True)
    before = {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers(0).items()}
    params = [p.detach().clone() for p in model.parameters()]
    loss = rm(_inputs(1, torch.float16)[0]).float().pow(2).mean() * float("inf")
    with amp.scale_loss(loss, opt) as scaled:
        scaled.backward()
    rm.clip_grad_norm(0.05)
    opt.step()
    for k, v in opt.state_buffers(0).items():
        assert torch.equal(v.view(torch.uint8), before[k]), k
    for p, q in zip(model.parameters(), params):
        assert torch.equal(p, q)


def test_loss_scale_on_the_device():
    """Count, gate and scale on the device give the bits of the host's."""
    outs = []
    for on_device in (False, True):
        _pyrannc.clear()
        model = _base()
        opt = FusedAdam(model.parameters(), lr=1e-2, state_bits=8, capturable=on_device)
        model, opt = amp.initialize(model, opt, opt_level="O2", max_loss_scale=2.0 ** 7, min_loss_scale=None, device_loss_scale=on_device)
        rm = rannc_amd.RaNNCModule(model, opt, enable_apex_amp=True)
        _train(rm, opt, _inputs(5, torch.float16), True)
        outs.append(([p.detach().cpu() for p in model.parameters()], {k: v.view(torch.uint8).cpu() for k, v in opt.state_buffers(0).items()}))
    for a, b in zip(outs[0][0], outs[1][0]):
        assert_bits_equal(a, b, "parameter")
    for k, v in outs[0][1].items():
        assert torch.equal(v, outs[1][1][k]), k


def test_parameters_on_the_host_between_steps():
    """What the offload wrapper does: parameters move to the GPU for the step and back; states stay on the GPU, checkpoints are
    written and read meanwhile."""
    def build():
        torch.manual_seed(5)
        return [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((300,), (33, 7), (5,))]

    def give(ps, step):
        gen = torch.Generator().manual_seed(step)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(DEV)

    stay, move = build(), build()
    a, b = FusedAdam(stay, lr=1e-2, state_bits=8), FusedAdam(move, lr=1e-2, state_bits=8)
    for step in range(6):
        for p in move:
            p.grad = None
            p.data = p.data.to(DEV)
        b.invalidate_tables()
        give(stay, step)
        give(move, step)
        a.step()
        b.step()
        for p in move:
            p.grad = None
            p.data = p.data.cpu()
        if step == 2:
            sd = b.state_dict()
            assert all(e["exp_avg"].is_cuda for e in sd["state"].values())
            b.load_state_dict(sd)                     # the parameters are on the host: converted by the next step
            with pytest.raises(RuntimeError, match="not there yet"):
                b.state_buffers()
            assert b.state_dict()["state"][0]["exp_avg"].dtype == torch.float32
    for p, q in zip(stay, move):
        assert_bits_equal(p.detach().cpu(), q.detach().cpu(), "moved parameter")
    _same_moments(a.state_dict()["state"], b.state_dict()["state"])


@pytest.mark.parametrize("bits", [8, 32])
def test_refused_step_counts_for_nothing(bits):
    params = [torch.nn.Parameter(torch.ones(10, device=DEV)), torch.nn.Parameter(torch.zeros(4, 6, device=DEV).t())]
    other = torch.nn.Parameter(torch.ones(10, device=DEV))
    opt, ref = FusedAdam(params, state_bits=bits), FusedAdam([other], state_bits=bits)
    params[1].grad = torch.ones(6, 4, device=DEV)
    for p in (params[0], other):
        p.grad = torch.full((10,), 0.25, device=DEV)
    for _ in range(2):
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
    params[1].grad = None
    for step in range(3):
        opt.step()
        ref.step()
        assert torch.equal(params[0], other) and float(opt.state[params[0]]["step"]) == step + 1


def test_refused_step_leaves_no_half_made_state():
    params = [torch.nn.Parameter(torch.zeros(10, device=DEV)), torch.nn.Parameter(torch.zeros(4, 6, device=DEV).t())]
    opt = FusedAdam(params, state_bits=8)
    params[0].grad = torch.ones(10, device=DEV)
    params[1].grad = torch.ones(6, 4, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    params[1].grad = None
    opt.step()
    assert opt.state[params[0]]["exp_avg"].dtype == torch.float8_e4m3fn
    sd = opt.state_dict()
    sd["state"][0]["exp_avg"] = torch.zeros(11)
    with pytest.raises((ValueError, RuntimeError)):
        opt.load_state_dict(sd)


def test_failed_conversion_keeps_the_loaded_moments(monkeypatch):
    """What a conversion that fails leaves behind is the float32 moments, not zeros."""
    def trained(opt, p):
        p.grad = torch.randn(700, generator=torch.Generator().manual_seed(1)).to(DEV)
        opt.step()
        return opt.state_dict()

    p, q = (torch.nn.Parameter(torch.ones(700, device=DEV)) for _ in range(2))
    sd = trained(FusedAdam([p], state_bits=8), p)
    opt = FusedAdam([q], state_bits=8)
    with monkeypatch.context() as m:
        m.setattr(State8Plan, "quantize", lambda self: (_ for _ in ()).throw(MemoryError("no memory")))
        with pytest.raises(MemoryError):
            opt.load_state_dict(sd)
    assert opt.state[q]["exp_avg"].dtype == torch.float32 and torch.equal(opt.state[q]["exp_avg"], sd["state"][0]["exp_avg"])
    q.grad = torch.zeros(700, device=DEV)
    opt.step()                                     # converts now
    assert opt.state[q]["exp_avg"].dtype == torch.float8_e4m3fn and float(opt.state[q]["step"]) == 2
    back = opt.state_dict()["state"][0]["exp_avg"]
    want = 0.9 * sd["state"][0]["exp_avg"]
    assert bool(((back - want).abs() <= want.abs() / 8 * (1 + 1e-5) + want.abs().max() * 2.0 ** -17).all())


def test_learning_rate_as_a_tensor_and_by_a_schedule():
    p, q = (torch.nn.Parameter(torch.ones(300, device=DEV)) for _ in range(2))
    lr = torch.tensor(0.1)
    a, b = FusedAdam([p], lr=0.1, state_bits=8), FusedAdam([q], lr=0.1, state_bits=8)
    b.param_groups[0]["lr"] = lr
    for step in range(6):
        a.param_groups[0]["lr"] = float(lr)
        for x in (p, q):
            x.grad = torch.full((300,), 0.5 + step, device=DEV)
        a.step()
        b.step()
        lr.mul_(0.5)                              # in place: the same object with another value
        assert torch.equal(p, q), step


# ---------------------------------------------------------------- sizes and alignments of large tables

@pytest.mark.parametrize("grad,copy", [(torch.float32, None), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_streaming_table_equals_small_ones_at_any_alignment(grad, copy, lead):
    """A table large enough to bypass the caches against one table per tensor that does not: the same bits, and nothing
    outside the tensors is touched."""
    sizes = [4_000_001, 255, 3_900_000, 1, 2_700_003, 770]
    gen = torch.Generator(device=DEV).manual_seed(lead)
    total = lead + sum(sizes) + 7 * len(sizes)
    starts = np.cumsum([lead] + [n + 7 for n in sizes])[:-1].tolist()
    p0 = torch.randn(total, generator=gen, device=DEV)
    g0 = (torch.randn(total, generator=gen, device=DEV) * 1e-2).to(grad)
    cut = lambda t: [t[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
    outs = []
    for together in (True, False):
        p = p0.clone()
        copies = torch.zeros(total, dtype=copy, device=DEV) if copy else None
        codes1, scales1, c1, s1 = allocate_state8(cut(p0))
        codes2, scales2, c2, s2 = allocate_state8(cut(p0))
        rows = [list(range(len(sizes)))] if together else [[i] for i in range(len(sizes))]
        for step in (1, 2):
            for r in rows:
                pick = lambda ts: [ts[i].data_ptr() for i in r]  # noqa: E731
                table = _lib.OptimTable(0, pick(cut(p)), pick(cut(g0)), pick(codes1), pick(codes2), pick(cut(copies)) if copy else None,
                                        [sizes[i] for i in r], [_code(grad)] * len(r), [_code(copy)] * len(r) if copy else None,
                                        pick(scales1), pick(scales2))
                table.adam_step(1e-3, 0.9, 0.999, 1e-8, 0.01, step, stream=stream_handle(torch.device(DEV)))
                torch.cuda.synchronize()
                table.close()
        outs.append([p, c1.view(torch.uint8), s1, c2.view(torch.uint8), s2] + ([copies] if copy else []))
    assert sum(sizes) * 10 > 96 << 20 > max(sizes) * 10
    for a, b in zip(*outs):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    outside = torch.ones(total, dtype=torch.bool, device=DEV)
    for v in cut(outside):
        v.fill_(False)
    assert torch.equal(outs[0][0][outside], p0[outside])
    if copy:
        assert not outs[0][5][outside].any()
        assert_bits_equal(outs[0][5][~outside].cpu(), outs[0][0][~outside].cpu().to(copy), "copies")


def _code(dtype):
    return {torch.float32: _lib.RG_F32, torch.float16: _lib.RG_F16, torch.bfloat16: _lib.RG_BF16}[dtype]


def test_a_tensor_beyond_two_to_the_31_elements():
    """Step and conversions on 2^31 + 4099 elements; compared with the oracle around the places where 31 bits end."""
    n = 2 ** 31 + 4099
    gen = torch.Generator(device=DEV).manual_seed(9)
    p = torch.empty(n, device=DEV)
    g = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    part = 2 ** 28
    for a in range(0, n, part):
        b = min(n, a + part)
        p[a:b] = torch.randn(b - a, generator=gen, device=DEV)
        g[a:b] = torch.randn(b - a, generator=gen, device=DEV).to(torch.bfloat16)
    spans = [(0, 2048), (2 ** 30 - 256, 2 ** 30 + 512), (2 ** 31 - 1024, 2 ** 31 + 1024), (n - 4099 - 256, n)]
    before = [p[a:b].cpu().numpy() for a, b in spans]
    codes1, scales1, _, _ = allocate_state8([p])
    codes2, scales2, _, _ = allocate_state8([p])
    table = _lib.OptimTable(0, [p.data_ptr()], [g.data_ptr()], [codes1[0].data_ptr()], [codes2[0].data_ptr()], None, [n], [_lib.RG_BF16],
                            None, [scales1[0].data_ptr()], [scales2[0].data_ptr()])
    table.adam_step(1e-3, 0.9, 0.999, 1e-8, 0.0, 1, stream=stream_handle(torch.device(DEV)))
    torch.cuda.synchronize()
    for (a, b), x in zip(spans, before):
        blocks = -(-(b - a) // 256)
        zero, none = np.zeros(b - a, dtype=np.uint8), np.zeros(blocks)
        want = oracle.adam_step(x, g[a:b].double().cpu().numpy(), zero, none, zero, none, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, first=a)
        assert (np.abs(p[a:b].double().cpu().numpy() - want["p"]) <= want["p_tol"]).all(), a
        for codes, scales, tag in ((codes1, scales1, "1"), (codes2, scales2, "2")):
            got = codes[0][a:b].view(torch.uint8).cpu().numpy()
            assert (got == want["codes" + tag])[want["sure" + tag]].all(), (a, tag)
            s = scales[0][a // 256:a // 256 + blocks].double().cpu().numpy()
            assert (np.abs(s - want["scales" + tag]) <= want["scale_tol" + tag]).all(), (a, tag)
    table.close()
    del g, codes2, scales2
    values = torch.empty(n, device=DEV)
    plan = State8Plan([values], codes1, scales1)
    plan.dequantize()
    for a, b in spans:
        want = oracle.read_back(codes1[0][a:b].view(torch.uint8).cpu().numpy(), scales1[0][a // 256:a // 256 - (-(b - a) // 256)].cpu().numpy())
        assert (np.abs(values[a:b].double().cpu().numpy() - want) <= np.abs(want) * oracle.EPS * 1.01).all(), a
    kept = [codes1[0][a:b].view(torch.uint8).clone() for a, b in spans]
    codes1[0].view(torch.uint8).fill_(0x11)
    plan.quantize()
    torch.cuda.synchronize()
    for (a, b), k in zip(spans, kept):
        # what was read back has the codes it came from, unless the dither had left the block's largest below 256
        got = codes1[0][a:b].view(torch.uint8)
        back = oracle.read_back(got.cpu().numpy(), scales1[0][a // 256:a // 256 - (-(b - a) // 256)].cpu().numpy())
        x = values[a:b].double().cpu().numpy()
        assert (np.abs(back - x) <= np.abs(x) / 16 * (1 + 1e-6) + np.abs(x).max() * 2.0 ** -18).all(), a
    plan.close()


def test_roots_of_every_magnitude():
    """Square roots of all of fp32's magnitudes, subnormal numbers among them: each number in a block of its own (so that the scale
    is its root), correctly rounded; and blocks whose numbers straddle the range of the quick square root."""
    rng = np.random.default_rng(3)
    bits = np.concatenate([np.arange(1, 300), (1 << np.arange(0, 23)), np.arange(0, 255 << 23, 1 << 23) + 0x2AAAAA, [0x7F7FFFFF, 0x00800000, 0x007FFFFF],
                           rng.integers(1, 0x7F800000, 3000)]).astype(np.uint32)
    bits = bits[(bits > 0) & (bits < 0x7F800000)]
    x = np.zeros((bits.size, 256), dtype=np.float32)
    x[:, 17] = bits.view(np.float32)
    v = torch.from_numpy(x.reshape(-1)).to(DEV)
    codes, scales, _, _ = allocate_state8([v])
    plan = State8Plan([v], codes, scales, root=True)
    plan.quantize()
    want = np.sqrt(bits.view(np.float32).astype(np.float64)).astype(np.float32)
    assert np.array_equal(scales[0].cpu().numpy(), want)
    c = codes[0].view(torch.uint8).cpu().numpy().reshape(-1, 256)
    assert (c[:, 17] == 0x78).all() and not np.delete(c, 17, axis=1).any()
    plan.close()
    full = rng.integers(0x00000001, 0x7F000000, 256 * 64).astype(np.uint32).view(np.float32)        # no zeros: all magnitudes in a block
    v = torch.from_numpy(full).to(DEV)
    codes, scales, _, _ = allocate_state8([v])
    plan = State8Plan([v], codes, scales, root=True)
    plan.quantize()
    wc, ws, tie = oracle.quantize(full, True)
    assert np.array_equal(scales[0].cpu().numpy(), ws.astype(np.float32))
    got = codes[0].view(torch.uint8).cpu().numpy()
    assert (got == wc)[tie > 48 * oracle.EPS].all() and (got >= 1).all()
    plan.close()


def test_zero_eps():
    """eps = 0: elements without any gradient give 0 / 0 as in torch.optim.Adam, the others a finite step."""
    p = torch.nn.Parameter(torch.ones(600, device=DEV))
    g = torch.randn(600, generator=torch.Generator().manual_seed(0)).to(DEV)
    g[100:110] = 0.0
    p.grad = g
    opt = FusedAdam([p], lr=0.1, eps=0.0, state_bits=8)
    opt.step()
    nan = torch.isnan(p.detach())
    assert nan.nonzero().flatten().tolist() == list(range(100, 110))
    torch.testing.assert_close(p.detach()[~nan], 1.0 - 0.1 * torch.sign(g[~nan]), rtol=1e-6, atol=1e-6)
    assert all(math.isfinite(float(s.sum())) for s in (opt.state[p]["exp_avg_scale"], opt.state[p]["exp_avg_sq_scale"]))
