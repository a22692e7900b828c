"""The steady-state check of the fused optimizers: gradient addresses collected by the compiled module or in Python, on
the CPU for what counts as usable, on the GPU for steps whose gradients move, change type, go missing and come back."""
import struct

import pytest
import torch

from rannc_amd import fused_optim
from rannc_amd.fused_optim import FusedAdam, FusedAdamW, FusedSGD

native = fused_optim._native


@pytest.fixture(params=["compiled", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(fused_optim, "_native", None)
    elif native is None:
        pytest.skip("the compiled module is not built")
    return request.param


def test_what_counts_as_usable(route):
    a, b, empty = torch.zeros(3, 4), torch.zeros(5), torch.zeros(0)
    words = lambda x: struct.unpack(f"{len(x) // 8}Q", x)  # noqa: E731
    assert words(fused_optim._addresses([a, b, empty], torch.float32)) == (a.data_ptr(), b.data_ptr(), 0)
    assert fused_optim._addresses([], torch.float32) == b""
    assert words(fused_optim._addresses([b[1:]], torch.float32)) == (b.data_ptr() + 4,)
    for bad in ([a, None], [a.half()], [a.t()], [torch.zeros(4).to_sparse()]):
        assert fused_optim._addresses(bad, torch.float32) is None
    assert fused_optim._addresses([a.half()], torch.float16) is not None


@pytest.mark.skipif(native is None, reason="the compiled module is not built")
def test_lists_read_the_gradients_of_the_moment():
    ps = [torch.nn.Parameter(torch.zeros(4)) for _ in range(3)]
    held = native.TensorList(ps)
    assert held.grad_addresses(torch.float32) is None
    for p in ps:
        p.grad = torch.ones(4)
    assert struct.unpack("3Q", held.grad_addresses(torch.float32)) == tuple(p.grad.data_ptr() for p in ps)
    assert held.grad_addresses(torch.float16) is None
    ps[1].grad = torch.ones(4)
    assert struct.unpack("3Q", held.grad_addresses(torch.float32))[1] == ps[1].grad.data_ptr()
    ps[1].grad = None
    assert held.grad_addresses(torch.float32) is None
    with pytest.raises(ValueError):
        native.tensor_addresses([3], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda ps: FusedAdam(ps, lr=1e-2), lambda ps: FusedAdamW(ps, lr=1e-2, state_bits=8),
                                  lambda ps: FusedSGD(ps, lr=0.05, momentum=0.9)], ids=["adam", "adamw8", "sgd"])
@pytest.mark.parametrize("sources", [False, True])
def test_steps_follow_their_gradients(route, make, sources):
    """Against a twin that forgets everything before every step."""
    dev = "cuda:0"
    gen = torch.Generator().manual_seed(7)
    shapes = [(257,), (64, 33), (5,), (0,)]
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dev)) for s in shapes]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, twin = make(ps), make(qs)
    sets = [[torch.zeros(s, device=dev) for s in shapes] for _ in range(2)]
    half = [torch.zeros(s, device=dev, dtype=torch.float16) for s in shapes]
    # which set of addresses the gradients lie in at each step, and whether one is missing
    for step, (where, missing) in enumerate([(0, None), (0, None), (1, None), (1, 1), (0, None), (2, None), (2, None), (0, None), (1, None), (1, None)]):
        grads = (sets + [half])[where]
        if where == 2 and not sources:
            grads = sets[0]                        # torch refuses half gradients on float parameters
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen))
        given = [None if i == missing else g for i, g in enumerate(grads)]
        fresh = [None if g is None else g.clone() for g in given]
        for o, params, gs in ((opt, ps, given), (twin, qs, fresh)):
            if sources:
                o.set_grad_sources([p for p, g in zip(params, gs) if g is not None], [g for g in gs if g is not None])
            else:
                for p, g in zip(params, gs):
                    p.grad = g
        twin.invalidate_tables()
        opt.step()
        twin.step()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(ps, qs)):
            assert torch.equal(p, q), (step, i)
        if not sources and step == 4:
            opt.zero_grad()
            assert all(p.grad is None for p in ps)
