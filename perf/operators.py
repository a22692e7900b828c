"""Optimizer states in 8 bits: the workloads by which the operators are timed and compared.

Three operators over many tensors at once, reached as a training program reaches them:

* ``adam``: one Adam / AdamW step whose two moments are held in 8 bits (``FusedAdam`` / ``FusedAdamW`` with
  ``state_bits=8``),
* ``quantize``: 32-bit moments into that form, as a loaded checkpoint is (``State8Plan.quantize``),
* ``dequantize``: back to 32 bits, as a checkpoint is written (``State8Plan.dequantize``).

The 8-bit form.  A tensor is cut into blocks of 256 consecutive elements (the last one may be shorter).  A block keeps
its largest magnitude ``s`` in 32 bits and, for every element ``x``, the e4m3 number that ``256 x / s`` is rounded to.  The
first moment is stored as it is, the second as its square root.  A block whose ``s`` is below 2^-100 is stored as zeros,
one with an infinity or a NaN has ``s`` = NaN; a root that is not zero is stored as at least 2^-9, e4m3's smallest
number.  ``quantize`` rounds to nearest (ties to even).  The step rounds with a dither: with ``q`` the distance of the
two e4m3 numbers around ``y`` and ``t`` = ``|y| / q``, the stored number is ``floor(t + u / 2^20) q``, where ``u`` is the
upper 20 bits of ``i A + step B`` (first moment) or ``i A + step C`` (root), mod 2^32; ``i`` is the element's place in its
tensor and A, B, C are the three fractions of the additive recurrence with the real root of x^4 = x + 1.

Tensors lie in flat buffers, each at a multiple of 256 elements; what is between them stays zero.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 256
A, B, C = 0xD1B54A33, 0xABC98389, 0x8CB92BA7
TINY = 2.0 ** -100
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- tensor lists

def _mlp(layers=4, width=1024):
    return [n for _ in range(layers) for n in (width * width, width)]


def _bert(layers, hidden, ffn, share=1, vocab=30522):
    one = [hidden * hidden, hidden] * 4 + [hidden] * 4 + [ffn * hidden, ffn, hidden * ffn, hidden]
    every = [vocab * hidden, 512 * hidden, 2 * hidden, hidden, hidden, hidden * hidden, hidden] + one * layers
    return [max(1, n // share) for n in every]


def _resnet152(width=2, split=2):
    """ResNet-152 with twice the channels, every tensor cut into two along its first dimension."""
    out = []

    def conv_bn(cout, cin, k):
        out.extend([cout // split * cin * k * k, cout // split, cout // split] * split)

    conv_bn(64 * width, 3, 7)
    cin = 64 * width
    for planes, blocks in ((64, 3), (128, 8), (256, 36), (512, 3)):
        planes *= width
        for b in range(blocks):
            conv_bn(planes, cin, 1)
            conv_bn(planes, planes, 3)
            conv_bn(planes * 4, planes, 1)
            if b == 0:
                conv_bn(planes * 4, cin, 1)
            cin = planes * 4
    return out + [1000 // split * cin] * split + [1000 // split] * split


def _ragged(tensors, total, seed):
    """Sizes spread over their logarithm that add up to about ``total``, three of four odd."""
    rng = np.random.RandomState(seed % (1 << 31))
    raw = np.exp(rng.uniform(0.0, math.log(4096.0), size=tensors))
    sizes = np.maximum(1, np.floor(raw * (total / raw.sum()))).astype(np.int64)
    return [int(n) | int(j % 4 != 3) for j, n in enumerate(sizes)]


def _numels(case):
    kind = case["layout"]
    if kind == "small_net":           # Linear(40, 64), Linear(64, 64), Linear(64, 3): the test suite's model
        return [64 * 40, 64, 64 * 64, 64, 3 * 64, 3]
    if kind == "mlp":
        return _mlp()
    if kind == "bert_large":
        return _bert(24, 1024, 4096)
    if kind == "bert_enlarged_quarter":
        return _bert(48, 2048, 8192, share=4)
    if kind == "resnet152x2":
        return _resnet152()
    return _ragged(case["tensors"], case["total"], case["layout_seed"])


def _starts(numels):
    """Where each tensor begins in the flat buffers, and their length."""
    padded = -(-np.array(numels, dtype=np.int64) // BLOCK) * BLOCK
    ends = np.cumsum(padded)
    return [int(x) for x in ends - padded], int(ends[-1])


# ---------------------------------------------------------------- cases

def listed():
    adam = {"op": "adam", "lr": 1e-4, "eps": 1e-8, "weight_decay": 0.01, "decoupled": True, "first": False}
    return [
        # a handful of small tensors, first steps from zero states: what one call costs
        dict(adam, name="adam small net", layout="small_net", grad="f32", copy="none", grad_scale=1.0, first=True),
        # four Linear(1024, 1024) in full precision
        dict(adam, name="adam mlp", layout="mlp", grad="f32", copy="none", grad_scale=1.0),
        # 934 tensors, most of them vectors of 64 to 2048 elements; L2 decay as vision models use it
        dict(adam, name="adam resnet152x2", layout="resnet152x2", grad="f32", copy="none", grad_scale=1.0, weight_decay=1e-4, decoupled=False),
        # mixed precision: scaled bf16 gradients in, bf16 model weights out
        dict(adam, name="adam bert large", layout="bert_large", grad="bf16", copy="bf16", grad_scale=2.0 ** -16),
        # segments of odd length, as a sharded flat buffer has them
        dict(adam, name="adam ragged", layout="ragged", tensors=512, total=150_000_000, layout_seed=3, grad="f16", copy="f16", grad_scale=2.0 ** -12),
        # one of four ranks' share of the 2.5e9-parameter stage
        dict(adam, name="adam bert enlarged quarter", layout="bert_enlarged_quarter", grad="f16", copy="f16", grad_scale=2.0 ** -12),
        # a checkpoint is loaded: first moments of the large model, second moments of the small and the ragged one
        {"op": "quantize", "name": "quantize bert large first", "layout": "bert_large", "root": False},
        {"op": "quantize", "name": "quantize mlp second", "layout": "mlp", "root": True},
        {"op": "quantize", "name": "quantize ragged second", "layout": "ragged", "tensors": 512, "total": 150_000_000, "layout_seed": 3, "root": True},
        # a checkpoint is written
        {"op": "dequantize", "name": "dequantize mlp first", "layout": "mlp", "root": False},
        {"op": "dequantize", "name": "dequantize bert large second", "layout": "bert_large", "root": True},
        {"op": "dequantize", "name": "dequantize ragged first", "layout": "ragged", "tensors": 512, "total": 150_000_000, "layout_seed": 3, "root": False},
    ]


def draw(rng):
    total = int(math.exp(rng.uniform(math.log(3000), math.log(3.3e8))))
    tensors = min(max(1, total // 512), int(math.exp(rng.uniform(0.0, math.log(900)))))
    case = {"op": rng.choice(("adam", "adam", "quantize", "dequantize")), "layout": "ragged", "tensors": tensors, "total": total,
            "layout_seed": rng.randrange(1 << 30)}
    if case["op"] != "adam":
        return dict(case, root=rng.random() < 0.5)
    grad = rng.choice(("f32", "f16", "bf16"))
    return dict(case, grad=grad, copy=rng.choice(("none", "bf16", "f16") if grad == "f32" else ("none", grad)),
                lr=10.0 ** rng.uniform(-5, -3), eps=10.0 ** rng.uniform(-9, -6), weight_decay=rng.choice((0.0, 0.01, 0.1)),
                decoupled=rng.random() < 0.5, first=rng.random() < 0.25, grad_scale=2.0 ** -rng.randrange(0, 17))


def work(case):
    numels = _numels(case)
    n, scales = sum(numels), sum(-(-x // BLOCK) for x in numels)
    if case["op"] != "adam":
        return {"bytes": 5 * n + 4 * scales, "flops": 2 * n}
    size = {"none": 0, "f32": 4, "f16": 2, "bf16": 2}
    # parameters and both moments in and out, the gradient in, the model copy out
    return {"bytes": n * (8 + 4 + size[case["grad"]] + size[case["copy"]]) + 16 * scales, "flops": 30 * n}


# ---------------------------------------------------------------- inputs

def _moments(gen, blocks, std):
    """First moments and roots of second moments as training leaves them: magnitudes that differ by rows and by
    elements, some rows that no gradient has reached yet."""
    dev = gen.device
    row = torch.exp(torch.randn(blocks, 1, generator=gen, device=dev)) * std
    row *= torch.rand(blocks, 1, generator=gen, device=dev) > 0.02
    root = torch.exp(0.7 * torch.randn(blocks, BLOCK, generator=gen, device=dev)) * row
    first = 0.4 * torch.randn(blocks, BLOCK, generator=gen, device=dev) * root
    return first, root


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    numels = _numels(case)
    starts, total = _starts(numels)
    blocks = total // BLOCK
    first_block = np.array(starts, dtype=np.int64) // BLOCK
    counts = np.diff(np.append(first_block, blocks))
    # the place of each block in its tensor, and the elements of the buffers that belong to a tensor
    place = torch.from_numpy(np.arange(blocks) - np.repeat(first_block, counts)).cuda()
    inside = torch.from_numpy(np.repeat(np.array(numels, dtype=np.int64), counts)).cuda()
    live = place[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < inside[:, None]
    s = {"case": case, "place": place}
    std = 1e-3
    if case["op"] != "adam":
        first, root = _moments(gen, blocks, std)
        values = torch.where(live, root.square() if case["root"] else first, 0.0)
        s["codes"] = torch.zeros(total, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.zeros(blocks, device="cuda")
        if case["op"] == "dequantize":
            codes, scales = _quantize(values, case["root"])
            s["codes"].copy_(codes.view(-1))
            s["scales"].copy_(scales)
            values.zero_()
        s["values"] = values.view(-1)
        if own:
            from rannc_amd.multi_tensor import State8Plan
            views = [s["values"][a:a + n] for a, n in zip(starts, numels)]
            codes = [s["codes"][a:a + n] for a, n in zip(starts, numels)]
            scales = [s["scales"][a // BLOCK:a // BLOCK + -(-n // BLOCK)] for a, n in zip(starts, numels)]
            s["plan"] = State8Plan(views, codes, scales, root=case["root"])
        return s
    s["params"] = torch.where(live, 0.05 * torch.randn(blocks, BLOCK, generator=gen, device="cuda"), 0.0).view(-1)
    grads = torch.randn(blocks, BLOCK, generator=gen, device="cuda") * (std / case["grad_scale"])
    s["grads"] = torch.where(live, grads, 0.0).to(DTYPES[case["grad"]]).view(-1)
    del grads
    if case["copy"] != "none":
        s["copies"] = torch.zeros(total, dtype=DTYPES[case["copy"]], device="cuda")
    if case["first"]:
        s["step"] = 0
        s["exp_avg"] = torch.zeros(total, dtype=torch.float8_e4m3fn, device="cuda")
        s["exp_avg_sq"] = torch.zeros_like(s["exp_avg"])
        s["exp_avg_scale"] = torch.zeros(blocks, device="cuda")
        s["exp_avg_sq_scale"] = torch.zeros(blocks, device="cuda")
    else:
        s["step"] = 1000 + seed % 100
        first, root = _moments(gen, blocks, std)
        for name, values, is_root in (("exp_avg", first, False), ("exp_avg_sq", root.square(), True)):
            codes, scales = _quantize(torch.where(live, values, 0.0), is_root)
            s[name], s[name + "_scale"] = codes.view(-1), scales
    if own:
        from rannc_amd.fused_optim import FusedAdam, FusedAdamW
        cut = lambda flat: [flat[a:a + n] for a, n in zip(starts, numels)]  # noqa: E731
        params = cut(s["params"])
        kind = FusedAdamW if case["decoupled"] else FusedAdam
        opt = kind(params, lr=case["lr"], eps=case["eps"], weight_decay=case["weight_decay"], state_bits=8)
        opt.grad_scale = case["grad_scale"]
        opt.set_grad_sources(params, cut(s["grads"]))
        if case["copy"] != "none":
            opt.set_model_copies(params, cut(s["copies"]))
        moments = [cut(_dequantize(s[k].view(-1, BLOCK), s[k + "_scale"], r).view(-1)) for k, r in (("exp_avg", False), ("exp_avg_sq", True))]
        state = {i: {"step": torch.tensor(float(s["step"])), "exp_avg": m, "exp_avg_sq": v} for i, (m, v) in enumerate(zip(*moments))}
        opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
        s["opt"] = opt
        s.update(opt.state_buffers(0))         # the optimizer's own buffers, laid out as the ones above
    return s


# ---------------------------------------------------------------- plain forms

def _scale_of(x):
    """Largest magnitude of every block (0 below 2^-100, NaN where something is not finite) and 256 over it (0 there)."""
    s = x.abs().amax(dim=1)
    s = torch.where(s < TINY, 0.0, s)
    s = torch.where(torch.isfinite(s), s, math.nan)
    inv = torch.where(s > 0, 256.0 * torch.reciprocal(s), 0.0)
    return s, inv[:, None]


def _quantize(values, root):
    x = torch.sqrt(values) if root else values
    s, inv = _scale_of(x)
    y = torch.where(inv > 0, x * inv, 0.0)
    if root:
        y = torch.where(y > 0, y.clamp(min=2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn), s


def _dequantize(codes, scales, root):
    x = codes.to(torch.float32) * (scales * 2.0 ** -8)[:, None]
    return x * x if root else x


def _dithered(y, u):
    """``floor(|y| / q + u / 2^20) q`` with the sign of ``y``; the quotient has no bits that matter below 2^-20."""
    exponent = torch.frexp(y)[1].clamp(min=-5) - 4                 # q = 2^exponent, at least 2^-9
    power = lambda n: ((n + 127) << 23).view(torch.float32)        # noqa: E731
    t = (y.abs() * power(20 - exponent)).to(torch.int32)
    k = (t + u) >> 20
    return torch.copysign(k.to(torch.float32) * power(exponent), y).to(torch.float8_e4m3fn)


def _plain_adam(s):
    case = s["case"]
    s["step"] += 1
    t, b1, b2 = s["step"], 0.9, 0.999
    g = s["grads"].to(torch.float32).view(-1, BLOCK) * case["grad_scale"]
    p = s["params"].view(-1, BLOCK)
    if case["decoupled"]:
        p = p * (1.0 - case["lr"] * case["weight_decay"])
    elif case["weight_decay"]:
        g = g + p * case["weight_decay"]
    m = _dequantize(s["exp_avg"].view(-1, BLOCK), s["exp_avg_scale"], False)
    v = _dequantize(s["exp_avg_sq"].view(-1, BLOCK), s["exp_avg_sq_scale"], True)
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * (1.0 - b2)) * g
    r = torch.sqrt(v)
    inv_bias = float(np.float32(1.0) / np.float32(math.sqrt(1.0 - b2 ** t)))
    p = p + (m * (-(case["lr"] / (1.0 - b1 ** t)))) / (r * inv_bias + case["eps"])
    s["params"].copy_(p.view(-1))
    if "copies" in s:
        s["copies"].copy_(p.view(-1))
    del g, p, v
    i = (s["place"][:, None] * BLOCK + torch.arange(BLOCK, device=s["params"].device)) * A
    for name, x, step_factor in (("exp_avg", m, B), ("exp_avg_sq", r, C)):
        scale, inv = _scale_of(x)
        y = torch.where(inv > 0, x * inv, 0.0)
        if step_factor == C:
            y = torch.where(y > 0, y.clamp(min=2.0 ** -9), y)
        u = (((i + t * step_factor) & 0xFFFFFFFF) >> 12).to(torch.int32)
        s[name].copy_(_dithered(y, u).view(-1))
        s[name + "_scale"].copy_(scale)



def _outputs(s):
    if s["case"]["op"] == "quantize":
        return {"codes": s["codes"], "scales": s["scales"]}
    if s["case"]["op"] == "dequantize":
        return {"values": s["values"]}
    names = ("params", "copies", "exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
    return {k: s[k] for k in names if k in s}


def run(state):
    case = state["case"]
    if case["op"] == "adam":
        if own:
            state["opt"].step()
        else:
            _plain_adam(state)
    elif case["op"] == "quantize":
        if own:
            state["plan"].quantize()
        else:
            codes, scales = _quantize(state["values"].view(-1, BLOCK), case["root"])
            state["codes"].copy_(codes.view(-1))
            state["scales"].copy_(scales)
    elif own:
        state["plan"].dequantize()
    else:
        state["values"].copy_(_dequantize(state["codes"].view(-1, BLOCK), state["scales"], case["root"]).view(-1))
    return _outputs(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _grid():
    """The numbers of e4m3 that are not negative."""
    return torch.tensor([f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)][:-1],
                        dtype=torch.float64, device="cuda")


def _neighbours(y):
    grid = _grid()
    a = y.abs()
    k = (torch.searchsorted(grid, a, right=True) - 1).clamp(0, len(grid) - 2)
    low, high = grid[k], grid[k + 1]
    return k, low, high, (a - low) / (high - low)


def _exact_scaled(x, root):
    s = x.abs().amax(dim=1)
    s = torch.where(s < TINY, 0.0, s)
    y = torch.where(s[:, None] > 0, 256.0 * x / s[:, None].clamp(min=TINY), 0.0)
    if root:
        y = torch.where(y > 0, y.clamp(min=2.0 ** -9), y)
    return s, y


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    held = lambda name: s[name].view(-1, BLOCK).double() * s[name + "_scale"].double()[:, None] / 256.0  # noqa: E731
    if case["op"] == "dequantize":
        x = s["codes"].view(-1, BLOCK).double() * s["scales"].double()[:, None] / 256.0
        return {"values": (x * x if case["root"] else x).view(-1)}
    if case["op"] == "quantize":
        x = s["values"].view(-1, BLOCK).double()
        scale, y = _exact_scaled(x.sqrt() if case["root"] else x, case["root"])
        k, low, high, part = _neighbours(y)
        up = (part > 0.5) | ((part == 0.5) & (k % 2 == 1))
        return {"codes": torch.copysign(torch.where(up, high, low), y).view(-1), "scales": scale}
    t, b1, b2 = s["step"] + 1, 0.9, 0.999
    g = s["grads"].view(-1, BLOCK).double() * case["grad_scale"]
    p = s["params"].view(-1, BLOCK).double()
    if not case["decoupled"]:
        g += case["weight_decay"] * p
    m = b1 * held("exp_avg") + (1 - b1) * g
    r = (b2 * held("exp_avg_sq").square() + (1 - b2) * g.square()).sqrt()
    step = case["lr"] * (m / (1 - b1 ** t)) / (r / math.sqrt(1 - b2 ** t) + case["eps"])
    p = (p * (1 - case["lr"] * case["weight_decay"]) if case["decoupled"] else p) - step
    del g, step
    out = {"params": p.view(-1)}
    if "copies" in s:
        out["copies"] = out["params"]
    i = s["place"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    for name, x, factor in (("exp_avg", m, B), ("exp_avg_sq", r, C)):
        out[name + "_scale"], y = _exact_scaled(x, factor == C)
        _, low, high, part = _neighbours(y)
        up = part * 2.0 ** 20 + (((i * A + t * factor) % (1 << 32)) // 4096) >= 2.0 ** 20
        out[name] = torch.copysign(torch.where(up, high, low), y).view(-1)
    return out
