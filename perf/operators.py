"""The 4-bit operators, as a serving program calls them: weights are quantised once, then every projection of a step reads them.

  linear    y = x W^T + b                   (``linear_w4``: the q|k|v, output and down projections, the output head)
  gated     y = f(x Wg^T) * (x Wu^T)        (``gated_w4``: gate and up projection, activation and product of a feed-forward)
  quantize  4-bit codes, scales and zero points of a matrix (``quantize_w4``: once for every weight of a checkpoint)

A weight is W[n][k] = (code[n][k] - zero) * scale, with a bf16 scale, and in the asymmetric form a zero point of 0..15, for every `group`
consecutive k of a row; the symmetric form has 8 for every zero point. ``packed`` is int32 [out][in / 8]: of eight consecutive k, number 2i is in
bits 4i .. 4i + 3 and number 2i + 1 in bits 16 + 4i .. 19 + 4i. ``scales`` (bf16) and ``zeros`` (uint8) are [in / group][out].

The packed words are whole numbers and returned as such: every code has to be the nearest one, ties going to the even one.
"""
from __future__ import annotations

import math

import torch

own = False

SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # of the eight codes in a word
SMALLEST = 2.0 ** -126  # scales below this are 0
MOST_FLOPS = 9.7e11  # of a drawn case: the largest listed one's


def listed():
    return [
        # one user in a chat: q|k|v of the Llama-3-8B shape; the smallest call of a decode step, latency counts
        dict(name="linear 1 x 4096 to 6144", op="linear", rows=1, k=4096, n=6144, group=128, zeros=False, bias=False, dtype="bf16"),
        # a small batch through the down projection of the same shape
        dict(name="linear 16 x 14336 to 4096", op="linear", rows=16, k=14336, n=4096, group=128, zeros=True, bias=False, dtype="bf16"),
        # the output head over the vocabulary, finer groups
        dict(name="linear 8 x 4096 to 128256", op="linear", rows=8, k=4096, n=128256, group=64, zeros=False, bias=False, dtype="bf16"),
        # the headline batch through q|k|v of the Qwen2-7B shape, which has biases
        dict(name="linear 64 x 3584 to 4608", op="linear", rows=64, k=3584, n=4608, group=128, zeros=True, bias=True, dtype="bf16"),
        # a prompt through the output projection
        dict(name="linear 2048 x 4096 to 4096", op="linear", rows=2048, k=4096, n=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # the f32 build at odd sizes: a ragged handful of rows, an odd number of outputs, the finest groups
        dict(name="linear f32 5 x 2048 to 1001", op="linear", rows=5, k=2048, n=1001, group=32, zeros=True, bias=True, dtype="f32"),
        # a short prompt in the f32 build
        dict(name="linear f32 211 x 2048 to 5504", op="linear", rows=211, k=2048, n=5504, group=64, zeros=False, bias=False, dtype="f32"),
        # one user in a chat: the feed-forward of the Llama-3-8B shape
        dict(name="gated 1 x 4096 to 14336", op="gated", rows=1, k=4096, n=14336, group=128, zeros=False, act="silu", dtype="bf16"),
        # a full batch in the feed-forward of the Qwen2-7B shape
        dict(name="gated 64 x 3584 to 18944", op="gated", rows=64, k=3584, n=18944, group=64, zeros=True, act="gelu_tanh", dtype="bf16"),
        # prompts of a continuous batch, the largest product
        dict(name="gated 4096 x 4096 to 14336", op="gated", rows=4096, k=4096, n=14336, group=128, zeros=False, act="silu", dtype="bf16"),
        # loading a checkpoint: an output projection of the Llama-3-8B shape
        dict(name="quantize 4096 x 4096", op="quantize", n=4096, k=4096, group=128, zeros=False, dtype="bf16"),
        # loading a checkpoint kept in f32: one half of a gated feed-forward, zero points, the finest groups
        dict(name="quantize f32 14336 x 4096", op="quantize", n=14336, k=4096, group=32, zeros=True, dtype="f32"),
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["linear", "linear", "gated", "gated", "quantize"])
    group = rng.choice([32, 64, 128])
    case = dict(op=op, k=max(1, spread(256, 14336) // group) * group, group=group, zeros=rng.random() < 0.5,
                dtype="bf16" if rng.random() < 0.75 else "f32")
    if op == "quantize":
        return dict(case, n=min(spread(256, 65536), 14336 * 4096 // case["k"]))
    case["n"] = spread(256, 65536 if op == "linear" else 28672)
    most = 2048 if case["dtype"] == "bf16" else 512
    fits = MOST_FLOPS / (2 if op == "linear" else 4) / case["n"] / case["k"] / (1 if case["dtype"] == "bf16" else 4)
    case["rows"] = min(spread(1, most), max(1, int(fits)))
    return dict(case, bias=rng.random() < 0.5) if op == "linear" else dict(case, act=rng.choice(["silu", "gelu_tanh"]))


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _inputs(case, seed):
    """The tensors of a case: weights N(0, 1/k) quantised to codes, activations with a few strong channels and the last row a padded one."""
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    n, k, group = case["n"], case["k"], case["group"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "quantize":
        w = normal(n, k) * (1.0 / math.sqrt(k))
        w += 0.002 * normal(n, 1)  # rows are not centred
        return dict(weight=w.to(_dtype(case)))

    def weight():
        packed = torch.randint(-(1 << 31), 1 << 31, (n, k // 8), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        # codes are near uniform where a group is scaled to its largest value; the groups' largest values differ by a factor of a few
        scales = ((0.3 / math.sqrt(k)) * torch.exp(0.3 * normal(k // group, n))).to(torch.bfloat16)
        zeros = torch.clamp((7.5 + 1.2 * normal(k // group, n)).round(), 0, 15).to(torch.uint8) if case["zeros"] else None
        return dict(packed=packed, scales=scales, zeros=zeros)

    x = normal(case["rows"], k) * (1.0 + 9.0 * (torch.rand(1, k, generator=gen, device="cuda") < 0.01))
    if case["rows"] > 1:
        x[-1] = 0.0
    state = dict(x=x.to(_dtype(case)), w=weight())
    if case["op"] == "gated":
        state["up"] = weight()
    elif case["bias"]:
        state["bias"] = normal(n)
    return state


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        from __graft_entry__ import load_package

        orion = load_package()
        state["orion"], state["backend"] = orion, orion.CudaBackend(torch.cuda.current_device())
        for name in ("w", "up"):
            if name in state:  # the handle that a program keeps for each of its weights
                state[name] = orion.W4Weight(**state[name], group=case["group"])
    return state


# ---- plain forms: 32 bits, 64 where a value may lie next to a border between two codes


def _dequantized(w, group):
    n, words = w["packed"].shape
    codes = (w["packed"][:, :, None] >> torch.tensor(SHIFTS, device="cuda", dtype=torch.int32)) & 15
    codes = codes.view(n, words * 8 // group, group).float()
    zeros = 8.0 if w["zeros"] is None else w["zeros"].float().t()[:, :, None]
    return ((codes - zeros) * w["scales"].float().t()[:, :, None]).view(n, words * 8)


def _activation(name, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _nearest_bf16(x):
    """64-bit values of 0 or more, rounded once to the 8 significant bits of bf16 (ties to even); 0 below the smallest normal number."""
    bits = x.view(torch.int64)
    bits = (bits + ((1 << 44) - 1) + ((bits >> 45) & 1)) >> 45 << 45
    x = bits.view(torch.float64)
    return torch.where(x < SMALLEST, torch.zeros_like(x), x)


def _quantized(weight, group, with_zeros):
    n, k = weight.shape
    w = weight.double().view(n, k // group, group)
    if with_zeros:
        low, high = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        scale = _nearest_bf16((high - low) / 15.0)
        per = torch.where(scale > 0, scale, torch.full_like(scale, math.inf))
        zero = torch.clamp(torch.round(-low / per), 0, 15)
    else:
        scale = _nearest_bf16(w.abs().amax(-1) / 7.0)
        per = torch.where(scale > 0, scale, torch.full_like(scale, math.inf))
        zero = torch.full_like(scale, 8.0)
    codes = torch.clamp(torch.round(w / per[:, :, None]) + zero[:, :, None], 0, 15)
    codes = codes.to(torch.int32).view(n, k // 8, 8)
    packed = (codes << torch.tensor(SHIFTS, device="cuda", dtype=torch.int32)).sum(-1, dtype=torch.int32)
    out = dict(packed=packed, scales=scale.t().contiguous().to(torch.bfloat16))
    return dict(out, zeros=zero.t().contiguous().to(torch.uint8)) if with_zeros else out


def run(state):
    case = state["case"]
    if own:
        orion, backend = state["orion"], state["backend"]
        if case["op"] == "linear":
            return orion.linear_w4(backend, state["x"], state["w"], bias=state.get("bias"))
        if case["op"] == "gated":
            return orion.gated_w4(backend, state["x"], state["w"], state["up"], activation=case["act"])
        w = orion.quantize_w4(backend, state["weight"], group=case["group"], zeros=case["zeros"])
        out = dict(packed=w.packed, scales=w.scales)
        return dict(out, zeros=w.zeros) if case["zeros"] else out
    if case["op"] == "quantize":
        return _quantized(state["weight"], case["group"], case["zeros"])
    x = state["x"].float()
    y = x @ _dequantized(state["w"], case["group"]).t()
    if case["op"] == "gated":
        y = _activation(case["act"], y) * (x @ _dequantized(state["up"], case["group"]).t())
    elif case["bias"]:
        y = y + state["bias"]
    return y.to(state["x"].dtype)


def work(case):
    n, k, size = case["n"], case["k"], 2 if case["dtype"] == "bf16" else 4
    weight = n * k // 2 + n * (k // case["group"]) * (3 if case["zeros"] else 2)
    if case["op"] == "quantize":
        return dict(bytes=n * k * size + weight, flops=4 * n * k)
    matrices = 2 if case["op"] == "gated" else 1
    total = matrices * weight + case["rows"] * (k + n) * size + (4 * n if case.get("bias") else 0)
    return dict(bytes=total, flops=2 * case["rows"] * n * k * matrices)


# ---- the definition in 64 bits


def _product64(x, w, group):
    """x W^T group by group: the codes less their zero point against the group's columns of x, then times the group's scale."""
    total = None
    for g in range(x.shape[1] // group):
        words = w["packed"][:, g * group // 8:(g + 1) * group // 8].long()
        at = torch.stack([(words // (1 << s)) % 16 for s in SHIFTS], dim=-1).reshape(words.shape[0], group).double()
        at -= 8.0 if w["zeros"] is None else w["zeros"][g][:, None].double()
        part = torch.matmul(x[:, g * group:(g + 1) * group], at.t()) * w["scales"][g].double()
        total = part if total is None else total.add_(part)
    return total


def _closest_bf16(x):
    """The bf16 number next to each 64-bit value, found among a guess and its two neighbours."""
    guess = x.to(torch.bfloat16)
    best = guess.double()
    for step in (-1, 1):
        other = (guess.view(torch.int16) + step).view(torch.bfloat16)
        closer = (other.double() - x).abs() - (best - x).abs()
        even = (other.view(torch.int16) & 1) == 0
        best = torch.where(((closer < 0) | ((closer == 0) & even)) & (guess > 0), other.double(), best)
    return torch.where(best < SMALLEST, torch.zeros_like(best), best)


def _rounded(v, scale, lowest, highest):
    """v / scale to the nearest whole number, ties to even, within lowest .. highest: the number of borders below v, with the sum taken border by border."""
    code = torch.full(v.shape, lowest, dtype=torch.int32, device=v.device)
    for j in range(lowest, highest):
        border = (j + 0.5) * scale
        code += ((v >= border) if j % 2 else (v > border)).int()
    return code


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quantize":
        n, k, group = case["n"], case["k"], case["group"]
        w = s["weight"].double().view(n, k // group, group)
        low, high = w.min(-1).values, w.max(-1).values
        if case["zeros"]:
            low, high = torch.minimum(low, torch.zeros_like(low)), torch.maximum(high, torch.zeros_like(high))
            scale = _closest_bf16((high - low) / 15.0)
            zero = torch.where(scale > 0, _rounded(-low, scale, 0, 15), torch.zeros_like(scale, dtype=torch.int32))
        else:
            scale = _closest_bf16(torch.maximum(-low, high) / 7.0)
            zero = torch.full_like(scale, 8, dtype=torch.int32)
        code = torch.where(scale[:, :, None] > 0, _rounded(w, scale[:, :, None], -16, 16), torch.zeros_like(w, dtype=torch.int32))
        code = torch.clamp(code + zero[:, :, None], 0, 15).long().view(n, k // 8, 8)
        packed = torch.zeros(n, k // 8, dtype=torch.int64, device="cuda")
        for i, shift in enumerate(SHIFTS):
            packed += code[:, :, i] * (1 << shift)
        packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        out = dict(packed=packed, scales=scale.t().contiguous().to(torch.bfloat16))
        return dict(out, zeros=zero.t().contiguous().to(torch.uint8)) if case["zeros"] else out
    x = s["x"].double()
    y = _product64(x, s["w"], case["group"])
    if case["op"] == "gated":
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        else:
            y = y * torch.sigmoid(math.sqrt(8.0 / math.pi) * (y + 0.044715 * y ** 3))
        y = y * _product64(x, s["up"], case["group"])
    elif case["bias"]:
        y = y + s["bias"].double()
    return y
