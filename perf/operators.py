"""Activation operators: what is measured, their plain forms, and their values in 64 bits.

Activations that a training step keeps for its backward pass are held as 8-bit codes, one shared power of two for
every 32 neighbouring channels of a token.  Four operators read or write that format:

  checkpoint       an activation stored in 8 bits and restored (what a checkpoint does between forward and backward)
  norm             residual addition and root-mean-square norm, forward only (serving: one token up to a prompt)
  norm_train       the same forward and backward; the normalised row is kept in 8 bits and the backward pass reads it
  weight_gradient  dW = dY^T X of a linear layer whose input X is held in 8 bits (straight from the codes)

Sizes are those of this repository's workloads: the 24-layer GPT-style decoder (d 1024, FFN 4096, batch 8 x 1024 tokens),
the Llama-shaped lists (hidden 1024 / 2048 / 4096, FFN 2816 / 5632 / 14336) and the test models (d 128, vocabulary 1000).
"""

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# smallest and largest power of two a group may carry, so that code * 2^k is exact and finite in the type
LOWEST = {"bf16": -126, "fp16": -24, "fp32": -126}
HIGHEST = {"bf16": 121, "fp16": 9, "fp32": 121}
EPS = 1e-5


def listed():
    return [
        # the input of one small layer of the test models: 8 sequences of 64 tokens, kept in 8 bits
        dict(name="checkpoint small", op="checkpoint", tokens=512, channels=128, dtype="bf16"),
        # the FFN activation of an 8 B-parameter decoder at 8 x 1024 tokens
        dict(name="checkpoint ffn", op="checkpoint", tokens=8192, channels=14336, dtype="bf16"),
        # a ragged packed batch in float32, a width that no group divides
        dict(name="checkpoint ragged fp32", op="checkpoint", tokens=4999, channels=2815, dtype="fp32"),
        # one token of a decoder that answers
        dict(name="norm one token", op="norm", tokens=1, channels=4096, dtype="bf16"),
        # a prompt of several sequences
        dict(name="norm prompt", op="norm", tokens=16384, channels=4096, dtype="bf16"),
        # a norm of the 24-layer decoder, one step of 8 x 1024 tokens
        dict(name="norm_train gpt", op="norm_train", tokens=8192, channels=1024, dtype="bf16"),
        # the hidden size of the 8 B-parameter decoder, 16 x 1024 tokens
        dict(name="norm_train wide", op="norm_train", tokens=16384, channels=4096, dtype="bf16"),
        # a packed batch of odd length in float16, width not a multiple of a group
        dict(name="norm_train ragged fp16", op="norm_train", tokens=3001, channels=1000, dtype="fp16"),
        # a layer of the test models: latency counts
        dict(name="weight_gradient small", op="weight_gradient", tokens=512, outputs=512, channels=128, dtype="bf16"),
        # the up projection of the 24-layer decoder, 8 x 1024 tokens
        dict(name="weight_gradient gpt up", op="weight_gradient", tokens=8192, outputs=4096, channels=1024, dtype="bf16"),
        # the up projection of the 8 B-parameter decoder: hidden 4096, FFN 14336, 8 x 1024 tokens
        dict(name="weight_gradient ffn", op="weight_gradient", tokens=8192, outputs=14336, channels=4096, dtype="bf16"),
        # a head over the test vocabulary on a packed batch of odd length, float16
        dict(name="weight_gradient ragged fp16", op="weight_gradient", tokens=4999, outputs=1001, channels=2815, dtype="fp16"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm spread evenly; half of them multiples of 8 where that fits."""
    n = int(round(low * (high / low) ** rng.random()))
    return max(low, n // 8 * 8) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["checkpoint", "norm", "norm_train", "weight_gradient"])
    if op == "weight_gradient":
        while True:
            case = dict(op=op, tokens=_spread(rng, 1, 16384), outputs=_spread(rng, 16, 14336), channels=_spread(rng, 16, 14336))
            if case["tokens"] * case["outputs"] * case["channels"] <= 8192 * 14336 * 4096:
                break
        return dict(case, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    most = 8192 * 14336 if op == "checkpoint" else 16384 * 4096
    while True:
        case = dict(op=op, tokens=_spread(rng, 1, 65536), channels=_spread(rng, 16, 16384))
        if case["tokens"] * case["channels"] <= most // 2:  # float32 holds twice the bytes
            break
    return dict(case, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _activation(shape, gen, dtype):
    """Activations as decoders have them: near normal, a few channels far louder than the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 0.005
    return x.mul_(torch.where(loud, 20.0, 1.0)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, t, c = DTYPES[case["dtype"]], case["tokens"], case["channels"]
    x = _activation((t, c), gen, dtype)
    if case["op"] == "checkpoint":
        return dict(case, x=x)
    if case["op"] == "weight_gradient":
        # the checkpoint that the forward pass left, in the documented layout, and the gradient that arrives
        codes, exponents = _encode(x.float(), case["dtype"])
        grad = (torch.randn((t, case["outputs"]), generator=gen, device="cuda") * 1e-2).to(dtype)
        pitch = (c + GROUP - 1) // GROUP * GROUP
        held = torch.zeros((t, pitch), dtype=torch.int8, device="cuda")
        held[:, :c] = codes.to(torch.int8)
        return dict(case, codes=held, exponents=exponents.to(torch.uint8), grad=grad)
    state = dict(case, x=x, residual=torch.randn((t, c), generator=gen, device="cuda").mul_(2.0).to(dtype))
    state["weight"] = (1.0 + 0.1 * torch.randn(c, generator=gen, device="cuda")).to(dtype)
    if case["op"] == "norm_train":
        state["grad"] = (torch.randn((t, c), generator=gen, device="cuda") * 1e-2).to(dtype)
        state["grad_residual"] = (torch.randn((t, c), generator=gen, device="cuda") * 1e-2).to(dtype)
        for name in ("x", "residual", "weight"):
            state[name].requires_grad_(True)
    return state


def _encode(v, dtype):
    """Codes in -127..127 (as numbers of v's type) and the groups' exponent bytes of the rows of v."""
    t, c = v.shape
    groups = (c + GROUP - 1) // GROUP
    padded = torch.zeros((t, groups * GROUP), dtype=v.dtype, device=v.device)
    padded[:, :c] = v
    padded = padded.view(t, groups, GROUP)
    # the power of two 2^k with the group's largest magnitude in [63.75, 127.5) of it
    mantissa, exponent = torch.frexp(padded.abs().amax(dim=2))
    k = torch.where(mantissa * 128 >= 127.5, exponent - 6, exponent - 7).clamp(LOWEST[dtype], HIGHEST[dtype])
    codes = (padded * _power(-k).unsqueeze(2)).round().clamp(-127, 127)
    empty = codes.abs().amax(dim=2) == 0
    return codes.view(t, groups * GROUP)[:, :c], torch.where(empty, 0, k + 127)


def _power(k):
    """2^k in 32 bits, k from -126 to 127."""
    return ((k + 127).to(torch.int32) << 23).view(torch.float32)


def _decode(codes, exponents):
    t, c = codes.shape
    scale = (exponents.to(torch.int32) << 23).view(torch.float32)
    return codes * scale.repeat_interleave(GROUP, dim=1)[:, :c]


def run(s):
    if own:
        return _run_own(s)
    dtype = DTYPES[s["dtype"]]
    if s["op"] == "checkpoint":
        return _decode(*_encode(s["x"].float(), s["dtype"])).to(dtype)
    if s["op"] == "weight_gradient":
        x = _decode(s["codes"][:, : s["channels"]].float(), s["exponents"])
        return (s["grad"].float().t() @ x).to(dtype)
    with torch.no_grad():
        # the sum is rounded to the stream's type, and that is what is normalised
        h = (s["x"].float() + s["residual"].float()).to(dtype)
        wide = h.double() if dtype == torch.float32 else h.float()  # a code next to a border needs more than 32 bits
        rstd = torch.rsqrt(wide.square().mean(dim=1, keepdim=True) + EPS)
        normed = wide * rstd
        w = s["weight"].to(wide.dtype)
        y = (normed * w).to(dtype)
        if s["op"] == "norm":
            return {"output": y, "residual": h}
        codes, exponents = _encode(normed, s["dtype"])
        kept = _decode(codes.float(), exponents)
        g = s["grad"].float()
        gw = g * w.float()
        mean = (gw * kept).mean(dim=1, keepdim=True)
        dx = (rstd.float() * (gw - kept * mean) + s["grad_residual"].float()).to(dtype)
        # a sum over all tokens: in 64 bits for float32 results
        dw = (g.to(wide.dtype) * kept.to(wide.dtype)).sum(dim=0).to(dtype)
        return {"output": y, "residual": h, "grad_input": dx, "grad_weight": dw}


def _run_own(s):
    from optimi_b200 import activations

    if s["op"] == "checkpoint":
        return activations.decompress(activations.compress(s["x"]))
    if s["op"] == "weight_gradient":
        saved = activations.CompressedActivation(s["codes"], s["exponents"], (s["tokens"], s["channels"]), DTYPES[s["dtype"]])
        return activations.weight_gradient(s["grad"], saved)
    if s["op"] == "norm":
        with torch.no_grad():
            out = activations.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return {"output": out.output, "residual": out.residual}
    out = activations.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    dx, dw = torch.autograd.grad((out.output, out.residual), (s["x"], s["weight"]), (s["grad"], s["grad_residual"]))
    return {"output": out.output, "residual": out.residual, "grad_input": dx, "grad_weight": dw}


def work(case):
    """One read of every input, one write of every result; the 8-bit form (33 bytes for 32 values) where it has to exist
    between two passes or is an input."""
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["tokens"] * case["channels"]
    if case["op"] == "checkpoint":
        return {"bytes": 2 * n * size + 2 * n * 33 / 32, "flops": 4 * n}
    if case["op"] == "norm":
        return {"bytes": 4 * n * size + case["channels"] * size, "flops": 5 * n}
    if case["op"] == "norm_train":
        return {"bytes": 7 * n * size + 2 * n * 33 / 32 + 2 * case["channels"] * size, "flops": 16 * n}
    o = case["outputs"]
    return {"bytes": case["tokens"] * o * size + n * 33 / 32 + o * case["channels"] * size, "flops": 2 * n * o}


def exact(case, seed):
    """The same from the definitions, in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "checkpoint":
            return _held(s["x"].double(), case)
        if case["op"] == "weight_gradient":
            e = s["exponents"].double()
            unit = torch.where(e > 0, _two_to(e - 127), 0.0)
            group = torch.arange(case["channels"], device="cuda") // GROUP
            x = s["codes"].double()[:, : case["channels"]] * unit[:, group]
            return torch.einsum("to,tc->oc", s["grad"].double(), x)
        h = s["x"].double() + s["residual"].double()
        h = h.to(DTYPES[case["dtype"]]).double()  # the definition normalises the rounded sum
        c = case["channels"]
        root = torch.sqrt((h * h).sum(dim=1) / c + EPS)
        normed = h / root[:, None]
        w = s["weight"].double()
        if case["op"] == "norm":
            return {"output": normed * w, "residual": h}
        kept = _held(normed, case)
        g = s["grad"].double()
        along = torch.einsum("tc,tc,c->t", g, kept, w) / c
        dx = (g * w - kept * along[:, None]) / root[:, None] + s["grad_residual"].double()
        return {"output": normed * w, "residual": h, "grad_input": dx, "grad_weight": torch.einsum("tc,tc->c", g, kept)}


def _two_to(k):
    """2^k in 64 bits, to the bit (pow is off by a unit, which tips values that lie halfway between two codes)."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _held(v, case):
    """What the 8-bit form keeps of v (64 bits): the nearest multiple, ties to even, of the group's power of two, which is the
    smallest one of which the group's largest magnitude, rounded, is at most 127."""
    t, c = v.shape
    out = torch.empty_like(v)
    for first in range(0, c, GROUP):
        part = v[:, first : first + GROUP]
        top = part.abs().amax(dim=1, keepdim=True)
        unit = _two_to(torch.floor(torch.log2(top.clamp_min(2.0**-160))) - 6)
        unit = torch.where(torch.round(top / unit) > 127, unit * 2, unit)
        unit = torch.where(torch.round(top / (unit / 2)) <= 127, unit / 2, unit)  # log2 may round up at a power of two
        unit = unit.clamp(2.0 ** LOWEST[case["dtype"]], 2.0 ** HIGHEST[case["dtype"]])
        out[:, first : first + GROUP] = torch.round(part / unit).clamp(-127, 127) * unit
    return out
