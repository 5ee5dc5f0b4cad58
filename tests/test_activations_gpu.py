"""Activation kernels against their definitions in 64 bits (activation_reference.py).

Tolerances count roundings.  One rounding to the result's type is off by at most u = eps / 2 of it (or half a subnormal
step); a float32 operation by U32 = 2^-24 of its result; a float32 sum of n terms by depth(n) * U32 of the sum of
magnitudes, depth(n) being the most additions one term goes through.
"""

import copy

import pytest
import torch
from torch import nn

from activation_reference import GROUP, RANGE, U32, decode, depth, encode, smallest_half_step, unit_roundoff, units

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = [torch.bfloat16, torch.float16]
IDS = {torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "fp32"}


def name_of(dtype):
    return IDS.get(dtype, str(dtype))


def act():
    from optimi_b200 import activations

    return activations


def normal(shape, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(dtype)


def loud(shape, dtype, seed=0):
    """Near normal with a few loud channels, as decoders' activations are."""
    x = normal(shape, torch.float64, seed)
    x[..., :: max(1, shape[-1] // 3)] *= 20
    return x.to(dtype)


def same_bits(a, b):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def same_values(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


# ---------------------------------------------------------------------------------------------
# compress / decompress: no rounding but the one to codes, so everything is equal
# ---------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 64), (7, 100), (2, 8, 1000), (129, 128), (33, 2816), (4, 4097), (1, 16384), (300, 16), (2, 3, 5, 72)]


def check_compressed(x, saved, out):
    x = x.detach().cpu()
    m = x.reshape(-1, x.shape[-1])
    codes, exps = encode(m, x.dtype)
    assert torch.equal(saved.exponents.cpu(), exps)
    assert torch.equal(saved.codes.cpu(), codes)
    want = decode(codes, exps, m.shape[1]).to(x.dtype)
    assert out.shape == x.shape and out.dtype == x.dtype
    assert same_values(out.cpu().reshape(m.shape), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_compress_and_restore(shape, dtype):
    x = loud(shape, dtype).cuda()
    saved = act().compress(x)
    check_compressed(x, saved, act().decompress(saved))
    assert saved.nbytes == saved.codes.shape[0] * (saved.codes.shape[1] * 33 // 32)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("cols", [32, 45, 256])
def test_compress_borders(cols, dtype):
    """Zeros, subnormals, the largest values, ties of the rounding, the border of the exponent, infinities and NaNs."""
    info = torch.finfo(dtype)
    tiny, top = info.smallest_normal, info.max
    rows = []
    for a in [0.0, tiny, tiny * info.eps, top, top / 2, 1.9921875, 1.984375, 127.5, 127.0, 63.75, 1.0, 2.0**-10, 2.0**-40 if dtype != torch.float16 else 2.0**-12,
              float("inf"), float("-inf"), float("nan")]:  # fmt: skip
        for sign in (1.0, -1.0):
            row = (torch.arange(cols, dtype=torch.float64) - cols / 2) / cols * (a if abs(a) < float("inf") else 1.0)
            row[cols // 2] = sign * a
            rows.append(row)
    half = torch.arange(cols, dtype=torch.float64) - 16.5  # exact ties beside 127: 100.5 rounds to 100, 101.5 to 102
    half[0] = 127.0
    rows.append(half)
    x = torch.stack(rows).to(dtype).cuda()
    saved = act().compress(x)
    check_compressed(x, saved, act().decompress(saved))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_a_restored_tensor_is_kept_exactly(dtype):
    x = loud((50, 1000), dtype).cuda()
    once = act().decompress(act().compress(x))
    assert same_bits(act().decompress(act().compress(once)), once)
    # half a step of the group at most
    unit = units(act().compress(x).exponents).repeat_interleave(GROUP, 1)[:, :1000]
    assert bool(((once.double() - x.double()).abs() <= unit / 2).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_compress_strides_and_empty_tensors(dtype):
    a = act()
    base = loud((64, 192), dtype).cuda()
    for x in [base[:, :100], base[:, 1:33], base[::2, 8:72], base.t(), base[3:4].expand(7, 192), base[:, :1], base[5], base[:, 4].contiguous(), base[:1, ::2]]:
        saved = a.compress(x)
        check_compressed(x.contiguous(), saved, a.decompress(saved))
    for shape in [(0, 64), (4, 0), (0,), (2, 0, 5)]:
        out = a.decompress(a.compress(torch.empty(shape, dtype=dtype, device="cuda")))
        assert out.shape == shape and out.dtype == dtype


def test_codes_of_a_wider_buffer_and_channel_scale():
    a = act()
    x = loud((9, 100), torch.bfloat16).cuda()
    scale = normal((100,), torch.bfloat16, 3).cuda()
    s = a.compress(x)
    codes = torch.full((12, 160), 77, dtype=torch.int8, device="cuda")
    exps = torch.full((12, 7), 201, dtype=torch.uint8, device="cuda")
    codes[2:11, :128], exps[2:11, :4] = s.codes, s.exponents
    wide = a.CompressedActivation(codes[2:11], exps[2:11], (3, 3, 100), torch.bfloat16, scale)
    want = (decode(s.codes.cpu(), s.exponents.cpu(), 100) * scale.cpu().double()).to(torch.bfloat16).view(3, 3, 100)
    assert same_bits(wide.decompress(), want)
    grad = normal((9, 24), torch.bfloat16, 4).cuda()
    plain = a.CompressedActivation(s.codes, s.exponents, (9, 100), torch.bfloat16, scale)
    assert same_bits(a.weight_gradient(grad, wide), a.weight_gradient(grad, plain))


# ---------------------------------------------------------------------------------------------
# rms_norm
# ---------------------------------------------------------------------------------------------

EPS = 1e-5


def norm_reference(h, weight, eps):
    h = h.double()
    rstd = 1 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    n = h * rstd
    return rstd, n, n if weight is None else n * weight.double()


def check_kept(saved, n, dtype):
    """The codes stand for n up to half a step and the float32 roundings before it; exponents are the definition's, or one
    off where the largest magnitude lies within those roundings of the border."""
    rows, cols = n.shape
    slack = (depth(cols) / 2 + 4) * U32
    v = decode(saved.codes.cpu(), saved.exponents.cpu(), cols)
    unit = units(saved.exponents.cpu()).repeat_interleave(GROUP, 1)[:, :cols]
    assert bool(((v - n).abs() <= unit / 2 + n.abs() * slack).all())
    _, low = encode(n * (1 - slack), dtype)
    _, high = encode(n * (1 + slack), dtype)
    e = saved.exponents.cpu()
    assert bool(((e >= low) & (e <= high)).all())
    assert bool((saved.codes.cpu()[:, cols:] == 0).all())
    return v


def run_norm(x, weight, residual, dy, dh, need_weight=True):
    a = act()
    leaf = lambda t, need=True: None if t is None else t.clone().requires_grad_(need)  # noqa: E731
    x, weight, residual = leaf(x), leaf(weight, need_weight), leaf(residual)
    out = a.rms_norm(x, weight, residual, eps=EPS)
    outs, grads = [out.output], [dy]
    if residual is not None and dh is not None:
        outs.append(out.residual)
        grads.append(dh)
    wanted = [t for t in (x, weight if need_weight else None, residual) if t is not None]
    got = torch.autograd.grad(outs, wanted, grads)
    it = iter(got)
    return out, next(it), next(it) if weight is not None and need_weight else None, next(it) if residual is not None else None


def check_norm(x, weight, residual, dy, dh):
    check_norm_results(x, weight, residual, dy, dh, run_norm(*(None if t is None else t.cuda() for t in (x, weight, residual, dy, dh))))


def check_norm_results(x, weight, residual, dy, dh, results):
    dtype = x.dtype
    u, floor = unit_roundoff(dtype), smallest_half_step(dtype)
    out, dx, dw, dr = results
    cols = x.shape[-1]
    flat = lambda t: t.detach().cpu().reshape(-1, cols)  # noqa: E731
    h = x if residual is None else x + residual
    if residual is not None:
        assert same_bits(out.residual.detach(), h)
    else:
        assert out.residual is None
    rstd, n, y = norm_reference(flat(h), weight, EPS)
    near = (depth(cols) / 2 + 4) * U32  # of rstd, and of what is multiplied by it
    assert out.output.shape == x.shape and out.output.dtype == dtype
    err = (flat(out.output).double() - y).abs()
    assert bool((err <= y.abs() * (u + near + 2 * U32) + floor).all()), (err / y.abs()).max()
    v = check_kept(out.saved, n, dtype)

    g = flat(dy).double()
    gw = g if weight is None else g * weight.double()
    m = (gw * v).mean(dim=1, keepdim=True)
    extra = torch.zeros_like(g) if dh is None or residual is None else flat(dh).double()
    want = rstd * (gw - v * m) + extra
    # g*w and v*m round once, their difference, the product and the sum once each; m is a sum of cols terms; rstd as above
    off = rstd * (gw.abs() + (v * m).abs()) * (near + 6 * U32) + extra.abs() * 2 * U32
    off += rstd * v.abs() * (gw * v).abs().mean(dim=1, keepdim=True) * (depth(cols) + 3) * U32
    err = (flat(dx).double() - want).abs()
    assert bool((err <= want.abs() * u + off * (1 + u) + floor).all()), (err - want.abs() * u - off).max()
    if residual is not None:
        assert same_bits(dr, dx)
    if weight is not None:
        want = (g * v).sum(dim=0)
        # a sum over the tokens in any order: every term goes through at most all additions, and one rounding of its own
        off = (g * v).abs().sum(dim=0) * (g.shape[0] + 1) * U32
        assert bool(((dw.cpu().double() - want).abs() <= want.abs() * u + off * (1 + u) + floor).all())


NORM_SHAPES = [(1, 1), (1, 4096), (5, 31), (3, 32), (2, 9, 64), (65, 100), (300, 128), (17, 1000), (9, 1024), (4, 2816), (3, 4099), (700, 256), (2, 16384), (2, 20000), (1, 40001)]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm_with_residual(shape, dtype):
    w = (1 + 0.1 * normal(shape[-1:], torch.float64, 9)).to(dtype)
    check_norm(loud(shape, dtype, 1), w, normal(shape, dtype, 2, 2.0), normal(shape, dtype, 3, 0.1), normal(shape, dtype, 4, 0.1))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("shape", [(7, 64), (33, 1000), (4, 4097)], ids=str)
@pytest.mark.parametrize("variant", ["no residual", "no weight", "neither", "residual unused"])
def test_norm_variants(shape, dtype, variant):
    w = None if variant in ("no weight", "neither") else (1 + 0.1 * normal(shape[-1:], torch.float64, 9)).to(dtype)
    r = None if variant in ("no residual", "neither") else normal(shape, dtype, 2, 2.0)
    dh = None if r is None or variant == "residual unused" else normal(shape, dtype, 4, 0.1)
    check_norm(loud(shape, dtype, 1), w, r, normal(shape, dtype, 3, 0.1), dh)


@pytest.mark.parametrize("channels", [1, 17, 64, 9000])
def test_norm_weight_gradient_of_many_tokens_keeps_its_digits(channels):
    """float32: terms of either sign all but cancel; added up in 64 bits and rounded once, the result is off by half a step of itself."""
    tokens = 60_000 if channels < 1000 else 3000
    x, dy = normal((tokens, channels), torch.float32, 1).cuda().requires_grad_(), normal((tokens, channels), torch.float32, 2).cuda()
    w = torch.ones(channels, device="cuda").requires_grad_()
    out = act().rms_norm(x, w, eps=EPS)
    (dw,) = torch.autograd.grad(out.output, w, dy)
    v = out.saved.decompress().double()
    want = (dy.double() * v).sum(dim=0)
    # 64-bit sums are off by at most tokens * 2^-53 of the sum of magnitudes, here 7e-12
    slack = (dy.double() * v).abs().sum(dim=0) * tokens * 2.0**-53
    assert bool(((dw.double() - want).abs() <= want.abs() * U32 + slack * 2).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_norm_strides(dtype):
    base, other = loud((40, 3, 160), dtype, 1).cuda(), normal((40, 3, 160), dtype, 2).cuda()
    w = (1 + 0.1 * normal((96,), torch.float64, 9)).to(dtype).cuda()
    for pick in [lambda t: t[:, 1, :96], lambda t: t[:, :, 1:97], lambda t: t[::3, 2, 8:104], lambda t: t[:, 0, :96].unsqueeze(1).expand(40, 2, 96)]:
        x, r = pick(base), pick(other)
        dy, dh = pick(other * 0.1), pick(base * 0.1)
        # rows that begin on 16 bytes are dealt out to the threads in another way than others, and so summed in another order: held to
        # the formula, like every call (clone() would give dense rows, so the leaves are the strided tensors themselves)
        leaves = [t.detach().requires_grad_() for t in (x, w, r)]
        out = act().rms_norm(*leaves, eps=EPS)
        dx, dw, dr = torch.autograd.grad((out.output, out.residual), leaves, (dy, dh))
        check_norm_results(*(t.cpu().contiguous() for t in (x, w, r, dy, dh)), (out, dx, dw, dr))
        assert same_bits(act().rms_norm(x, w, r, eps=EPS).output, out.output.detach())


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_norm_forward_only_and_its_eight_bit_output(dtype):
    a = act()
    x, r = loud((6, 1000), dtype, 1).cuda(), normal((6, 1000), dtype, 2).cuda()
    w = (1 + 0.1 * normal((1000,), torch.float64, 9)).to(dtype).cuda()
    plain = a.rms_norm(x, w, r)
    kept = a.rms_norm(x, w, r, compress=True)
    assert plain.saved is None and same_bits(plain.output, kept.output) and same_bits(plain.residual, kept.residual)
    train = a.rms_norm(x.clone().requires_grad_(), w, r)
    assert same_bits(train.output.detach(), plain.output)
    assert torch.equal(train.saved.codes, kept.saved.codes) and torch.equal(train.saved.exponents, kept.saved.exponents)
    # restored, the output is off by at most half a step of its group times the channel's weight, and two roundings of each
    unit = units(kept.saved.exponents).repeat_interleave(GROUP, 1)[:, :1000]
    back = kept.saved.decompress().double()
    u = unit_roundoff(dtype)
    bound = unit / 2 * w.double().abs() * (1 + 4 * u) + kept.output.double().abs() * (2 * u + depth(1000) * U32)
    assert bool(((back - kept.output.double()).abs() <= bound).all())
    with torch.no_grad():
        assert a.rms_norm(x.clone().requires_grad_(), w, r).saved is None


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_norm_of_rows_with_infinities_nans_and_zeros(dtype):
    x = loud((6, 200), dtype, 1)
    x[1, 5], x[2, 199], x[3] = float("inf"), float("nan"), 0.0
    w = (1 + 0.1 * normal((200,), torch.float64, 9)).to(dtype)
    dy = normal((6, 200), dtype, 3, 0.1)
    out, dx, dw, _ = run_norm(x.cuda(), w.cuda(), None, dy.cuda(), None)
    y, e, dx = out.output.detach().cpu(), out.saved.exponents.cpu(), dx.cpu()
    for row in (0, 4, 5):
        assert torch.isfinite(y[row]).all() and torch.isfinite(dx[row]).all()
    assert bool((y[3] == 0).all()) and bool((e[3] == 0).all())
    # a row of zeros: rstd = eps^-1/2 and no projection
    want = dy[3].double() * w.double() / EPS**0.5
    got = dx[3].double()
    fits = want.abs() < torch.finfo(dtype).max
    assert bool(((got - want).abs()[fits] <= want.abs()[fits] * (unit_roundoff(dtype) + 6 * U32) + smallest_half_step(dtype)).all())
    assert bool(y[1, 5].isnan()) and bool(y[2].isnan().all()) and bool(dx[2].isnan().all()) and bool(dw.isnan().any())


def test_norm_gradient_against_differences():
    """float32: the kernel's gradient of sum(dy * y) + sum(dh * h) against central differences of the 64-bit formula.  What separates
    them is the 8-bit row in the projection: half a step of every value."""
    rows, cols = 3, 64
    x, r = loud((rows, cols), torch.float32, 1), normal((rows, cols), torch.float32, 2)
    w = (1 + 0.1 * normal((cols,), torch.float64, 9)).to(torch.float32)
    dy, dh = normal((rows, cols), torch.float32, 3), normal((rows, cols), torch.float32, 4)
    out, dx, dw, _ = run_norm(*(t.cuda() for t in (x, w, r, dy, dh)))
    h = (x + r).double()

    def value(h, w):
        _, _, y = norm_reference(h, w, EPS)
        return (y * dy.double()).sum(dim=1) + (h * dh.double()).sum(dim=1)

    step = 1e-5
    rstd, n, _ = norm_reference(h, w, EPS)
    unit = units(out.saved.exponents.cpu()).repeat_interleave(GROUP, 1)[:, :cols]
    g = dy.double() * w.double()
    for c in range(cols):
        d = torch.zeros(cols, dtype=torch.float64)
        d[c] = step
        num = (value(h + d, w) - value(h - d, w)) / (2 * step)
        err = (dx.cpu().double()[:, c] - num).abs()
        half = unit / 2
        shift = rstd[:, 0] * (half[:, c] * ((g * n).mean(1).abs() + (g.abs() * half).mean(1)) + n[:, c].abs() * (g.abs() * half).mean(1))
        # differences: third derivative (order rstd^3 * |g| * cols) * step^2, cancellation 1e-16 * |value| / step; float32: 1e-5
        scale = value(h, w).abs() + g.abs().sum(1) * (1 + rstd[:, 0]) ** 3
        assert bool((err <= shift + 1e-5 * scale).all())
        numw = (value(h, (w.double() + d)) - value(h, (w.double() - d))).sum() / (2 * step)
        bound = (dy.double()[:, c].abs() * half[:, c]).sum() + 1e-5 * (1 + scale.sum())
        assert float((dw.cpu().double()[c] - numw).abs()) <= float(bound)


# ---------------------------------------------------------------------------------------------
# weight_gradient
# ---------------------------------------------------------------------------------------------


def check_weight_gradient(grad, saved, dw):
    tokens, outputs = grad.reshape(-1, grad.shape[-1]).shape
    channels = saved.shape[-1]
    u = unit_roundoff(grad.dtype)
    dev = grad.device
    x = decode(saved.codes.cpu(), saved.exponents.cpu(), channels).to(dev)
    g = grad.reshape(tokens, outputs).double()
    want, size = g.t() @ x, g.abs().t() @ x.abs()
    if saved.channel_scale is not None:
        want, size = want * saved.channel_scale.double(), size * saved.channel_scale.double().abs()
    assert dw.shape == (outputs, channels) and dw.dtype == grad.dtype
    # products are exact; the tensor cores add in float32 and may cut off instead of rounding (2^-23 an addition)
    off = size * (2 * tokens + 4) * U32
    err = (dw.double() - want).abs()
    assert bool((err <= want.abs() * u + off * (1 + u) + smallest_half_step(grad.dtype)).all()), (err - want.abs() * u - off).max()
    # over all results together the additions' errors do not pile up in one direction: the result's own rounding dominates
    if tokens and bool(want.norm() > 0):
        assert float(err.norm() / want.norm()) <= u


WG_SHAPES = [  # tokens, outputs, channels
    (1, 1, 1), (1, 16, 16), (1, 512, 4096), (2, 8, 32), (7, 40, 72), (15, 100, 33), (16, 128, 128), (63, 129, 257), (64, 256, 256),
    (65, 255, 300), (128, 1000, 128), (512, 512, 128), (777, 1001, 96), (1000, 64, 2816), (4096, 256, 256), (9000, 72, 40), (300, 4096, 1024),
    # tiles of 384 outputs, the last one 256 wide or less, whole turns and a cut one
    (640, 9600, 1000), (200, 14336, 2048), (2048, 3900, 2900), (64, 6144, 3000), (130, 385, 257), (20000, 400, 130),
]  # fmt: skip


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
@pytest.mark.parametrize("shape", WG_SHAPES, ids=str)
def test_weight_gradient(shape, dtype):
    tokens, outputs, channels = shape
    a = act()
    x, grad = loud((tokens, channels), dtype, 1).cuda(), normal((tokens, outputs), dtype, 2, 0.1).cuda()
    saved = a.compress(x)
    check_weight_gradient(grad, saved, a.weight_gradient(grad, saved))


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_weight_gradient_is_exact_where_no_rounding_happens(dtype):
    """Whole numbers small enough for every sum to be exact in every order: equal to the last bit, so no token, channel or
    output is dropped, doubled or misplaced."""
    a = act()
    gen = torch.Generator().manual_seed(5)
    for tokens, outputs, channels in [(130, 200, 300), (257, 131, 515), (64, 600, 64), (1, 77, 1000), (96, 264, 520)]:
        x = torch.randint(-3, 4, (tokens, channels), generator=gen).to(dtype).cuda()
        grad = (torch.randint(0, 12, (tokens, outputs), generator=gen) == 0).to(dtype).cuda()
        saved = a.compress(x)
        assert same_bits(a.decompress(saved), x)
        want = grad.double().t() @ x.double()
        assert float(want.abs().max()) < 256
        assert torch.equal(a.weight_gradient(grad, saved).double(), want)


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_weight_gradient_strides_and_shapes(dtype):
    a = act()
    x = loud((4, 30, 200), dtype, 1).cuda()
    saved = a.compress(x)
    base = normal((4, 30, 300), dtype, 2, 0.1).cuda()
    for grad in [base, base[..., :104], base[..., 3:104], base[..., 8:80], normal((4, 30, 1), dtype, 3).cuda().expand(4, 30, 64),
                 base.transpose(0, 1).contiguous().transpose(0, 1), normal((), dtype, 4).cuda().expand(4, 30, 40)]:  # fmt: skip
        want = a.weight_gradient(grad.contiguous(), saved)
        assert same_bits(a.weight_gradient(grad, saved), want)
        check_weight_gradient(grad, saved, want)


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_weight_gradient_without_tokens_outputs_or_channels(dtype):
    a = act()
    empty = lambda *s: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    dw = a.weight_gradient(empty(0, 72), a.compress(empty(0, 100)))
    assert dw.shape == (72, 100) and bool((dw == 0).all())
    assert a.weight_gradient(empty(5, 0), a.compress(empty(5, 100))).shape == (0, 100)
    assert a.weight_gradient(empty(5, 72), a.compress(empty(5, 0))).shape == (72, 0)


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_weight_gradient_keeps_nans_where_they_belong(dtype):
    a = act()
    x = normal((70, 256), dtype, 1)
    x[3, 40] = float("inf")
    grad = normal((70, 136), dtype, 2, 0.1)
    grad[60, 17] = float("nan")
    saved = a.compress(x.cuda())
    dw = a.weight_gradient(grad.cuda(), saved).cpu()
    bad = torch.zeros(136, 256, dtype=torch.bool)
    bad[:, 32:64] = True  # the group of the infinity
    bad[17] = True
    assert torch.equal(dw.isnan(), bad)
    assert torch.isfinite(dw[~bad]).all()


def test_no_wait_ran_out():
    import ctypes

    from optimi_b200 import _lib

    flag = ctypes.c_int(-1)
    assert _lib.LIB.optimi_b200_weight_gradient_status(ctypes.byref(flag)) == 0 and flag.value == 0


def test_weight_gradient_same_bits_every_time():
    a = act()
    x, grad = loud((5000, 320), torch.bfloat16, 1).cuda(), normal((5000, 200), torch.bfloat16, 2).cuda()
    saved = a.compress(x)
    first = a.weight_gradient(grad, saved)
    for _ in range(5):
        assert same_bits(a.weight_gradient(grad, saved), first)


# ---------------------------------------------------------------------------------------------
# linear, checkpoint, models
# ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
@pytest.mark.parametrize("bias", [True, False], ids=["bias", "no bias"])
def test_linear(dtype, bias):
    a = act()
    x = loud((3, 50, 96), dtype, 1).cuda().requires_grad_()
    w = normal((72, 96), dtype, 2, 0.1).cuda().requires_grad_()
    b = normal((72,), dtype, 3).cuda().requires_grad_() if bias else None
    dy = normal((3, 50, 72), dtype, 4).cuda()
    y = a.linear(x, w, b)
    assert same_bits(y.detach(), nn.functional.linear(x, w, b).detach())
    got = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy)
    assert same_bits(got[0], dy @ w.detach())
    assert same_bits(got[1], a.weight_gradient(dy, a.compress(x.detach())))
    if bias:
        want = dy.double().sum((0, 1))
        off = dy.double().abs().sum((0, 1)) * 151 * U32
        assert bool(((got[2].double() - want).abs() <= want.abs() * unit_roundoff(dtype) + off * 1.01 + smallest_half_step(dtype)).all())
    # frozen weights keep nothing and give nothing; a frozen input gets no gradient
    y = a.linear(x, w.detach(), b)
    assert same_bits(torch.autograd.grad(y, x, dy)[0], got[0])
    y = a.linear(x.detach(), w, b)
    assert same_bits(torch.autograd.grad(y, w, dy)[0], got[1])
    with torch.no_grad():
        assert same_bits(a.linear(x, w, b), nn.functional.linear(x, w, b))
    vector = x.detach()[0, 0].requires_grad_()
    gw, gx = torch.autograd.grad(a.linear(vector, w, b), (w, vector), dy[0, 0])
    check_weight_gradient(dy[0, :1], a.compress(vector.detach().view(1, -1)), gw)
    assert gx.shape == vector.shape


def test_linear_refusals():
    a = act()
    x, w = torch.zeros(4, 40, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 40, dtype=torch.bfloat16, device="cuda")
    saved = a.compress(x)
    for call, match in [
        (lambda: a.linear(x.float(), w.float()), "float32 is not supported"),
        (lambda: a.linear(x, w.half()), "does not match"),
        (lambda: a.linear(x, w[:, :39]), "do not match"),
        (lambda: a.linear(x, w, torch.zeros(7, dtype=torch.bfloat16, device="cuda")), "do not match|does not match"),
        (lambda: a.linear(x[:3], w, saved=saved), "does not stand for"),
        (lambda: a.linear(x.half(), w.half(), saved=saved), "does not stand for"),
        (lambda: a.weight_gradient(x.float(), saved), "float32"),
        (lambda: a.weight_gradient(x.half(), saved), "does not match"),
        (lambda: a.weight_gradient(x[:3], saved), "numbers of tokens"),
        (lambda: a.compress(x.double()), "unsupported dtype"),
        (lambda: a.compress(torch.zeros((), device="cuda")), "at least one dimension"),
        (lambda: a.rms_norm(x, w[0, :39]), "last dimension"),
        (lambda: a.rms_norm(x, w[0].float()), "does not match"),
        (lambda: a.rms_norm(x, None, x[:2]), "does not match"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
    with pytest.raises(ValueError, match="negative"):
        a.rms_norm(x, eps=-1.0)


def test_norm_and_linears_share_one_kept_row():
    """rms_norm -> three linear layers, as in an attention block: one 8-bit row serves the norm's backward pass and all three
    weight gradients, which take the norm's weight from the columns."""
    a = act()
    dtype = torch.bfloat16
    x, r = loud((100, 256), dtype, 1).cuda().requires_grad_(), normal((100, 256), dtype, 2).cuda().requires_grad_()
    w = (1 + 0.1 * normal((256,), torch.float64, 9)).to(dtype).cuda().requires_grad_()
    mats = [normal((o, 256), dtype, 10 + o, 0.05).cuda().requires_grad_() for o in (64, 32, 32)]
    dys = [normal((100, o), dtype, 20 + o, 0.1).cuda() for o in (64, 32, 32)]
    out = a.rms_norm(x, w, r, eps=EPS)
    ys = [a.linear(out.output, m, saved=out.saved) for m in mats]
    got = torch.autograd.grad(ys + [out.residual], [x, r, w, *mats], dys + [x.detach() * 0.01])
    for m, dy, dw in zip(mats, dys, got[3:]):
        check_weight_gradient(dy, out.saved, dw)
    # the gradient that reaches the norm is the sum of three rounded products
    dy = sum(d @ m.detach() for d, m in zip(dys[1:], mats[1:])) * 0  # shape only
    dy = torch.zeros_like(dy, dtype=torch.float64)
    size = torch.zeros_like(dy)
    for d, m in zip(dys, mats):
        p = d.double() @ m.detach().double()
        dy, size = dy + p, size + p.abs() + d.double().abs() @ m.detach().double().abs() * 65 * U32 / unit_roundoff(dtype)
    h = (x + r).detach()
    rstd, n, _ = norm_reference(h.cpu(), w.detach().cpu(), EPS)
    v = decode(out.saved.codes.cpu(), out.saved.exponents.cpu(), 256)
    g = dy.cpu() * w.detach().cpu().double()
    want = rstd * (g - v * (g * v).mean(1, keepdim=True)) + (x.detach() * 0.01).cpu().double()
    u = unit_roundoff(dtype)
    slack = (size.cpu() * w.detach().cpu().double().abs()) * 3 * u  # three products and two sums, each rounded: 3u of their size covers 5 half steps of parts
    off = rstd * (slack * 2 + v.abs() * (slack * v.abs()).mean(1, keepdim=True) * 2)
    err = (got[0].cpu().double() - want).abs()
    assert bool((err <= off + want.abs() * 2 * u + 1e-6).all())
    assert same_bits(got[0], got[1])


class Block(nn.Module):
    def __init__(self, d, f):
        super().__init__()
        self.norm, self.up, self.gate, self.down = nn.RMSNorm(d), nn.Linear(d, f), nn.Linear(d, f), nn.Linear(f, d)

    def forward(self, x):
        y = self.norm(x)
        return x + self.down(nn.functional.silu(self.gate(y)) * self.up(y))


class Decoder(nn.Module):
    def __init__(self, vocab=200, d=128, f=320, layers=2):
        super().__init__()
        self.embed, self.blocks = nn.Embedding(vocab, d), nn.ModuleList(Block(d, f) for _ in range(layers))
        self.norm, self.head = nn.RMSNorm(d), nn.Linear(d, vocab, bias=False)

    def forward(self, idx, through=None):
        x = self.embed(idx).to(self.head.weight.dtype)
        for b in self.blocks:
            x = b(x) if through is None else through(b, x)
        return self.head(self.norm(x))


def loss_of(model, idx, **kw):
    return nn.functional.cross_entropy(model(idx, **kw).float().flatten(0, 1), idx.flatten())


def decoder(dtype=torch.bfloat16):
    import optimi_b200

    torch.manual_seed(0)
    return optimi_b200.to_low_precision(Decoder(), dtype=dtype, device="cuda")


def saved_bytes(model, idx):
    """Bytes autograd keeps for the backward pass of one step, parameters apart."""
    held = {}
    params = {p.untyped_storage().data_ptr() for p in model.parameters()}

    def pack(t):
        s = t.untyped_storage()
        if s.data_ptr() not in params:
            held[s.data_ptr()] = s.nbytes()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        loss = loss_of(model, idx)
    total = sum(held.values())
    loss.backward()
    return total


def relative(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
def test_prepared_model_forward_gradients_and_memory(dtype):
    import optimi_b200

    idx = torch.randint(0, 200, (8, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    plain, packed = decoder(dtype), decoder(dtype)
    optimi_b200.prepare_for_compressed_activations(packed)
    before = loss_of(plain, idx)
    # the products are the same calls; the norm's last bit may differ from torch's: one rounding of the logits either way
    assert abs(float(loss_of(packed, idx)) - float(before)) <= float(before) * 8 * unit_roundoff(dtype)
    less, more = saved_bytes(packed, idx), saved_bytes(plain, idx)
    # per token, a block keeps 33 bytes for 32 values of the norm's row and of the down projection's input, where it kept two
    # 16-bit rows around the norm and the 16-bit input (the gated activation's own factors stay); so do the last norm and the head
    d, f, tokens = 128, 320, 8 * 64
    assert more - less == tokens * (2 * (2 * (2 * d + f) - (d + f) * 33 // 32) + 2 * 2 * d - d * 33 // 32)
    for (name, p), q in zip(packed.named_parameters(), plain.parameters()):
        # 8 bits off by half a step of 1/64 to 1/127 of a group's largest value, averaged over the tokens: a few percent at most
        assert relative(p.grad, q.grad) < 0.05, (name, relative(p.grad, q.grad))
    optimi_b200.remove_compressed_activations(packed)
    assert float(loss_of(packed, idx)) == float(before)


def test_prepared_model_under_gradient_release_and_accumulation():
    """The framework's own path: gradients released into the optimizer inside the backward pass, activations in 8 bits.  The same
    step as collecting the gradients first, bit for bit."""
    import optimi_b200

    idx = [torch.randint(0, 200, (4, 32), device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(4)]
    results = []
    for release in (False, True):
        model = optimi_b200.prepare_for_compressed_activations(decoder())
        opt = optimi_b200.AdamW(model.parameters(), lr=1e-3, gradient_release=release)
        if release:
            optimi_b200.prepare_for_gradient_release(model, opt)
        for batch in idx:
            loss_of(model, batch).backward()
            if not release:
                opt.step()
                opt.zero_grad()
        torch.cuda.synchronize()
        results.append([p.detach().clone() for p in model.parameters()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_prepared_model_under_autocast():
    import optimi_b200

    torch.manual_seed(0)
    model = Decoder().cuda()
    twin = optimi_b200.prepare_for_compressed_activations(copy.deepcopy(model))
    idx = torch.randint(0, 200, (4, 32), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for m in (model, twin):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = loss_of(m, idx)
        loss.backward()
    for (name, p), q in zip(twin.named_parameters(), model.parameters()):
        assert p.grad.dtype == torch.float32 and relative(p.grad, q.grad) < 0.05, name
    # float32: the linear layers' own forward; a norm's output is within 20 * U32 of torch's, which a logit (a sum of 128 products of
    # about 0.05) sees as 128 * 0.05 * 3 * 20 * U32 = 2.3e-5 at most, three norms together
    assert abs(float(loss_of(twin, idx)) - float(loss_of(model, idx))) < 7e-5


@pytest.mark.parametrize("through", ["torch", "8 bits"])
def test_prepared_model_recomputed_in_the_backward_pass(through):
    """Recomputation makes the same kept rows again: the gradients of the prepared model, bit for bit where the block's input is
    kept as it is."""
    import optimi_b200

    idx = torch.randint(0, 200, (8, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    model = optimi_b200.prepare_for_compressed_activations(decoder())
    loss_of(model, idx).backward()
    want = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    if through == "torch":
        loss_of(model, idx, through=lambda b, x: torch.utils.checkpoint.checkpoint(b, x, use_reentrant=False)).backward()
    else:
        loss_of(model, idx, through=act().checkpoint).backward()
    for n, p in model.named_parameters():
        if through == "torch":
            # (an embedding's gradient is a scatter of additions in no fixed order)
            assert same_bits(p.grad, want[n]) or "embed" in n and relative(p.grad, want[n]) < 1e-5, n
        else:
            assert relative(p.grad, want[n]) < 0.05, n


def test_prepared_norm_without_weight_and_copies_of_a_prepared_model():
    import io

    import optimi_b200

    model = nn.Sequential(nn.RMSNorm(64, elementwise_affine=False), nn.Linear(64, 32)).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    x, dy = normal((40, 64), torch.bfloat16, 1).cuda().requires_grad_(), normal((40, 32), torch.bfloat16, 2).cuda()
    want = torch.autograd.grad(model(x), [x, *model.parameters()], dy)
    out = act().rms_norm(x)
    assert same_bits(want[1], act().weight_gradient(dy, out.saved))
    buf = io.BytesIO()
    torch.save(model, buf)
    buf.seek(0)
    for twin in (copy.deepcopy(model), torch.load(buf, weights_only=False)):
        for a, b in zip(torch.autograd.grad(twin(x), [x, *twin.parameters()], dy), want):
            assert same_bits(a, b)
        optimi_b200.remove_compressed_activations(twin)
        assert type(twin[0]) is nn.RMSNorm and type(twin[1]) is nn.Linear
    assert type(model[1]) is not nn.Linear


def test_a_norm_output_that_was_written_to_is_not_mistaken_for_the_kept_one():
    import optimi_b200

    model = nn.Sequential(nn.RMSNorm(64), nn.Linear(64, 32, bias=False)).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    x, dy = normal((40, 64), torch.bfloat16, 1).cuda(), normal((40, 32), torch.bfloat16, 2).cuda()
    y = model[0](x)
    y.mul_(2)
    model[1](y).backward(dy)
    assert same_bits(model[1].weight.grad, act().weight_gradient(dy, act().compress(y.detach())))


def test_a_norm_output_given_other_memory_is_not_mistaken_for_the_kept_one():
    import optimi_b200

    model = nn.Sequential(nn.RMSNorm(64), nn.Linear(64, 32, bias=False)).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    x, dy = normal((40, 64), torch.bfloat16, 1).cuda(), normal((40, 32), torch.bfloat16, 2).cuda()
    y = model[0](x)
    y.data = y.data * 3
    model[1](y).backward(dy)
    assert same_bits(model[1].weight.grad, act().weight_gradient(dy, act().compress(y.detach())))


def small_chain(dtype=torch.bfloat16):
    a = act()
    x, r = loud((50, 96), dtype, 1).cuda().requires_grad_(), normal((50, 96), dtype, 2).cuda().requires_grad_()
    w = (1 + 0.1 * normal((96,), torch.float64, 9)).to(dtype).cuda().requires_grad_()
    m = normal((40, 96), dtype, 3, 0.1).cuda().requires_grad_()
    b = normal((40,), dtype, 4).cuda().requires_grad_()

    def run():
        out = a.rms_norm(x, w, r, eps=EPS)
        return a.linear(out.output, m, b, saved=out.saved), out.residual

    return [x, r, w, m, b], run, (normal((50, 40), dtype, 5, 0.1).cuda(), normal((50, 96), dtype, 6, 0.1).cuda())


def test_leaf_gradients_are_tensors_of_their_own_and_accumulate():
    leaves, run, grads = small_chain()
    once = [g.clone() for g in torch.autograd.grad(run(), leaves, grads)]
    for _ in range(2):
        torch.autograd.backward(run(), grads)
    assert len({t.grad.data_ptr() for t in leaves}) == len(leaves)
    for t, g in zip(leaves, once):
        assert same_bits(t.grad, g + g)


def test_backward_twice_and_only_through_the_residual():
    leaves, run, grads = small_chain()
    outs = run()
    first = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(outs, leaves, grads)):
        assert same_bits(a, b)
    x, r, w, _, _ = leaves
    gx, gr, gw = torch.autograd.grad(run()[1], (x, r, w), grads[1])
    assert same_bits(gx, grads[1]) and same_bits(gr, grads[1]) and bool((gw == 0).all())


def test_differentiating_a_gradient_is_refused():
    leaves, run, grads = small_chain()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(run(), leaves, grads, create_graph=True)
    x = leaves[0]
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(act().rms_norm(x).output.sum(), x, create_graph=True)


def test_what_is_kept_may_travel_through_saved_tensor_hooks():
    leaves, run, grads = small_chain()
    want = torch.autograd.grad(run(), leaves, grads)
    with torch.autograd.graph.save_on_cpu():
        outs = run()
    for a, b in zip(torch.autograd.grad(outs, leaves, grads), want):
        assert same_bits(a, b)


def test_kept_rows_written_to_are_noticed():
    a = act()
    x = loud((50, 96), torch.bfloat16, 1).cuda().requires_grad_()
    out = a.rms_norm(x)
    out.saved.codes.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.output.sum().backward()


def test_lazily_negated_views():
    a = act()
    z = torch.complex(normal((6, 40), torch.float32, 1), normal((6, 40), torch.float32, 2)).cuda()
    view = z.conj().imag
    assert view.is_neg()
    want = a.compress(view.clone())
    got = a.compress(view)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.exponents, want.exponents)


def test_first_call_of_a_thread():
    """A thread that made no CUDA call yet (as autograd's own, when the input needs no gradient) has no current context."""
    import threading

    a = act()
    x, dy = loud((96, 128), torch.bfloat16, 1).cuda(), normal((96, 64), torch.bfloat16, 2).cuda()
    saved = a.compress(x)
    want = a.weight_gradient(dy, saved)
    torch.empty_like(want), torch.empty_like(want)
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(a.weight_gradient(dy, saved))
        except RuntimeError as e:
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert same_bits(got[0], want)


def test_calls_from_two_threads():
    import threading

    a = act()
    x, dy = loud((300, 512), torch.bfloat16, 1).cuda(), normal((300, 128), torch.bfloat16, 2).cuda()
    saved = a.compress(x)
    want = a.weight_gradient(dy, saved)
    torch.cuda.synchronize()
    failures = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                s = a.compress(x)
                dw = a.weight_gradient(dy, s)
                if not torch.equal(dw, want):
                    failures.append("differs")
                if a.rms_norm(x, eps=EPS).output.shape != x.shape:
                    failures.append("shape")

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_checkpoint_recomputes_from_eight_bits():
    a = act()
    model = decoder()
    idx = torch.randint(0, 200, (8, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    before = loss_of(model, idx)
    loss = loss_of(model, idx, through=a.checkpoint)
    assert float(loss) == float(before)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    before.backward()
    for n, p in model.named_parameters():
        assert relative(got[n], p.grad) < 0.05, n

    # what a block sees the second time is the restored input; masks and leaves are handed over as they are
    x = loud((4, 64), torch.bfloat16, 1).cuda().requires_grad_()
    mask = torch.full((4, 64), float("-inf"), dtype=torch.bfloat16, device="cuda").triu(1)
    seen = []

    def f(t, m):
        seen.append((t.detach().clone(), m))
        return (t * t + m).exp()

    inner = x * 1.5
    a.checkpoint(f, inner, mask).sum().backward()
    assert same_bits(seen[0][0], inner.detach()) and same_bits(seen[1][0], a.decompress(a.compress(inner.detach())))
    assert seen[1][1] is mask or same_bits(seen[1][1], mask)


# ---------------------------------------------------------------------------------------------
# streams, graphs, sizes
# ---------------------------------------------------------------------------------------------


def test_operators_on_a_side_stream():
    a = act()
    x, dy = loud((500, 1024), torch.bfloat16, 1).cuda(), normal((500, 256), torch.bfloat16, 2).cuda()
    want = a.compress(x)
    want_dw, want_back = a.weight_gradient(dy, want), a.decompress(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = a.compress(x)
        dw, back = a.weight_gradient(dy, s), a.decompress(s)
    torch.cuda.current_stream().wait_stream(side)
    assert same_bits(dw, want_dw) and same_bits(back, want_back)


def test_forward_and_backward_inside_a_graph():
    """Captured once and replayed on new inputs: the bits of the eager calls.  Two graphs at once share no scratch."""
    a = act()
    dtype = torch.bfloat16
    w = (1 + 0.1 * normal((512,), torch.float64, 9)).to(dtype).cuda().requires_grad_()
    m = normal((200, 512), dtype, 3, 0.05).cuda().requires_grad_()

    def step(x, r, dy, dh):
        out = a.rms_norm(x, w, r, eps=EPS)
        y = a.linear(out.output, m, saved=out.saved)
        return [y.detach(), out.residual.detach(), *torch.autograd.grad((y, out.residual), (x, r, w, m), (dy, dh))]

    def inputs(seed):
        return [loud((3000, 512), dtype, seed).cuda(), normal((3000, 512), dtype, seed + 1).cuda(), normal((3000, 200), dtype, seed + 2).cuda(),
                normal((3000, 512), dtype, seed + 3).cuda()]  # fmt: skip

    def leaves(ts):
        return [ts[0].clone().requires_grad_(), ts[1].clone().requires_grad_(), ts[2].clone(), ts[3].clone()]

    first, second = inputs(10), inputs(20)
    eager = [[t.clone() for t in step(*leaves(i))] for i in (first, second)]
    static = [leaves(first), leaves(second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            step(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for swap in (0, 1):
        with torch.no_grad():
            for k in (0, 1):
                for dst, src in zip(static[k], (first, second)[k ^ swap]):
                    dst.copy_(src)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, st in zip(graphs, streams):  # both at once
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for k in (0, 1):
            for got, want in zip(outs[k], eager[k ^ swap]):
                assert same_bits(got, want)


def test_kernels_count_as_the_librarys_launches():
    from optimi_b200 import _lib

    a = act()
    x = loud((10, 64), torch.bfloat16).cuda()
    before = _lib.LIB.optimi_b200_launch_count()
    saved = a.compress(x)
    a.decompress(saved)
    a.weight_gradient(x, saved)
    a.rms_norm(x)
    assert _lib.LIB.optimi_b200_launch_count() >= before + 4


def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last rows are the bits of the same rows taken alone."""
    a = act()
    rows, cols = 70_000, 32_768
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for part in x.split(10_000):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.bfloat16))
    assert x.numel() > 2**31
    saved = a.compress(x)
    tail = a.compress(x[-5:])
    assert torch.equal(saved.codes[-5:], tail.codes) and torch.equal(saved.exponents[-5:], tail.exponents)
    back = a.decompress(saved)
    assert same_bits(back[-5:], a.decompress(tail))
    del back
    odd = a.compress(x[:, 1:])  # rows that begin anywhere
    tail = a.compress(x[-5:, 1:].contiguous())
    assert torch.equal(odd.codes[-5:], tail.codes) and torch.equal(odd.exponents[-5:], tail.exponents)
    back = a.decompress(odd)
    assert same_bits(back[-5:], a.decompress(tail))
    del back, odd
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    xg = x.requires_grad_()
    out = a.rms_norm(xg, w)
    dx = torch.autograd.grad(out.output, xg, x.detach())[0]
    xt = x.detach()[-5:].clone().requires_grad_()
    small = a.rms_norm(xt, w)
    assert same_bits(out.output.detach()[-5:], small.output.detach())
    assert same_bits(dx[-5:], torch.autograd.grad(small.output, xt, xt.detach())[0])
    del dx, out, small
    # a gradient whose last tokens lie beyond 32 bits, and codes likewise: zero but for one early and one late token
    grad = x.detach()
    grad[2:-2] = 0
    narrow = a.compress(normal((rows, 64), torch.bfloat16, 4).cuda())
    keep = torch.tensor([0, 1, rows - 2, rows - 1], device="cuda")
    few = a.CompressedActivation(narrow.codes[keep], narrow.exponents[keep], (4, 64), torch.bfloat16)
    check_weight_gradient(grad[keep], few, a.weight_gradient(grad, narrow))
    some = normal((rows, 16), torch.bfloat16, 5).cuda()
    some[2:-2] = 0
    few = a.CompressedActivation(saved.codes[keep], saved.exponents[keep], (4, cols), torch.bfloat16)
    check_weight_gradient(some[keep], few, a.weight_gradient(some, saved))
    del x, xg, xt, saved, some, grad
    # a result of more than 2^31 values: its last rows are those of the last outputs taken alone
    dy, kept = normal((16, 70_008), torch.bfloat16, 6).cuda(), a.compress(normal((16, cols), torch.bfloat16, 7).cuda())
    dw = a.weight_gradient(dy, kept)
    assert dw.numel() > 2**31
    check_weight_gradient(dy[:, -8:].contiguous(), kept, dw[-8:])
