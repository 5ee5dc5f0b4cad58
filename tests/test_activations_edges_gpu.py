"""Activation operators at the edges of what they accept, against their definitions in 64 bits (activation_reference.py)."""

import copy
import ctypes
import io
import threading

import pytest
import torch
from torch import nn

import test_activations_gpu as common
from activation_reference import U32, depth, smallest_half_step, unit_roundoff
from test_activations_gpu import DTYPES, HALF, act, loud, name_of, normal, same_bits

pytestmark = pytest.mark.gpu


def gave_up():
    from optimi_b200 import _lib

    flag = ctypes.c_int(-1)
    assert _lib.LIB.optimi_b200_weight_gradient_status(ctypes.byref(flag)) == 0
    return flag.value


def test_weight_gradients_one_behind_another():
    """Both blocks of a pair stay until the last arrival at their own barriers: blocks as short as they come (one step and two, one
    tile and several), each started where another one has just ended, exact in whole numbers."""
    a = act()
    gen = torch.Generator().manual_seed(5)
    calls = []
    for tokens, outputs, channels in [(1, 8, 32), (64, 8, 32), (65, 264, 40), (130, 600, 300)]:
        x = torch.randint(-3, 4, (tokens, channels), generator=gen).to(torch.bfloat16).cuda()
        grad = (torch.randint(0, 12, (tokens, outputs), generator=gen) == 0).to(torch.bfloat16).cuda()
        calls.append((grad, a.compress(x), (grad.double().t() @ x.double()).to(torch.bfloat16)))
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        for grad, saved, want in calls:
            wrong += (a.weight_gradient(grad, saved) != want).sum()
    assert int(wrong) == 0 and gave_up() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name_of)
def test_exponents_that_are_columns_of_a_table_beyond_32_bits(dtype):
    """Codes close together and exponents 32 KB from row to row: the last rows' lie beyond 2^31 bytes."""
    a = act()
    rows, cols = 70_000, 31
    x = torch.randn((rows, cols), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    dense = a.compress(x)
    table = torch.zeros((rows, 32_768), dtype=torch.uint8, device="cuda")
    table[:, 5:6] = dense.exponents
    wide = a.CompressedActivation(dense.codes, table[:, 5:6], (rows, cols), dtype)
    assert torch.equal(wide.decompress(), dense.decompress())


SCALES = [1e-3, 0.01, 0.02, 1.0, 100.0]  # 0.02: a usual embedding


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("scale", SCALES)
def test_norm_with_the_default_epsilon(scale, dtype, monkeypatch):
    """The formula with 2^-23, forward, kept row and gradients."""
    monkeypatch.setattr(common, "EPS", 2.0**-23)
    x, dy = normal((40, 256), dtype, 1, scale), normal((40, 256), dtype, 3, 0.01)
    w = (1 + 0.1 * normal((256,), torch.float64, 9)).to(dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w)]
    out = act().rms_norm(*leaves)
    common.check_norm_results(x, w, None, dy, None, (out, *torch.autograd.grad(out.output, leaves, dy.cuda()), None))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("eps", [None, 1e-6, 1e-2])
def test_a_prepared_norm_is_the_plain_one(eps, scale, dtype):
    """Value by value, with gradients and without: both are the formula's, off by the float32 operations before the result and by
    one rounding to the type here and two at most there (the normalised value, its product with the weight)."""
    import optimi_b200

    plain = nn.RMSNorm(256, eps=eps)
    with torch.no_grad():
        plain.weight.copy_(1 + 0.1 * normal((256,), torch.float64, 9))
    plain = plain.to(device="cuda", dtype=dtype)
    x = normal((40, 256), dtype, 1, scale).cuda()
    want = plain(x).detach().double()
    prepared = optimi_b200.prepare_for_compressed_activations(plain)
    bound = want.abs() * (3 * unit_roundoff(dtype) + 2 * (depth(256) / 2 + 6) * U32) * 1.01 + 3 * smallest_half_step(dtype)
    trained = prepared(x)
    assert trained.requires_grad and bool(((trained.detach().double() - want).abs() <= bound).all())
    with torch.no_grad():
        assert bool(((prepared(x).double() - want).abs() <= bound).all())


@pytest.mark.parametrize("carrier", ["x", "weight", "residual"])
@pytest.mark.parametrize("grads", [True, False])
def test_forward_mode_tangents_are_refused(carrier, grads):
    """Not dropped: the result would come without a tangent."""
    import torch.autograd.forward_ad as fw

    args = dict(x=normal((5, 64), torch.float32, 1).cuda(), weight=torch.ones(64, device="cuda"), residual=normal((5, 64), torch.float32, 2).cuda())
    want = act().rms_norm(**args)
    with fw.dual_level(), torch.set_grad_enabled(grads):
        dual = dict(args, **{carrier: fw.make_dual(args[carrier], torch.ones_like(args[carrier]))})
        with pytest.raises(RuntimeError, match=f"`{carrier}` carries a forward-mode tangent"):
            act().rms_norm(**dual)
        assert same_bits(act().rms_norm(**args).output, want.output)


def test_autocast_leaves_float64_alone():
    """As it does with the plain layer."""
    import optimi_b200

    model, x = nn.Linear(64, 32).cuda().double(), normal((5, 64), torch.float64, 1).cuda().requires_grad_()
    leaves = [x, *model.parameters()]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = model(x)
        grads = torch.autograd.grad(want.square().sum(), leaves)
        got = optimi_b200.prepare_for_compressed_activations(model)(x)
        assert got.dtype == torch.float64 and torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got.square().sum(), leaves), grads):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="unsupported dtype torch.float64"):
            act().linear(x, model.weight)
        with pytest.raises(RuntimeError, match="`weight` has unsupported dtype torch.float64"):
            act().linear(x.bfloat16(), model.weight)
        with pytest.raises(RuntimeError, match="unsupported dtype"):
            act().linear(torch.zeros(5, 64, dtype=torch.int32, device="cuda"), model.weight.float())
        # float32 and the other 16-bit type are cast, the layer's as the operator's
        y = act().linear(x.float(), model.weight.half(), model.bias.float())
        assert same_bits(y.detach(), nn.functional.linear(x.bfloat16(), model.weight.half().bfloat16(), model.bias.bfloat16()).detach())


@pytest.mark.parametrize("dtype", HALF, ids=name_of)
@pytest.mark.parametrize("cols", [32, 20, 45, 64])
def test_strides_without_meaning(cols, dtype):
    """Those of one row, and that of one group: any number may stand there."""
    a = act()
    x, grad = normal((1, cols), dtype, 1).cuda(), normal((1, 24), dtype, 2).cuda()
    dense = a.compress(x)
    padded, groups = dense.codes.shape[1], dense.exponents.shape[1]
    wider = torch.zeros((1, padded + 16), dtype=torch.int8, device="cuda")
    wider[:, :padded] = dense.codes
    upright = torch.empty_like(dense.codes[0]).copy_(dense.codes[0]).view(-1, 1).t(), dense.exponents[0].clone().view(-1, 1).t()
    assert upright[0].stride() == (1, 1)
    odd = dense.codes.as_strided((1, padded), (7, 1)), dense.exponents.as_strided((1, groups), (0, 1))
    for codes, exponents in [(wider, dense.exponents), upright, odd]:
        saved = a.CompressedActivation(codes, exponents, (cols,), dtype)
        assert same_bits(saved.decompress(), dense.decompress()[0])
        assert same_bits(a.weight_gradient(grad, saved), a.weight_gradient(grad, dense))
        w = normal((24, cols), dtype, 3).cuda().requires_grad_()
        assert same_bits(torch.autograd.grad(a.linear(x, w, saved=saved), w, grad)[0], a.weight_gradient(grad, dense))
    if groups == 1:
        many = a.compress(normal((9, cols), dtype, 4).cuda())
        lying = torch.zeros((1, 9), dtype=torch.uint8, device="cuda")
        lying[0] = many.exponents[:, 0]
        assert lying.t().stride() == (1, 9)
        assert same_bits(a.CompressedActivation(many.codes, lying.t(), (9, cols), dtype).decompress(), many.decompress())


@pytest.mark.parametrize("shape", [(5, 40, 0), (5, 0, 7), (0, 40, 7), (0, 0, 0)], ids=str)
def test_a_linear_layer_without_tokens_channels_or_outputs(shape):
    tokens, channels, outputs = shape
    x, w, b = (torch.ones(s, dtype=torch.bfloat16, device="cuda", requires_grad=True) for s in ((tokens, channels), (outputs, channels), (outputs,)))
    y = act().linear(x, w, b)
    for got, want in zip(torch.autograd.grad(y, (x, w, b), torch.ones_like(y)), torch.autograd.grad(nn.functional.linear(x, w, b), (x, w, b), torch.ones_like(y))):
        assert got.shape == want.shape and got.dtype == want.dtype and torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_lazily_negated_weights_and_scales(dtype):
    """Views whose memory holds the opposite, as the imaginary part of a conjugate is."""
    a = act()
    x, r, dy, w = (normal(s, dtype, i).cuda() for i, s in enumerate([(6, 40), (6, 40), (6, 40), (40,)]))
    negated = torch._neg_view(-w)
    assert negated.is_neg() and negated.is_contiguous() and same_bits(negated.clone(), w)
    saved = a.compress(x)
    assert same_bits(a.CompressedActivation(saved.codes, saved.exponents, (6, 40), dtype, negated).decompress(),
                     a.CompressedActivation(saved.codes, saved.exponents, (6, 40), dtype, w).decompress())  # fmt: skip
    results = []
    for weight in (negated, w):
        leaves = [t.detach().requires_grad_() for t in (x, weight, r)]
        out = a.rms_norm(*leaves)
        results.append([out.output.detach(), out.saved.decompress(), *torch.autograd.grad(out.output, leaves, dy)])
        results[-1].append(a.rms_norm(torch._neg_view(-x), weight, torch._neg_view(-r)).output)
        if dtype != torch.float32:
            results[-1].append(a.weight_gradient(torch._neg_view(-dy), out.saved))
    for got, want in zip(*results):
        assert same_bits(got, want)


def test_a_norms_output_is_saved_and_copied_without_its_row():
    import optimi_b200

    model = nn.Sequential(nn.RMSNorm(64), nn.Linear(64, 32, bias=False)).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    y = model[0](normal((40, 64), torch.bfloat16, 1).cuda())
    files = [io.BytesIO(), io.BytesIO()]
    torch.save(y, files[0])
    torch.save(y.detach().clone(), files[1])
    assert abs(files[0].tell() - files[1].tell()) < 1000  # the row is 40 * 66 bytes
    files[0].seek(0)
    loaded = torch.load(files[0], weights_only=True)
    assert same_bits(loaded.detach(), y.detach())
    dy = normal((40, 32), torch.bfloat16, 2).cuda()
    for other in (loaded, copy.copy(y)):
        (dw,) = torch.autograd.grad(model[1](other), model[1].weight, dy)
        assert same_bits(dw, act().weight_gradient(dy, act().compress(other.detach())))


def through_torch(function, x):
    return torch.utils.checkpoint.checkpoint(function, x, use_reentrant=False)


def through_torch_on_cpu(function, x):
    with torch.autograd.graph.save_on_cpu():
        return through_torch(function, x)


def through_eight_bits(function, x):
    return act().checkpoint(function, x)


def through_both(function, x):
    return through_eight_bits(lambda t: through_torch(function, t), x)


@pytest.mark.parametrize("through", [through_torch, through_torch_on_cpu, through_eight_bits, through_both])
def test_recomputed_layers_behind_a_norm(through):
    """The norm within the block that is run again: its row is shared, as without recomputation.  The norm before it: the layer keeps
    its input itself, in both runs."""
    import optimi_b200

    torch.manual_seed(0)
    norm, layers = nn.RMSNorm(64), nn.ModuleList([nn.Linear(64, 32), nn.Linear(64, 32)])
    model = nn.ModuleList([norm, layers]).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    a = act()
    x = a.decompress(a.compress(normal((40, 64), torch.bfloat16, 1).cuda()))  # 8 bits hold it exactly
    x.requires_grad_()
    leaves, dy = [x, *model.parameters()], normal((40, 32), torch.bfloat16, 2).cuda()

    def both(t):
        y = norm(t)
        return layers[0](y) + layers[1](y)

    plain = both(x * 1.0)
    want = torch.autograd.grad(plain, leaves, dy)
    again = through(both, x * 1.0)
    assert same_bits(again.detach(), plain.detach())
    for got, expected in zip(torch.autograd.grad(again, leaves, dy), want):
        assert same_bits(got, expected)

    y = norm(x * 1.0)
    outside = through(lambda t: layers[0](t) + layers[1](t), y)
    assert same_bits(outside.detach(), plain.detach())
    got = torch.autograd.grad(outside, leaves, dy)
    for i, layer in enumerate(layers):
        assert same_bits(got[2 + 2 * i], a.weight_gradient(dy, a.compress(y.detach())))
        assert same_bits(got[3 + 2 * i], want[3 + 2 * i])
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])


def test_a_norm_and_a_layer_under_the_same_hooks_share_the_row():
    import optimi_b200

    model = nn.Sequential(nn.RMSNorm(64), nn.Linear(64, 32, bias=False)).to(device="cuda", dtype=torch.bfloat16)
    optimi_b200.prepare_for_compressed_activations(model)
    x, dy = normal((40, 64), torch.bfloat16, 1).cuda(), normal((40, 32), torch.bfloat16, 2).cuda()
    row = act().rms_norm(x, model[0].weight, compress=True).saved
    with torch.autograd.graph.save_on_cpu():
        out = model(x)
    assert same_bits(torch.autograd.grad(out, model[1].weight, dy)[0], act().weight_gradient(dy, row))
    y = model[0](x)
    with torch.autograd.graph.save_on_cpu():
        out = model[1](y)
    assert same_bits(torch.autograd.grad(out, model[1].weight, dy)[0], act().weight_gradient(dy, act().compress(y.detach())))


@pytest.mark.parametrize("prepared", [True, False], ids=["prepared layers", "operators"])
def test_a_row_made_on_one_stream_and_read_on_another(prepared):
    """The weight gradient alone is asked for, late on the layer's stream; the graph and the row are dropped at once, and the norm's
    stream takes memory of the row's size and writes to it."""
    import optimi_b200

    a = act()
    norm, layer = nn.RMSNorm(512), nn.Linear(512, 256, bias=False)
    model = nn.Sequential(norm, layer).to(device="cuda", dtype=torch.bfloat16)
    if prepared:
        optimi_b200.prepare_for_compressed_activations(model)
    x, dy = normal((3000, 512), torch.bfloat16, 1).cuda().requires_grad_(), normal((3000, 256), torch.bfloat16, 2).cuda()
    row = a.rms_norm(x.detach(), norm.weight.detach(), eps=2.0**-23, compress=True).saved
    want, size = a.weight_gradient(dy, row), row._tensors()[0].numel()
    del row
    side = torch.cuda.Stream()
    for _ in range(3):
        if prepared:
            y, saved = norm(x), None
        else:
            y, _, saved = a.rms_norm(x, norm.weight)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y.record_stream(side), dy.record_stream(side)
            out = layer(y) if prepared else a.linear(y, layer.weight, saved=saved)
            torch.cuda._sleep(20_000_000)  # about ten milliseconds
            (dw,) = torch.autograd.grad(out, layer.weight, dy)
        del y, saved, out
        taken = [torch.full((size,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        assert same_bits(dw, want)
        del taken


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_norms_from_two_threads(dtype):
    """Forward, kept row and gradients on two streams at once: the bits of the calls alone."""
    a = act()
    leaves = [t.cuda().requires_grad_() for t in (loud((700, 512), dtype, 1), (1 + 0.1 * normal((512,), torch.float64, 9)).to(dtype), normal((700, 512), dtype, 2))]
    grads = normal((700, 512), dtype, 3).cuda(), normal((700, 512), dtype, 4).cuda()

    def call():
        out = a.rms_norm(*leaves)
        return [out.output.detach(), out.residual.detach(), out.saved.codes, out.saved.exponents, *torch.autograd.grad(out[:2], leaves, grads)]

    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    failures = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    failures.extend(i for i, (got, expected) in enumerate(zip(call(), want)) if not torch.equal(got, expected))
        except RuntimeError as e:
            failures.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
