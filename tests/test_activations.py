"""The activation operators' checks of arguments: everything here fails before a device is touched."""

import copy
import ctypes
import os
import subprocess
import warnings

import pytest
import torch
from torch import nn

import optimi_b200
from optimi_b200 import _lib, activations


def saved_on_cpu(rows=4, cols=40, dtype=torch.bfloat16, **kw):
    return activations.CompressedActivation(torch.zeros(rows, 64, dtype=torch.int8), torch.zeros(rows, 2, dtype=torch.uint8), (rows, cols), dtype, **kw)


@pytest.mark.parametrize("call", [
    lambda x: activations.compress(x),
    lambda x: activations.decompress(saved_on_cpu()),
    lambda x: activations.rms_norm(x),
    lambda x: activations.linear(x, torch.zeros(8, 40, dtype=torch.bfloat16)),
    lambda x: activations.weight_gradient(x, saved_on_cpu()),
], ids=["compress", "decompress", "rms_norm", "linear", "weight_gradient"])  # fmt: skip
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(torch.zeros(4, 40, dtype=torch.bfloat16))


def test_compressed_activation_checks_its_buffers():
    codes, exps = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    make = activations.CompressedActivation
    ok = make(codes, exps, (2, 2, 40), torch.float16)
    assert ok.nbytes == 4 * 66 and ok.shape == (2, 2, 40) and "float16" in repr(ok)
    for bad, match in [
        (lambda: make(codes, exps, (4, 40), torch.float64), "dtype"),
        (lambda: make(codes, exps, (), torch.float16), "dimension"),
        (lambda: make(codes.float(), exps, (4, 40), torch.float16), "codes must be int8"),
        (lambda: make(codes, exps, (5, 40), torch.float16), "codes must be int8"),
        (lambda: make(codes, exps, (4, 65), torch.float16), "codes must be int8"),
        (lambda: make(codes, exps[:, :1], (4, 40), torch.float16), "exponents must be uint8"),
        (lambda: make(codes, exps.char(), (4, 40), torch.float16), "exponents must be uint8"),
        (lambda: make(torch.zeros(64, 4, dtype=torch.int8).t(), exps, (4, 40), torch.float16), "contiguous"),
        (lambda: make(torch.zeros(4, 80, dtype=torch.int8), exps, (4, 40), torch.float16), "multiple of 32"),
        (lambda: make(torch.zeros(4, 96, dtype=torch.int8)[:, 1:65], exps, (4, 40), torch.float16), "16-byte aligned"),
        (lambda: make(torch.zeros(1, 64, dtype=torch.int8).expand(4, 64), exps, (4, 40), torch.float16), "overlap"),
        (lambda: make(codes, exps, (4, 40), torch.float16, channel_scale=torch.zeros(41, dtype=torch.float16)), "channel_scale"),
        (lambda: make(codes, exps, (4, 40), torch.float16, channel_scale=torch.zeros(40)), "channel_scale"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_entry_points_reject_bad_arguments_without_launching():
    L = _lib.LIB
    before = L.optimi_b200_launch_count()
    p = ctypes.c_void_p(0x1000)  # never dereferenced
    odd = ctypes.c_void_p(0x1001)

    def refused(rc, text, code=-1):
        assert rc == code and text in L.optimi_b200_last_error(), L.optimi_b200_last_error()

    refused(L.optimi_b200_compress(p, 64, 4, 64, 9, p, 64, p, 2, None), b"dtype")
    refused(L.optimi_b200_compress(p, 64, -1, 64, 1, p, 64, p, 2, None), b"outside")
    refused(L.optimi_b200_compress(p, 64, 1 << 31, 64, 1, p, 64, p, 2, None), b"outside")
    refused(L.optimi_b200_compress(None, 64, 4, 64, 1, p, 64, p, 2, None), b"x is NULL")
    refused(L.optimi_b200_compress(p, 64, 4, 64, 1, None, 64, p, 2, None), b"codes or exponents is NULL")
    refused(L.optimi_b200_compress(p, 64, 4, 64, 1, odd, 64, p, 2, None), b"alignment")
    refused(L.optimi_b200_compress(p, 65, 4, 65, 1, p, 64, p, 3, None), b"pitch")
    refused(L.optimi_b200_compress(p, 64, 4, 64, 1, p, 80, p, 2, None), b"pitch")
    refused(L.optimi_b200_compress(p, 65, 4, 65, 1, p, 96, p, 2, None), b"exponent pitch")
    refused(L.optimi_b200_decompress(p, 64, p, 2, None, 4, 64, 1, None, None), b"out is NULL")
    refused(L.optimi_b200_decompress(p, 32, p, 2, None, 4, 64, 1, p, None), b"pitch")
    norm = [p, 64, None, 0, None, 4, 64, 1e-6, 1, p, None, None, 0, None, 0, None, None]

    def with_(base, **at):
        out = list(base)
        for i, v in at.items():
            out[int(i[1:])] = v
        return out

    refused(L.optimi_b200_rms_norm(*with_(norm, _0=None)), b"x or y is NULL")
    refused(L.optimi_b200_rms_norm(*with_(norm, _2=p)), b"residual and sum")
    refused(L.optimi_b200_rms_norm(*with_(norm, _7=-1.0)), b"eps")
    refused(L.optimi_b200_rms_norm(*with_(norm, _7=float("nan"))), b"eps")
    refused(L.optimi_b200_rms_norm(*with_(norm, _11=p, _12=64, _13=p, _14=2)), b"go together")
    refused(L.optimi_b200_rms_norm(*with_(norm, _15=p)), b"codes or exponents is NULL")
    back = [p, 64, None, 0, p, 64, p, 2, p, None, 400, 64, 1, p, p, p, 1 << 20, None]
    refused(L.optimi_b200_rms_norm_backward(*with_(back, _0=None)), b"grad or rstd is NULL")
    refused(L.optimi_b200_rms_norm_backward(*with_(back, _8=None)), b"grad or rstd is NULL")
    refused(L.optimi_b200_rms_norm_backward(*with_(back, _16=8)), b"workspace", -3)
    refused(L.optimi_b200_rms_norm_backward(*with_(back, _15=None)), b"workspace", -3)
    dw = [p, 64, p, 64, p, 2, None, 4, 64, 64, 1, p, p, 1 << 30, None]
    refused(L.optimi_b200_weight_gradient(*with_(dw, _10=0)), b"neither bfloat16 nor float16")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _8=-3)), b"outside")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _11=None)), b"grad_weight is NULL")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _0=None)), b"grad is NULL")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _3=32)), b"pitch")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _0=ctypes.c_void_p(0x1008))), b"begin on 16 bytes")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _1=68)), b"begin on 16 bytes")
    refused(L.optimi_b200_weight_gradient(*with_(dw, _1=56)), b"begin on 16 bytes")
    refused(L.optimi_b200_weight_gradient_status(None), b"gave_up is NULL")
    refused(L.optimi_b200_align_rows(p, 65, 4, 65, 1, p, 65, None), b"out_stride")
    refused(L.optimi_b200_align_rows(p, 65, 4, 65, 1, odd, 72, None), b"not 16-byte aligned")
    refused(L.optimi_b200_align_rows(None, 65, 4, 65, 1, p, 72, None), b"x or out is NULL")
    refused(L.optimi_b200_align_rows(p, 65, 4, 65, 5, p, 72, None), b"dtype")
    # nothing to do is not an error
    assert L.optimi_b200_compress(None, 0, 0, 64, 1, None, 0, None, 0, None) == 0
    assert L.optimi_b200_rms_norm(*with_(norm, _5=0)) == 0
    assert L.optimi_b200_weight_gradient(*with_(dw, _9=0)) == 0
    assert L.optimi_b200_launch_count() == before


def test_checkpoint_takes_only_the_non_reentrant_form():
    with pytest.raises(ValueError, match="use_reentrant"):
        activations.checkpoint(lambda x: x, torch.zeros(3), use_reentrant=True)


class Tied(nn.Linear):
    pass


def test_preparing_a_model_changes_only_what_it_says():
    model = nn.Sequential(nn.Linear(8, 8), nn.RMSNorm(8), nn.RMSNorm((4, 8)), Tied(8, 8), nn.LayerNorm(8), nn.Sequential(nn.Linear(8, 3)))
    keys = list(model.state_dict())
    x = torch.randn(2, 4, 8)
    want = model(x)
    assert optimi_b200.prepare_for_compressed_activations(model) is model
    kinds = [type(m).__name__ for m in model]
    assert kinds == ["_CompressedLinear", "_CompressedRMSNorm", "RMSNorm", "Tied", "LayerNorm", "Sequential"]
    assert isinstance(model[0], nn.Linear) and isinstance(model[1], nn.RMSNorm) and type(model[5][0]).__name__ == "_CompressedLinear"
    assert list(model.state_dict()) == keys
    with torch.no_grad():  # no gradients: the layers' own forward, wherever the model is
        assert torch.equal(model(x), want)
    assert torch.equal(model[0](x), nn.functional.linear(x, model[0].weight, model[0].bias))  # float32 stays as it is
    with pytest.raises(ValueError, match="already prepared"):
        optimi_b200.prepare_for_compressed_activations(model)
    twin = copy.deepcopy(model)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        twin[0].bfloat16()(x.bfloat16())
    optimi_b200.remove_compressed_activations(twin)
    assert type(twin[0]) is nn.Linear and type(model[0]) is not nn.Linear
    optimi_b200.remove_compressed_activations(model)
    assert [type(m) for m in model] == [nn.Linear, nn.RMSNorm, nn.RMSNorm, Tied, nn.LayerNorm, nn.Sequential]
    assert torch.equal(model(x), want)
    with warnings.catch_warnings(record=True) as caught:
        warnings.simplefilter("always")
        optimi_b200.remove_compressed_activations(model)
    assert any("does not have any compressed activations" in str(w.message) for w in caught)


def test_workspaces_grow_with_the_problem():
    L = _lib.LIB
    assert L.optimi_b200_rms_norm_backward_workspace_bytes(0, 64, 1) == 0
    assert L.optimi_b200_rms_norm_backward_workspace_bytes(1, 64, 1) == 0  # one block adds up the rows itself
    assert 0 < L.optimi_b200_rms_norm_backward_workspace_bytes(100, 64, 1) < L.optimi_b200_rms_norm_backward_workspace_bytes(1000, 64, 1)
    assert L.optimi_b200_rms_norm_backward_workspace_bytes(1000, 64, 9) == 0


@pytest.fixture(scope="module")
def small_offsets(tmp_path_factory):
    """The choice between offsets of 32 and 64 bits, from the header the kernels' launches include, through the host's compiler."""
    where = tmp_path_factory.mktemp("offsets")
    source, lib = where / "offsets.cpp", where / "offsets.so"
    header = os.path.join(os.path.dirname(optimi_b200.__file__), "csrc", "activation_offsets.h")
    source.write_text(f'#include "{header}"\nextern "C" int small(int64_t r, int64_t s, int64_t p, int64_t e) {{ return optimi::act::small_offsets(r, s, p, e); }}\n')
    subprocess.run([_lib._build.find_gxx(), "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(source)], check=True)
    fn = ctypes.CDLL(str(lib)).small
    fn.argtypes = [ctypes.c_int64] * 4
    return lambda *args: bool(fn(*args))


def test_offsets_of_32_bits_only_where_all_of_them_fit(small_offsets):
    assert small_offsets(4096, 4095, 4096, 128) and small_offsets(1, 1, 32, 1)
    assert small_offsets(70_000, 31, 32, 29_000)  # 2.03e9 bytes of exponents from the first row to the last
    # exponents that are columns of a wide table: rows 32 KB apart reach past 2^31
    assert not small_offsets(70_000, 31, 32, 32_768) and not small_offsets(65_536, 31, 32, 32_768)
    assert not small_offsets(70_000, 32_767, 32, 1) and not small_offsets(70_000, 31, 32_768, 1)
    for at in range(3):
        steps = [1, 32, 1]
        steps[at] = 1 << 62  # the product would not fit 64 bits
        assert not small_offsets(1 << 30, *steps)
    # and never where an offset of the last row reaches 2^31
    for rows in (1, 2, 3, 1000, 65_537, (1 << 31) - 1):
        for step in (1, 31, (1 << 31) // rows - 1, (1 << 31) // rows, (1 << 31) // rows + 1):
            for at in range(3):
                steps = [1, 1, 1]
                steps[at] = step
                assert not small_offsets(rows, *steps) or rows * step < 1 << 31


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_an_unaligned_workspace_is_refused(dtype):
    """The kernels write sums of 4 and 8 bytes there."""
    L = _lib.LIB
    p, before = ctypes.c_void_p(0x1000), L.optimi_b200_launch_count()
    for at in (0x1001, 0x1004, 0x1008):
        rc = L.optimi_b200_rms_norm_backward(p, 64, None, 0, p, 64, p, 2, p, None, 400, 64, dtype, p, p, ctypes.c_void_p(at), 1 << 20, None)
        assert rc == -3 and b"16-byte aligned" in L.optimi_b200_last_error()
        if dtype:
            tokens = 64 * 200  # one tile, cut into slices
            assert L.optimi_b200_weight_gradient_workspace_bytes(tokens, 64, 64) > 0
            rc = L.optimi_b200_weight_gradient(p, 64, p, 64, p, 2, None, tokens, 64, 64, dtype, p, ctypes.c_void_p(at), 1 << 30, None)
            assert rc == -3 and b"16-byte aligned" in L.optimi_b200_last_error()
    assert L.optimi_b200_launch_count() == before


@pytest.mark.parametrize("call, modes", [
    (lambda x: activations.compress(x).codes, (True, False)),
    (lambda x: activations.decompress(saved_on_cpu()), (True, False)),
    (lambda x: activations.rms_norm(x).output, (True, False)),
    (lambda x: activations.linear(x, torch.zeros(8, 40, dtype=torch.bfloat16)), (True,)),  # without gradients it is torch's own
    (lambda x: activations.weight_gradient(x, saved_on_cpu()), (True, False)),
], ids=["compress", "decompress", "rms_norm", "linear", "weight_gradient"])  # fmt: skip
def test_traces_are_refused(call, modes):
    """A trace would hold the buffers without the kernels that fill them."""
    for grads in modes:
        with torch.set_grad_enabled(grads), warnings.catch_warnings():
            warnings.simplefilter("ignore")
            with pytest.raises(RuntimeError, match="cannot be recorded by torch.jit.trace"):
                torch.jit.trace(call, (torch.zeros(4, 40, dtype=torch.bfloat16),), check_trace=False)


def test_a_prepared_model_is_traced_as_its_plain_layers():
    model = nn.Sequential(nn.RMSNorm(40), nn.Linear(40, 8)).bfloat16()
    x = torch.randn(4, 40).bfloat16()
    want = model(x)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(optimi_b200.prepare_for_compressed_activations(model), (x,))
    assert torch.equal(traced(x), want)


def test_a_prepared_model_in_float64_stays_as_it_is():
    for model in (nn.Sequential(nn.RMSNorm(40), nn.Linear(40, 8)), nn.Sequential(nn.RMSNorm(40, elementwise_affine=False), nn.Linear(40, 8))):
        model.double()
        x = torch.randn(4, 40, dtype=torch.float64, requires_grad=True)
        want = torch.autograd.grad(model(x).square().sum(), [x, *model.parameters()])
        optimi_b200.prepare_for_compressed_activations(model)
        for got, plain in zip(torch.autograd.grad(model(x).square().sum(), [x, *model.parameters()]), want):
            assert torch.equal(got, plain)
