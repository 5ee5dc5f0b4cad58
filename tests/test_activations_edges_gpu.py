"""Activation operators at the edges of what they accept, against their definitions in 64 bits (activation_reference.py)."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def act():
    from optimi_b200 import activations

    return activations


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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
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
