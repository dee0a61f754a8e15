"""The loss terms where their arithmetic goes to its ends: references far from zero, lists far from zero, sizes just past a kernel's, against 64 bits.

Tolerances are those of test_gpu_losses.py unless a test derives its own."""

import pytest
import torch

from oracle import loss_oracle
from tests.test_gpu_losses import DTYPES, IDS, check_distill, check_top, lists_for, made

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ references far from zero
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.5, 2.0, 2.5, 4.0])
def test_top_logits_with_as_many_groups_as_the_list_is_long(temperature, dtype):
    """The last segment of a row has k groups of neighbours, and in one of them all values are below -2: the bound that k of them reach is far below every value."""
    k = 20
    each = 128 // torch.finfo(dtype).bits                       # classes of a group: 16 bytes
    v = 16384 + k * each
    x = made(6, v, dtype, "normal").abs()
    for i, low in enumerate((-2.5, -3.0, -7.75, -20.0, -100.0)):
        x[i, 16384 + (3 * i) * each:16384 + (3 * i + 1) * each] = low
    check_top(x, k, temperature)
    check_top(x[:, :16384 + (k - 1) * each].contiguous(), k - 1, temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -3e29, -1e30, -1e37])
@pytest.mark.parametrize("v,k", [(40, 12), (300, 20), (1000, 64), (2500, 100), (9001, 64), (20000, 128), (70001, 50)])
def test_top_logits_of_classes_masked_with_a_number(v, k, mask, dtype):
    x = made(9, v, dtype, "normal")
    x[0] = mask
    x[1], x[1, v // 2] = mask, 0.25
    x[2, 7:] = mask
    x[3, : v - 7] = mask
    x[4, k - 1:] = mask
    x[5, k:] = mask
    x[6, k + 1:] = mask
    x[7, : v // 2] = mask
    x[8, :: 2] = mask
    for temperature in (1.0, 1.5, 4.0):
        check_top(x, k, temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -3e29, -1e30, -1e37])
@pytest.mark.parametrize("n,v", [(6, 40), (6, 1000), (6, 70001), (70, 2100), (70, 20000), (66, 70001)])
def test_distillation_of_classes_masked_with_a_number(n, v, mask, dtype):
    """The first and the last classes, and all that are not listed; by few rows and by many, which take other kernels."""
    k = 9
    x = made(n, v, dtype, "normal")
    values, indices, rest = lists_for(x, k, 1.5)
    row = torch.arange(n)
    x[:, : v // 3] = torch.where((row % 5 == 0)[:, None].cuda(), mask, x[:, : v // 3].float()).to(dtype)
    x[:, v // 4:] = torch.where((row % 5 == 1)[:, None].cuda(), mask, x[:, v // 4:].float()).to(dtype)
    for i in range(2, n, 5):
        keep = x[i, indices[i]].clone()
        x[i] = mask
        x[i, indices[i]] = keep
    x[3] = mask
    up = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    for with_rest in (True, False):
        top = (values, indices, rest if with_rest else None)
        check_distill(x, top, 1.5, None, "none", up)
        check_distill(x, top, 1.5, None, "sum", None)
