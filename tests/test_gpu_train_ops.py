"""Group norm, linear products with epilogues and AdamW: the HIP kernels against 64-bit definitions."""
import pytest
import torch

from tests import train_ops_cases as cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", cases.GN, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm(case, dtype):
    cases.check_group_norm(case, dtype, "cuda")


@pytest.mark.parametrize("case", cases.LINEAR, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear(case, dtype):
    cases.check_linear(case, dtype, "cuda")


@pytest.mark.parametrize("sizes", cases.ADAMW, ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(sizes, bits):
    cases.check_adamw(sizes, bits, "cuda")


@pytest.mark.parametrize("name", sorted(cases.REFUSALS))
def test_refusals(name):
    cases.check_refusal(name, "cuda")
