"""Every kernel of the group-norm and linear operators against 64-bit definitions."""
import pytest
import torch

from tests import train_ops_forms as forms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", forms.DRES, ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dresidual_without_a_residual(case, act, dtype):
    forms.check_dresidual_alone(case, act, dtype, "cuda")


@pytest.mark.parametrize("widths", forms.NARROW, ids=str)
def test_narrow_hidden_layers(widths):
    forms.check_narrow_mlp(widths, "cuda")
