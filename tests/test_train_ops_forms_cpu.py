"""Forms of the group-norm and linear operators: the checks on the CPU, and what the plans choose for the GPU."""
import pytest
import torch

from distributedpytorch_amd.models.factory import get_model
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import Mlp
from tests import train_ops_forms as forms
from tests import train_ops_nets as nets


@pytest.mark.parametrize("case", forms.DRES, ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dresidual_without_a_residual(case, act, dtype):
    forms.check_dresidual_alone(case, act, dtype, "cpu")


@pytest.mark.parametrize("widths", forms.NARROW, ids=str)
def test_narrow_hidden_layers(widths):
    forms.check_narrow_mlp(widths, "cpu")


@pytest.mark.parametrize("hidden", [(1,), (4,), (2, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_classifier_with_narrow_hidden_layers(hidden, dtype):
    dm = nets.model("cpu", dtype, "adamw", head_hidden=hidden)
    dm.train_step(*nets.batch(2, dm.net, dtype, 0))
    assert torch.isfinite(dm.net.store.p).all()


def test_widths_and_channels_are_refused():
    for hidden in ((0,), (8, -1)):
        with pytest.raises(ValueError, match="widths"):
            get_model("resnet", 10, norm="group", head_hidden=hidden)
    store = ParamStore("cpu")
    m = Mlp(store, "m", (16, 8))
    store.finalize()
    with pytest.raises(ValueError, match="m.weight takes 16 channels"):
        m(Context(store, True, Tape()), Act(torch.zeros(2, 1, 1, 24), False))


def test_no_group_norm_plan_is_larger_than_a_launch():
    """A launch has fewer than 2^32 threads; the kernels for any layout loop over images instead."""
    from distributedpytorch_amd.ops import hip_train_ops as h
    for n in (1 << 22, (1 << 23) + 1, 1 << 24, (1 << 27) + 5):
        for c, groups in ((8, 1), (8, 8), (64, 64), (512, 32), (30, 3), (7, 7)):
            for hw in (1, 4, 9):
                for v in (8, 4, 1, 0):
                    if v < 2 or c % v == 0:
                        for bwd in (0, 1):
                            way, threads, w, _, _, s, _ = h._gn_plan(n, hw, c, c // groups, v, bwd)
                            assert way == h._ANY or n * s * (c // (w if way == h._LONE else w * v)) * threads < 1 << 32


@pytest.mark.parametrize("case", forms.INF[:3], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_in_a_product(case, dtype):
    forms.check_infinities(case, dtype, "cpu")
