"""Forms of the group-norm and linear operators: the checks on the CPU, and what the plans choose for the GPU."""
import random

import pytest
import torch

from distributedpytorch_amd.models.factory import get_model
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import Mlp
from distributedpytorch_amd.ops import hip_train_ops as h
from tests import train_ops_cases as cases
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


def gn_kernels(n, hw, c, groups):
    """(fp32, backward, way, threads, vectors a thread, groups of whole vectors) of a contiguous call, and whether the sums of a wave
    stay in its registers."""
    out = set()
    for f32 in (False, True):
        v = 4 if f32 else 8
        v = 1 if c % v else v
        for bwd in (0, 1):
            way, threads, w, _, r, _, _ = h._gn_plan(n, hw, c, c // groups, v, bwd)
            vectors = way in (h._ONE, h._TWO)
            out.add((f32, bwd, way, threads, r, vectors and c // groups % v == 0))
            out.add((f32, bwd, way, "even" if vectors and w <= 64 and w & (w - 1) == 0 else "odd"))
    return out


def linear_kernels(m, n, k):
    """(direction, fp32, tile or rows of the kernel for few rows, split, way to the bias gradient) of contiguous calls."""
    out = set()
    for f32 in (False, True):
        if m <= (64 if f32 else 32) and k % (4 if f32 else 8) == 0:
            out.add(("fprop", f32, "rows", 16 if m <= 16 else 32 if m <= 32 else 64))
        else:
            tile, splits = h._plan(m, n, k, f32)
            out.add(("fprop", f32, tile, splits > 1))
        tile, splits = h._plan(m, k, n, f32)
        out.add(("dgrad", f32, tile, splits > 1))
        tile, splits = h._plan(n, k, m, f32)
        steps = h._cdiv(m, 32 if tile >= 4 else 64) * (6 if f32 and tile < 4 else 1)
        parts = h._cdiv(steps, h._cdiv(steps, splits))
        out.add(("wgrad", f32, tile, "a pass" if tile == 0 else "joined with the parts" if parts > 1 else "direct" if steps <= 16 else "joined"))
    return out


def test_every_kernel_of_a_plan_has_a_case():
    """Whatever the plans choose over wide ranges of sizes is compared with its 64-bit definition on the GPU."""
    rng = random.Random(1)
    size = lambda bits: int(2 ** rng.uniform(0, bits))  # noqa: E731
    there = set().union(*(gn_kernels(n, hh * w, c, g) for n, hh, w, c, g, *_ in cases.GN + forms.GN if n))
    for _ in range(40000):
        n, hw, per, groups = size(9), size(14), size(8), rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
        per = max(8, per // 8 * 8) if rng.random() < 0.6 else per
        missing = gn_kernels(n, hw, per * groups, groups) - there
        assert not missing, (missing, (n, hw, per * groups, groups))
    there = set().union(*(linear_kernels(m, n, k) for m, n, k, *_ in cases.LINEAR + forms.LINEAR if m))
    for _ in range(60000):
        m, n, k = size(15), size(14), size(14)
        if rng.random() < 0.6:
            n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
        missing = linear_kernels(m, n, k) - there
        assert not missing, (missing, (m, n, k))


@pytest.mark.parametrize("name", sorted(forms.SHARED))
def test_shared_memory_is_refused(name):
    forms.check_shared(name, "cpu")


def test_neighbours_in_a_buffer():
    forms.check_neighbours("cpu")


@pytest.mark.parametrize("case", forms.FAR, ids=str)
def test_means_far_from_zero(case):
    forms.check_far_means(case, "cpu")


def test_sums_over_many_rows():
    forms.check_long_sums("cpu")
