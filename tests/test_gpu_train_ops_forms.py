"""Every kernel of the group-norm and linear operators against 64-bit definitions."""
import pytest
import torch

from distributedpytorch_amd import ops
from tests import train_ops_cases as cases
from tests import train_ops_forms as forms
from tests import train_ops_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", forms.DRES, ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dresidual_without_a_residual(case, act, dtype):
    forms.check_dresidual_alone(case, act, dtype, "cuda")


@pytest.mark.parametrize("widths", forms.NARROW, ids=str)
def test_narrow_hidden_layers(widths):
    forms.check_narrow_mlp(widths, "cuda")


@pytest.mark.parametrize("dtype,n,c,groups", [(torch.bfloat16, (1 << 24) + 3, 8, 1), (torch.float32, (1 << 23) + 1, 16, 16)])
def test_group_norm_of_more_images_than_a_launch_has_blocks(dtype, n, c, groups):
    """One pixel an image: every 256 threads of a launch would have one of 2^24 chunks."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, 1, 1, c, device="cuda", generator=g).to(dtype) for _ in range(2))
    gamma, beta = torch.rand(c, device="cuda", generator=g) + 0.5, torch.randn(c, device="cuda", generator=g)
    y, dx = (torch.full_like(x, float("nan")) for _ in range(2))
    (mean, rstd), (dg, db) = torch.empty(2, n, groups, device="cuda"), torch.empty(2, c, device="cuda")
    ops.group_norm_fwd(x, gamma, beta, groups, 1e-5, y, mean, rstd, act="silu")
    ops.group_norm_bwd(dy, x, gamma, beta, groups, mean, rstd, dx, dg, db, act="silu")
    sums, few = torch.zeros(4, c, dtype=torch.float64), 1 << 14
    for lo in (0, n // 2, n - few):
        sl = slice(lo, lo + few)
        px, pdy, py, pdx, pm, pr, pg, pb = (t.cpu() for t in (x[sl], dy[sl], y[sl], dx[sl], mean[sl], rstd[sl], gamma, beta))
        want, wm, wr, e_y, e_m, e_r = O.gn_forward(px, pg, pb, groups, 1e-5, "silu", None)
        O.close("mean", pm, wm, e_m)
        O.close("rstd", pr, wr, e_r)
        O.close("y", py, want, e_y, dtype)
        want, err = O.gn_backward(pdy, px, pg, pb, groups, pm, pr, "silu", None, None)
        O.close("dx", pdx, want[0], err[0], dtype)
    for lo in range(0, n, 1 << 20):
        sl = slice(lo, lo + (1 << 20))
        per = lambda t: t[sl].double().repeat_interleave(c // groups, 1)  # noqa: E731
        xhat = (x[sl].double().view(-1, c) - per(mean)) * per(rstd)
        dz = dy[sl].double().view(-1, c) * O.phi(xhat * gamma.double() + beta.double(), "silu")[1]
        sums += torch.stack([t.cpu().sum(0) for t in (dz * xhat, dz, (dz * xhat).abs(), dz.abs())])
    # 64 rows of at most 2^18 images behind one another: as many roundings, each of at most half a step of the sum of magnitudes,
    # and 64 elementwise ones (a derivative's is relative to 1: 64 of |dy xhat|, at most four times |dz xhat| in the sum)
    for name, got, want, mag in (("dgamma", dg, sums[0], sums[2]), ("dbeta", db, sums[1], sums[3])):
        O.close(name, got, want, (2 ** 18 + 256) * O.E * mag)


def test_more_columns_than_a_launch_of_the_kernel_for_few_rows_has():
    n, k = (1 << 27) + 5, 8
    g = torch.Generator(device="cuda").manual_seed(2)
    w, x = torch.randn(n, k, device="cuda", generator=g, dtype=torch.bfloat16), torch.randn(1, k, device="cuda", generator=g, dtype=torch.bfloat16)
    y = torch.full((1, n), float("nan"), device="cuda", dtype=torch.bfloat16)
    ops.linear_fprop(x, w, y)
    for sl in (slice(0, 1 << 16), slice((1 << 26) - 77, (1 << 26) + 77), slice(n - (1 << 16), n)):
        want, err = O.product(x.cpu(), w[sl].cpu())
        O.close("y", y[:, sl], want, err, torch.bfloat16)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("case", forms.INF, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_in_a_product(case, dtype):
    forms.check_infinities(case, dtype, "cuda")


@pytest.mark.parametrize("case", forms.GN, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm(case, dtype):
    cases.check_group_norm(case, dtype, "cuda")


@pytest.mark.parametrize("case", forms.LINEAR, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear(case, dtype):
    cases.check_linear(case, dtype, "cuda")


@pytest.mark.parametrize("name", sorted(forms.SHARED))
def test_shared_memory_is_refused(name):
    forms.check_shared(name, "cuda")


def test_neighbours_in_a_buffer():
    forms.check_neighbours("cuda")


@pytest.mark.parametrize("case", forms.FAR, ids=str)
def test_means_far_from_zero(case):
    forms.check_far_means(case, "cuda")


def test_sums_over_many_rows():
    forms.check_long_sums("cuda")
