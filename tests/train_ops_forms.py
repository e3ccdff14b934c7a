"""Forms of the group-norm and linear operators that each kernel of theirs has to take, shared by the CPU and GPU tests."""
import torch

from distributedpytorch_amd import ops
from tests import train_ops_cases as cases
from tests import train_ops_oracle as O

# (n, h, w, c, groups): layouts without 16-byte vectors, small and large; with them, an image in one pass and in two
DRES = [(2, 40, 40, 30, 3), (2, 5, 5, 30, 3), (2, 6, 6, 64, 8), (1, 112, 112, 64, 32)]


def check_dresidual_alone(case, act, dtype, device):
    """The gradient under the activation is asked for, and there is no residual."""
    n, h, w, c, groups = case
    gen = torch.Generator().manual_seed(n + h + c)
    x, dy = (torch.randn(n, h, w, c, generator=gen).to(dtype) for _ in range(2))
    gamma, beta = torch.rand(c, generator=gen) + 0.5, 0.5 * torch.randn(c, generator=gen)
    xd, gd, bd = x.to(device), gamma.to(device), beta.to(device)
    y, (mean, rstd) = torch.empty_like(xd), torch.empty(2, n, groups, device=device)
    ops.group_norm_fwd(xd, gd, bd, groups, 1e-5, y, mean, rstd, act=act)
    for mask in (None, y) if act == "relu" else (None,):
        want, err = O.gn_backward(dy, x, gamma, beta, groups, mean.cpu(), rstd.cpu(), act, None if mask is None else mask.cpu(), None)
        dx, dres = (torch.full_like(xd, float("nan")) for _ in range(2))
        dg, db = torch.full((2, c), float("nan"), device=device)
        ops.group_norm_bwd(dy.to(device), xd, gd, bd, groups, mean, rstd, dx, dg, db, act=act, y=mask, dresidual=dres)
        for k, got in enumerate((dx, dg, db, dres)):
            O.close(("dx", "dgamma", "dbeta", "dresidual")[k], got, want[k], err[k], dtype if k in (0, 3) else torch.float32)
