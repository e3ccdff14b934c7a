"""Group norm, linear products and AdamW on the GPU as programs use them: layers, networks, captured graphs, streams, bad values
in one place, tensors beyond 2^31 elements."""
import pytest
import torch

from distributedpytorch_amd import ops
from distributedpytorch_amd.nn.optim import make_hyper
from tests import train_ops_nets as nets

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("act,mlp_act", [("relu", "relu"), ("silu", "gelu"), ("gelu", "silu"), ("none", "none")])
def test_layers_and_their_gradients(act, mlp_act):
    nets.check_layers("cuda", act, mlp_act)


def test_adamw_follows_torch():
    nets.check_adamw_torch("cuda")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_training(kind, dtype):
    nets.check_training("cuda", dtype, kind, n=16)


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_a_captured_step_equals_the_eager_one(kind):
    """Replays, with the program's own eager steps of the other model and synchronisations between them."""
    a, b = nets.model("cuda", BF, kind), nets.model("cuda", BF, kind)
    batches = [nets.batch(16, a.net, BF, s) for s in range(4)]
    assert b.capture_train_step(*batches[0])
    assert torch.equal(a.net.store.p, b.net.store.p)
    for x, y in batches:
        a.train_step(x, y)
        b.replay_train_step(x, y)
        torch.cuda.synchronize()
        assert torch.equal(a.net.store.p, b.net.store.p)
        for s, t in zip(a.opt.state_tensors(), b.opt.state_tensors()):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
    assert a.epoch_metrics() == b.epoch_metrics()


class Chain:
    """Every operator once: norm and its gradient, products, a step; all outputs in `out`."""

    def __init__(self, dtype, n=6, h=9, w=7, c=64, hid=136, rows=77, seed=0, act="silu"):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, dt=dtype: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
        e = lambda *s, dt=dtype: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
        self.act = act
        self.x, self.res, self.dy = r(n, h, w, c), r(n, h, w, c), r(n, h, w, c)
        self.gamma, self.beta = r(c, dt=F32), r(c, dt=F32)
        self.y, self.dx, self.dres = (e(n, h, w, c) for _ in range(3))
        self.mean, self.rstd, self.dg, self.db = e(n * 8, dt=F32), e(n * 8, dt=F32), e(c, dt=F32), e(c, dt=F32)
        self.a, self.w, self.g = r(rows, c), r(hid, c), r(rows, hid)
        self.bias, self.o, self.z, self.da = r(hid, dt=F32), e(rows, hid), e(rows, hid), e(rows, c)
        self.za = r(rows, c)
        self.dw, self.dbias = e(hid, c, dt=F32), e(hid, dt=F32)
        k = 64 * 37
        self.p, self.grad = r(k, dt=F32), r(k, dt=F32)
        self.m, self.v = torch.zeros(k, device="cuda", dtype=torch.float8_e4m3fn), torch.zeros(k, device="cuda", dtype=torch.float8_e5m2)
        self.ms, self.vs, self.p16 = torch.zeros(37, device="cuda"), torch.zeros(37, device="cuda"), e(k, dt=BF)
        self.hyper = make_hyper(1e-2, 0.9, 0.999, 1e-8, 0.1, 0.0, 0.0, 1.0, device="cuda")
        self.groups, self.ids = torch.ones(1, 2, device="cuda"), torch.zeros(37, device="cuda", dtype=torch.uint8)

    def run(self):
        s = self
        ops.group_norm_fwd(s.x, s.gamma, s.beta, 8, 1e-5, s.y, s.mean, s.rstd, act=s.act, residual=s.res)
        ops.group_norm_bwd(s.dy, s.x, s.gamma, s.beta, 8, s.mean, s.rstd, s.dx, s.dg, s.db, act=s.act, residual=s.res, dresidual=s.dres)
        ops.linear_fprop(s.a, s.w, s.o, s.bias, act=s.act, preact=s.z)
        ops.linear_dgrad(s.g, s.w, s.da, act=s.act, preact=s.za)
        ops.linear_wgrad(s.g, s.a, s.dw, s.dbias)
        ops.adamw8_step(s.p, s.grad, s.m, s.v, s.ms, s.vs, s.p16, s.hyper, s.groups, s.ids, 3)
        ops.advance_step(s.hyper)

    def out(self):
        return [t.clone() for t in (self.y, self.mean, self.rstd, self.dx, self.dres, self.dg, self.db, self.o, self.z, self.da, self.dw,
                                    self.dbias, self.p, self.m.view(torch.uint8), self.v.view(torch.uint8), self.ms, self.vs, self.p16)]

    def feed(self, seed):
        g = torch.Generator(device="cuda").manual_seed(100 + seed)
        for t in (self.x, self.dy, self.res, self.a, self.g, self.grad):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))


def same(a, b):
    for i, (s, t) in enumerate(zip(a, b)):
        assert torch.equal(s, t), i


def capture(c):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    return g


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", [dict(), dict(n=2, h=70, w=61, rows=1, c=64), dict(n=3, h=40, w=40, rows=700, hid=520), dict(c=24, hid=20, rows=5)], ids=str)
def test_two_graphs_and_eager_calls(dtype, shape):
    """Two captured graphs whose replays alternate, on two streams, with eager calls between: each has workspaces of its own."""
    e = [Chain(dtype, seed=i, **shape) for i in range(2)]
    c = [Chain(dtype, seed=i, **shape) for i in range(2)]
    graphs = []
    for i in range(2):
        e[i].run()
        graphs.append(capture(c[i]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for it in range(3):
        for i in range(2):
            for ch in (e[i], c[i]):
                ch.feed(10 * it + i)
        torch.cuda.synchronize()
        for i in range(2):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        for i in range(2):
            e[i].run()
        torch.cuda.synchronize()
        for i in range(2):
            same(e[i].out(), c[i].out())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_another_stream(dtype):
    """Inputs made and used on a side stream, while the current stream is busy; nothing waits for the default stream."""
    a, b = Chain(dtype), Chain(dtype)
    a.feed(1)
    a.run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b.feed(1)
        b.run()
        got = b.out()
    s.synchronize()
    same(a.out(), got)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("hw", [(7, 7), (28, 28), (80, 80)], ids=str)
@pytest.mark.parametrize("c,act", [(64, "relu"), (60, "silu")])
def test_a_bad_value_stays_in_its_group(dtype, hw, c, act):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(3, *hw, c, device="cuda", generator=g).to(dtype)
    dy = torch.randn(3, *hw, c, device="cuda", generator=g).to(dtype)
    gamma, beta = torch.rand(c, device="cuda", generator=g) + 0.5, torch.randn(c, device="cuda", generator=g)

    def run(x, dy):
        y, dx, (m, r) = torch.empty_like(x), torch.empty_like(x), torch.empty(2, 3 * 4, device="cuda")
        ops.group_norm_fwd(x, gamma, beta, 4, 1e-5, y, m, r, act=act)
        ops.group_norm_bwd(dy, x, gamma, beta, 4, m, r, dx, act=act)
        return y, dx
    want = run(x, dy)
    per = c // 4
    for value in (float("nan"), float("inf")):
        xb = x.clone()
        xb[1, 3, 2, per] = value                                   # image 1, group 1
        got = run(xb, dy)
        for a, b in zip(got, want):
            a, b = a.view(3, -1, 4, per), b.view(3, -1, 4, per)
            if act != "relu":                                      # (a ReLU's comparison with a NaN is false)
                assert a[1, :, 1].isnan().all()
            rest = torch.ones(3, 4, dtype=torch.bool, device="cuda")
            rest[1, 1] = False
            assert torch.equal(a.permute(0, 2, 1, 3)[rest], b.permute(0, 2, 1, 3)[rest])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("m,n,k", [(70, 130, 72), (300, 260, 264), (1000, 520, 4100)], ids=str)
def test_a_bad_value_stays_in_its_row(dtype, m, n, k):
    """A NaN in one row of x or one column of dy reaches that row of y and dx, that row of dw and that entry of db, and nothing else."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, dy = (torch.randn(*s, device="cuda", generator=g).to(dtype) for s in ((m, k), (n, k), (m, n)))
    bias = torch.randn(n, device="cuda", generator=g)

    def run(x, dy):
        y, dx, dw, db = torch.empty(m, n, device="cuda", dtype=dtype), torch.empty_like(x), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
        ops.linear_fprop(x, w, y, bias, act="gelu")
        ops.linear_dgrad(dy, w, dx)
        ops.linear_wgrad(dy, x, dw, db)
        return y, dx, dw, db
    want = run(x, dy)
    for value in (float("nan"), float("inf")):
        xb, dyb = x.clone(), dy.clone()
        xb[5, 3], dyb[7, 37] = value, value
        y, _, dwx, _ = run(xb, dy)
        _, dx, dw, db = run(x, dyb)
        rows, cols, outs = (torch.arange(s, device="cuda") for s in (m, k, n))
        for got, ref, rest in ((y, want[0], rows != 5), (dx, want[1], rows != 7), (dw, want[2], outs != 37), (db, want[3], outs != 37)):
            assert torch.equal(got[rest], ref[rest]) and not torch.isfinite(got[~rest]).all()
        assert torch.equal(dwx[:, cols != 3], want[2][:, cols != 3]) and not torch.isfinite(dwx[:, 3]).any()


def check_large(n, h, w, c, groups, dtype, view=lambda t: t):
    """Forward and backward against the formula in 64 bits, on the CPU: torch's sums over many blocks of the GPU do not repeat."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x, dy = (view(torch.randn(n, h, w, c, device="cuda", generator=g).to(dtype)) for _ in range(2))
    ga, be = torch.rand(c, device="cuda", generator=g) + 0.5, torch.randn(c, device="cuda", generator=g)
    y, dx = (view(torch.empty(n, h, w, c, device="cuda", dtype=dtype)) for _ in range(2))
    mean, rstd, dg, db = *torch.empty(2, n * groups, device="cuda"), *torch.empty(2, c, device="cuda")
    ops.group_norm_fwd(x, ga, be, groups, 1e-5, y, mean, rstd, act="silu")
    ops.group_norm_bwd(dy, x, ga, be, groups, mean, rstd, dx, dg, db, act="silu")
    half = nets.E if dtype == F32 else 2.0 ** -8
    tol = half + 1024 * nets.E          # (512 roundings of a statistic, each way)
    sg, sb, k = torch.zeros(c, dtype=torch.float64), torch.zeros(c, dtype=torch.float64), c // groups
    x, dy, y, dx, ga, be, dg, db = (t.cpu() for t in (x, dy, y, dx, ga, be, dg, db))
    for i in range(n):
        xd = x[i].double().reshape(-1, groups, k)
        mu = xd.mean((0, 2))
        rs = 1 / ((xd - mu[:, None]).square().mean((0, 2)) + 1e-5).sqrt()
        xh = ((xd - mu[:, None]) * rs[:, None]).reshape(-1, c)
        u = xh * ga + be
        s = torch.sigmoid(u)
        assert nets.rel(y[i].reshape(-1, c), u * s) <= tol
        dz = dy[i].double().reshape(-1, c) * s * (1 + u * (1 - s))
        t = (dz * ga).reshape(-1, groups, k)
        h2 = xh.reshape(-1, groups, k)
        want = rs[:, None] * (t - t.mean((0, 2))[:, None] - h2 * (t * h2).mean((0, 2))[:, None])
        assert nets.rel(dx[i].reshape(-1, c), want.reshape(-1, c)) <= tol
        sg += (dz * xh).sum(0)
        sb += dz.sum(0)
    # a sum of n random terms is near their root: 1024 roundings of sum |dz| are sqrt(n) times as many of the sum
    for got, want in ((dg, sg), (db, sb)):
        assert float((got.double() - want).abs().max()) <= 1024 * nets.E * n * h * w * 3


@pytest.mark.parametrize("dtype", [F32, BF])
def test_group_norm_of_a_large_image(dtype):
    check_large(1, 1500, 1050, 8, 2, dtype)
    check_large(2, 512, 999, 6, 3, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("wide", [(1 << 18) - 8, 1 << 18, (1 << 20) + 8])
def test_group_norm_of_pixels_far_apart(dtype, wide):
    check_large(2, 9, 3, 24, 3, dtype, lambda t: torch.zeros(2, 9, 3, wide, device="cuda", dtype=dtype)[..., 16: 40].copy_(t))


def test_group_norm_beyond_31_bits_of_elements():
    """A channel slice of a wide buffer whose last image starts behind 2^31 elements, against that image alone."""
    n, h, w, c, wide = 5, 640, 512, 16, 1704
    buf = torch.zeros(n, h, w, wide, device="cuda", dtype=BF)
    assert (n - 1) * h * w * wide > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(4)
    x = buf[..., 64: 64 + c]
    x.copy_(torch.randn(n, h, w, c, device="cuda", generator=g))
    y = buf[..., 1000: 1000 + c]
    ga, be = torch.rand(c, device="cuda", generator=g) + 0.5, torch.randn(c, device="cuda", generator=g)
    mean, rstd = torch.empty(2, n * 2, device="cuda")
    ops.group_norm_fwd(x, ga, be, 2, 1e-5, y, mean, rstd, act="gelu")
    dy = torch.randn(n, h, w, c, device="cuda", generator=g).to(BF)
    dx = buf[..., 96: 96 + c]
    ops.group_norm_bwd(dy, x, ga, be, 2, mean, rstd, dx, act="gelu")
    x1 = x[4:].contiguous()
    y1, dx1, (m1, r1) = torch.empty_like(x1), torch.empty_like(x1), torch.empty(2, 2, device="cuda")
    ops.group_norm_fwd(x1, ga, be, 2, 1e-5, y1, m1, r1, act="gelu")
    ops.group_norm_bwd(dy[4:], x1, ga, be, 2, m1, r1, dx1, act="gelu")
    # the split of an image's sums depends on the number of images: 512 roundings, and one of the output
    assert nets.rel(mean[8:], m1) <= 1024 * nets.E and nets.rel(rstd[8:], r1) <= 1024 * nets.E
    assert nets.rel(y[4:], y1) <= 2 ** -8 and nets.rel(dx[4:], dx1) <= 2 ** -8
    assert not buf[..., :64].any() and not buf[..., 1000 + c:].any()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_linear_beyond_31_bits_of_elements(dtype):
    """Rows of a wide buffer: the last ones lie behind 2^31 elements, and are computed as they are alone."""
    m, n, k, wide = (1 << 18) + 3, 24, 40, 8320
    assert (m - 64) * wide > 1 << 31
    buf = torch.zeros(m, wide, device="cuda", dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    x, y, dx = buf[:, :k], buf[:, 4096: 4096 + n], buf[:, 8192: 8192 + k]
    x.copy_(torch.randn(m, k, device="cuda", generator=g))
    w = torch.randn(n, k, device="cuda", generator=g).to(dtype)
    ops.linear_fprop(x, w, y, act="relu")
    ops.linear_dgrad(y, w, dx)
    tail = slice(m - 64, m)
    want = torch.relu(x[tail].double() @ w.double().t())
    half = nets.E if dtype == F32 else 2.0 ** -8
    assert nets.rel(y[tail], want) <= half + (k + 16) * nets.E
    assert nets.rel(dx[tail], y[tail].double() @ w.double()) <= half + (n + 16) * nets.E
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    ops.linear_wgrad(y, x, dw, db)
    a, b = y.float().cpu().double(), x.float().cpu().double()
    # sums of m products, in partial sums of at most 2^14 and one behind another: |error| <= 2^15 E sum |y x|, in fact its root
    assert nets.rel(dw, a.t() @ b) <= 2 ** 15 * nets.E and nets.rel(db, a.sum(0)) <= 2 ** 15 * nets.E
    assert not buf[:, k: 4096].any() and not buf[:, 8192 + k:].any()


def test_adamw_beyond_31_bits_of_elements():
    n, t = (1 << 31) + 64 * 1000, 64 * 1000
    hyper = make_hyper(1e-2, 0.9, 0.999, 1e-8, 0.1, 3.0, 0.0, 1.0, device="cuda")
    groups = torch.ones(1, 2, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(6)
    arenas = [torch.zeros(n, device="cuda") for _ in range(4)]
    small = [torch.randn(t, device="cuda", generator=gen) for _ in range(3)] + [torch.rand(t, device="cuda", generator=gen)]
    for a, s in zip(arenas, small):
        a[n - t:] = s
    ops.adamw_step(*arenas, None, hyper, groups, torch.zeros(n // 64, device="cuda", dtype=torch.uint8))
    ops.adamw_step(*small, None, hyper, groups, torch.zeros(t // 64, device="cuda", dtype=torch.uint8))
    for a, s in zip(arenas, small):
        assert torch.equal(a[n - t:], s) and not a[: n - t].any()
