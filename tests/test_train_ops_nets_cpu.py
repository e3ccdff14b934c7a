"""Group norm, linear products and AdamW as layers, networks and an optimizer use them, on the CPU."""
import os
import sys

import pytest
import torch
import torch.multiprocessing as mp

from distributedpytorch_amd.models.factory import get_model
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import GroupNorm2d, Mlp
from distributedpytorch_amd.nn.optim import ArenaOptimizer
from tests import train_ops_nets as nets
from tests.test_ddp_cpu import ROOT, _bring_up, _free_port


@pytest.mark.parametrize("act,mlp_act", [("relu", "relu"), ("silu", "gelu"), ("gelu", "silu"), ("none", "none")])
def test_layers_and_their_gradients(act, mlp_act):
    nets.check_layers("cpu", act, mlp_act)


def test_adamw_follows_torch():
    nets.check_adamw_torch("cpu")


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_training(kind):
    nets.check_training("cpu", torch.float32, kind, n=2)


def test_frozen_trunk_trains_the_classifier_alone():
    dm = nets.model("cpu", torch.float32, "adamw", feature_extract=True)
    st = dm.net.store
    before = {s.name: st.get_logical(s).clone() for s in st.params}
    dm.train_step(*nets.batch(2, dm.net, torch.float32, 0))
    changed = sorted(s.name for s in st.params if not torch.equal(before[s.name], st.get_logical(s)))
    assert changed == ["fc.0.bias", "fc.0.weight", "fc.2.bias", "fc.2.weight"]


def test_names_of_a_group_norm_network():
    names = set(nets.model("cpu", torch.float32, "adamw", head_hidden=()).net.state_dict(""))
    plain = get_model("resnet", 10, small_input=True)[0].state_dict("")
    assert names == {k for k in plain if not k.endswith(("running_mean", "running_var", "num_batches_tracked"))}


def test_8_bit_states_load_into_32_and_back():
    dm = nets.model("cpu", torch.float32, "adamw8")
    dm.train_step(*nets.batch(2, dm.net, torch.float32, 0))
    sd = dm.opt.state_dict()
    wide = ArenaOptimizer(dm.net.store, "adamw")
    wide.load_state_dict(sd)
    narrow = ArenaOptimizer(dm.net.store, "adamw8")
    narrow.load_state_dict(wide.state_dict())
    # the values of a block's codes are the same multiples of a scale that is off by at most two roundings
    for a, b in ((narrow.m, dm.opt.m), (narrow.v, dm.opt.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in ((narrow.m_scale, dm.opt.m_scale), (narrow.v_scale, dm.opt.v_scale)):
        assert bool(((a - b).abs() <= 4 * nets.E * b).all())


def test_8_bit_states_load_into_a_network_of_another_layout():
    """A bf16 network pads its input to 8 channels, an fp32 one to 4: arenas of different lengths, the same states."""
    a, b = nets.model("cpu", torch.float32, "adamw8"), nets.model("cpu", torch.bfloat16, "adamw8")
    assert a.opt.m.numel() != b.opt.m.numel()
    a.train_step(*nets.batch(2, a.net, torch.float32, 0))
    sd = a.opt.state_dict()
    b.opt.load_state_dict(sd)
    for i, s in b.opt.state_dict()["state"].items():
        for k in ("exp_avg", "exp_avg_sq"):          # blocks of 64 lie elsewhere: one more rounding, of half a step of the largest code
            want = sd["state"][i][k]
            if want.shape == s[k].shape:
                assert nets.rel(s[k], want) <= (2.0 ** -4 if k == "exp_avg" else 2.0 ** -3)


@pytest.mark.parametrize("make", [
    lambda: ArenaOptimizer(ParamStore("cpu").finalize(), "adamw16"),
    lambda: get_model("resnet", 10, norm="layer"),
    lambda: get_model("resnet", 10, norm="group", act="tanh"),
    lambda: get_model("resnet", 10, act="silu"),
    lambda: get_model("alexnet", 10, norm="group"),
    lambda: get_model("vgg", 10, head_hidden=(64,)),
    lambda: GroupNorm2d(ParamStore("cpu"), "n", 48, 32),
    lambda: GroupNorm2d(ParamStore("cpu"), "n", 12, 4),
    lambda: Mlp(ParamStore("cpu"), "m", (16,)),
], ids=["optimizer", "norm", "activation", "activation with batch norms", "model", "classifier", "groups", "padded channels", "widths"])
def test_refusals(make):
    with pytest.raises(ValueError):
        make()


def test_mlp_refuses_a_map():
    store = ParamStore("cpu")
    m = Mlp(store, "m", (16, 16))
    store.finalize()
    with pytest.raises(ValueError):
        m(Context(store, True, Tape()), Act(torch.zeros(2, 3, 3, 16), False))


def test_a_checkpoint_of_another_optimizer_is_refused():
    store = ParamStore("cpu")
    Mlp(store, "m", (16, 16))
    store.finalize()
    with pytest.raises(ValueError):
        ArenaOptimizer(store, "adamw").load_state_dict(ArenaOptimizer(store, "adam").state_dict())
    with pytest.raises(ValueError):
        ArenaOptimizer(store, "adam").load_state_dict(ArenaOptimizer(store, "adamw").state_dict())


def _rank(rank, world, port, out, backend):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    from distributedpytorch_amd.nn.loss import Criterion
    from distributedpytorch_amd.parallel.ddp import DistributedModel
    torch.set_num_threads(2)
    nc = _bring_up(backend, rank, world, port) if world > 1 else None
    torch.manual_seed(rank)                     # the wrap-time broadcast makes the ranks alike
    net, _ = get_model("resnet", 10, device="cpu", small_input=True, norm="group", act="gelu", head_hidden=(32,))
    opt = ArenaOptimizer(net.store, "adamw8", lr=1e-3, seed=3)
    dm = DistributedModel(net, Criterion(), opt, first_bucket_mb=0.05, bucket_cap_mb=2.0, native_comm=nc)
    x, y = nets.batch(4, net, torch.float32, 1)
    per, grads = 4 // world, None
    for _ in range(2):
        dm.train_step(x[rank * per: (rank + 1) * per], y[rank * per: (rank + 1) * per])
        grads = net.store.g.clone() if grads is None else grads
    torch.save({"g": grads / world, "p": net.store.p, "m": opt.m.view(torch.uint8), "s": opt.m_scale}, f"{out}/{world}.{rank}.pt")


@pytest.mark.parametrize("backend", ["gloo", "native"])
def test_two_ranks_train_as_one(backend, tmp_path):
    """A group norm knows nothing of the batch, so two half batches give the whole one's gradients; ranks stay bit for bit alike,
    their stochastic rounding included."""
    mp.spawn(_rank, args=(2, _free_port(), str(tmp_path), backend), nprocs=2)
    mp.spawn(_rank, args=(1, 0, str(tmp_path), backend), nprocs=1)
    a, b, one = (torch.load(tmp_path / f"{n}.pt", weights_only=True) for n in ("2.0", "2.1", "1.0"))
    for k in a:
        assert torch.equal(a[k], b[k]), k
    # 20 layers, 544 roundings each, and norms whose backward pass leaves at least a quarter of a gradient's size
    assert nets.rel(a["g"], one["g"]) <= 20 * 544 * nets.E * 4
