"""Group norm, linear products and AdamW as layers, networks and an optimizer use them, on the CPU."""
import pytest
import torch

from distributedpytorch_amd.models.factory import get_model
from distributedpytorch_amd.nn.engine import Act, Context, ParamStore, Tape
from distributedpytorch_amd.nn.layers import GroupNorm2d, Mlp
from distributedpytorch_amd.nn.optim import ArenaOptimizer
from tests import train_ops_nets as nets


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
