"""A layer with a gate refuses what its own router would have used, on the CPU: before any launch."""

import pytest
import torch

import keep_amd

INF = float("inf")


def _layer(gate=None, **kw):
    up, down = keep_amd.SwitchLinear(torch.zeros(4, 8, 16)), keep_amd.SwitchLinear(torch.zeros(4, 16, 8))
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=up, up_proj=up, down_proj=down)
    return keep_amd.RoutedVQMoE(glu, top_k=2, gate=keep_amd.MoEGate(torch.zeros(4, 16), top_k=2, **(gate or {})), **kw)


@pytest.mark.parametrize("over, msg", [
    (dict(bias_served=torch.zeros(4)), "bias_served"), (dict(bias_demand=torch.zeros(4)), "bias_served"), (dict(tau=0.3), "tau"),
    (dict(score_func="sigmoid"), "score_func"), (dict(renormalize=False), "renormalize"), (dict(route_scale=2.5), "route_scale"),
    (dict(one_launch=True), "one-launch"), (dict(slot_map=torch.zeros(4)), "slot_map"),
])
def test_settings_of_the_other_router(over, msg):
    with pytest.raises(ValueError, match=msg):
        _layer(**over)
    layer = _layer()
    for name, value in over.items():  # set afterwards, as a residency cache's are
        setattr(layer, name, value)
    with pytest.raises(ValueError, match=msg):
        layer(torch.zeros(2, 16))


def test_settings_of_the_gate_may_be_repeated():
    own = dict(score_func="sigmoid", renormalize=False, route_scale=2.5)
    _layer(own, **own)
    _layer(own)
    with pytest.raises(ValueError, match="route_scale"):
        _layer(own, **{**own, "route_scale": 2.0})


def test_logits():
    with pytest.raises(ValueError, match="forms its own logits"):
        _layer()(torch.zeros(2, 16), torch.zeros(2, 4))
