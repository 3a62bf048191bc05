"""GPU: outputs next to what a call reads, and in the room between a pool's slots, are taken and right; one in the gates is refused."""
import pytest
import torch

from batch_util import Layer, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_output_between_slots_and_gates(pkg, device, longest):
    spans, hv, dim = [3, 40], 4, 64
    layer = Layer(pkg, device, spans, dim=dim, raw_gates=False, seed=1)
    n, state = sum(spans), hv * dim * dim
    size = n * hv * dim // 2                                   # the output's, in floats
    assert size % 4 == 0
    room = torch.zeros((layer.recurrent.shape[0], state + size), device=device)
    pool = room[:, :state].unflatten(1, (hv, dim, dim))
    pool.copy_(layer.recurrent)
    out = room[2, state:].view(torch.bfloat16).view(n, hv, dim)
    layer.d["recurrent"] = pool
    layer.pool = layer.pool._replace(recurrent=pool)
    assert layer.rule(out, longest=longest) is out
    layer.check_rule(out)
    layer = Layer(pkg, device, spans, dim=dim, raw_gates=False, seed=2)
    gates = torch.zeros((2 * n * hv + size,), device=device)
    layer.d["decay"], layer.d["beta"] = gates[:n * hv].view(n, hv), gates[-n * hv:].view(n, hv)
    layer.d["decay"].copy_(layer.decay), layer.d["beta"].copy_(layer.beta)
    out = gates[n * hv:-n * hv].view(torch.bfloat16).view(n, hv, dim)
    layer.check_rule(layer.rule(out, longest=longest))


def test_output_in_the_gates(pkg, device):
    layer = Layer(pkg, device, [5, 9], dim=64, seed=3)
    wide = torch.zeros((14, 2 * 4 * 64 + 8), dtype=torch.bfloat16, device=device)
    out = wide.flatten()[:14 * 256].view(14, 4, 64)
    before = layer.d["recurrent"].clone()
    for name in ("decay", "beta"):
        kept = layer.d[name]
        layer.d[name] = wide[:, -8:-4] if name == "decay" else wide[:, -4:]
        with pytest.raises(pkg._lib.DflashError, match="gates"):
            layer.rule(out)
        layer.d[name] = kept
    assert same_bits(before, layer.d["recurrent"])
