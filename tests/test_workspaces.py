"""A caller's workspace: kernels write its bytes one after the other, so only a contiguous tensor is one.

An expanded byte has one byte of memory however many elements it counts, and a strided slice has another view's bytes
between its own: both would be written past.
"""
import pytest
import torch

import paged_util as pu


def _unlike(size, device):
    """Tensors of enough elements whose memory is not theirs from the first to the last byte."""
    room = torch.empty(2 * size, dtype=torch.uint8, device=device)
    return {"expanded": torch.empty(1, dtype=torch.uint8, device=device).expand(size), "strided": room[::2],
            "columns": room.view(size, 2)[:, 0], "transposed": room.view(2, size).t()}


@pytest.mark.parametrize("form", ["expanded", "strided", "columns", "transposed"])
def test_a_workspace_is_contiguous(pkg, form):
    cpu = torch.device("cpu")
    with pytest.raises(ValueError, match="contiguous"):
        pkg.ops._workspace(64, cpu, _unlike(64, cpu)[form])


def test_workspaces_that_are_taken(pkg):
    cpu = torch.device("cpu")
    for given in (torch.empty(64, dtype=torch.uint8), torch.empty((8, 9), dtype=torch.uint8), torch.empty(99, dtype=torch.uint8)[3:]):
        assert pkg.ops._workspace(64, cpu, given) is given
    with pytest.raises(ValueError, match="at least 65 bytes"):
        pkg.ops._workspace(65, cpu, torch.empty(64, dtype=torch.uint8))


@pytest.mark.gpu
def test_both_forms_refuse_a_workspace_with_gaps(pkg, device):
    """The native form leaves the call to the Python form, which refuses it: nothing is launched."""
    batch = pu.Batch(pkg, device, [(2, 20), (1, 3)], page=16, dtype=torch.bfloat16, seed=7, heads=4, kv=2, dim=128)
    c, q, s, native = batch.cache, batch.q, batch.s, pkg._lib.host()
    need = pkg.ops.paged_attention_workspace_bytes(3, 4, 2, 128, 2, False)
    layer = pkg.synthetic.moe_layer(4, hidden=512, inter=512, experts=16, seed=1)
    x, banks, router = layer.hidden.to(device), (layer.gate_up.to(device), layer.down.to(device)), layer.router_weight.to(device)
    room = pkg.ops.moe_workspace_bytes(4, 512, 512, 16, 4, 128, False)
    for given in _unlike(need, device).values():
        assert native.paged_attention(q, None, c, s, 0.1, True, None, given) is None
        with pytest.raises(ValueError, match="contiguous"):
            pkg.ops.paged_attention(q, c, s, scale=0.1, workspace=given)
    for given in _unlike(room, device).values():
        assert native.moe(x, *banks, 4, router, None, given, None) is None
        with pytest.raises(ValueError, match="contiguous"):
            pkg.ops.moe_w4a16(x, *banks, top_k=4, router_weight=router, workspace=given)
    own = torch.empty(need, dtype=torch.uint8, device=device)
    assert torch.equal(native.paged_attention(q, None, c, s, 0.1, True, None, own), pkg.ops.paged_attention(q, c, s, scale=0.1))
