"""GPU: the paged-cache operators at the ends of what they take: pools past 2^32 elements, many heads in a group, many KV heads."""
import pytest
import torch

import paged_util as pu
from test_gpu_paged import BF16, FP16, MODEL, SMALL, appended, attended

pytestmark = pytest.mark.gpu


def spread_out(batch, stride):
    """The batch's pages ``stride`` elements apart in buffers of their own."""
    moved = []
    for pool in (batch.cache.keys, batch.cache.values):
        buffer = torch.empty((pool.shape[0] - 1) * stride + pool[0].numel(), dtype=pool.dtype, device=pool.device)
        far = buffer.as_strided(pool.shape, (stride, *pool.stride()[1:]))
        far.copy_(pool)
        moved.append(far)
    batch.cache = batch.cache._replace(keys=moved[0], values=moved[1])
    return batch


@pytest.mark.parametrize("shape,dtype", [(MODEL, BF16), (SMALL, FP16)])
@pytest.mark.parametrize("spans", [[(1, 40), (2, 33)], [(70, 100)]], ids=["16 rows", "128 rows"])
def test_pools_past_32_bits(pkg, device, spans, shape, dtype):
    batch = spread_out(pu.Batch(pkg, device, spans, page=32, dtype=dtype, seed=1, spare=1, **shape), (1 << 30) + 4104)
    assert (batch.cache.keys.shape[0] - 1) * batch.cache.keys.stride(0) > 1 << 32
    attended(pkg, batch, True)
    prefix = spread_out(pu.Batch(pkg, device, [(0, 150)], page=32, dtype=dtype, seed=2, **shape), (1 << 30) + 64)
    attended(pkg, batch, False, prefix)
    appended(pkg, batch, device)


@pytest.mark.parametrize("shape", [dict(heads=1024, kv=1, dim=128), dict(heads=512, kv=2, dim=256), dict(heads=300, kv=100, dim=128),
                                   dict(heads=128, kv=128, dim=256)])
@pytest.mark.parametrize("spans", [[(1, 300), (0, 4), (1, 1)], [(3, 200), (2, 2)]])
def test_many_heads(pkg, device, spans, shape):
    batch = pu.Batch(pkg, device, spans, page=16, dtype=BF16, seed=3, spare=1, **shape)
    attended(pkg, batch, True, wide=True)
    attended(pkg, batch, True, pu.Batch(pkg, device, [(0, 100)], page=16, dtype=BF16, seed=4, **shape), wide=True)
    appended(pkg, batch, device)


def test_queries_far_apart(pkg, device):
    """Token rows more than 2^32 elements from the first."""
    batch = pu.Batch(pkg, device, [(1, 90), (4, 30)], page=16, dtype=BF16, seed=5, **SMALL)
    stride = (1 << 30) + 1032
    far = torch.empty(4 * stride + 512, dtype=BF16, device=device).as_strided((5, 4, 128), (stride, 128, 1))
    far.copy_(batch.q)
    batch.q = far
    attended(pkg, batch, True)
    near, want = batch.cache._replace(keys=batch.cache.keys.clone(), values=batch.cache.values.clone()), batch.cache
    assert torch.equal(pkg.ops.paged_append(near, far[:, :2], far[:, 2:], batch.s, query=far), far.contiguous())
    pkg.ops.paged_append(want, far[:, :2].contiguous(), far[:, 2:].contiguous(), batch.s)
    assert torch.equal(near.keys.view(torch.int16), want.keys.view(torch.int16))
    assert torch.equal(near.values.view(torch.int16), want.values.view(torch.int16))


def test_in_place_and_repeated_pages(pkg, device):
    """``out`` may be the query, and a page may stand in a table several times where it is only read."""
    for spans in ([(1, 300)] * 3, [(40, 600), (3, 9)]):
        batch = pu.Batch(pkg, device, spans, page=16, dtype=BF16, seed=6, **MODEL)
        want = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=0.06)
        given = batch.q.clone()
        assert pkg.ops.paged_attention(given, batch.cache, batch.s, scale=0.06, out=given) is given
        assert torch.equal(given, want)
        pool = torch.nan_to_num(batch.cache.keys), torch.nan_to_num(batch.cache.values)
        table = torch.full_like(batch.cache.table, 1)
        same = batch.cache._replace(keys=pool[0], values=pool[1], table=table)
        spread = batch.cache._replace(keys=pool[0][1:2].repeat(table.shape[1], 1, 1, 1), values=pool[1][1:2].repeat(table.shape[1], 1, 1, 1),
                                      table=torch.arange(table.shape[1], dtype=torch.int32, device=device).repeat(table.shape[0], 1))
        assert torch.equal(pkg.ops.paged_attention(batch.q, same, batch.s, scale=0.06),
                           pkg.ops.paged_attention(batch.q, spread, batch.s, scale=0.06))
