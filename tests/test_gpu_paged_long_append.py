"""GPU: appends of more tokens than one workgroup a slice of the heads is taken for (1024), where a workgroup turns all heads of its
token, several reads one behind the other."""
import pytest
import torch

import paged_util as pu
from test_gpu_paged import BF16, FP16, MODEL, SMALL, appended

pytestmark = pytest.mark.gpu
WIDE = dict(heads=32, kv=8, dim=128)


@pytest.mark.parametrize("shape,page,dtype,rotary", [(MODEL, 64, BF16, 64), (MODEL, 16, FP16, 256), (WIDE, 16, FP16, 128), (WIDE, 48, BF16, 16),
                                                     (SMALL, 16, BF16, 32), (dict(heads=1, kv=1, dim=128), 16, BF16, 32),
                                                     (dict(heads=31, kv=1, dim=256), 32, BF16, 64)])
@pytest.mark.parametrize("spans", [[(1024, 1024)], [(1025, 1025)], [(700, 900), (1, 40), (0, 5), (650, 650)],
                                   [(12, 12 + b % 7) for b in range(100)]], ids=["1024", "1025", "prompts", "blocks"])
def test_append_of_many_tokens(pkg, device, spans, shape, page, dtype, rotary):
    batch = pu.Batch(pkg, device, spans, page=page, dtype=dtype, seed=len(spans), spare=2, **shape)
    appended(pkg, batch, device, rotary=rotary)


@pytest.mark.parametrize("rotary,norms,query", [(0, False, True), (0, False, False), (0, True, True), (64, False, True), (64, True, False)])
def test_append_of_many_tokens_without_its_parts(pkg, device, rotary, norms, query):
    for shape in (MODEL, WIDE):
        batch = pu.Batch(pkg, device, [(900, 1000), (200, 200)], page=16, dtype=BF16, seed=1, **shape)
        appended(pkg, batch, device, rotary=rotary, norms=norms, query=query)


def test_append_of_many_tokens_leaves_out_what_has_no_place(pkg, device):
    """Rows before 0, past the table and on entries that are no pages, among 1200 tokens: all others go where they belong."""
    batch = pu.Batch(pkg, device, [(1200, 1264)], page=16, dtype=BF16, seed=6, **WIDE)
    rows = torch.randn((1200, 8, 128), device=device).to(BF16)
    table = batch.cache.table.clone()
    table[0, 20], table[0, 33] = -1, 1 << 30
    for length in (1264, 1100, 1200 + (batch.width - 1) * 16):
        cache = batch.cache._replace(table=table, lengths=torch.tensor([length], dtype=torch.int32, device=device))
        want = {name: getattr(cache, name).clone() for name in ("keys", "values")}
        row = torch.arange(length - 1200, length)
        entry = (row // 16).clamp(0, batch.width - 1)
        page = table.cpu()[0, entry]
        held = (row >= 0) & (row < batch.width * 16) & (page >= 0) & (page < cache.keys.shape[0])
        for pool in want.values():
            pool[page[held].long().to(device), :, (row[held] % 16).to(device)] = rows[held.to(device)]
        pkg.ops.paged_append(cache, rows, rows, batch.s)
        for name, pool in want.items():
            assert torch.equal(getattr(cache, name).view(torch.int16), pool.view(torch.int16)), (length, name)
