"""GPU: the paged-cache operators against plain 64-bit forms (``paged_util``).

Unused rows of every pool are NaN, table entries behind a sequence's last row are no pages, tokens behind the last sequence
keep what their rows of ``out`` held.  Tolerances are the error bounds that ``paged_util.bound`` derives, per element.
"""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
MODEL, SMALL = dict(heads=16, kv=2, dim=256), dict(heads=4, kv=2, dim=128)


def check(got, want, limit, what=""):
    over = (got.double().cpu() - want).abs() - limit
    assert torch.isfinite(got).all(), what
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, (what, worst)


def attended(pkg, batch, causal, prefix=None, scale=None, wide=False):
    """The operator's result over a batch, checked against 64 bits (``wide``: on the device); rows of tokens in no sequence stay."""
    scale = batch.dim ** -0.5 if scale is None else scale
    out = torch.full((batch.total, batch.heads, batch.dim), 7.0, dtype=batch.dtype, device=batch.q.device)
    if prefix is None:
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale, causal=causal, out=out)
    else:
        got = pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=scale, causal=causal, out=out)
    assert got is out
    want, size, most, keys = (pu.expected_wide(batch, scale, causal, batch.q.device, prefix) if wide
                              else pu.expected(batch, scale, causal, prefix))
    check(got[:batch.tokens], want, pu.bound(batch.dtype, batch.dim, scale, size, most, keys), str(batch.spans[:4]))
    assert (got[batch.tokens:] == 7.0).all()
    return got


SPANS = {
    "one key": [(1, 1)],
    "one token": [(1, 100)],
    "unit edges": [(1, 31), (1, 32), (1, 33), (1, 127), (1, 128), (1, 129), (1, 255), (1, 257)],
    "empty": [(1, 0), (0, 5), (0, 0), (3, 3), (1, 17)],
    "longer than its rows": [(5, 3), (2, 1), (4, 0), (20, 7)],
    "blocks": [(16, 127), (2, 129), (17, 17), (3, 300)],
    "prompt": [(130, 200), (1, 64), (67, 67)],
}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("spans", SPANS.values(), ids=SPANS.keys())
@pytest.mark.parametrize("shape,page,dtype", [(MODEL, 16, BF16), (MODEL, 64, FP16), (SMALL, 48, BF16), (SMALL, 16, FP16),
                                              (dict(heads=6, kv=2, dim=128), 32, BF16), (dict(heads=3, kv=3, dim=256), 16, BF16),
                                              (dict(heads=20, kv=1, dim=128), 16, FP16)])
def test_attention(pkg, device, spans, shape, page, dtype, causal):
    attended(pkg, pu.Batch(pkg, device, spans, page=page, dtype=dtype, seed=len(spans), spare=2, **shape), causal)


@pytest.mark.parametrize("shape", [MODEL, SMALL])
def test_attention_over_many_chunks(pkg, device, shape):
    attended(pkg, pu.Batch(pkg, device, [(1, 5003)], page=64, dtype=BF16, seed=1, **shape), True)
    attended(pkg, pu.Batch(pkg, device, [(3, 4099), (1, 9), (16, 700)], page=16, dtype=FP16, seed=2, **shape), True)


# Row tiles of 128: chunks longer than 16 and 32 steps of 64 keys, chunks that end inside a step and inside a page
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape,page,spans", [
    (MODEL, 64, [(600, 4100)]), (MODEL, 16, [(513, 2900), (40, 41), (129, 1411)]), (SMALL, 64, [(1500, 4100)]),
    (dict(heads=32, kv=8, dim=128), 16, [(700, 2950)]), (dict(heads=1, kv=1, dim=128), 16, [(333, 700)]),
    (dict(heads=7, kv=1, dim=256), 32, [(90, 9001)])])
def test_attention_of_many_rows(pkg, device, shape, page, spans, causal):
    attended(pkg, pu.Batch(pkg, device, spans, page=page, dtype=BF16, seed=len(spans), spare=1, **shape), causal, wide=True)


@pytest.mark.parametrize("shape", [dict(heads=32, kv=8, dim=128), MODEL, dict(heads=8, kv=8, dim=256)])
@pytest.mark.parametrize("spans", [[(900, 900), (130, 1000), (0, 0), (1800, 1800), (5, 5)], [(60, 64 + 7 * b) for b in range(66)],
                                   [(33, 33)] * 64])
def test_more_row_tiles_than_workgroups_at_once(pkg, device, shape, spans):
    """Several to a place, of more and of fewer sequences than lanes, and more than 16384 rows to merge."""
    attended(pkg, pu.Batch(pkg, device, spans, page=16, dtype=FP16, seed=3, spare=1, **shape), True, wide=True)


@pytest.mark.parametrize("shape", [MODEL, SMALL])
@pytest.mark.parametrize("tokens,rows", [(20, 301), (40, 1003), (128, 4001)])
def test_many_rows_over_a_page_of_any_size(pkg, device, shape, tokens, rows):
    batch = pu.Batch(pkg, device, [(tokens, rows), (tokens, tokens + 5)], page=rows, dtype=BF16, seed=5, one_page=True, **shape)
    attended(pkg, batch, True, wide=True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shape", [MODEL, SMALL, dict(heads=2, kv=2, dim=256)])
def test_a_value_among_many_counts_only_where_it_is_seen(pkg, device, shape, bad):
    """Values that are NaN or infinite inside blocks of hundreds of tokens, in the first, an inner and the last step and chunk."""
    tokens, keys = 500, 2113
    batch = pu.Batch(pkg, device, [(tokens, keys), (1, 9)], page=16, dtype=BF16, seed=17, **shape)
    scale, pool = batch.dim ** -0.5, batch.cache.values
    for i in (0, 1, 63, 64, 250, 498, 499):
        row = keys - tokens + i
        at = (batch.table[0, row // 16].item(), slice(None), row % 16, 5)
        kept = pool[at].clone()
        pool[at] = 0.0
        want = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale)
        pool[at] = bad
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale)
        pool[at] = kept
        assert not torch.isfinite(got[i:tokens, :, 5]).any(), i
        got[i:tokens, :, 5] = want[i:tokens, :, 5]
        assert torch.equal(got, want), i


@pytest.mark.parametrize("count", [64, 65, 150])
def test_attention_over_more_sequences_than_lanes(pkg, device, count):
    spans = [((b * 7) % 3, (b * 53) % 290) for b in range(count)]
    attended(pkg, pu.Batch(pkg, device, spans, page=16, dtype=BF16, seed=3, spare=1, **SMALL), True)


@pytest.mark.parametrize("page,rows", [(37, 37), (37, 20), (4001, 333), (1, 1)])
def test_a_page_that_holds_a_whole_sequence_has_any_size(pkg, device, page, rows):
    batch = pu.Batch(pkg, device, [(1, rows), (1, min(rows, 5))], page=page, dtype=BF16, seed=4, one_page=True, **SMALL)
    attended(pkg, batch, True)


@pytest.mark.parametrize("spans", [SPANS["blocks"], SPANS["empty"]])
def test_attention_over_row_major_pages_and_strided_queries(pkg, device, spans):
    """Pages [pages, rows, heads, dim] seen with heads first, queries inside wider rows, a table with spare columns."""
    batch = pu.Batch(pkg, device, spans, page=16, dtype=BF16, seed=5, layout="rows", **SMALL)
    assert not batch.cache.keys.is_contiguous()
    wide = torch.full((batch.total, batch.heads, 2 * batch.dim), float("nan"), dtype=BF16, device=device)
    wide[..., :batch.dim] = batch.q
    batch.q = wide[..., :batch.dim]
    table = torch.full((len(spans), batch.width + 3), 1 << 30, dtype=torch.int32, device=device)
    table[:, :batch.width] = batch.cache.table
    batch.cache = batch.cache._replace(table=table[:, :batch.width])
    attended(pkg, batch, True)
    odd = torch.empty((batch.total, batch.heads, batch.dim + 1), dtype=BF16, device=device)[..., 1:]   # copied: misaligned
    odd.copy_(batch.q)
    batch.q = odd
    attended(pkg, batch, True)


def test_keys_and_values_may_share_one_tensor(pkg, device):
    batch = pu.Batch(pkg, device, SPANS["blocks"], page=16, dtype=FP16, seed=6, **SMALL)
    both = torch.stack((batch.cache.keys, batch.cache.values), 1)
    batch.cache = batch.cache._replace(keys=both[:, 0], values=both[:, 1])
    attended(pkg, batch, True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("shape", [MODEL, dict(heads=3, kv=3, dim=128)])
def test_a_key_counts_only_where_it_is_seen(pkg, device, shape, tokens, bad):
    """A NaN or infinite value (and key) at the block's token 1 leaves token 0 as it was and reaches the later ones."""
    batch = pu.Batch(pkg, device, [(tokens, tokens + 60), (1, 9)], page=16, dtype=BF16, seed=7, **shape)
    scale = batch.dim ** -0.5
    before = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale)
    row = 61
    page = batch.table[0, row // 16].item()
    for name in ("values", "keys"):
        pool = getattr(batch.cache, name)
        kept = pool[page, :, row % 16].clone()
        pool[page, :, row % 16, 5] = bad
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale)
        assert torch.equal(got[0], before[0]) and torch.equal(got[tokens:], before[tokens:]), name
        if name == "values":
            assert not torch.isfinite(got[1:tokens, :, 5]).any()
            got[1:tokens, :, 5] = before[1:tokens, :, 5]
            assert torch.equal(got, before)
        elif bad != bad:
            assert torch.isnan(got[1:tokens]).all()
        pool[page, :, row % 16] = kept


def test_a_row_whose_scores_are_all_minus_infinity_gives_zeros(pkg, device):
    batch = pu.Batch(pkg, device, [(1, 40)], page=16, dtype=BF16, seed=8, **SMALL)
    batch.q[..., 3] = 1.0
    for r in range(40):
        batch.cache.keys[batch.table[0, r // 16].item(), :, r % 16, 3] = -float("inf")
    assert (pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=0.1) == 0).all()


def test_peaked_and_large_scores(pkg, device):
    """Scores of several hundred: the softmax is a choice of one key, and no exponent overflows."""
    batch = pu.Batch(pkg, device, [(16, 700), (1, 300)], page=64, dtype=BF16, seed=9, **MODEL)
    attended(pkg, batch, True, scale=8.0)
    attended(pkg, batch, True, scale=2.0 ** -20)


def test_entries_that_are_no_pages_stay_inside_the_pool(pkg, device):
    """A table of rubbish reads the nearest page: as with the entries clamped."""
    batch = pu.Batch(pkg, device, [(2, 90), (1, 33)], page=16, dtype=BF16, seed=10, **SMALL)
    pool = torch.randn_like(batch.cache.keys)
    cache = batch.cache._replace(keys=pool, values=torch.randn_like(pool))
    pages = pool.shape[0]
    wild = torch.tensor([[-1, pages, 1 << 30, -(1 << 31), 2, (1 << 31) - 1, 3], [0, pages + 1, -5, 1, 1, 1, 1]],
                        dtype=torch.int32, device=device)[:, :batch.width]
    got = pkg.ops.paged_attention(batch.q, cache._replace(table=wild.contiguous()), batch.s, scale=0.1)
    want = pkg.ops.paged_attention(batch.q, cache._replace(table=wild.clamp(0, pages - 1).contiguous()), batch.s, scale=0.1)
    assert torch.equal(got, want)


PREFIXES = [1, 63, 128, 1000]


@pytest.mark.parametrize("rows", PREFIXES)
@pytest.mark.parametrize("spans", [[(1, 1)], [(1, 5), (1, 200), (0, 3), (1, 0)], [(16, 16)] * 3, [(7, 90), (140, 150)]])
@pytest.mark.parametrize("shape,page,dtype", [(MODEL, 64, BF16), (SMALL, 16, FP16), (dict(heads=3, kv=3, dim=128), 16, BF16)])
def test_shared_prefix(pkg, device, spans, rows, shape, page, dtype):
    batch = pu.Batch(pkg, device, spans, page=page, dtype=dtype, seed=rows, spare=1, **shape)
    prefix = pu.Batch(pkg, device, [(0, rows)], page=48, dtype=dtype, seed=rows + 1, **shape)
    attended(pkg, batch, True, prefix)
    attended(pkg, batch, False, prefix)


def test_a_sessions_contiguous_cache_is_a_prefix(pkg, device):
    """[1, kv heads, capacity, dim] with a capacity that is no multiple of 16: one page; a prefix without rows counts for nothing."""
    batch = pu.Batch(pkg, device, [(16, 16)] * 4, page=16, dtype=BF16, seed=11, **MODEL)
    prefix = pu.Batch(pkg, device, [(0, 301)], page=1003, dtype=BF16, seed=12, one_page=True, **MODEL)
    attended(pkg, batch, True, prefix)
    prefix.cache.lengths.zero_()
    scale = batch.dim ** -0.5
    got = pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=scale)
    want, size, most, keys = pu.expected(batch, scale, True)
    check(got, want, pu.bound(BF16, batch.dim, scale, size, most, keys))


def test_many_sequences_behind_a_long_prefix(pkg, device):
    batch = pu.Batch(pkg, device, [(1, b % 40) for b in range(90)], page=16, dtype=BF16, seed=13, **SMALL)
    prefix = pu.Batch(pkg, device, [(0, 2500)], page=64, dtype=BF16, seed=14, **SMALL)
    attended(pkg, batch, True, prefix)


@pytest.mark.parametrize("shape", [MODEL, dict(heads=32, kv=8, dim=128)])
@pytest.mark.parametrize("spans,rows", [([(1, 300 + b) for b in range(64)], 4097), ([(1, (37 * b) % 600) for b in range(130)], 2003),
                                        ([(50, 50 + 9 * b) for b in range(12)], 3003), ([(1, 2)] * 3, 7000),
                                        ([(300, 2500)], 40), ([(1, 5000), (1, 1)], 33)])
def test_prefixes_and_own_keys_of_many_sizes(pkg, device, shape, spans, rows):
    """Much of the one and little of the other: their shares of the workgroups."""
    batch = pu.Batch(pkg, device, spans, page=16, dtype=BF16, seed=rows, spare=1, **shape)
    prefix = pu.Batch(pkg, device, [(0, rows)], page=64, dtype=BF16, seed=rows + 1, **shape)
    attended(pkg, batch, True, prefix, wide=True)


# ------------------------------------------------------------------ append
def appended(pkg, batch, device, *, rotary=32, norms=True, positions=None, query=True, key_dtype_rows=None):
    gen = torch.Generator().manual_seed(99)
    total, kv, dim, dtype = batch.total, batch.kv, batch.dim, batch.dtype
    proj = torch.randn((total, 2 * (batch.heads + kv) * dim), generator=gen).to(dtype)
    gated, k, v = proj.split((2 * batch.heads * dim, kv * dim, kv * dim), dim=-1)
    host = {"query": gated.reshape(total, batch.heads, 2 * dim)[..., :dim], "key": k.reshape(total, kv, dim),
            "value": v.reshape(total, kv, dim)}
    d = proj.to(device)
    gated, k, v = d.split((2 * batch.heads * dim, kv * dim, kv * dim), dim=-1)
    q_norm, k_norm = (torch.rand((dim,), generator=gen) * 0.2 - 0.1 for _ in range(2)) if norms else (None, None)
    inv = 10000.0 ** -(torch.arange(rotary // 2) / (rotary // 2)) if rotary else None
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    before = {n: getattr(batch.cache, n).clone() for n in ("keys", "values")}
    got = pkg.ops.paged_append(batch.cache, k.reshape(total, kv, dim), v.reshape(total, kv, dim), batch.s,
                               query=gated.reshape(total, batch.heads, 2 * dim)[..., :dim] if query else None,
                               inv_freq=dev(inv), positions=dev(positions), q_norm=dev(q_norm) if query else None,
                               k_norm=dev(k_norm), eps=1e-6)
    row = torch.cat([torch.arange(n - t, n) for t, n in batch.spans] or [torch.zeros(0)]).long()
    where = row if positions is None else positions[:batch.tokens]
    # the norm's and rotation's fp32 roundings are far under the rounding of the result: |y| <= |a| + |b| of two features, a
    # couple of dozen roundings of 2^-24 (the sum of squares adds dim / 2 of them under the root)
    unit = pu.UNIT[dtype]

    def near(got, x, weight):
        want = pu.turned(x, weight, inv, where, 1e-6)
        size = want.abs()
        if inv is not None:
            h = inv.shape[0]
            pair = pu.turned(x, weight, None, where, 1e-6)[..., :2 * h].abs()
            pair = pair[..., :h] + pair[..., h:]
            size[..., :2 * h] = torch.cat((pair, pair), -1)
        check(got, want, unit * want.abs() + (24 + dim / 2) * 2.0 ** -24 * size + pu.TINY[dtype])

    n = batch.tokens
    if query:
        near(got[:n], host["query"][:n], q_norm)
    else:
        assert got is None
    # rows of the block, and every other row as it was
    sequence = torch.cat([torch.full((t,), b) for b, (t, _) in enumerate(batch.spans)] or [torch.zeros(0)]).long()
    held = row >= 0
    page = batch.table[sequence[held], row[held] // batch.page].long()
    inside = row[held] % batch.page
    keys, values = batch.cache.keys.cpu(), batch.cache.values.cpu()
    if norms or inv is not None:
        where = where[held]
        near(keys[page, :, inside], host["key"][:n][held], k_norm)
    else:
        assert torch.equal(keys[page, :, inside], host["key"][:n][held])
    assert torch.equal(values[page, :, inside], host["value"][:n][held])
    for name, now in (("keys", keys), ("values", values)):
        then = before[name].cpu()
        now[page, :, inside] = 0
        then[page, :, inside] = 0
        assert torch.equal(now.view(torch.int16), then.view(torch.int16)), name
    return got


@pytest.mark.parametrize("spans", SPANS.values(), ids=SPANS.keys())
@pytest.mark.parametrize("shape,page,dtype,rotary", [(MODEL, 16, BF16, 64), (MODEL, 64, FP16, 256), (SMALL, 48, BF16, 32),
                                                     (SMALL, 16, FP16, 128), (dict(heads=20, kv=1, dim=128), 16, BF16, 16)])
def test_append(pkg, device, spans, shape, page, dtype, rotary):
    batch = pu.Batch(pkg, device, spans, page=page, dtype=dtype, seed=len(spans), spare=2, **shape)
    appended(pkg, batch, device, rotary=rotary)


@pytest.mark.parametrize("rotary,norms,query", [(0, False, True), (0, False, False), (0, True, True), (64, False, True),
                                                (64, True, False)])
def test_append_without_its_parts(pkg, device, rotary, norms, query):
    batch = pu.Batch(pkg, device, SPANS["blocks"], page=16, dtype=BF16, seed=1, **MODEL)
    appended(pkg, batch, device, rotary=rotary, norms=norms, query=query)


@pytest.mark.parametrize("far", [0, 4097, 1_000_003, (1 << 31) - 40, -17])
def test_append_at_far_positions(pkg, device, far):
    """Angles of positions up to 2^31: 64-bit products, so that the cosine is as exact as at position 0."""
    batch = pu.Batch(pkg, device, [(16, 16), (3, 40)], page=16, dtype=FP16, seed=2, **SMALL)
    gen = torch.Generator().manual_seed(3)
    appended(pkg, batch, device, positions=(torch.randint(0, 39, (batch.total,), generator=gen) + far).to(torch.int32))


def test_append_of_many_tokens_and_sequences(pkg, device):
    batch = pu.Batch(pkg, device, [(b % 5, b % 5 + b % 31) for b in range(200)], page=16, dtype=BF16, seed=4, spare=3, **SMALL)
    appended(pkg, batch, device)


def test_append_into_row_major_pages(pkg, device):
    batch = pu.Batch(pkg, device, SPANS["blocks"], page=16, dtype=BF16, seed=5, layout="rows", **SMALL)
    appended(pkg, batch, device)


def test_append_leaves_out_rows_without_a_page(pkg, device):
    batch = pu.Batch(pkg, device, [(20, 40)], page=16, dtype=BF16, seed=6, **SMALL)
    rows = torch.randn((20, 2, 128), device=device).to(BF16)
    before = batch.cache.keys.clone()
    for wild in (-1, batch.cache.keys.shape[0], (1 << 31) - 1, -(1 << 31)):
        table = batch.cache.table.clone()
        table[0, 1] = wild
        batch.cache.keys.copy_(before)
        assert pkg.ops.paged_append(batch.cache._replace(table=table), rows, rows, batch.s) is None
        want = before.clone()
        want[table[0, 2].long(), :, :8] = rows[12:].transpose(0, 1)
        assert torch.equal(batch.cache.keys.view(torch.int16), want.view(torch.int16)), wild


@pytest.mark.parametrize("length", [48, 49, 55, 67, 68, 1 << 30, (1 << 31) - 1])
def test_append_past_the_last_page_leaves_the_rest_alone(pkg, device, length):
    """A sequence longer than its table has pages for: rows that have a place go there, no other row changes."""
    batch = pu.Batch(pkg, device, [(20, 48)], page=16, dtype=BF16, seed=6, **SMALL)
    rows = torch.randn((20, 2, 128), device=device).to(BF16)
    cache = batch.cache._replace(table=batch.cache.table[:, :3].contiguous(),
                                 lengths=torch.tensor([length], dtype=torch.int32, device=device))
    want = {name: getattr(cache, name).clone() for name in ("keys", "values")}
    for i in range(20):
        row = length - 20 + i
        if row < 48:
            for pool in want.values():
                pool[cache.table[0, row // 16].item(), :, row % 16] = rows[i]
    pkg.ops.paged_append(cache, rows, rows, batch.s)
    for name, pool in want.items():
        assert torch.equal(getattr(cache, name).view(torch.int16), pool.view(torch.int16)), name


# ------------------------------------------------------------------ refusals, streams, graphs, runs
def test_python_refusals(pkg, device):
    ops = pkg.ops
    batch = pu.Batch(pkg, device, [(2, 20), (1, 3)], page=16, dtype=BF16, seed=7, **SMALL)
    c, q, s = batch.cache, batch.q, batch.s
    rows = torch.zeros((3, 2, 128), dtype=BF16, device=device)
    attend = lambda q=q, c=c, s=s, **kw: ops.paged_attention(q, c, s, **{"scale": 0.1, **kw})  # noqa: E731
    append = lambda c=c, k=rows, v=rows, s=s, **kw: ops.paged_append(c, k, v, s, **kw)  # noqa: E731
    for call, message in [
            (lambda: attend(c=c._replace(values=c.values.half())), "one dtype"), (lambda: attend(q=q.half()), "query"),
            (lambda: attend(c=c._replace(keys=c.keys.float(), values=c.values.float())), "bfloat16 or float16"),
            (lambda: attend(c=c._replace(keys=c.keys[..., :100], values=c.values[..., :100])), "heads, 100"),
            (lambda: attend(c=c._replace(keys=c.keys[..., 4:], values=c.values[..., 4:])), "aligned"),
            (lambda: attend(c=c._replace(table=c.table.long())), "int32"), (lambda: attend(c=c._replace(lengths=c.lengths[:1])), "lengths"),
            (lambda: attend(s=s[:2]), "starts"), (lambda: attend(s=s.long()), "starts"), (lambda: attend(s=s.cpu()), "starts"),
            (lambda: attend(q=q[:, :3]), "multiple"), (lambda: attend(q=q[..., :64]), "query"), (lambda: attend(q=q[0]), "query"),
            (lambda: attend(out=q[:2]), "out"), (lambda: attend(out=q.float()), "out"), (lambda: attend(scale=None), "scale"),
            (lambda: attend(causal=1), "causal"), (lambda: attend(workspace=torch.empty(8, dtype=torch.uint8, device=device)), "workspace"),
            (lambda: attend(q=q.clone().requires_grad_()), "no_grad"),
            (lambda: ops.shared_prefix_attention(q, c, c, s, scale=0.1), "one sequence"),
            (lambda: append(k=rows[:2]), "value"), (lambda: append(k=rows[:, :1]), "key"), (lambda: append(query=q[:2]), "query"),
            (lambda: append(query=q[:, :0]), "head"), (lambda: append(q_norm=torch.zeros(128, device=device)), "needs a query"),
            (lambda: append(k_norm=torch.zeros(64, device=device)), "k_norm"), (lambda: append(inv_freq=torch.zeros(16)), "inv_freq"),
            (lambda: append(positions=torch.zeros(3, dtype=torch.int32, device=device)), "inv_freq"),
            (lambda: append(positions=torch.zeros(2, dtype=torch.int32, device=device), inv_freq=torch.ones(16, device=device)),
             "positions"),
            (lambda: append(c=c._replace(keys=c.keys[:1].expand(4, -1, -1, -1), values=c.values[:4])), "overlap"),
            (lambda: append(k=rows.clone().requires_grad_()), "no_grad")]:
        with pytest.raises(ValueError, match=message):
            call()
    for call, message in [(lambda: attend(scale=0.0), "scale"), (lambda: append(inv_freq=torch.ones(12, device=device)), "rotary_dim"),
                          (lambda: append(eps=-1.0), "eps")]:
        with pytest.raises(pkg._lib.DflashError, match=message):
            call()


def test_empty_calls(pkg, device):
    batch = pu.Batch(pkg, device, [(0, 5)], page=16, dtype=BF16, seed=8, **SMALL)
    rows = torch.zeros((0, 2, 128), dtype=BF16, device=device)
    assert pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=0.1).shape == (0, 4, 128)
    assert pkg.ops.paged_append(batch.cache, rows, rows, batch.s, query=batch.q).shape == (0, 4, 128)
    none = batch.cache._replace(table=batch.cache.table[:0], lengths=batch.cache.lengths[:0])
    out = torch.ones((2, 4, 128), dtype=BF16, device=device)
    assert (pkg.ops.paged_attention(out, none, batch.s[:1], scale=0.1, out=out.clone()) == 1).all()


def test_starts_that_are_no_such_thing_stay_inside(pkg, device):
    """Offsets out of order or past the block fault nothing and leave rows behind the block alone."""
    batch = pu.Batch(pkg, device, [(4, 40), (5, 33), (7, 7)], page=16, dtype=BF16, seed=9, **SMALL)
    rows = torch.randn((16, 2, 128), device=device).to(BF16)
    keep = torch.full((20, 4, 128), 3.0, dtype=BF16, device=device)
    for bad in ([0, 16, 2, 16], [-5, 3, 1 << 30, -(1 << 31)], [16, 0, 16, 0], [9, 9, 9, 9], [1 << 30] * 4):
        s = torch.tensor(bad, dtype=torch.int32, device=device)
        for lengths in ([40, 33, 7], [-1, 1 << 30, 0]):
            cache = batch.cache._replace(lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
            pkg.ops.paged_attention(batch.q, cache, s, scale=0.1, out=keep[:16])
            pkg.ops.paged_append(cache, rows, rows, s)
    torch.cuda.synchronize()
    assert (keep[16:] == 3).all()


@pytest.mark.parametrize("shape,tokens", [(MODEL, 700), (SMALL, 40), (MODEL, 12)])
def test_overlapping_blocks_stay_inside_the_workspace(pkg, device, shape, tokens):
    """Starts out of order, so that sequences' blocks hold more rows than the batch: nothing behind the workspace is written."""
    batch = pu.Batch(pkg, device, [(tokens, 3 * tokens + 900)] + [(0, 1200)] * 7, page=16, dtype=BF16, seed=19, **shape)
    prefix = pu.Batch(pkg, device, [(0, 500)], page=16, dtype=BF16, seed=20, **shape)
    wild = torch.tensor([0, tokens] * 4 + [0], dtype=torch.int32, device=device)
    for front in (None, prefix):
        size = pkg.ops.paged_attention_workspace_bytes(tokens, batch.heads, batch.kv, batch.dim, 8, front is not None)
        room = torch.full((size + (1 << 24),), 0x5A, dtype=torch.uint8, device=device)
        out = torch.zeros((tokens + 64, batch.heads, batch.dim), dtype=BF16, device=device)
        if front is None:
            pkg.ops.paged_attention(batch.q, batch.cache, wild, scale=0.1, out=out[:tokens], workspace=room)
        else:
            pkg.ops.shared_prefix_attention(batch.q, front.cache, batch.cache, wild, scale=0.1, out=out[:tokens], workspace=room)
        assert (room[size:] == 0x5A).all() and (out[tokens:] == 0).all()


def test_two_streams_at_once(pkg, device):
    """Calls on two streams side by side, each with what it allocates itself, give what they give alone."""
    big = pu.Batch(pkg, device, [(600, 2100)], page=16, dtype=BF16, seed=21, **MODEL)
    small = pu.Batch(pkg, device, [(1, 900 + b) for b in range(24)], page=16, dtype=BF16, seed=22, **MODEL)
    prefix = pu.Batch(pkg, device, [(0, 1500)], page=64, dtype=BF16, seed=23, **MODEL)
    calls = (lambda: pkg.ops.paged_attention(big.q, big.cache, big.s, scale=0.06),
             lambda: pkg.ops.shared_prefix_attention(small.q, prefix.cache, small.cache, small.s, scale=0.06))
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    for one, many in zip(alone, got):
        assert all(torch.equal(one, other) for other in many)


def test_other_stream_and_repeats(pkg, device):
    """A call on a stream of its own gives the default stream's result; every call the same bits."""
    batch = pu.Batch(pkg, device, [(1, 3000), (16, 900), (1, 40)], page=16, dtype=BF16, seed=10, **MODEL)
    prefix = pu.Batch(pkg, device, [(0, 800)], page=64, dtype=BF16, seed=11, **MODEL)
    run = lambda: (pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=0.06),  # noqa: E731
                   pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=0.06))
    first = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        others = [run() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_decode_steps_of_a_captured_graph(pkg, device):
    """Append and both attentions captured once, replayed while lengths, tables and tokens change; a second graph of the same
    calls between the replays; every replay as the eager calls."""
    batch = pu.Batch(pkg, device, [(1, 30), (1, 700), (1, 17)], page=16, dtype=BF16, seed=12, **MODEL)
    prefix = pu.Batch(pkg, device, [(0, 500)], page=64, dtype=BF16, seed=13, **MODEL)
    pool = [torch.randn_like(batch.cache.keys) for _ in range(2)]
    cache = pkg.ops.PagedKV(*pool, torch.arange(180, device=device, dtype=torch.int32).reshape(3, 60) % pool[0].shape[0],
                            torch.tensor([30, 700, 17], dtype=torch.int32, device=device))
    k, v = (torch.randn((3, 2, 256), device=device).to(BF16) for _ in range(2))
    q = torch.randn((3, 16, 256), device=device).to(BF16)
    inv = 10000.0 ** -(torch.arange(32, device=device) / 32)

    def step():
        turned = pkg.ops.paged_append(cache, k, v, batch.s, query=q, inv_freq=inv)
        return (turned, pkg.ops.paged_attention(turned, cache, batch.s, scale=0.06),
                pkg.ops.shared_prefix_attention(turned, prefix.cache, cache, batch.s, scale=0.06))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    memory = torch.cuda.graph_pool_handle()
    for g in graphs:
        with torch.cuda.graph(g, pool=memory):
            outs.append(step())
    for i in range(6):
        cache.lengths.add_(torch.tensor([1, -37, 90], dtype=torch.int32, device=device))
        cache.table.copy_(cache.table.roll(1, 0))
        q.copy_(torch.randn(q.shape, device=device))
        eager = [t.clone() for t in step()]
        torch.randn(1 << 20, device=device).sum().item()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i % 2], eager)), i


@pytest.mark.parametrize("shared", [False, True])
def test_a_run_of_prompt_and_decode_steps(pkg, device, shared):
    """Prompts, then decoded tokens, of three sequences in one pool against attention over each sequence's whole history."""
    heads, kv, dim, page, dtype = 16, 2, 256, 16, BF16
    gen = torch.Generator().manual_seed(14)
    prefix = pu.Batch(pkg, device, [(0, 70)], heads=heads, kv=kv, dim=dim, page=page, dtype=dtype, seed=15) if shared else None
    offset = 70 if shared else 0
    pool = torch.full((40, kv, page, dim), float("nan"), dtype=dtype, device=device)
    table = torch.randperm(39, generator=gen)[:36].to(torch.int32).reshape(3, 12).to(device)
    inv = 10_000_000.0 ** -(torch.arange(32) / 32)
    keys, values = pool, pool.clone()
    lengths, history = [0, 0, 0], [[], [], []]
    scale = dim ** -0.5
    for block in ([37, 5, 64], [1, 1, 1], [1, 0, 1], [16, 1, 3], [1, 1, 1]):
        total = sum(block)
        q, k, v = (torch.randn((total, h, dim), generator=gen).to(dtype) for h in (heads, kv, kv))
        lengths = [n + t for n, t in zip(lengths, block)]
        starts = torch.tensor([sum(block[:b]) for b in range(4)], dtype=torch.int32, device=device)
        cache = pkg.ops.PagedKV(keys, values, table, torch.tensor(lengths, dtype=torch.int32, device=device))
        rows = torch.cat([torch.arange(n - t, n) for n, t in zip(lengths, block)]) + offset
        turned = pkg.ops.paged_append(cache, k.to(device), v.to(device), starts, query=q.to(device), inv_freq=inv.to(device),
                                      positions=rows.to(torch.int32).to(device))
        if shared:
            got = pkg.ops.shared_prefix_attention(turned, prefix.cache, cache, starts, scale=scale)
        else:
            got = pkg.ops.paged_attention(turned, cache, starts, scale=scale)
        # the operators' own rounded rows are the inputs of the 64-bit form: the append is checked on its own above
        at = 0
        for b, t in enumerate(block):
            where = torch.arange(lengths[b], device=device)
            page_of = table[b].long()[where // page]
            kk, vv = (x[page_of, :, where % page].double().cpu() for x in (keys, values))
            ref_k = pu.turned(k[at:at + t], None, inv, rows[at:at + t], 0.0)
            check(kk[lengths[b] - t:], ref_k, pu.UNIT[dtype] * ref_k.abs() + 64 * 2.0 ** -24 * 8)
            if shared:
                kk, vv = torch.cat((prefix.rows(0), kk)), torch.cat((prefix.rows(0, "values"), vv))
            seen = torch.arange(kk.shape[0] - t, kk.shape[0]) + 1
            for h in range(heads):
                want, size, most = pu.attend(turned[at:at + t, h].double().cpu(), kk[:, h // 8], vv[:, h // 8], seen, scale)
                check(got[at:at + t, h], want, pu.bound(dtype, dim, scale, size, most, kk.shape[0]))
            at += t


def test_the_native_and_the_python_form_take_the_same_calls(pkg, device, monkeypatch):
    """Bit for bit the same result; what the native form leaves to the Python form comes out as there."""
    native = pkg._lib.host()
    batch = pu.Batch(pkg, device, SPANS["blocks"], page=16, dtype=BF16, seed=16, spare=1, **SMALL)
    prefix = pu.Batch(pkg, device, [(0, 90)], page=16, dtype=BF16, seed=17, **SMALL)
    rows = torch.randn((batch.total, 2, 128), device=device).to(BF16)
    inv, norm = 10000.0 ** -(torch.arange(16, device=device) / 16), torch.rand((128,), device=device)
    where = torch.arange(batch.total, dtype=torch.int32, device=device)
    c, q, s = batch.cache, batch.q, batch.s

    def calls():
        got = [pkg.ops.paged_append(c, rows, rows, s, query=q, inv_freq=inv, positions=where, q_norm=norm, k_norm=norm),
               pkg.ops.paged_append(c, rows, rows, s), c.keys.clone()]
        out = torch.zeros_like(q)
        got += [pkg.ops.paged_attention(q, c, s, scale=0.1, causal=False), pkg.ops.paged_attention(q, c, s, scale=0.1, out=out), out,
                pkg.ops.shared_prefix_attention(q, prefix.cache, c, s, scale=0.1)]
        return got

    got = calls()
    assert native.paged_append(c, rows, rows, s, q, inv, where, norm, norm, 1e-6) is not None
    assert native.paged_append(c, rows, rows, s, None, None, None, None, None, 1e-6) is True
    assert native.paged_attention(q, prefix.cache, c, s, 0.1, True, None, None) is not None
    with monkeypatch.context() as m:
        m.setattr(pkg.ops, "_plain", lambda x: False)
        want = calls()
    for a, b in zip(got, want):
        assert a is b is None or torch.equal(a[:batch.tokens].view(torch.int16), b[:batch.tokens].view(torch.int16))
    odd = torch.empty((batch.total, 4, 129), dtype=BF16, device=device)[..., 1:]
    odd.copy_(q)
    wide = torch.zeros((4, 6), dtype=torch.int32, device=device)
    for args in ((odd, None, c, s, 0.1, True, None, None), (q, None, tuple(c), s, 0.1, True, None, None),
                 (q, None, c, wide[:, 0], 0.1, True, None, None), (q, None, c, s, 1, True, None, None),
                 (q, c, c, s, 0.1, True, None, None), (q.clone().requires_grad_(), None, c, s, 0.1, True, None, None),
                 (q, None, c._replace(lengths=c.lengths.long()), s, 0.1, True, None, None)):
        assert native.paged_attention(*args) is None
    for args in ((c, rows, rows[:3], s, None, None, None, None, None, 1e-6), (c, rows, rows, s, None, None, where, None, None, 1e-6),
                 (c, rows, rows, s, None, None, None, norm, None, 1e-6), (c, rows, rows, s, None, None, None, None, norm[:64], 1e-6),
                 (c._replace(keys=c.keys[:1].expand(4, -1, -1, -1), values=c.values[:4]), rows, rows, s, None, None, None, None, None,
                  1e-6)):
        assert native.paged_append(*args) is None
