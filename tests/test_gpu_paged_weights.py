"""GPU: how exact the paged attention's weights are, against the 64-bit forms of ``paged_util``.

Sinks: one key of the sequence takes nearly all of the softmax and has a value of zeros, so that the result is what the other
keys' small weights make of their values.  Features 1 on are zero in queries and keys: a score is the key's feature 0, exactly.
"""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
MODEL, SMALL, WIDE = dict(heads=16, kv=2, dim=256), dict(heads=4, kv=2, dim=128), dict(heads=32, kv=8, dim=128)


def sink_batch(pkg, device, spans, where, gap, spread, dtype, shape, seed):
    """Sequences whose keys score N(0, spread), but ``gap`` at row ``where`` (None: nowhere), whose value is 0; the other values lie
    in [1/2, 3/2]."""
    batch = pu.Batch(pkg, device, spans, page=64, dtype=dtype, seed=seed, **shape)
    gen = torch.Generator().manual_seed(seed)
    keys, values = batch.host["keys"], batch.host["values"]
    score = (torch.randn(keys.shape[:3], generator=gen) * spread).to(dtype)
    used = ~torch.isnan(keys)
    keys[used] = 0.0
    keys[..., 0] = torch.where(used[..., 0], score, keys[..., 0])
    values.copy_(torch.where(used, (torch.rand(values.shape, generator=gen) + 0.5).to(dtype), values))
    if where is not None:
        for b, (_, n) in enumerate(spans):
            if n > where:
                at = (batch.table[b, where // 64].item(), slice(None), where % 64)
                keys[at], values[at] = 0.0, 0.0
                keys[(*at, 0)] = gap
    batch.query[..., 0], batch.query[..., 1:] = 1.0, 0.0
    batch.q = batch.query.to(device)
    batch.cache = batch.cache._replace(keys=keys.to(device), values=values.to(device))
    return batch


def attend_checked(pkg, batch, prefix, weight_unit):
    """Scale 1.  A score is exact, so a weight is off by two roundings of |score| log2 e (at most 64) and 2^-22 for the exponential;
    ``weight_unit``: its rounding for the product with V.  Sums add 2^-24 a term.  All relative to the sum of weights times |v|, all
    positive; then the output's rounding.  Weights are not rounded to multiples of anything that the result could show: 2^-30 of the
    largest |v| is left for the few that share 64 keys with the sink."""
    if prefix is None:
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=1.0)
    else:
        got = pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=1.0)
    want, size, _, keys = pu.expected_wide(batch, 1.0, True, batch.q.device, prefix)
    weight = 2 * 64 * 2.0 ** -24 + 2.0 ** -22 + weight_unit
    relative = 2 * weight + 2 * (keys + 16) * 2.0 ** -24
    limit = relative * size + 2.0 ** -30 * 1.5
    limit = limit + pu.UNIT[batch.dtype] * (want.abs() + limit) + pu.TINY[batch.dtype]
    over = (got[:batch.tokens].double().cpu() - want).abs() - limit
    assert float(over.max()) <= 0, (float(over.max()), float(want.abs().max()))


SPANS = {"decode": [(1, 20_011)], "decode of two": [(1, 4099), (1, 9000)], "blocks": [(40, 9001), (33, 2000)], "prompt": [(300, 300)]}


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("gap", [11.0, 14.0, 17.5, 22.0, 25.0])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("spans,shape,where", [("decode", SMALL, 0), ("decode", MODEL, 9000), ("decode of two", WIDE, 40),
                                               ("blocks", SMALL, 0), ("blocks", MODEL, 100), ("prompt", SMALL, 5)])
def test_small_weights_behind_a_sink(pkg, device, spans, shape, where, spread, gap, dtype):
    attend_checked(pkg, sink_batch(pkg, device, SPANS[spans], where, gap, spread, dtype, shape, 1), None, 2 * pu.UNIT[dtype])


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("gap", [14.0, 17.5, 25.0])
@pytest.mark.parametrize("spans,shape,front,first,second", [
    ([(1, 700)] * 3, SMALL, 6000, 0, None), ([(1, 700)] * 3, SMALL, 6000, None, 300), ([(16, 500)] * 4, MODEL, 5000, 70, None),
    ([(16, 500)] * 4, MODEL, 5000, None, 1), ([(1, 900)] * 40, WIDE, 4000, 4, None), ([(1, 900)] * 40, WIDE, 4000, None, 4)])
def test_a_sink_in_the_prefix_or_behind_it(pkg, device, spans, shape, front, first, second, gap, dtype):
    batch = sink_batch(pkg, device, spans, second, gap, 1.0, dtype, shape, 2)
    prefix = sink_batch(pkg, device, [(0, front)], first, gap, 1.0, dtype, shape, 3)
    attend_checked(pkg, batch, prefix, 2 * pu.UNIT[dtype])


@pytest.mark.parametrize("shape,tokens", [(SMALL, 1), (SMALL, 64), (MODEL, 64)])
def test_sinks_that_come_and_go(pkg, device, shape, tokens):
    """A key ahead of the rest in every 200th place, each further ahead than the last: the reference falls and rises many times."""
    batch = sink_batch(pkg, device, [(tokens, 12_001)], None, 0.0, 1.0, FP16, shape, 4)
    keys, values = batch.host["keys"], batch.host["values"]
    for i, r in enumerate(range(7, 12_000, 200)):
        at = (batch.table[0, r // 64].item(), slice(None), r % 64)
        keys[(*at, 0)], values[at] = 8.0 + i / 4, 0.0
    batch.cache = batch.cache._replace(keys=keys.to(device), values=values.to(device))
    attend_checked(pkg, batch, None, 2 * pu.UNIT[FP16])


def exact_to_the_rounding(got, want, limit, dtype):
    """``want``, 64 bits, is off ``got`` by the output's rounding and ``limit`` before it; and over all elements no further than the
    rounding alone is, but 1%: independent errors add as squares, so what comes before it is at most a seventh of the rounding."""
    got = got.double().cpu()
    over = (got - want).abs() - limit - pu.UNIT[dtype] * (want.abs() + limit) - pu.TINY[dtype]
    assert float(over.max()) <= 0, float(over.max())
    alone = (want.to(dtype).double() - want).square().sum().sqrt()
    assert float((got - want).square().sum().sqrt()) <= 1.01 * float(alone), float((got - want).square().sum().sqrt() / alone)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [MODEL, WIDE])
@pytest.mark.parametrize("spans,front", [([(1, 1500)] * 3, 0), ([(1, 20_000)], 0), ([(16, 900), (3, 77)], 0), ([(700, 2900), (90, 90)], 0),
                                         ([(1, 300)] * 8, 900), ([(16, 400)] * 3, 2000), ([(130, 200)], 500)])
def test_weights_are_as_exact_as_the_sums(pkg, device, spans, front, shape, causal, dtype):
    """N(0, 1) rows.  A weight is held in two parts, each off by half a step: UNIT^2 of it is left out; in fp16 also up to
    2^-25 where the second part is as small as that, which for 64 keys whose largest weighs 2^3 at least is 2^-22 of it (|v| < 8)."""
    batch = pu.Batch(pkg, device, spans, page=64, dtype=dtype, seed=5, **shape)
    prefix = pu.Batch(pkg, device, [(0, front)], page=64, dtype=dtype, seed=6, **shape) if front else None
    scale = batch.dim ** -0.5
    if prefix is None:
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale, causal=causal)
    else:
        got = pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=scale, causal=causal)
    want, size, most, keys = pu.expected_wide(batch, scale, causal, device, prefix)
    weight = (batch.dim + 6) * 2.0 ** -24 * scale * most + 2.0 ** -22 + pu.UNIT[dtype] ** 2
    limit = (2 * weight + 2 * (keys + 16) * 2.0 ** -24) * size + (2.0 ** -22 * 8 if dtype == FP16 else 0.0)
    exact_to_the_rounding(got, want, limit, dtype)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("scale", [2.0 ** 10, 2.0 ** 12, 2.0 ** 40])
@pytest.mark.parametrize("spans,shape,front", [([(1, 5000), (1, 333)], SMALL, 0), ([(1, 700)] * 20, MODEL, 0), ([(33, 3001)], SMALL, 0),
                                               ([(40, 900)] * 3, MODEL, 0), ([(1, 400)] * 8, WIDE, 900), ([(16, 300)] * 3, MODEL, 700)])
def test_scores_of_many_millions_choose_their_largest_keys(pkg, device, spans, shape, front, scale, dtype):
    """Scores past 2^25, where a step of fp32 is more than a binade of the weights: keys differ by more than 1000 or not at all, so a
    row is the mean of the values at its largest score, whichever way the reference was rounded."""
    gen = torch.Generator().manual_seed(8)

    def steep(batch):
        keys = batch.host["keys"]
        keys[..., 0] = torch.where(torch.isnan(keys[..., 0]), keys[..., 0], (32.0 * torch.randint(-2000, 2000, keys.shape[:3], generator=gen)).to(dtype))
        batch.cache = batch.cache._replace(keys=keys.to(device))
        return batch

    batch = steep(sink_batch(pkg, device, spans, None, 0.0, 1.0, dtype, shape, 7))
    prefix = steep(sink_batch(pkg, device, [(0, front)], None, 0.0, 1.0, dtype, shape, 8)) if front else None
    if prefix is None:
        got = pkg.ops.paged_attention(batch.q, batch.cache, batch.s, scale=scale)
    else:
        got = pkg.ops.shared_prefix_attention(batch.q, prefix.cache, batch.cache, batch.s, scale=scale)
    want, size, _, keys = pu.expected_wide(batch, scale, True, device, prefix)
    # equal weights of equal keys: the roundings of the sums, the parts and the output are left
    limit = (2 * pu.UNIT[dtype] ** 2 + 2 * (keys + 16) * 2.0 ** -24) * size
    over = (got.double().cpu() - want).abs() - limit - pu.UNIT[dtype] * (want.abs() + limit)
    assert torch.isfinite(got).all() and float(over.max()) <= 0, float(over.max())
