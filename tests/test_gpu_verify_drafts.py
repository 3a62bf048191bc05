"""GPU: the check of drafted tokens against a plain 64-bit form (``batch_util.verified``).

Whole numbers have to be equal.  ``margin`` says how near the reference's nearest comparison was: inputs are seeded, and none
is nearer than fp32 sums (acceptance) and 64-bit sums (draws) can tell.
"""
import math

import pytest
import torch

from batch_util import verified

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(spans, vocab, dtype, seed, noise=0.7, spare=0, temperature=None, one=False):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(spans) + spare
    target = torch.randn((rows, vocab), generator=gen) * 2
    target[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=gen)] += 4 + 10 * torch.rand((rows,), generator=gen)
    draft = target + noise * torch.randn((rows, vocab), generator=gen)
    target, draft = target.to(dtype), draft.to(dtype)
    starts = [sum(spans[:b]) for b in range(len(spans) + 1)]
    drafted = torch.empty((rows,), dtype=torch.int32)
    for r in range(rows):
        b = next((b for b in range(len(spans)) if starts[b] <= r < starts[b + 1]), 0)
        t = 1.0 if temperature is None else float(temperature[b])
        if one or not t > 0:
            drafted[r] = int(draft[r].float().argmax())
        else:
            drafted[r] = int(torch.multinomial(torch.softmax(draft[r].double() / min(t, 1e30), 0), 1, generator=gen))
    return dict(target=target, drafted=drafted, starts=torch.tensor(starts, dtype=torch.int32),
                uniforms=torch.rand((rows,), generator=gen), draft=None if one else draft, temperature=temperature)


def check(pkg, device, c, what="", **moved):
    dev = {k: None if v is None else moved.get(k, v.to(device)) for k, v in c.items()}
    got = pkg.ops.verify_drafts(dev["target"], dev["drafted"], dev["starts"], dev["uniforms"], draft=dev["draft"], temperature=dev["temperature"])
    accepted, token, margin = verified(**c)
    assert margin > 1e-12, (what, margin)
    assert torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.token.cpu(), token), (what, got, accepted, token)
    return got


SPANS = [[1], [16], [5, 1, 9, 2], [0, 3, 0, 1, 0], [2] * 70, [33, 7]]


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("spans", SPANS, ids=str)
@pytest.mark.parametrize("vocab", [1, 7, 8, 2049])
def test_sizes(pkg, device, vocab, spans, dtype, one):
    for seed in range(3):
        check(pkg, device, make(spans, vocab, dtype, seed, spare=seed, one=one), f"seed {seed}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [4096, 32_001, 248_320])
def test_vocabularies(pkg, device, vocab, dtype):
    for seed, (spans, one) in enumerate((([1], True), ([4, 1, 3], False), ([5], False))):
        t = torch.tensor([0.8, 1.3, 0.6][:len(spans)])
        check(pkg, device, make(spans, vocab, dtype, seed, temperature=t, one=one))


def test_flat_rows(pkg, device):
    """Every token about alike: a running sum stands 4e-6 from the next, and fp32 sums would miss."""
    for seed in range(4):
        c = make([3, 1], 248_320, FP32, seed)
        c["target"], c["draft"] = c["target"] * 0.02, c["draft"] * 0.02
        check(pkg, device, c)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_temperatures(pkg, device, dtype):
    values = [0.0, 1.0, 1e-3, 0.05, 3.0, -1.0, math.nan, 1e-38, 1e-45, 1e38, 0.9, math.inf]
    for seed in range(3):
        for one in (False, True):
            c = make([4, 1, 3] * 4, 509, dtype, seed, temperature=torch.tensor(values), one=one)
            check(pkg, device, c, f"seed {seed} {one}")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_masks(pkg, device, dtype):
    """Rows with nothing left, tokens of the type's lowest value, infinities and NaN."""
    low, inf = torch.finfo(dtype).min, math.inf
    for temperature in (None, torch.tensor([0.0] * 8), torch.tensor([0.7] * 8)):
        for seed in range(4):
            c = make([4] * 8, 301, dtype, seed, temperature=temperature)
            gen = torch.Generator().manual_seed(seed)
            t, d = c["target"], c["draft"]
            hide = torch.rand(t.shape, generator=gen) < 0.9
            t[0:4][hide[0:4]], d[0:4][hide[0:4]] = -inf, -inf     # the same filter on both sides
            t[4:8][hide[4:8]] = -inf                              # on the target's alone
            d[8:12][hide[8:12]] = low
            t[12], d[13], t[15] = -inf, -inf, -inf                # rows with nothing
            t[16:18], d[17] = low, low                            # all at the lowest value: all alike
            t[20][hide[20]], d[21][~hide[21]] = math.nan, math.nan
            t[23], d[22] = math.nan, math.nan
            t[24, 5], t[24, 9], d[24, 9], t[27, 300] = inf, inf, inf, inf
            t[28, 1:], d[28, 1:] = -inf, -inf                     # one token left
            check(pkg, device, c, f"seed {seed}")


def test_equal_distributions_accept_everything(pkg, device):
    for dtype in (BF16, FP32):
        c = make([9, 2, 17], 5003, dtype, 1, noise=0.0)
        c["uniforms"].fill_(1.0 - 2.0 ** -24)
        got = check(pkg, device, c)
        assert got.accepted.tolist() == [8, 1, 16]


def test_random_numbers_at_their_ends(pkg, device):
    for value in (0.0, 2.0 ** -149, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan):
        for one in (False, True):
            c = make([4, 1, 3], 777, FP32, 2, one=one)
            c["uniforms"].fill_(value)
            got = pkg.ops.verify_drafts(*(c[k].to(device) for k in ("target", "drafted", "starts", "uniforms")),
                                        draft=None if one else c["draft"].to(device))
            accepted, token, _ = verified(**c)
            assert torch.equal(got.accepted.cpu(), accepted)
            if value < 1:      # a number that no generator gives still draws a token that can be drawn
                assert torch.equal(got.token.cpu(), token), value
            assert bool(((got.token >= 0) & (got.token < 777)).all())


def test_drafted_tokens_outside_the_vocabulary(pkg, device):
    for one in (False, True):
        c = make([3, 3, 3], 64, BF16, 3, one=one)
        c["drafted"] = torch.tensor([-1, 5, 0, 64, 1, 0, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32)
        assert check(pkg, device, c).accepted.tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shift", [1, 3, 4, 7])
def test_strides_and_alignment(pkg, device, dtype, shift):
    c = make([6, 1, 5], 1003, dtype, shift)
    place = {}
    for i, name in enumerate(("target", "draft")):
        wide = torch.full((12, 1003 + 13 + shift + i), math.nan, dtype=dtype, device=device)
        place[name] = wide[:, shift + 2 * i:shift + 2 * i + 1003]
        place[name].copy_(c[name])
    check(pkg, device, c, **place)
    check(pkg, device, c, target=c["target"].t().contiguous().to(device).t())     # rows that are no rows: copied


def test_rows_behind_the_last_sequence_take_no_part(pkg, device):
    c = make([3, 4], 500, BF16, 5, spare=3)
    c["target"][7:], c["draft"][7:] = math.nan, math.nan
    c["drafted"][7:] = -7
    check(pkg, device, c)


def test_repeats(pkg, device):
    c = make([7] * 20, 32_001, BF16, 6)
    dev = {k: None if v is None else v.to(device) for k, v in c.items()}
    first = pkg.ops.verify_drafts(**dev)
    for _ in range(3):
        again = pkg.ops.verify_drafts(**dev)
        assert torch.equal(first.accepted, again.accepted) and torch.equal(first.token, again.token)


def test_frequencies(pkg, device):
    """Tokens of one drafted row and its successor follow the target's distribution, whatever the drafter's: over n draws a count
    strays from n p by more than 6 sqrt(n p (1 - p)) once in 5e8 (a binomial's tail)."""
    n, vocab = 20_000, 6
    gen = torch.Generator().manual_seed(0)
    p, q = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.2, 0.1]), torch.tensor([0.4, 0.1, 0.1, 0.05, 0.05, 0.3])
    drafted = torch.multinomial(q, n, True, generator=gen).to(torch.int32)
    rows = torch.stack((drafted, torch.zeros_like(drafted)), 1).reshape(-1)
    got = pkg.ops.verify_drafts(p.log().expand(2 * n, vocab).to(device), rows.to(device),
                                (2 * torch.arange(n + 1)).to(torch.int32).to(device), torch.rand((2 * n,), generator=gen).to(device),
                                draft=q.log().expand(2 * n, vocab).to(device))
    first = torch.where(got.accepted.cpu() == 1, drafted, got.token.cpu())
    counts = torch.bincount(first.long(), minlength=vocab).double()
    assert bool(((counts - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all()), counts
