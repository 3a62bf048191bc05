"""GPU: acceptance tests and draws of ``verify_drafts`` next to their limits, which sums of 64 bits decide, alone or among others."""
import math

import pytest
import torch

from batch_util import chances
from test_gpu_verify_drafts import check, make

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def at_the_limit(c, seed):
    """Every row's random number is one of the two fp32 numbers next to p(x) / q(x), or to p(x) where the token was chosen outright."""
    gen = torch.Generator().manual_seed(seed)
    starts, rows = c["starts"].tolist(), c["target"].shape[0]
    for b in range(len(starts) - 1):
        t = 1.0 if c["temperature"] is None else float(c["temperature"][b])
        for r in range(starts[b], starts[b + 1] - 1):
            limit = float(chances(c["target"][r], t)[int(c["drafted"][r])])
            if c["draft"] is not None:
                limit /= float(chances(c["draft"][r], t)[int(c["drafted"][r])])
            near = torch.tensor(limit, dtype=torch.float32)
            other = torch.nextafter(near, torch.tensor(0.0 if float(near) > limit else math.inf))
            c["uniforms"][r] = near if torch.rand((), generator=gen) < 0.5 else other
    return c


def rows_of(c, b):
    lo, hi = int(c["starts"][b]), int(c["starts"][b + 1])
    return {k: None if v is None else v[lo:hi].clone() for k, v in c.items() if k not in ("starts", "temperature")} | {
        "starts": torch.tensor([0, hi - lo], dtype=torch.int32), "temperature": None if c["temperature"] is None else c["temperature"][b:b + 1]}


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("vocab,dtype", [(509, FP16), (32_001, BF16), (32_001, FP32), (100_277, FP32)])
def test_acceptance_at_its_limit(pkg, device, vocab, dtype, one):
    """Off by a step of fp32 at most, so that sums have to tell 6e-8 of them apart: all sequences in a call, and single ones alone."""
    spans = [2, 3, 2, 4] * 10
    c = make(spans, vocab, dtype, 5, noise=0.3, one=one, temperature=0.6 + 0.02 * torch.arange(40.0))
    c["target"] = c["target"] * 0.2 if vocab == 509 else c["target"]
    check(pkg, device, at_the_limit(c, 1))
    for b in range(0, 40, 5):
        check(pkg, device, rows_of(c, b), f"sequence {b}")


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("stop", [None, 0, 15, 16, 20, 33])
def test_long_blocks_at_their_limits(pkg, device, stop, one):
    """Blocks of more rows than are looked at together: every row's number is the last below its limit, or in row `stop` the first that is
    not, so that each test has to be made in 64 bits."""
    c = make([40, 17, 35], 5003, BF16, 7, noise=0.3, one=one)
    for b in range(3):
        lo, hi = int(c["starts"][b]), int(c["starts"][b + 1])
        for r in range(lo, hi - 1):
            x = int(c["drafted"][r])
            limit = float(chances(c["target"][r], 1.0)[x]) / (1.0 if one else float(chances(c["draft"][r], 1.0)[x]))
            near = torch.tensor(limit, dtype=torch.float32)
            under, above = ((near, torch.nextafter(near, torch.tensor(math.inf))) if float(near) < limit else
                            (torch.nextafter(near, torch.tensor(0.0)), near))
            c["uniforms"][r] = above if r - lo == stop else under
    want = [min(hi - 1 if stop is None else stop, hi - 1) for hi in (40, 17, 35)]
    assert check(pkg, device, c).accepted.tolist() == want


@pytest.mark.parametrize("order", [1, -1])
def test_acceptance_of_sorted_rows(pkg, device, order):
    """Logits that rise or fall all along: a running maximum that moves with every token, or never."""
    vocab, spans = 248_320, [2, 2, 3]
    c = make(spans, vocab, FP32, 6, one=True)
    line = torch.linspace(-6.0, 1.0, vocab)
    for r in range(sum(spans)):
        c["target"][r] = line if order > 0 else line.flip(0)
        c["target"][r] += 1e-3 * r
        c["drafted"][r] = vocab // 2 + r
    check(pkg, device, at_the_limit(c, 2))


def test_numbers_exactly_at_the_limit(pkg, device):
    """p is a power of two and the random number the same: not below it, so not accepted; q of one half beside it."""
    for vocab in (1024, 65_536):
        for dtype in (BF16, FP16, FP32):
            c = make([2, 2], vocab, dtype, 0, one=True)
            c["target"][:] = 1.5
            c["uniforms"][:] = torch.tensor([1.0 / vocab, 0.25, (1.0 - 2.0 ** -24) / vocab, 0.25])
            dev = {k: None if v is None else v.to(device) for k, v in c.items()}
            assert pkg.ops.verify_drafts(**dev).accepted.tolist() == [0, 1], (vocab, dtype)


def test_a_part_whose_end_the_sum_hides(pkg, device):
    """A draw at the end of a part of the row, where the part's sum and the sum along it round to the two sides of the number drawn.

    Token 0 weighs 1, tokens 1 to 7 0.77 * 2^-53 each: added one by one to 1 they vanish, added up first they do not.  Three more tokens
    weigh 1, in other parts, so a quarter of the whole is the sum up to the first part's end, to a rounding: the token is one of the
    part's, or the next that weighs anything, and never a later one.
    """
    line = torch.full((8192,), -math.inf)
    line[0], line[1:8] = 0.0, -37.0
    line[[5000, 6000, 8000]] = 0.0
    for dtype in (BF16, FP16, FP32):
        got = pkg.ops.verify_drafts(line.to(dtype)[None].to(device), torch.zeros((1,), dtype=torch.int32, device=device),
                                    torch.tensor([0, 1], dtype=torch.int32, device=device), torch.tensor([0.25], device=device))
        assert got.token.tolist()[0] in (*range(8), 5000), (dtype, got)
