"""GPU: the check of drafted tokens where logits tie at temperature 0: the first of the largest is the one, wherever a row starts."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
VOCAB = 5003


def placed(line, ahead, rows, device):
    """``rows`` times the row ``line``, which starts ``ahead`` values behind a 16-byte boundary."""
    room = torch.full((ahead + line.numel() + 64,), math.nan, dtype=line.dtype, device=device)
    assert room.data_ptr() % 16 == 0
    row = room[ahead:ahead + line.numel()]
    row.copy_(line)
    return row[None].expand(rows, -1)


def ties(ahead, dtype):
    """Rows and the places of their largest logit: everywhere, or in the row's first eight and in some behind it."""
    yield torch.full((VOCAB,), 0.5, dtype=dtype), [0, 1, 8, VOCAB - 1]
    yield torch.full((VOCAB,), torch.finfo(dtype).min, dtype=dtype), [0, 2, 4096, VOCAB - 1]
    gen = torch.Generator().manual_seed(ahead)
    quiet = torch.randn((VOCAB,), generator=gen).clamp(max=2.0).to(dtype)
    start = lambda eight: 8 * eight - ahead  # noqa: E731
    some = [start(e) + i for e in (1, 255, 256, 257, 513) for i in (0, 5)]
    last = [max(start(1) - 1, 0), 0]        # the row's first eight: its last and first token
    for places in [[last[0], p] for p in some] + [[0, p] for p in some] + [some, last + some, [start(513), start(256) + 7], [start(257), start(1) + 3],
                                                                          [VOCAB - 1, start(512)], [VOCAB - 1, VOCAB - 2]]:
        row = quiet.clone()
        row[places] = 7.0
        yield row, sorted(set(places))


@pytest.mark.parametrize("sequences", [1, 1100], ids=["several parts a row", "one part a row"])
@pytest.mark.parametrize("dtype,ahead", [(t, a) for t in (BF16, FP16) for a in range(8)] + [(FP32, a) for a in range(4)])
def test_first_of_the_largest(pkg, device, dtype, ahead, sequences):
    """Sequences of two rows alike: the first tied token drafted is accepted and drawn again behind it, a later one is not."""
    starts = (2 * torch.arange(sequences + 1)).to(torch.int32).to(device)
    uniforms, cold = torch.full((2 * sequences,), 0.5, device=device), torch.zeros((sequences,), device=device)
    for line, places in ties(ahead, dtype):
        target = placed(line, ahead, 2 * sequences, device)
        for at, accepted in ((places[0], 1), (places[-1], int(len(places) == 1))):
            drafted = torch.full((2 * sequences,), at, dtype=torch.int32, device=device)
            got = pkg.ops.verify_drafts(target, drafted, starts, uniforms, temperature=cold)
            assert bool((got.token == places[0]).all()) and bool((got.accepted == accepted).all()), (places, at, got.token[:4], got.accepted[:4])


@pytest.mark.parametrize("vocab", [1009, 32_001])
def test_many_ties_in_rows_of_an_odd_vocabulary(pkg, device, vocab):
    """Rows one behind the other start anywhere; logits of a few values tie often."""
    gen = torch.Generator().manual_seed(vocab)
    for dtype in (BF16, FP32):
        target = torch.randint(-3, 4, (60, vocab), generator=gen).to(dtype)
        target[::3, 10:] = target[::3, 10:].clamp(max=2)      # the largest near the row's start, or nowhere else
        first = torch.tensor([int((row == row.max()).nonzero()[0]) for row in target.float()], dtype=torch.int32)
        got = pkg.ops.verify_drafts(target.to(device), first.to(device), torch.tensor([0, 20, 21, 60], dtype=torch.int32, device=device),
                                    torch.full((60,), 0.5, device=device), temperature=torch.zeros((3,), device=device))
        assert got.accepted.tolist() == [19, 0, 38] and got.token.tolist() == [int(first[r]) for r in (19, 20, 59)]
