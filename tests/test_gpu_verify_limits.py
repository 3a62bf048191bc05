"""GPU: draws of ``verify_drafts`` next to their limits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


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
