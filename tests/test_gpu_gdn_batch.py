"""GPU: convolution, delta rule and advance of a batch of sequences against plain 64-bit forms (``batch_util``).

Tokens behind the last sequence keep what their rows of ``out`` held, other slots their bits, and a slot that a fresh sequence
does not read is NaN.
"""
import pytest
import torch

from batch_util import Layer, same_bits

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SPANS = {
    "one token": [1],
    "decode": [1] * 7,
    "empty": [0, 3, 0, 0, 1, 0],
    "short": [1, 2, 3, 4, 5],
    "verify": [16, 9, 1, 15, 2],
    "edges": [15, 16, 17, 31, 33],
    "prompt": [70, 1, 130, 0, 64],
    "chunk edges": [63, 64, 65, 127, 129],
}
SHAPES = [dict(key_heads=2, value_heads=4, dim=128, dtype=BF16), dict(key_heads=3, value_heads=3, dim=64, dtype=FP16),
          dict(key_heads=1, value_heads=5, dim=128, dtype=FP16), dict(key_heads=2, value_heads=6, dim=64, dtype=BF16)]


def filled(layer, *shape):
    return torch.full((layer.total, *shape), 7.0, dtype=layer.dtype, device=layer.device)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("spans", SPANS.values(), ids=SPANS.keys())
def test_conv(pkg, device, spans, shape):
    layer = Layer(pkg, device, spans, seed=len(spans), spare=2, missing=(1,), fresh=(0, 3), **shape)
    out = filled(layer, layer.channels)
    assert layer.conv(out) is out
    layer.check_conv(out)
    assert (out[layer.tokens:] == 7.0).all()


@pytest.mark.parametrize("counts", [[0, 0, 0, 0, 0], [1, 2, 3, 4, 5], [2, 1, 0, -5, 99]])
def test_conv_counts(pkg, device, counts):
    layer = Layer(pkg, device, [5, 2, 3, 4, 5], counts=counts, strided=False)
    layer.check_conv(layer.conv())


def test_conv_of_many_tokens(pkg, device):
    """Tiles of several tokens: blocks that start at every place of a tile, and histories used across its end."""
    for seed in range(3):
        layer = Layer(pkg, device, [7 + seed, 1, 2, 9, 1, 1, 4100, 3, 8, 8, 16, 801], key_heads=1, value_heads=1, dim=64, seed=seed, spare=3,
                      fresh=(2, 6))
        out = filled(layer, layer.channels)
        layer.conv(out)
        layer.check_conv(out, str(seed))
        assert (out[layer.tokens:] == 7.0).all()
    layer = Layer(pkg, device, [700, 1, 3, 2, 900, 5], key_heads=16, value_heads=32, seed=5, fresh=(0,), counts=[700, 1, 0, 1, 899, 5])
    layer.check_conv(layer.conv())


@pytest.mark.parametrize("longest", [None, 1, 16, 200])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("spans", SPANS.values(), ids=SPANS.keys())
def test_rule(pkg, device, spans, shape, longest):
    layer = Layer(pkg, device, spans, seed=len(spans), spare=2, missing=(1,), fresh=(0, 3), **shape)
    out = filled(layer, layer.hv, layer.dim)
    assert layer.rule(out, longest=longest) is out
    layer.check_rule(out)
    assert (out[layer.tokens:] == 7.0).all()


@pytest.mark.parametrize("longest", [1, 16, 200])
@pytest.mark.parametrize("counts", [[0] * 6, [1, 20, 64, 65, 128, 129], [70, 16, 63, 1, 127, 400], [-1, 36, 0, 2, 191, 300]])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP16)])
def test_rule_counts(pkg, device, counts, dim, dtype, longest):
    """The state stops at any token while the outputs go on."""
    layer = Layer(pkg, device, [70, 36, 64, 66, 192, 300], dim=dim, dtype=dtype, counts=counts, fresh=(2,))
    layer.check_rule(layer.rule(longest=longest))


@pytest.mark.parametrize("longest", [1, 16, 200])
@pytest.mark.parametrize("kind", [torch.float32, BF16, FP16])
def test_rule_gates_given(pkg, device, kind, longest):
    """Gates as they are, from hardly any decay to states that vanish within a token."""
    for seed, scale in enumerate((0.0, 0.01, 1.0, 40.0)):
        layer = Layer(pkg, device, [3, 150, 1, 17], raw_gates=False, gates_dtype=kind, seed=seed, decay_scale=scale, strided=seed % 2 == 0)
        layer.check_rule(layer.rule(longest=longest), f"decay {scale}")


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_rule_without_norm(pkg, device, longest):
    layer = Layer(pkg, device, [5, 100, 64], seed=3)
    for t in (layer.key, layer.d["key"]):    # of norm about one, as the bound asks: a power of two takes nothing off
        t.mul_(1 / 16)
    layer.check_rule(layer.rule(normalise=False, scale=0.5, longest=longest), normalise=False, scale=0.5)


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_rule_repeated_keys(pkg, device, longest):
    """One key in every token: the chunk's system is as far from the identity as it gets."""
    layer = Layer(pkg, device, [200, 64], raw_gates=False, decay_scale=0.001, seed=8)
    for t in (layer.key, layer.d["key"]):
        t[:] = t[:1].clone()
    layer.check_rule(layer.rule(longest=longest))


def test_rule_gates_at_their_ends(pkg, device):
    """Decays of zero and -infinity, writes of zero and one; a key of zeros."""
    for longest in (1, 16, 200):
        layer = Layer(pkg, device, [80, 5], raw_gates=False, seed=4)
        for t in (layer.decay, layer.d["decay"]):
            t[3], t[10], t[70], t[82] = float("-inf"), 0.0, float("-inf"), float("-inf")
        for t in (layer.beta, layer.d["beta"]):
            t[5], t[11], t[83] = 0.0, 1.0, 0.0
        for t in (layer.key, layer.d["key"]):
            t[6], t[84] = 0.0, 0.0
        layer.check_rule(layer.rule(longest=longest))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("spans,counts", [([1], [1]), ([16, 9, 1, 15, 2], [16, 4, 0, 1, 2]), ([0, 3, 40], [5, 2, 33]),
                                          ([5, 5, 5], [-1, 77, 3])])
def test_advance(pkg, device, spans, counts, shape):
    layer = Layer(pkg, device, spans, counts=counts, missing=(2,) if len(spans) > 3 else (), fresh=(1,) if len(spans) > 1 else (), spare=1,
                  **shape)
    layer.advance()
    _, _, recurrent, bound = layer.expected_rule()
    layer.check_state(recurrent, bound)
    assert same_bits(layer.d["history"].cpu(), layer.expected_conv()[2])


def test_advance_is_what_the_forward_leaves(pkg, device):
    """A verify block taken without advancing, then committed whole, leaves what a forward that advances does."""
    spans = [16, 3, 1, 12]
    kept = Layer(pkg, device, spans, counts=[0] * 4, seed=2)
    ahead = Layer(pkg, device, spans, seed=2)
    out = (kept.conv(), kept.rule(longest=16)), (ahead.conv(), ahead.rule(longest=16))
    assert all(same_bits(a.cpu(), b.cpu()) for a, b in zip(*out))
    assert same_bits(kept.d["history"].cpu(), kept.history) and same_bits(kept.d["recurrent"].cpu(), kept.recurrent)
    kept.d["counts"] = torch.tensor(spans, dtype=torch.int32, device=device)
    kept.advance()
    assert same_bits(kept.d["history"].cpu(), ahead.d["history"].cpu())
    want, bound = ahead.expected_rule()[2:]
    kept.counts = torch.tensor(spans)
    kept.check_state(want, bound)


@pytest.mark.parametrize("longest", [1, 16, 500])
def test_repeats_bit_for_bit(pkg, device, longest):
    spans = [1, 16, 200, 65, 0, 3]
    a, b = (Layer(pkg, device, spans, seed=6, key_heads=4, value_heads=8) for _ in range(2))
    assert same_bits(a.rule(longest=longest).cpu(), b.rule(longest=longest).cpu())
    assert same_bits(a.d["recurrent"].cpu(), b.d["recurrent"].cpu())


def test_blocks_in_pieces(pkg, device):
    """A prompt in pieces leaves the state and gives the outputs of the whole, to the roundings."""
    whole = Layer(pkg, device, [150, 90], seed=9, fresh=(0, 1))
    want = whole.expected_rule()
    for cut in (1, 16, 64, 77):
        layer = Layer(pkg, device, [150, 90], seed=9, fresh=(0, 1))
        d, got = layer.d, torch.zeros((240, layer.hv, layer.dim), dtype=layer.dtype, device=device)
        for first, last, fresh in ((0, cut, True), (cut, None, False)):
            rows = torch.cat([torch.arange(s, e)[first:last] for s, e in ((0, 150), (150, 240))]).to(device)
            n = [len(torch.arange(e)[first:last]) for e in (150, 90)]
            starts = torch.tensor([0, n[0], n[0] + n[1]], dtype=torch.int32, device=device)
            got[rows] = pkg.ops.gdn_rule(d["query"][rows], d["key"][rows], d["value"][rows], d["decay"][rows], d["beta"][rows], layer.pool,
                                         starts, a_log=d["a_log"], dt_bias=d["dt_bias"], fresh=torch.tensor([fresh] * 2, device=device))
        assert float(((got.double().cpu() - want[0]).abs() - want[1]).max()) <= 0
        layer.check_state(want[2], want[3], str(cut))


@pytest.mark.parametrize("longest", [60, 200])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (128, FP16), (64, BF16), (64, FP16)])
def test_rule_of_prompts_with_many_heads(pkg, device, dim, dtype, longest):
    """Sequences and heads enough that a workgroup takes 32 columns of the state (at 60, which says that all are about alike); blocks that
    end at every place of a chunk, empty and fresh ones among them, counts inside."""
    spans = [70, 1, 130, 0, 64, 200, 33, 129] * (1 if dim == 128 else 2)
    for counts in (None, [min(n, 65) - b % 3 for b, n in enumerate(spans)]):
        layer = Layer(pkg, device, spans, key_heads=4, value_heads=8, dim=dim, dtype=dtype, seed=11, spare=2, missing=(2,), fresh=(0, 5),
                      counts=counts)
        out = filled(layer, layer.hv, dim)
        layer.rule(out, longest=longest)
        layer.check_rule(out)
        assert (out[layer.tokens:] == 7.0).all()


@pytest.mark.parametrize("longest", [None, 1, 16, 250])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (128, FP16), (64, BF16), (64, FP16)])
def test_rule_of_long_and_short_blocks(pkg, device, dim, dtype, longest):
    """Prompts among verify blocks and single tokens, whose launches share the batch: every sequence in exactly one of them."""
    spans = [1, 2, 200, 0, 3, 33, 32, 16, 70, 1, 34, 31, 1, 5, 250, 0, 4, 17, 64, 65, 1, 1, 12, 40, 1, 2] * (1 if dim == 128 else 3)
    for counts in (None, [(n * 3) // 4 + b % 2 for b, n in enumerate(spans)], [0] * len(spans)):
        layer = Layer(pkg, device, spans, value_heads=6, dim=dim, dtype=dtype, seed=12, spare=2, missing=(1, 8), fresh=(0, 2, 6, 20), counts=counts)
        out = filled(layer, layer.hv, dim)
        layer.rule(out, longest=longest)
        layer.check_rule(out)
        assert (out[layer.tokens:] == 7.0).all()


def test_rule_of_many_sequences(pkg, device):
    """More sequences than are searched at a time, prompts at the search's ends."""
    spans = [1] * 200
    for b, n in ((0, 40), (63, 70), (64, 65), (127, 33), (130, 130), (199, 99)):
        spans[b] = n
    layer = Layer(pkg, device, spans, value_heads=2, seed=13, fresh=(63, 199), missing=(64,))
    layer.check_rule(layer.rule(longest=130))
    layer.d["starts"][:] = 0   # every block empty
    assert layer.rule(longest=130).shape == (layer.total, 2, 128)
