"""GPU: the delta rule's products where terms cancel, and states that are kept over thousands of tokens, against 64 bits."""
import pytest
import torch

from batch_util import EPS, TINY, UNIT, Layer

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SHAPES = [(128, BF16), (128, FP16), (64, BF16), (64, FP16)]
WAYS = [1, 16, 200]      # token after token, 16 at a time, 64 at a time


def put(layer, name, value):
    """A changed tensor of the layer on both sides."""
    t = getattr(layer, name)
    t.copy_(value)
    layer.d[name].copy_(t)


@pytest.mark.parametrize("longest", WAYS)
@pytest.mark.parametrize("dim,dtype", SHAPES)
def test_outputs_of_states_that_cancel(pkg, device, dim, dtype, longest):
    """o = S^T q of two of the state's rows that take all but 2^-14 of each other off.

    A product of q's 16 bits and S is as exact as fp32: S stands in parts that hold it to EPS / 2, its at most twelve part products
    are exact, and each sum of them is off by at most 2 EPS (a matrix instruction may cut off) of |q||S|; factors are 1.  2 * 12 + 1 and
    one more for the factor: 26 EPS of the sum of |q||S|, and the output's own rounding.
    """
    layer = Layer(pkg, device, [20, 70], dim=dim, dtype=dtype, raw_gates=False, seed=3, strided=False)
    gen = torch.Generator().manual_seed(4)
    s = torch.randn(layer.recurrent.shape, generator=gen)
    s[:, :, 1::2] = -s[:, :, 0::2] + 2.0 ** -14 * s[:, :, 1::2]
    put(layer, "recurrent", s)
    for name in ("key", "value", "decay", "beta"):
        put(layer, name, 0.0)
    q = torch.zeros(layer.query.shape)
    for t in range(layer.total):
        at = 2 * int(torch.randint(0, dim // 2, (), generator=gen))
        q[t, :, at:at + 2] = 1.0 + float(torch.rand((), generator=gen))
    put(layer, "query", q.to(dtype))
    got = layer.rule(longest=longest, normalise=False, scale=1.0).double().cpu()
    rep = layer.hv // layer.hk
    for b, at in enumerate((0, 20)):
        n, state, rows = layer.spans[b], layer.recurrent[int(layer.slots[b])].double(), layer.query.double().repeat_interleave(rep, 1)
        rows = rows[at:at + n].transpose(0, 1)
        want, size = rows @ state, rows.abs() @ state.abs()
        over = (got[at:at + n].transpose(0, 1) - want).abs() - (26 * EPS * size + UNIT[dtype] * want.abs() + TINY[dtype])
        assert float(over.max()) <= 0, (b, float((over / size).max()) / EPS)


@pytest.mark.parametrize("longest", WAYS)
@pytest.mark.parametrize("dim,dtype", SHAPES)
def test_outputs_of_tokens_that_cancel(pkg, device, dim, dtype, longest):
    """o = P_0 u_0 + P_1 u_1 of two tokens of one block that take all but 2^-14 of each other off: k of one feature each, q of both.

    u = beta v is off by at most 3 EPS (its factors' product, and as parts of an operand), P_0 = e^g by 6 (the exponent's rounding and
    product, g >= -1, and the exponential's two steps; its parts), the at most twelve part products' sums by 2 EPS each: with |P_0 u_0| the
    size of both terms 2 (3 + 6 + 24) = 66 EPS of it, and the output's own rounding.
    """
    layer = Layer(pkg, device, [20, 70], dim=dim, dtype=dtype, raw_gates=False, seed=5, strided=False, fresh=(0, 1))
    gen = torch.Generator().manual_seed(6)
    n, hv = layer.total, layer.hv
    for t in range(0, n, 2):     # pairs of tokens, each with two features of its own (the others' keys are at right angles)
        a, b = (t % (dim // 2)) * 2, (t % (dim // 2)) * 2 + 1
        k, q, v = torch.zeros((2, layer.hk, dim)), torch.zeros((2, layer.hk, dim)), torch.randn((hv, dim), generator=gen).to(dtype)
        k[0, :, a], k[1, :, b], q[1, :, a], q[1, :, b] = 1.0, 1.0, 1.0, 1.0
        layer.key[t:t + 2], layer.query[t:t + 2] = k.to(dtype), q.to(dtype)
        layer.value[t], layer.value[t + 1] = v, -v
        g = -torch.rand((hv,), generator=gen)
        layer.decay[t], layer.decay[t + 1] = float("-inf"), g      # nothing of the pairs before
        layer.beta[t] = 0.5 + 0.5 * torch.rand((hv,), generator=gen)
        layer.beta[t + 1] = layer.beta[t].double() * g.double().exp() * (1 - 2.0 ** -14)
    for name in ("key", "query", "value", "decay", "beta"):
        layer.d[name].copy_(getattr(layer, name))
    got = layer.rule(longest=longest, normalise=False, scale=1.0).double().cpu()
    old = layer.value.double()[0::2] * layer.beta.double()[0::2, :, None] * layer.decay.double()[1::2, :, None].exp()
    new = layer.value.double()[1::2] * layer.beta.double()[1::2, :, None]
    want = old + new
    over = (got[1::2] - want).abs() - (66 * EPS * old.abs() + UNIT[dtype] * want.abs() + TINY[dtype])
    assert float(over.max()) <= 0, float((over / old.abs()).max()) / EPS
    assert not bool(got[0::2].any())      # a query of zeros


GATES = torch.tensor([-1 / 4000, -1 / 3000, -1e-4, -1 / 2500, -1 / 7000, -2e-4])


def kept(layer, calls):
    """The norm of what the states are off by, over theirs, after their decays alone; and what roundings that act independently leave:
    each of `calls` steps rounds an element at most three times, by at most EPS."""
    return (16 + 3 * calls ** 0.5) * EPS


@pytest.mark.parametrize("spans,count", [([4, 1, 16], 1), ([7, 3, 2], 2), ([16, 5, 9], 3)])
@pytest.mark.parametrize("dim,dtype", SHAPES)
def test_states_after_thousands_of_commits(pkg, device, dim, dtype, spans, count):
    """A speculative run's commits of a token or a few at a time: a decay that is rounded near 1 would add up over what a head remembers.
    The decays' own part alone has a closed form: nothing is written (beta 0), and S is e^(sum of g) of what it was."""
    calls = 6000
    layer = Layer(pkg, device, spans, value_heads=6, dim=dim, dtype=dtype, raw_gates=False, seed=7, counts=[count] * len(spans))
    put(layer, "beta", 0.0)
    put(layer, "decay", GATES.expand(layer.total, 6))
    for _ in range(calls):
        layer.advance()
    got = layer.d["recurrent"].double().cpu()
    for b, n in enumerate(spans):
        tokens, was = calls * min(count, n), layer.recurrent[int(layer.slots[b])].double()
        want = was * (GATES.float().double() * tokens).exp()[:, None, None]
        off = (got[int(layer.slots[b])] - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
        assert float(off.max()) <= kept(layer, calls), (b, off / kept(layer, calls))


@pytest.mark.parametrize("longest,spans", [(1, [1, 1]), (16, [5, 16]), (16, [1, 9]), (16, [17, 4]), (200, [64, 70]), (200, [33, 130])])
@pytest.mark.parametrize("dim,dtype", SHAPES)
def test_states_after_thousands_of_blocks(pkg, device, dim, dtype, longest, spans):
    """The same through the rule, which advances by its blocks: token after token, 16 and 64 at a time."""
    steps = {1: 1, 16: 16, 200: 64}[longest]
    calls = 4000 if longest < 200 else 1500
    layer = Layer(pkg, device, spans, value_heads=6, dim=dim, dtype=dtype, raw_gates=False, seed=8)
    gates = GATES * (1.0 if longest == 1 else 0.2 if longest == 16 else 0.02)
    put(layer, "beta", 0.0)
    put(layer, "decay", gates.expand(layer.total, 6))
    for _ in range(calls):
        layer.rule(longest=longest)
    got = layer.d["recurrent"].double().cpu()
    for b, n in enumerate(spans):
        was = layer.recurrent[int(layer.slots[b])].double()
        want = was * (gates.float().double() * (calls * n)).exp()[:, None, None]
        off = (got[int(layer.slots[b])] - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
        limit = kept(layer, calls * -(-n // steps))
        assert float(off.max()) <= limit, (b, off / limit)


@pytest.mark.parametrize("dim,dtype", SHAPES)
def test_a_run_of_commits(pkg, device, dim, dtype):
    """Commits of one token each with keys, values and writes: the state against the 64-bit recurrence."""
    calls = 4000
    layer = Layer(pkg, device, [4], key_heads=3, value_heads=6, dim=dim, dtype=dtype, raw_gates=False, seed=9, counts=[1])
    ops, d = pkg.ops, layer.d
    gen = torch.Generator().manual_seed(10)
    rows = torch.randn((calls + 3, layer.channels), generator=gen).to(dtype)
    key, value = rows[:, :3 * dim].unflatten(-1, (3, dim)), rows[:, 6 * dim:].unflatten(-1, (6, dim))
    beta, decay = torch.rand((calls + 3, 6), generator=gen) * 0.1, GATES.expand(calls + 3, 6).contiguous()
    dev = [t.to(device) for t in (rows, rows, beta, decay)]
    dkey, dvalue = dev[0][:, :3 * dim].unflatten(-1, (3, dim)), dev[0][:, 6 * dim:].unflatten(-1, (6, dim))
    for i in range(calls):
        part = slice(i, i + 4)
        ops.gdn_advance(layer.pool, dev[0][part], dkey[part], dvalue[part], dev[3][part], dev[2][part], d["starts"], d["counts"])
    s = layer.recurrent[int(layer.slots[0])].double()
    k = key.double()
    k = (k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(2, 1)
    fade = GATES.double().exp()[:, None, None]
    for i in range(calls):
        s = fade * s
        u = beta[i].double()[:, None] * (value[i].double() - (s * k[i][..., None]).sum(1))
        s = s + k[i][..., None] * u[:, None, :]
    got = d["recurrent"][int(layer.slots[0])].double().cpu()
    off = (got - s).flatten(1).norm(dim=1) / s.flatten(1).norm(dim=1)
    memory = float((1 - (GATES.double() * calls).exp()).div(-GATES.double()).max())
    assert float(off.max()) <= (16 + 3 * memory ** 0.5) * EPS, off / EPS
