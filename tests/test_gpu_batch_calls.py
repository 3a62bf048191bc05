"""GPU: how the operators of a batch's states and drafts are called: refusals, odd calls, streams, captured graphs, far strides, NaN of
other sequences, and a run of them together."""
import pytest
import torch

from batch_util import Layer, same_bits, verified

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def drafts(device, spans, vocab=1009, dtype=BF16, seed=0, spare=0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(spans) + spare
    target = (torch.randn((rows, vocab), generator=gen) * 3).to(dtype)
    draft = (target.float() + torch.randn((rows, vocab), generator=gen)).to(dtype)
    c = dict(target=target, drafted=draft.float().argmax(1).to(torch.int32), starts=torch.tensor([sum(spans[:b]) for b in range(len(spans) + 1)],
                                                                                                 dtype=torch.int32),
             uniforms=torch.rand((rows,), generator=gen), draft=draft, temperature=torch.full((len(spans),), 0.9))
    return c, {k: v.to(device) for k, v in c.items()}


@pytest.fixture
def python_form(pkg, monkeypatch):
    """Calls a function with the native form switched off."""
    def call(fn, *args, **kw):
        with monkeypatch.context() as m:
            m.setattr(pkg.ops, "_plain", lambda x: False)
            return fn(*args, **kw)
    return call


def twins(pkg, device, *args, **kw):
    return Layer(pkg, device, *args, **kw), Layer(pkg, device, *args, **kw)


def same_states(a, b):
    return same_bits(a.d["history"].cpu(), b.d["history"].cpu()) and same_bits(a.d["recurrent"].cpu(), b.d["recurrent"].cpu())


# ------------------------------------------------------------------ refusals
def test_refusals_of_the_states(pkg, device, python_form):
    ops, layer = pkg.ops, Layer(pkg, device, [3, 2], counts=[3, 2])
    d, pool, before = layer.d, layer.pool, Layer(pkg, device, [3, 2])
    other = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
    conv = lambda x=d["x"], w=d["weight"], pool=pool, s=d["starts"], **kw: ops.gdn_conv(x, w, pool, s, **kw)  # noqa: E731
    rule = lambda q=d["query"], k=d["key"], v=d["value"], g=d["decay"], b=d["beta"], pool=pool, s=d["starts"], **kw: ops.gdn_rule(  # noqa: E731
        q, k, v, g, b, pool, s, **{"a_log": d["a_log"], "dt_bias": d["dt_bias"], **kw})
    advance = lambda pool=pool, x=d["x"], k=d["key"], counts=d["counts"], **kw: ops.gdn_advance(  # noqa: E731
        pool, x, k, d["value"], d["decay"], d["beta"], d["starts"], counts, **{"a_log": d["a_log"], "dt_bias": d["dt_bias"], **kw})
    part = lambda **kw: pool._replace(**kw)  # noqa: E731
    calls = [
        (lambda: conv(pool=(pool.history, None, pool.slots)), "StatePool"), (lambda: conv(x=d["x"].half()), "history must be"),
        (lambda: conv(x=d["x"].float(), w=d["weight"].float()), "history must be"), (lambda: conv(x=d["x"][:, :512]), "x must be"),
        (lambda: conv(x=d["x"][0]), "x must be"), (lambda: conv(x=d["x"].cpu()), "x must be"), (lambda: conv(w=d["weight"][:, 0]), "weight"),
        (lambda: conv(w=d["weight"].half()), "weight"), (lambda: conv(s=d["starts"][:2]), "starts"), (lambda: conv(s=d["starts"].long()), "starts"),
        (lambda: conv(counts=other(3)), "counts"), (lambda: conv(counts=other(2).long()), "counts"),
        (lambda: conv(fresh=other(2)), "fresh"), (lambda: conv(fresh=torch.zeros(3, dtype=torch.bool, device=device)), "fresh"),
        (lambda: conv(fresh=torch.zeros(2, dtype=torch.bool)), "fresh"), (lambda: conv(out=torch.zeros((4, 1024), dtype=BF16, device=device)), "out"),
        (lambda: conv(out=torch.zeros((1024, 5), dtype=BF16, device=device).t()), "out"),
        (lambda: conv(pool=part(history=pool.history[..., :2])), "contiguous slots|four taps"),
        (lambda: conv(pool=part(history=pool.history[0])), "history"), (lambda: conv(pool=part(history=None)), "history"),
        (lambda: conv(pool=part(history=pool.history[:1].expand(5, -1, -1))), "overlap"),
        (lambda: conv(pool=part(history=pool.history.transpose(1, 2).contiguous().transpose(1, 2))), "contiguous slots"),
        (lambda: conv(pool=part(slots=pool.slots.long())), "slots"), (lambda: conv(pool=part(slots=pool.slots[None])), "slots"),
        (lambda: conv(x=d["x"].clone().requires_grad_()), "no_grad"), (lambda: conv(w=d["weight"].clone().requires_grad_()), "no_grad"),
        (lambda: rule(q=None), "query"), (lambda: rule(q=d["query"][:, :1]), "query"), (lambda: rule(k=d["key"][:4]), "key"),
        (lambda: rule(q=d["query"][..., :64]), "query"), (lambda: rule(v=d["value"][:, :3]), "value"), (lambda: rule(v=d["value"].float()), "bfloat16 or float16|key"),
        (lambda: rule(q=d["value"][:, :3], k=d["value"][:, :3]), "multiple"), (lambda: rule(q=d["query"][:, :0], k=d["key"][:, :0]), "multiple"),
        (lambda: rule(g=d["decay"][:, :2]), "decay"), (lambda: rule(g=d["decay"].float()), "one dtype"), (lambda: rule(b=d["beta"].double()), "beta"),
        (lambda: rule(a_log=None), "go together"), (lambda: rule(dt_bias=d["dt_bias"].to(BF16)), "dt_bias"),
        (lambda: rule(a_log=d["a_log"][:2]), "a_log"), (lambda: rule(normalise=1), "normalise"), (lambda: rule(scale="1"), "scale"),
        (lambda: rule(longest=-1), "longest"), (lambda: rule(longest=2.0), "longest"), (lambda: rule(out=d["value"].float()), "out"),
        (lambda: rule(pool=part(recurrent=pool.recurrent.to(BF16))), "recurrent"),
        (lambda: rule(pool=part(recurrent=pool.recurrent[..., :64])), "recurrent"),
        (lambda: rule(pool=part(recurrent=pool.recurrent.transpose(2, 3))), "contiguous slots"),
        (lambda: rule(pool=part(recurrent=pool.recurrent[:1].expand(5, -1, -1, -1))), "overlap"),
        (lambda: rule(q=d["query"].clone().requires_grad_()), "no_grad"), (lambda: rule(g=d["decay"].clone().requires_grad_()), "no_grad"),
        (lambda: advance(counts=None), "counts"), (lambda: advance(x=d["x"][:4]), "x must be"), (lambda: advance(x=d["x"].half()), "x must be"),
        (lambda: advance(pool=part(recurrent=pool.recurrent[:4])), "as many slots"), (lambda: advance(pool=part(history=None)), "history"),
        (lambda: advance(k=d["key"].clone().requires_grad_()), "no_grad")]
    for i, (call, message) in enumerate(calls):
        for form in (lambda c: c(), python_form):
            with pytest.raises(ValueError, match=message):
                form(call)
                print("not refused:", i)
    whole = d["value"].contiguous()
    for call, message in [(lambda: rule(scale=float("nan")), "scale"), (lambda: rule(v=whole, out=whole), "out cannot be")]:
        with pytest.raises(pkg._lib.DflashError, match=message):
            call()
    torch.cuda.synchronize()
    assert same_states(layer, before)


def test_workspaces(pkg, device):
    layer = Layer(pkg, device, [300, 70], seed=1)
    size = pkg.ops.gdn_rule_workspace_bytes(370, 2, 4, 128, 2, 300)
    assert size > 0
    room = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=device)
    for bad in (room[:size - 1], room.view(torch.int8), torch.zeros((size,), dtype=torch.uint8), room[:1].expand(size), room[::2]):
        with pytest.raises(ValueError, match="workspace"):
            layer.rule(longest=300, workspace=bad)
    layer.check_rule(layer.rule(longest=300, workspace=room[:size]))
    assert (room[size:] == 0x5A).all()
    c, dev = drafts(device, [3, 2])
    size = pkg.ops.verify_drafts_workspace_bytes(5, 1009, 2, True)
    room = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=device)
    with pytest.raises(ValueError, match="workspace"):
        pkg.ops.verify_drafts(**dev, workspace=room[:size - 1])
    got = pkg.ops.verify_drafts(**dev, workspace=room[:size])
    assert got.accepted.tolist() == verified(**c)[0].tolist() and got.token.tolist() == verified(**c)[1].tolist()
    assert (room[size:] == 0x5A).all()


def test_refusals_of_the_drafts(pkg, device, python_form):
    _, dev = drafts(device, [3, 2])
    for name, value, message in [
            ("target", dev["target"].double(), "target"), ("target", dev["target"][0], "target"), ("target", dev["target"].cpu(), "ROCm"),
            ("target", dev["target"][:, :0], "target"), ("draft", dev["draft"].half(), "draft"), ("draft", dev["draft"][:, :5], "draft"),
            ("drafted", dev["drafted"].long(), "drafted"), ("drafted", dev["drafted"][:4], "drafted"), ("starts", dev["starts"][:0], "starts"),
            ("starts", dev["starts"].long(), "starts"), ("uniforms", dev["uniforms"].double(), "uniforms"),
            ("uniforms", dev["uniforms"][:4], "uniforms"), ("temperature", dev["temperature"][:1], "temperature"),
            ("temperature", dev["temperature"].double(), "temperature"), ("temperature", 0.7, "temperature"),
            ("target", dev["target"].clone().requires_grad_(), "no_grad"), ("draft", dev["draft"].clone().requires_grad_(), "no_grad")]:
        for form in (lambda f, **kw: f(**kw), python_form):
            with pytest.raises(ValueError, match=message):
                form(pkg.ops.verify_drafts, **{**dev, name: value})


# ------------------------------------------------------------------ odd calls
def test_empty_calls(pkg, device, python_form):
    for form in (lambda f, *a, **kw: f(*a, **kw), python_form):
        layer, before = twins(pkg, device, [0, 0])
        assert form(layer.conv).shape == (0, 1024) and form(layer.rule).shape == (0, 4, 128)
        layer.d["counts"] = torch.ones(2, dtype=torch.int32, device=device)
        form(layer.advance)
        none = Layer(pkg, device, [], spare=3)
        out = torch.full((3, 4, 128), 7.0, dtype=BF16, device=device)
        assert (form(none.rule, out) == 7.0).all()
        assert (form(none.conv, torch.full((3, 1024), 7.0, dtype=BF16, device=device)) == 7.0).all()
        assert same_states(layer, before)
        _, dev = drafts(device, [0, 0])
        got = form(pkg.ops.verify_drafts, **dev)
        assert got.accepted.tolist() == [0, 0] and got.token.tolist() == [-1, -1]
        _, dev = drafts(device, [], spare=2)
        assert form(pkg.ops.verify_drafts, **dev).accepted.shape == (0,)


@pytest.mark.parametrize("longest", [1, 16, 200, None])
def test_starts_that_are_no_such_thing_stay_inside(pkg, device, longest):
    """Offsets out of order or past the block, counts and slots of any value: nothing behind the block, the workspace or the pool."""
    layer = Layer(pkg, device, [64, 70, 66], seed=3, counts=[0, 0, 0])
    d = layer.d
    rows, mixed, heads = 200, torch.full((264, 1024), 3.0, dtype=BF16, device=device), torch.full((264, 4, 128), 3.0, dtype=BF16, device=device)
    size = pkg.ops.gdn_rule_workspace_bytes(rows, 2, 4, 128, 3, longest or 0)
    room = torch.full((size + (1 << 20),), 0x5A, dtype=torch.uint8, device=device)
    d["slots"].copy_(torch.tensor([2, -1, 0], dtype=torch.int32))
    held = d["recurrent"][3:].clone(), d["history"][3:].clone()
    for bad in ([0, 200, 2, 200], [-5, 3, 1 << 30, -(1 << 31)], [200, 0, 200, 0], [9, 9, 9, 9], [1 << 30] * 4):
        d["starts"].copy_(torch.tensor(bad, dtype=torch.int32))
        for counts in ([1 << 30, 5, -(1 << 31)], [64, 64, 65]):
            d["counts"] = torch.tensor(counts, dtype=torch.int32, device=device)
            layer.conv(mixed[:rows])
            layer.rule(heads[:rows], longest=longest, workspace=room[:max(size, 1)])
            layer.advance()
    torch.cuda.synchronize()
    assert (mixed[rows:] == 3).all() and (heads[rows:] == 3).all() and (room[size:] == 0x5A).all()
    assert same_bits(d["recurrent"][3:].cpu(), held[0].cpu()) and same_bits(d["history"][3:].cpu(), held[1].cpu())


def test_starts_of_many_sequences_that_are_no_such_thing_stay_inside(pkg, device):
    """The same of a batch whose long and short blocks have launches of their own: more long blocks than the tokens could hold."""
    layer = Layer(pkg, device, [20] * 30, seed=3, counts=[0] * 30)
    d, heads = layer.d, torch.full((664, 4, 128), 3.0, dtype=BF16, device=device)
    size = pkg.ops.gdn_rule_workspace_bytes(600, 2, 4, 128, 30, 300)
    assert size > 0
    room = torch.full((size + (1 << 20),), 0x5A, dtype=torch.uint8, device=device)
    before = d["recurrent"].clone()
    for bad in ([0, 600] * 15 + [0], [0] + [600, 0] * 15, [0] + [40, 600] * 15, list(range(600, -20, -20)), [1 << 30] * 31, [-(1 << 31), 1 << 30] * 15 + [5]):
        d["starts"].copy_(torch.tensor(bad, dtype=torch.int32))
        layer.rule(heads[:600], longest=300, workspace=room[:size])
    torch.cuda.synchronize()
    assert (heads[600:] == 3).all() and (room[size:] == 0x5A).all() and same_bits(before.cpu(), d["recurrent"].cpu())


def test_rows_of_drafts_that_are_no_such_thing_stay_inside(pkg, device):
    _, dev = drafts(device, [5, 4, 7], vocab=3001)
    size = pkg.ops.verify_drafts_workspace_bytes(16, 3001, 3, True)
    room = torch.full((size + (1 << 20),), 0x5A, dtype=torch.uint8, device=device)
    for bad in ([0, 16, 2, 16], [-5, 3, 1 << 30, -(1 << 31)], [16, 0, 16, 0], [9, 9, 9, 9], [1 << 30] * 4):
        dev["starts"] = torch.tensor(bad, dtype=torch.int32, device=device)
        got = pkg.ops.verify_drafts(**dev, workspace=room[:size])
        assert bool(((got.accepted >= 0) & (got.accepted <= 16)).all())
    assert (room[size:] == 0x5A).all()


def test_far_strides(pkg, device):
    """Rows, slots and logits whose offsets pass 32 bits."""
    rows, each = 70, 1 << 26
    space = torch.empty((rows * each,), dtype=BF16, device=device)
    states = torch.empty((4 * (1 << 29) + (1 << 20),), dtype=FP32, device=device)
    pasts = torch.empty((4 * (1 << 29) + (1 << 20),), dtype=BF16, device=device)
    for longest in (1, 16, 200):
        layer = Layer(pkg, device, [40, 30], seed=4, counts=[40, 7])
        d = layer.d
        at = 0
        for name in ("x", "query", "key", "value"):
            wide = d[name].flatten(1)
            place = space.as_strided((rows, wide.shape[1]), (each, 1), at)
            place.copy_(wide)
            d[name], at = place.unflatten(1, d[name].shape[1:]), at + wide.shape[1]
        for name, memory in (("recurrent", states), ("history", pasts)):
            place = memory.as_strided(d[name].shape, (1 << 29, *d[name].stride()[1:]))
            place.copy_(d[name])
            d[name] = place
        d["slots"].copy_(torch.tensor([4, 3], dtype=torch.int32))
        layer.slots = torch.tensor([4, 3], dtype=torch.int32)
        layer.pool = pkg.ops.StatePool(d["history"], d["recurrent"], d["slots"])
        layer.check_conv(layer.conv())
        layer.check_rule(layer.rule(longest=longest))
    kept = Layer(pkg, device, [40, 30], seed=4, counts=[40, 7])
    kept.slots, old = layer.slots, (layer.d["recurrent"], layer.d["history"])
    old[0].copy_(kept.d["recurrent"]), old[1].copy_(kept.d["history"])
    layer.advance()
    kept.d["recurrent"], kept.d["history"] = old
    kept.check_state(*kept.expected_rule()[2:])
    assert same_bits(kept.d["history"].cpu(), kept.expected_conv()[2])
    c, dev = drafts(device, [3, 1], seed=2)
    for i, name in enumerate(("target", "draft")):
        place = space.as_strided((4, 1009), (1 << 30, 1), 5000 * i + i)
        place.copy_(dev[name])
        dev[name] = place
    got = pkg.ops.verify_drafts(**dev)
    assert got.accepted.tolist() == verified(**c)[0].tolist() and got.token.tolist() == verified(**c)[1].tolist()


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_nan_stays_in_its_sequence(pkg, device, longest):
    spans, rows = [20, 35, 70], slice(20, 55)
    clean, dirty = twins(pkg, device, spans, seed=5)
    bad = int(dirty.slots[1])
    for name in ("x", "query", "key", "value", "decay", "beta"):
        dirty.d[name][20:55] = float("nan")
    dirty.d["recurrent"][bad], dirty.d["history"][bad] = float("nan"), float("inf")
    for one, other in ((clean.conv(), dirty.conv()), (clean.rule(longest=longest), dirty.rule(longest=longest))):
        one[rows], other[rows] = 0, 0
        assert same_bits(one.cpu(), other.cpu())
    for name in ("recurrent", "history"):
        clean.d[name][bad], dirty.d[name][bad] = 0, 0
    assert same_states(clean, dirty)


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_infinities_stay_in_their_head(pkg, device, longest):
    clean, dirty = twins(pkg, device, [20, 70], seed=5)
    dirty.d["value"][30, 1], dirty.d["decay"][31, 1], dirty.d["beta"][2, 1] = float("inf"), float("nan"), float("inf")
    a, b = clean.rule(longest=longest), dirty.rule(longest=longest)
    a[:, 1], b[:, 1], clean.d["recurrent"][:, 1], dirty.d["recurrent"][:, 1] = 0, 0, 0, 0
    assert same_bits(a.cpu(), b.cpu()) and same_states(clean, dirty)


# ------------------------------------------------------------------ forms, streams, graphs
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_native_and_python_forms(pkg, device, python_form, dtype):
    """Both enqueue the same kernels with the same arguments."""
    for kw in (dict(), dict(fresh=(1,), counts=[2, 0, 70]), dict(raw_gates=False, missing=(0,))):
        a, b = twins(pkg, device, [2, 1, 70], seed=6, dtype=dtype, spare=1, **kw)
        zero = lambda layer, *shape: torch.zeros((74, *shape), dtype=dtype, device=device)  # noqa: E731
        d = a.d
        assert pkg._lib.host().gdn_conv(d["x"], d["weight"], a.pool, d["starts"], d["fresh"], None, None) is not None
        python_form(b.conv)
        for longest in (None, 16):
            assert same_bits(a.conv(zero(a, 1024)).cpu(), python_form(b.conv, zero(b, 1024)).cpu())
            assert same_bits(a.rule(zero(a, 4, 128), longest=longest).cpu(), python_form(b.rule, zero(b, 4, 128), longest=longest).cpu())
        a.d["counts"] = b.d["counts"] = torch.tensor([1, 1, 33], dtype=torch.int32, device=device)
        a.advance()
        python_form(b.advance)
        assert same_states(a, b)
    _, dev = drafts(device, [3, 5, 1], dtype=dtype)
    for draft in (dev["draft"], None):
        for temperature in (dev["temperature"], None):
            kw = {**dev, "draft": draft, "temperature": temperature}
            one, other = pkg.ops.verify_drafts(**kw), python_form(pkg.ops.verify_drafts, **kw)
            assert torch.equal(one.accepted, other.accepted) and torch.equal(one.token, other.token)


def test_streams_side_by_side(pkg, device):
    """Calls on streams side by side, each with what it allocates itself, give what they give alone."""
    prompt, block = Layer(pkg, device, [900, 500], seed=7, counts=[0, 0]), Layer(pkg, device, [16] * 20, seed=8, counts=[0] * 20)
    _, dev = drafts(device, [8] * 16, vocab=32_001)
    calls = (lambda: (prompt.conv(), prompt.rule(longest=900)), lambda: (block.conv(), block.rule(longest=16)),
             lambda: tuple(pkg.ops.verify_drafts(**dev)))
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    for one, many in zip(alone, got):
        assert all(torch.equal(a, b) for other in many for a, b in zip(one, other))


@pytest.mark.parametrize("longest", [1, 16, 200])
def test_steps_of_a_captured_graph(pkg, device, longest):
    """Conv, rule, check and advance captured once, replayed while rows, starts, slots, drafts and random numbers change; a second
    graph of the same calls between the replays; every replay as the eager calls."""
    layer = Layer(pkg, device, [40, 30, 30], seed=9, counts=[0, 0, 0])
    d = layer.d
    _, dev = drafts(device, [40, 30, 30], vocab=701, seed=9)
    out = torch.zeros((2, 100, 1024), dtype=BF16, device=device), torch.zeros((2, 100, 4, 128), dtype=BF16, device=device)
    stay = d["counts"]

    def step(i):
        d["counts"] = stay
        layer.conv(out[0][i])
        layer.rule(out[1][i], longest=longest)
        got = pkg.ops.verify_drafts(**{**dev, "starts": d["starts"]})
        d["counts"] = got.accepted + 1
        layer.advance()
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    memory = torch.cuda.graph_pool_handle()
    for g in graphs:
        with torch.cuda.graph(g, pool=memory):
            outs.append(step(1))
    gen = torch.Generator().manual_seed(1)
    for i in range(6):
        cuts = sorted(torch.randint(0, 101, (2,), generator=gen).tolist())
        d["starts"].copy_(torch.tensor([0, *cuts, 100], dtype=torch.int32))
        d["slots"].copy_(torch.randperm(6, generator=gen)[:3].to(torch.int32))
        dev["uniforms"].copy_(torch.rand((100,), generator=gen))
        d["x"].copy_(d["x"].roll(1, 0))
        d["value"].copy_(d["value"].roll(1, 0))
        held = d["history"].clone(), d["recurrent"].clone()
        got = step(0)
        after = d["history"].clone(), d["recurrent"].clone()
        d["history"].copy_(held[0]), d["recurrent"].copy_(held[1])
        torch.randn(1 << 20, device=device).sum().item()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2].accepted, got.accepted) and torch.equal(outs[i % 2].token, got.token), i
        assert torch.equal(out[0][0], out[0][1]) and torch.equal(out[1][0], out[1][1]), i
        assert torch.equal(d["history"], after[0]) and torch.equal(d["recurrent"], after[1]), i


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_run_of_prompts_and_speculative_steps(pkg, device, dtype):
    """Three sequences of one pool: prompts, then blocks of drafted tokens, of which each step commits what the check accepts.  The rows that were
    committed give, in 64 bits, the states and outputs that the run left."""
    vocab, hk, hv, dim = 97, 2, 4, 128
    layer = Layer(pkg, device, [1, 1, 1], key_heads=hk, value_heads=hv, dim=dim, dtype=dtype, seed=10, fresh=(0, 1, 2))
    gen = torch.Generator().manual_seed(11)
    table = (torch.randn((vocab, layer.channels), generator=gen)).to(dtype).to(device)
    gates = torch.randn((2, vocab, hv), generator=gen).to(dtype).to(device)
    lift = (torch.randn((hv * dim, vocab), generator=gen)).to(device)
    guess = torch.randn((vocab, vocab), generator=gen) * 1.5
    d, kept = layer.d, [[] for _ in range(3)]

    def forward(blocks, fresh, counts):
        ids = torch.tensor(sum(blocks, []), dtype=torch.int64, device=device)
        d["starts"] = torch.tensor([sum(len(o) for o in blocks[:b]) for b in range(4)], dtype=torch.int32, device=device)
        d["fresh"], d["counts"] = torch.tensor(fresh, device=device), counts
        d["x"], (d["decay"], d["beta"]) = table[ids], gates[:, ids]
        mixed = layer.conv()
        d["query"], d["key"], d["value"] = (t.unflatten(-1, (-1, dim)) for t in mixed.split((hk * dim, hk * dim, hv * dim), -1))
        out = layer.rule(longest=max(map(len, blocks)))
        return d["x"], mixed, d["decay"], d["beta"], out

    def commit(rows, blocks, counts):
        at = 0
        for b, n in enumerate(counts):
            kept[b].append([t[at:at + n].cpu() for t in rows])
            at += len(blocks[b])

    prompts = [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in (70, 5, 1)]
    first = [p[:-1] for p in prompts]
    commit(forward(first, [True] * 3, None), first, [len(p) for p in first])
    last, empty = [p[-1] for p in prompts], [False, False, True]   # the third slot still holds nothing
    for step in range(8):
        blocks, draft = [], []
        for b, n in enumerate((3, 0, 6)):
            line = [last[b]]
            for _ in range(n):
                line.append(int(torch.multinomial(torch.softmax(guess[line[-1]].double(), 0), 1, generator=gen)))
            blocks.append(line)
            draft.append(guess[line])
        rows = forward(blocks, empty, torch.zeros(3, dtype=torch.int32, device=device))
        drafted = torch.tensor(sum((line[1:] + [0] for line in blocks), []), dtype=torch.int32)
        given = dict(target=(rows[4].flatten(1).float() @ lift * 2.0 + torch.cat(draft).to(device)).contiguous(), drafted=drafted.to(device),
                     starts=d["starts"], uniforms=torch.rand((len(drafted),), generator=gen).to(device), draft=torch.cat(draft).to(device))
        got = pkg.ops.verify_drafts(**given)
        accepted, token, margin = verified(**{k: v.cpu() for k, v in given.items()})
        assert margin > 1e-12 and torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.token.cpu(), token), step
        d["counts"] = got.accepted + 1
        layer.advance()
        commit(rows, blocks, (accepted + 1).tolist())
        last, empty = token.tolist(), [False] * 3
    assert sum(len(k[0]) for one in kept for k in one[1:]) > 3 * 8   # some drafts were accepted
    layer.spans = [sum(len(k[0]) for k in one) for one in kept]
    layer.tokens = layer.total = sum(layer.spans)
    layer.starts = torch.tensor([sum(layer.spans[:b]) for b in range(4)], dtype=torch.int32)
    layer.x, mixed, layer.decay, layer.beta, out = (torch.cat([k[i] for one in kept for k in one]) for i in range(5))
    layer.query, layer.key, layer.value = (t.unflatten(-1, (-1, dim)) for t in mixed.split((hk * dim, hk * dim, hv * dim), -1))
    layer.counts = None
    layer.check_conv(mixed)
    layer.check_rule(out)
