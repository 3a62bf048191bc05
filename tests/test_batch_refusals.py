"""CPU: calls that the entries of a batch's states and drafts refuse.  None of them launches anything."""
import ctypes

import pytest
import torch

ADDRESS = 1 << 20    # an address that is never followed


def _pool(lib, **kw):
    base = dict(history=ADDRESS, recurrent=ADDRESS, slots=ADDRESS, sequences=2, pool_slots=5, history_stride=1536, recurrent_stride=65536,
                channels=512, value_heads=4, head_dim=64, dtype=lib.DTYPE_BF16)
    base.update(kw)
    return lib.PoolDesc(**base)


def _rows(lib, data=ADDRESS, token_stride=512, head_stride=64):
    return lib.RowsDesc(data, token_stride, head_stride)


def _rule(lib, **kw):
    base = dict(query=_rows(lib), key=_rows(lib), value=_rows(lib), decay=ADDRESS, beta=ADDRESS, decay_stride=4, beta_stride=4, a_log=None,
                dt_bias=None, key_heads=2, scale=0.1, normalise=1, gates_dtype=lib.DTYPE_F32)
    base.update(kw)
    return lib.RuleDesc(**base)


def _conv(lib, pool=None, x=None, weight=ADDRESS, starts=ADDRESS, tokens=3, out=2 * ADDRESS):
    lib.call("dflash_gdn_conv", None if pool == 0 else ctypes.byref(pool or _pool(lib)), None if x == 0 else ctypes.byref(x or _rows(lib)),
             weight, starts, None, None, tokens, out, None)


def _delta(lib, pool=None, rule=None, starts=ADDRESS, tokens=3, longest=0, out=2 * ADDRESS, ws=ADDRESS, size=1 << 40):
    lib.call("dflash_gdn_rule", None if pool == 0 else ctypes.byref(pool or _pool(lib)),
             None if rule == 0 else ctypes.byref(rule or _rule(lib)), starts, None, None, tokens, longest, out, ws, size, None)


def _advance(lib, pool=None, x=None, rule=None, starts=ADDRESS, counts=ADDRESS, tokens=3):
    lib.call("dflash_gdn_advance", None if pool == 0 else ctypes.byref(pool or _pool(lib)), ctypes.byref(x or _rows(lib)),
             None if rule == 0 else ctypes.byref(rule or _rule(lib)), starts, counts, None, tokens, None)


def refused(lib, call, message, status=None, **kw):
    with pytest.raises(lib.DflashError, match=message) as e:
        call(lib, **kw)
    assert status is None or e.value.status == status


@pytest.mark.parametrize("change,status,message", [
    (dict(dtype=1), 2, "BF16 or F16"), (dict(dtype=7), 2, "BF16 or F16"), (dict(sequences=-1), 1, "out of range"),
    (dict(sequences=(1 << 20) + 1), 1, "out of range"), (dict(pool_slots=-1), 1, "out of range"), (dict(pool_slots=1 << 31), 1, "out of range"),
    (dict(slots=None), 1, "slots")])
def test_bad_pools(pkg, change, status, message):
    lib = pkg._lib
    for call in (_conv, _delta, _advance):
        refused(lib, call, message, status, pool=_pool(lib, **change))
        refused(lib, call, "NULL", 1, pool=0)


def test_bad_histories_and_states(pkg):
    lib = pkg._lib
    for change, message in [(dict(channels=0), "channels"), (dict(channels=12), "channels"), (dict(channels=(1 << 16) + 8), "channels"),
                            (dict(history=None), "history"), (dict(history=ADDRESS + 8), "history"), (dict(history_stride=12), "multiple of 8"),
                            (dict(history_stride=-8), "multiple of 8")]:
        refused(lib, _conv, message, pool=_pool(lib, **change))
        refused(lib, _advance, message, pool=_pool(lib, **change))
    for change, message in [(dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(value_heads=0), "value_heads"),
                            (dict(value_heads=1025), "value_heads"), (dict(sequences=1 << 19, value_heads=8), "2\\^19"),
                            (dict(recurrent=None), "recurrent"), (dict(recurrent=ADDRESS + 4), "recurrent"),
                            (dict(recurrent_stride=6), "multiple of 4"), (dict(recurrent_stride=-4), "multiple of 4")]:
        refused(lib, _delta, message, pool=_pool(lib, **change))
        refused(lib, _advance, message, pool=_pool(lib, **change))


def test_conv_refusals(pkg):
    lib = pkg._lib
    for kw, message in [(dict(x=0), "x"), (dict(x=_rows(lib, None)), "x"), (dict(x=_rows(lib, ADDRESS + 2)), "x"),
                        (dict(x=_rows(lib, token_stride=508)), "multiples of 8"), (dict(x=_rows(lib, token_stride=-512)), "multiples of 8"),
                        (dict(weight=None), "weight"), (dict(weight=ADDRESS + 8), "weight"), (dict(out=None), "out"),
                        (dict(out=ADDRESS + 8), "out"), (dict(out=ADDRESS), "out cannot be x"), (dict(starts=None), "starts"),
                        (dict(out=ADDRESS + 2 * 512 * 3 - 16), "overlap"), (dict(out=ADDRESS - 2 * 512 * 3 + 16), "overlap"),
                        (dict(tokens=-1), "2\\^20"), (dict(tokens=(1 << 20) + 1), "2\\^20"), (dict(tokens=1 << 62), "2\\^20")]:
        refused(lib, _conv, message, **kw)
    _conv(lib, tokens=0)                                         # nothing to do
    _conv(lib, pool=_pool(lib, sequences=0, slots=None))


def test_rule_refusals(pkg):
    lib = pkg._lib
    rules = [(dict(key_heads=3), "multiple of key_heads"), (dict(key_heads=0), "multiple of key_heads"), (dict(key=_rows(lib, None)), "key"),
             (dict(value=_rows(lib, ADDRESS + 8)), "value"), (dict(value=_rows(lib, head_stride=60)), "multiples of 8"),
             (dict(decay=None), "decay"), (dict(beta=None), "beta"), (dict(decay=ADDRESS + 2), "misaligned"), (dict(decay_stride=-4), "negative"),
             (dict(gates_dtype=3), "gates_dtype"), (dict(a_log=ADDRESS), "go together"), (dict(dt_bias=ADDRESS), "go together"),
             (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")]
    for change, message in rules:
        refused(lib, _delta, message, rule=_rule(lib, **change))
        refused(lib, _advance, message, rule=_rule(lib, **change))
    for kw, message in [(dict(rule=0), "NULL"), (dict(rule=_rule(lib, query=_rows(lib, None))), "query"), (dict(starts=None), "starts"),
                        (dict(tokens=-1), "2\\^20"), (dict(tokens=1 << 62), "2\\^20"), (dict(longest=-1), "longest"), (dict(out=None), "out"),
                        (dict(out=ADDRESS + 8), "out"), (dict(out=ADDRESS), "out cannot be"), (dict(tokens=500, ws=None), "workspace"),
                        (dict(rule=_rule(lib, value=_rows(lib, 2 * ADDRESS - 2 * (2 * 512 + 256) + 16))), "overlap"),
                        (dict(rule=_rule(lib, query=_rows(lib, 2 * ADDRESS + 2 * 3 * 256 - 16))), "overlap"),
                        (dict(tokens=500, ws=ADDRESS + 8), "workspace"), (dict(longest=33, tokens=33, size=100), "workspace"), (dict(tokens=1 << 20, pool=_pool(lib, value_heads=512)), "2\\^28")]:
        refused(lib, _delta, message, **kw)
    for kw, message in [(dict(rule=0), "NULL"), (dict(counts=None), "counts"), (dict(starts=None), "starts"),
                        (dict(x=_rows(lib, ADDRESS + 2)), "x"), (dict(tokens=1 << 21), "2\\^20")]:
        refused(lib, _advance, message, **kw)
    refused(lib, _advance, "too many", pool=_pool(lib, sequences=1 << 19, value_heads=1, channels=1 << 16, history_stride=3 << 16),
            rule=_rule(lib, key_heads=1), x=_rows(lib, token_stride=1 << 16))
    _delta(lib, tokens=0)
    _delta(lib, pool=_pool(lib, sequences=0))
    _advance(lib, tokens=0)
    _advance(lib, pool=_pool(lib, sequences=0))


def _verify(lib, drafted=ADDRESS, starts=ADDRESS, sequences=2, uniforms=ADDRESS, accepted=ADDRESS, token=ADDRESS, ws=ADDRESS, size=1 << 40, **kw):
    base = dict(target=ADDRESS, draft=ADDRESS, target_stride=100, draft_stride=100, rows=5, vocab=100, dtype=lib.DTYPE_BF16)
    base.update(kw)
    lib.call("dflash_verify_drafts", ctypes.byref(lib.LogitsDesc(**base)), drafted, starts, sequences, uniforms, None, accepted, token, ws, size,
             None)


def test_verify_refusals(pkg):
    lib = pkg._lib
    need = lib.load().dflash_verify_drafts_workspace_bytes(5, 100, 2, 1)
    assert need > 0
    for kw, message in [(dict(rows=-1), "2\\^20"), (dict(rows=1 << 62), "2\\^20"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"),
                        (dict(sequences=-1), "2\\^20"), (dict(sequences=(1 << 20) + 1), "2\\^20"), (dict(dtype=3), "dtype"),
                        (dict(target=None), "target"), (dict(target=ADDRESS + 1), "misaligned"), (dict(draft=ADDRESS + 1), "misaligned"),
                        (dict(target=ADDRESS + 2, dtype=lib.DTYPE_F32), "misaligned"), (dict(target_stride=-1), "strides"),
                        (dict(drafted=None), "drafted"), (dict(uniforms=None), "uniforms"), (dict(starts=None), "starts"),
                        (dict(accepted=None), "accepted"), (dict(token=None), "token"), (dict(ws=None), "workspace"),
                        (dict(ws=ADDRESS + 8), "workspace"), (dict(size=need - 1), "workspace")]:
        refused(lib, _verify, message, **kw)
    _verify(lib, sequences=0)
    with pytest.raises(lib.DflashError, match="NULL"):
        lib.call("dflash_verify_drafts", None, ADDRESS, ADDRESS, 2, ADDRESS, None, ADDRESS, ADDRESS, ADDRESS, 1 << 40, None)


def test_workspace_queries(pkg):
    ops, lib = pkg.ops, pkg._lib.load()
    q = lib.dflash_verify_drafts_workspace_bytes
    assert q(-1, 100, 2, 0) == 0 and q(5, 0, 2, 0) == 0 and q(5, 1 << 40, 2, 0) == 0 and q(5, 100, 1 << 40, 0) == 0
    assert 0 < q(5, 248320, 2, 0) < q(5, 248320, 2, 1)
    assert ops.verify_drafts_workspace_bytes(5, 100, 2, True) == q(5, 100, 2, 1)
    r = lib.dflash_gdn_rule_workspace_bytes
    for args in ((-1, 2, 4, 128, 2, 0), (5, 3, 4, 128, 2, 0), (5, 2, 4, 96, 2, 0), (1 << 62, 2, 4, 128, 2, 0), (5, 2, 4, 128, 1 << 40, 0),
                 (5, 0, 4, 128, 2, 0), (5, 2, 4, 128, 2, -1)):
        assert r(*args) == 0, args
    assert ops.gdn_rule_workspace_bytes(500, 2, 4, 128, 3) == r(500, 2, 4, 128, 3, 0)


def test_python_forms_refuse_host_tensors(pkg):
    ops = pkg.ops
    ints = torch.zeros((2,), dtype=torch.int32)
    pool = ops.StatePool(torch.zeros((3, 256, 3), dtype=torch.bfloat16), torch.zeros((3, 2, 64, 64)), ints[:1])
    x, rows, gates = torch.zeros((1, 256), dtype=torch.bfloat16), torch.zeros((1, 2, 64), dtype=torch.bfloat16), torch.zeros((1, 2))
    for call in (lambda: ops.gdn_conv(x, torch.zeros((256, 1, 4), dtype=torch.bfloat16), pool, ints),
                 lambda: ops.gdn_rule(rows, rows, rows, gates, gates, pool, ints),
                 lambda: ops.gdn_advance(pool, x, rows, rows, gates, gates, ints, ints[:1]),
                 lambda: ops.verify_drafts(gates, ints[:1], ints, gates[:, 0])):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="StatePool"):
        ops.gdn_rule(rows, rows, rows, gates, gates, tuple(pool), ints)
    with pytest.raises(ValueError, match="StatePool"):
        ops.gdn_conv(x, x, None, ints)
    with pytest.raises(ValueError, match="longest"):
        ops.gdn_rule(rows, rows, rows, gates, gates, pool, ints, longest=True)
    with pytest.raises(ValueError, match="query"):
        ops.gdn_rule(None, rows, rows, gates, gates, pool, ints)
    with pytest.raises(ValueError, match="counts"):
        ops.gdn_advance(pool, x, rows, rows, gates, gates, ints, None)
