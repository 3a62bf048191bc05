"""CPU: calls that the paged-cache entries refuse.  None of them launches anything."""
import ctypes

import pytest
import torch

ADDRESS = 1 << 20    # an address that is never followed


def _cache(lib, **kw):
    base = dict(keys=ADDRESS, values=ADDRESS, table=ADDRESS, lengths=ADDRESS, sequences=2, table_width=4, table_stride=4, pages=9,
                page_size=16, kv_heads=2, head_dim=128, key_page_stride=4096, key_head_stride=2048, key_row_stride=128,
                value_page_stride=4096, value_head_stride=2048, value_row_stride=128, dtype=lib.DTYPE_BF16)
    base.update(kw)
    return lib.PagedDesc(**base)


def _rows(lib, data=ADDRESS, token_stride=512, head_stride=128):
    return ctypes.byref(lib.RowsDesc(data, token_stride, head_stride))


BAD_CACHES = [
    (dict(head_dim=64), 2, "head_dim"), (dict(dtype=1), 2, "dtype"), (dict(page_size=24), 2, "multiple of 16"),
    (dict(page_size=0), 1, "out of range"), (dict(pages=0), 1, "out of range"), (dict(table_width=0), 1, "out of range"),
    (dict(table_width=1 << 27), 2, "2\\^30"), (dict(table_width=1 << 62, page_size=1 << 30), 2, "2\\^30"),
    (dict(kv_heads=0), 1, "out of range"), (dict(kv_heads=1025), 1, "out of range"), (dict(sequences=-1), 1, "out of range"),
    (dict(sequences=(1 << 20) + 1), 1, "out of range"), (dict(pages=1 << 31), 1, "out of range"),
    (dict(table_stride=-4), 1, "out of range"), (dict(key_row_stride=129), 1, "multiples of 8"),
    (dict(value_page_stride=-8), 1, "multiples of 8"), (dict(key_row_stride=(1 << 26) + 8), 2, "2\\^26"),
    (dict(value_row_stride=1 << 40), 2, "2\\^26"), (dict(keys=0), 1, "NULL"), (dict(lengths=0), 1, "NULL"),
    (dict(values=ADDRESS + 8), 1, "aligned")]


@pytest.mark.parametrize("change,status,message", BAD_CACHES)
def test_bad_caches(pkg, change, status, message):
    lib, d = pkg._lib, _cache(pkg._lib, **change)
    calls = (lambda: lib.call("dflash_paged_append", ctypes.byref(d), _rows(lib), _rows(lib), ADDRESS, 3, None, 0, None, None,
                              None, 0, None, 1e-6, None, None),
             lambda: lib.call("dflash_paged_attention", ctypes.byref(d), None, _rows(lib), ADDRESS, 3, 4, 0.1, 1, ADDRESS, ADDRESS,
                              1 << 40, None),
             lambda: lib.call("dflash_paged_attention", ctypes.byref(_cache(lib)), ctypes.byref(d), _rows(lib), ADDRESS, 3, 4,
                              0.1, 1, ADDRESS, ADDRESS, 1 << 40, None))
    for call in calls:
        with pytest.raises(lib.DflashError, match=message) as e:
            call()
        assert e.value.status == status


def _append(lib, cache=None, key=None, value=None, starts=ADDRESS, tokens=3, query=None, heads=0, inv_freq=None, rotary=0,
            eps=1e-6, out=None):
    lib.call("dflash_paged_append", ctypes.byref(cache or _cache(lib)), key or _rows(lib), value or _rows(lib), starts, tokens,
             query, heads, None, None, inv_freq, rotary, None, eps, out, None)


def test_append_refusals(pkg):
    lib = pkg._lib
    for kw, message in [
            (dict(key=_rows(lib, 0)), "key"), (dict(value=_rows(lib, ADDRESS + 2)), "value"),
            (dict(key=_rows(lib, token_stride=508)), "multiples of 8"), (dict(value=_rows(lib, head_stride=-128)), "multiples of 8"),
            (dict(starts=None), "starts"), (dict(tokens=-1), "2\\^24"), (dict(tokens=1 << 23), "2\\^24"),
            (dict(tokens=1 << 62), "2\\^24"), (dict(heads=4), "without"), (dict(query=_rows(lib)), "without"),
            (dict(query=_rows(lib), heads=1025, out=ADDRESS), "1024"), (dict(query=_rows(lib), heads=4), "query_out"),
            (dict(query=_rows(lib), heads=4, out=ADDRESS + 4), "query_out"), (dict(rotary=32), "rotary_dim"),
            (dict(inv_freq=ADDRESS), "rotary_dim"), (dict(inv_freq=ADDRESS, rotary=24), "rotary_dim"),
            (dict(inv_freq=ADDRESS, rotary=144), "rotary_dim"), (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"),
            (dict(eps=float("inf")), "eps")]:
        with pytest.raises(lib.DflashError, match=message):
            _append(lib, **kw)
    _append(lib, tokens=0)                                       # nothing to do
    _append(lib, cache=_cache(lib, sequences=0))


def _attend(lib, cache=None, prefix=None, query=None, starts=ADDRESS, tokens=3, heads=4, scale=0.1, out=ADDRESS, ws=ADDRESS,
            size=1 << 40):
    lib.call("dflash_paged_attention", ctypes.byref(cache or _cache(lib)), None if prefix is None else ctypes.byref(prefix),
             query or _rows(lib), starts, tokens, heads, scale, 1, out, ws, size, None)


def test_attention_refusals(pkg):
    lib = pkg._lib
    need = lib.load().dflash_paged_attention_workspace_bytes(3, 4, 2, 128, 2, 0)
    assert need > 0
    for kw, message in [
            (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(heads=2048), "at most 1024"),
            (dict(tokens=-1), "at most"), (dict(tokens=1 << 21), "2\\^22"), (dict(tokens=1 << 62), "2\\^22"),
            (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
            (dict(scale=float("inf")), "scale"), (dict(scale=2.5e38), "scale"), (dict(query=_rows(lib, 0)), "query"), (dict(starts=None), "starts"),
            (dict(out=None), "out"), (dict(out=ADDRESS + 8), "out"), (dict(ws=None), "workspace"),
            (dict(ws=ADDRESS + 8), "workspace"), (dict(size=need - 1), "workspace"),
            (dict(prefix=_cache(lib)), "one sequence"), (dict(prefix=_cache(lib, sequences=1, kv_heads=4)), "kv_heads"),
            (dict(prefix=_cache(lib, sequences=1, head_dim=256)), "head_dim"),
            (dict(prefix=_cache(lib, sequences=1, dtype=lib.DTYPE_F16)), "dtype")]:
        with pytest.raises(lib.DflashError, match=message):
            _attend(lib, **kw)
    _attend(lib, tokens=0)
    _attend(lib, cache=_cache(lib, sequences=0))


def test_workspace_queries(pkg):
    lib = pkg._lib.load()
    q = lib.dflash_paged_attention_workspace_bytes
    assert q(3, 3, 2, 128, 1, 0) == 0 and q(-1, 4, 2, 128, 1, 0) == 0 and q(3, 4, 2, 96, 1, 0) == 0
    assert q(1 << 62, 4, 2, 128, 1, 0) == 0 and q(3, 4, 2, 128, 1 << 40, 0) == 0 and q(3, 4, 0, 128, 1, 0) == 0
    assert 0 < q(1, 4, 2, 128, 1, 0) < q(1, 4, 2, 128, 1, 1)
    assert pkg.ops.paged_attention_workspace_bytes(3, 4, 2, 128, 2, False) == q(3, 4, 2, 128, 2, 0)


def test_python_forms_refuse_host_tensors(pkg):
    ints = torch.zeros((1, 2), dtype=torch.int32)
    pool = torch.zeros((3, 2, 16, 128), dtype=torch.bfloat16)
    cache = pkg.ops.PagedKV(pool, pool.clone(), ints, ints[:, 0].contiguous())
    rows = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        pkg.ops.paged_append(cache, rows, rows, ints[0])
    with pytest.raises(ValueError, match="ROCm device"):
        pkg.ops.paged_attention(rows, cache, ints[0], scale=0.1)
    with pytest.raises(ValueError, match="PagedKV"):
        pkg.ops.paged_attention(rows, tuple(cache), ints[0], scale=0.1)
    with pytest.raises(ValueError, match="needs a prefix"):
        pkg.ops.shared_prefix_attention(rows, None, cache, ints[0], scale=0.1)
