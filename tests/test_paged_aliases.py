"""CPU: an append whose key pages are its value pages is refused: a token's K and V rows would be written to one place, in no order."""
import ctypes

import pytest

from test_paged_refusals import ADDRESS, _append, _cache, _rows


def test_keys_and_values_in_one_place_are_not_appended_to(pkg):
    lib = pkg._lib
    for kw in ({}, dict(query=_rows(lib), heads=4, out=ADDRESS)):
        with pytest.raises(lib.DflashError, match="same memory") as e:
            _append(lib, **kw)
        assert e.value.status == 1
    _append(lib, tokens=0)          # nothing is written


def test_the_same_pages_are_read_as_keys_and_values(pkg):
    """Attention over them is no conflict: it is refused for what it lacks, not for that."""
    lib = pkg._lib
    with pytest.raises(lib.DflashError, match="starts"):
        lib.call("dflash_paged_attention", ctypes.byref(_cache(lib)), None, _rows(lib), None, 3, 4, 0.1, 1, ADDRESS, ADDRESS, 1 << 40, None)
