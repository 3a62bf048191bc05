"""CPU: outputs of the batch's convolution and delta rule that lie in what the call reads are refused.  None of the calls launches anything:
each output shares at least a byte with the input that its case names."""
import ctypes

import pytest

from test_batch_refusals import ADDRESS, _conv, _delta, _pool, _rule, refused

OUT = 16 * ADDRESS           # three tokens of four heads of 64, or of 512 channels
RULE, CONV = 2 * 3 * 256, 2 * 3 * 512


def around(size, length, step):
    """Addresses of ``size`` bytes that share the first or the last ``step`` of the output's ``length`` bytes."""
    return OUT - size + step, OUT + length - step


@pytest.mark.parametrize("name", ["decay", "beta"])
@pytest.mark.parametrize("kind,size", [("DTYPE_F32", 4), ("DTYPE_BF16", 2)])
@pytest.mark.parametrize("stride", [4, 20])
def test_gates_in_the_output(pkg, name, kind, size, stride):
    lib = pkg._lib
    for at in around(size * (2 * stride + 4), RULE, size):
        refused(lib, _delta, "gates", 1, rule=_rule(lib, gates_dtype=getattr(lib, kind), **{name: at, f"{name}_stride": stride}), out=OUT)
    refused(lib, _delta, "gates", 1, rule=_rule(lib, gates_dtype=getattr(lib, kind), **{name: OUT + 512, f"{name}_stride": 4}), out=OUT)


@pytest.mark.parametrize("name", ["a_log", "dt_bias"])
def test_gate_vectors_in_the_output(pkg, name):
    lib = pkg._lib
    other = {"a_log": "dt_bias", "dt_bias": "a_log"}[name]
    for at in around(16, RULE, 4):
        refused(lib, _delta, "gates", 1, rule=_rule(lib, **{name: at, other: ADDRESS}), out=OUT)


@pytest.mark.parametrize("slot", [0, 1, 4])
def test_slots_in_the_output(pkg, slot):
    """Five slots, 65536 floats or 1536 16-bit values apart, with room between them."""
    lib = pkg._lib
    for at in around(4 * 4 * 64 * 64, RULE, 16):
        refused(lib, _delta, "states", 1, pool=_pool(lib, recurrent=at - slot * 4 * 65536), out=OUT)
    for at in around(6 * 512, CONV, 16):
        refused(lib, _conv, "histories", 1, pool=_pool(lib, history=at - slot * 2 * 4096, history_stride=4096), out=OUT)


def test_the_rest_in_the_output(pkg):
    lib = pkg._lib
    for at in around(8 * 512, CONV, 16):
        refused(lib, _conv, "weight", 1, weight=at, out=OUT)
    for call, length in ((_conv, CONV), (_delta, RULE)):
        for at in around(8, length, 4):
            refused(lib, call, "slots, starts", 1, pool=_pool(lib, slots=at), out=OUT)
        for at in around(12, length, 4):
            refused(lib, call, "slots, starts", 1, starts=at, out=OUT)
    entry = lambda counts, fresh, out=OUT: lib.call(  # noqa: E731
        "dflash_gdn_rule", ctypes.byref(_pool(lib)), ctypes.byref(_rule(lib)), ADDRESS, counts, fresh, 3, 0, out, ADDRESS, 1 << 40, None)
    for counts, fresh in ((OUT, None), (OUT - 4, None), (None, OUT + RULE - 1), (None, OUT - 1)):
        with pytest.raises(lib.DflashError, match="counts and fresh"):
            entry(counts, fresh)


def test_strides_beyond_any_memory(pkg):
    lib = pkg._lib
    refused(lib, _delta, "states", 1, pool=_pool(lib, recurrent=OUT, recurrent_stride=1 << 62), out=OUT)
    refused(lib, _delta, "gates", 1, rule=_rule(lib, beta=ADDRESS, beta_stride=(1 << 62) + 1), out=OUT)
