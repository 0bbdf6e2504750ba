"""Where the layer calls with adapters may hand the logits out to: nowhere that the layer still reads, or writes something else
(csrc/tune_host.c on a stand-in for the CUDA shim, no GPU)."""
import ctypes as C

import pytest

from picoforge_b200 import abi
from test_tuning_checks import AT, adapters, lib  # noqa: F401

TOKENS, HIDDEN, EXPERTS, TOP_K = 64, 32, 24, 4


def status(lib, ad="own", **change):  # noqa: F811
    v = dict(AT, weights=AT["weights_grad"]) | change
    ad = adapters() if isinstance(ad, str) else ad
    fn = lib.qw4tune_logits_out
    fn.argtypes = [C.c_void_p] + [C.c_size_t] * 4 + [C.c_void_p] * 7
    err = abi.Qwen4Error()
    st = fn(v["logits"], TOKENS, HIDDEN, EXPERTS, TOP_K, v["x"], v["y"], v["ids"], v["weights"], C.byref(ad) if ad else None, v["slots"], C.byref(err))
    assert err.code == st
    return st


def test_taken(lib):  # noqa: F811
    for change in ({}, {"logits": None}, {"y": None, "ids": None, "weights": None}, {"logits": AT["x"] + TOKENS * HIDDEN * 4},
                   {"logits": AT["x"] - TOKENS * EXPERTS * 4}, {"logits": AT["ids"] + TOKENS * TOP_K * 4}):
        assert status(lib, **change) == abi.OK, change
    assert status(lib, None, logits=AT["slots"]) == abi.OK                                 # slots are not looked at without adapters
    assert status(lib, adapters(scale=None)) == abi.OK


@pytest.mark.parametrize("logits", [AT["logits"] + 2, AT["x"], AT["x"] + TOKENS * HIDDEN * 4 - 4, AT["y"] + 128, AT["ids"] - TOKENS * EXPERTS * 4 + 4, AT["weights_grad"],
                                    AT["slots"] + 4 * TOKENS - 4, AT["a"], AT["b"], AT["scale"]])
def test_refused(lib, logits):  # noqa: F811
    assert status(lib, logits=logits) == abi.INVALID_ARGUMENT
