"""What the adapter and balance entry points refuse, and with which status: csrc/tune_host.c on a stand-in for the CUDA shim
(tests/tune_shim_stub.c), so no GPU is needed and nothing wrong can reach one."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from picoforge_b200 import abi

ROOT = Path(__file__).resolve().parent.parent
P, Z = C.c_void_p, C.c_size_t


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("tune") / "libtune_host.so"
    subprocess.run(["gcc", "-std=c11", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared", "-D_DEFAULT_SOURCE",
                    str(ROOT / "picoforge_b200" / "csrc" / "tune_host.c"), str(ROOT / "tests" / "tune_shim_stub.c"), "-o", str(out)], check=True)
    lib = C.CDLL(str(out))
    lib.qw4cu_tune_work_device_bytes.restype = Z
    lib.qw4cu_tune_work_device_bytes.argtypes = [P]
    lib.qw4cu_tune_work_destroy.argtypes = [P]
    lib.qw4cu_tune_work_sync.argtypes = lib.qw4cu_tune_work_reset.argtypes = [P, P]
    lib.qw4cu_adapter_forward_device.argtypes = [P, P, Z, P, P, Z, P, Z, Z, P, P]
    lib.qw4cu_adapter_backward_device.argtypes = [P, P, Z, P, P, Z, P, Z, P, Z, P, P, Z, P, P]
    lib.qw4cu_balance_forward_device.argtypes = [P, P, Z, P, P, Z, P, P, P, P, P]
    lib.qw4cu_balance_backward_device.argtypes = [P, P, Z, P, P, Z, P, C.c_float, P, P, Z, P, P]
    return lib


def create(lib, tokens=64, slots=4, rank=8, experts=16):
    handle, err = P(), abi.Qwen4Error()
    limits = abi.QW4CuTuneLimits(tokens, slots, rank, experts)
    st = lib.qw4cu_tune_work_create(C.byref(limits), C.byref(handle), C.byref(err))
    assert err.code == st and (err.subject == b"tune" and err.detail if st else not err.detail)
    return st, handle


@pytest.fixture
def work(lib):
    st, handle = create(lib)
    assert st == abi.OK
    yield handle
    lib.qw4cu_tune_work_destroy(handle)


def launches(lib):
    return C.c_int.in_dll(lib, "stub_launches").value


def test_limits_of_a_workspace(lib):
    assert create(lib, tokens=0)[0] == abi.RANGE
    assert create(lib, tokens=(1 << 20) + 1)[0] == abi.RANGE
    assert create(lib, slots=0, experts=0)[0] == abi.RANGE
    assert create(lib, slots=1025)[0] == abi.RANGE
    assert create(lib, rank=0)[0] == abi.RANGE
    assert create(lib, rank=129)[0] == abi.RANGE
    assert create(lib, experts=4097)[0] == abi.RANGE
    assert lib.qw4cu_tune_work_create(None, C.byref(P()), None) == abi.INVALID_ARGUMENT
    for kwargs in ({"slots": 0, "rank": 0}, {"experts": 0}, {"tokens": 1, "slots": 1024, "rank": 128, "experts": 4096}):
        st, handle = create(lib, **kwargs)
        assert st == abi.OK and lib.qw4cu_tune_work_device_bytes(handle) > 0
        lib.qw4cu_tune_work_destroy(handle)
    fail = C.c_int.in_dll(lib, "stub_fail_malloc")
    fail.value = 1
    try:
        assert create(lib)[0] == abi.OOM
    finally:
        fail.value = 0
    assert lib.qw4cu_tune_work_device_bytes(None) == 0
    lib.qw4cu_tune_work_destroy(None)


# addresses that nothing reads: apart from one another, on 16-byte boundaries
AT = {name: (i + 1) << 32 for i, name in enumerate(("a", "b", "scale", "x", "slots", "base", "y", "dy", "dx", "da", "db", "logits", "ids", "mask",
                                                    "counts", "prob_sums", "loss", "weights_grad", "grad"))}


def adapters(**change):
    v = {"a": AT["a"], "b": AT["b"], "scale": AT["scale"], "type": abi.BF16, "slots": 4, "rank": 8, "k": 32, "n": 24} | change
    return abi.QW4CuAdapters(v["a"], v["b"], v["scale"], v["type"], v["slots"], v["rank"], v["k"], v["n"])


def forward(lib, work, ad=None, **change):
    v = dict(AT, x_pitch=128, base_pitch=96, y_pitch=96, tokens=64) | change
    ad = adapters() if ad is None else ad
    before, err = launches(lib), abi.Qwen4Error()
    st = lib.qw4cu_adapter_forward_device(C.byref(ad) if ad else None, v["x"], v["x_pitch"], v["slots"], v["base"], v["base_pitch"], v["y"],
                                          v["y_pitch"], v["tokens"], work, C.byref(err))
    assert err.code == st and launches(lib) - before == (1 if st == abi.OK and v["tokens"] else 0)
    return st


def backward(lib, work, ad=None, **change):
    v = dict(AT, x_pitch=128, dy_pitch=96, base_pitch=128, dx_pitch=128, tokens=64) | change
    ad = adapters() if ad is None else ad
    before, err = launches(lib), abi.Qwen4Error()
    st = lib.qw4cu_adapter_backward_device(C.byref(ad), v["x"], v["x_pitch"], v["slots"], v["dy"], v["dy_pitch"], v["base"], v["base_pitch"],
                                           v["dx"], v["dx_pitch"], v["da"], v["db"], v["tokens"], work, C.byref(err))
    assert err.code == st and launches(lib) - before == (1 if st == abi.OK else 0)
    return st


BAD_ADAPTERS = [({"a": None}, abi.INVALID_ARGUMENT), ({"b": None}, abi.INVALID_ARGUMENT), ({"a": AT["a"] + 1}, abi.INVALID_ARGUMENT),
                ({"type": abi.F32, "b": AT["b"] + 2}, abi.INVALID_ARGUMENT), ({"scale": AT["scale"] + 2}, abi.INVALID_ARGUMENT),
                ({"type": abi.Q4_K}, abi.TYPE), ({"slots": 5}, abi.CAPACITY), ({"rank": 9}, abi.CAPACITY), ({"rank": 0}, abi.SHAPE),
                ({"slots": 0}, abi.SHAPE), ({"k": 0}, abi.SHAPE), ({"n": (1 << 24) + 1}, abi.SHAPE)]


@pytest.mark.parametrize("change,status", BAD_ADAPTERS)
def test_adapters_refused(lib, work, change, status):
    assert forward(lib, work, adapters(**change)) == status
    assert backward(lib, work, adapters(**change)) == status


@pytest.mark.parametrize("change,status", [
    ({"x": None}, abi.INVALID_ARGUMENT), ({"slots": None}, abi.INVALID_ARGUMENT), ({"y": None}, abi.INVALID_ARGUMENT),
    ({"x": AT["x"] + 2}, abi.INVALID_ARGUMENT), ({"slots": AT["slots"] + 1}, abi.INVALID_ARGUMENT),
    ({"x_pitch": 124}, abi.STRIDE), ({"x_pitch": 130}, abi.STRIDE), ({"y_pitch": 92}, abi.STRIDE), ({"base_pitch": 92}, abi.STRIDE),
    ({"x_pitch": 1 << 60}, abi.OVERFLOW), ({"tokens": 65}, abi.CAPACITY),
    ({"y": AT["x"]}, abi.INVALID_ARGUMENT), ({"y": AT["x"] + 128 * 63 + 124}, abi.INVALID_ARGUMENT), ({"y": AT["a"]}, abi.INVALID_ARGUMENT),
    ({"y": AT["slots"]}, abi.INVALID_ARGUMENT), ({"y": AT["scale"] + 4}, abi.INVALID_ARGUMENT),
    ({"y": AT["base"] + 4}, abi.INVALID_ARGUMENT), ({"y": AT["base"], "y_pitch": 192}, abi.INVALID_ARGUMENT)])
def test_forward_refused(lib, work, change, status):
    assert forward(lib, work, **change) == status


def test_forward_taken(lib, work):
    for change in ({}, {"base": None, "base_pitch": 0}, {"base": AT["y"]}, {"x_pitch": 132}, {"x": AT["x"] + 4}, {"tokens": 1},
                   {"tokens": 0}, {"tokens": 0, "x": None, "y": None, "slots": None, "base": None}):
        assert forward(lib, work, **change) == abi.OK, change
    assert forward(lib, work, adapters(scale=None)) == abi.OK
    assert forward(lib, None) == abi.INVALID_ARGUMENT
    assert lib.qw4cu_adapter_forward_device(None, AT["x"], 128, AT["slots"], None, 0, AT["y"], 96, 1, work, None) == abi.INVALID_ARGUMENT


@pytest.mark.parametrize("change,status", [
    ({"dy": None}, abi.INVALID_ARGUMENT), ({"x": None}, abi.INVALID_ARGUMENT), ({"da": None}, abi.INVALID_ARGUMENT), ({"db": None}, abi.INVALID_ARGUMENT),
    ({"da": None, "db": None, "dx": None}, abi.INVALID_ARGUMENT), ({"dy_pitch": 92}, abi.STRIDE), ({"dx_pitch": 124}, abi.STRIDE),
    ({"dx": AT["x"]}, abi.INVALID_ARGUMENT), ({"da": AT["db"]}, abi.INVALID_ARGUMENT), ({"da": AT["a"]}, abi.INVALID_ARGUMENT),
    ({"dx": AT["da"] + 4 * 8 * 32 * 4 - 4}, abi.INVALID_ARGUMENT), ({"tokens": 65}, abi.CAPACITY)])
def test_backward_refused(lib, work, change, status):
    assert backward(lib, work, **change) == status


def test_backward_taken(lib, work):
    for change in ({}, {"base": None}, {"base": AT["dx"]}, {"dx": None, "base": None}, {"da": None, "db": None, "x": None},
                   {"tokens": 0, "x": None, "dy": None, "slots": None, "dx": None}):
        assert backward(lib, work, **change) == abi.OK, change


def config(**change):
    v = {"experts": 16, "top_k": 4, "norm_topk_prob": True} | change
    return abi.Qwen4MoeConfig(**v)


def balance(lib, work, cfg=None, back=False, **change):
    v = dict(AT, pitch=64, grad_pitch=64, tokens=64) | change
    cfg = config() if cfg is None else cfg
    before, err = launches(lib), abi.Qwen4Error()
    if back:
        st = lib.qw4cu_balance_backward_device(C.byref(cfg), v["logits"], v["pitch"], v["ids"], v["mask"], v["tokens"], v["counts"], 0.5,
                                               v["weights_grad"], v["grad"], v["grad_pitch"], work, C.byref(err))
    else:
        st = lib.qw4cu_balance_forward_device(C.byref(cfg), v["logits"], v["pitch"], v["ids"], v["mask"], v["tokens"], v["counts"], v["prob_sums"],
                                              v["loss"], work, C.byref(err))
    assert err.code == st and launches(lib) - before == (1 if st == abi.OK and (v["tokens"] or not back) else 0)
    return st


@pytest.mark.parametrize("back", [False, True])
def test_balance_refused_and_taken(lib, work, back):
    for change, status in ([({"logits": None}, abi.INVALID_ARGUMENT), ({"ids": None}, abi.INVALID_ARGUMENT), ({"counts": None}, abi.INVALID_ARGUMENT),
                            ({"logits": AT["logits"] + 2}, abi.INVALID_ARGUMENT), ({"pitch": 60}, abi.STRIDE), ({"pitch": 66}, abi.STRIDE),
                            ({"pitch": 1 << 62}, abi.OVERFLOW), ({"tokens": 65}, abi.CAPACITY)]
                           + ([({"grad": None}, abi.INVALID_ARGUMENT), ({"grad_pitch": 60}, abi.STRIDE), ({"grad": AT["logits"]}, abi.INVALID_ARGUMENT),
                               ({"grad": AT["counts"] + 8}, abi.INVALID_ARGUMENT), ({"grad": AT["weights_grad"]}, abi.INVALID_ARGUMENT)] if back else
                              [({"loss": None}, abi.INVALID_ARGUMENT), ({"prob_sums": AT["counts"] + 64}, abi.INVALID_ARGUMENT),
                               ({"loss": AT["mask"] + 60}, abi.INVALID_ARGUMENT), ({"counts": AT["ids"]}, abi.INVALID_ARGUMENT)])):
        assert balance(lib, work, back=back, **change) == status, change
    for cfg, status in ((config(experts=17), abi.CAPACITY), (config(top_k=17), abi.RANGE), (config(top_k=0), abi.RANGE), (config(experts=0, top_k=0), abi.RANGE)):
        assert balance(lib, work, cfg, back=back) == status
    for change in ({}, {"mask": None}, {"mask": AT["mask"] + 3}, {"pitch": 68}, {"tokens": 0, "logits": None, "ids": None, "mask": None},
                   {"weights_grad": None}):
        assert balance(lib, work, back=back, **change) == abi.OK, change
    assert balance(lib, None, back=back) == abi.INVALID_ARGUMENT


def test_parts_that_a_workspace_lacks(lib):
    _, handle = create(lib, slots=0, rank=0)
    assert forward(lib, handle) == abi.CAPACITY and balance(lib, handle) == abi.OK
    lib.qw4cu_tune_work_destroy(handle)
    _, handle = create(lib, experts=0)
    assert forward(lib, handle) == abi.OK and balance(lib, handle) == abi.CAPACITY
    lib.qw4cu_tune_work_destroy(handle)


def test_latch_device_and_launch_failure(lib, work):
    err = abi.Qwen4Error()
    status = (C.c_uint32 * 2).in_dll(lib, "stub_status")
    assert lib.qw4cu_tune_work_sync(work, C.byref(err)) == abi.OK
    status[0], status[1] = 1, 7
    assert lib.qw4cu_tune_work_sync(work, C.byref(err)) == abi.NONFINITE and err.row == 7
    assert forward(lib, work) == abi.BAD_STATE and backward(lib, work) == abi.BAD_STATE and balance(lib, work) == abi.BAD_STATE
    status[0], status[1] = 0, 0xFFFFFFFF
    assert lib.qw4cu_tune_work_reset(work, C.byref(err)) == abi.OK
    assert forward(lib, work) == abi.OK
    status[0] = 2
    assert lib.qw4cu_tune_work_sync(work, C.byref(err)) == abi.RANGE
    status[0] = 0
    assert lib.qw4cu_tune_work_reset(work, C.byref(err)) == abi.OK
    device = C.c_int.in_dll(lib, "stub_device")
    device.value = 1
    try:
        assert forward(lib, work) == abi.OWNER and balance(lib, work) == abi.OWNER
        assert lib.qw4cu_tune_work_sync(work, C.byref(err)) == abi.OWNER
    finally:
        device.value = 0
    fail = C.c_int.in_dll(lib, "stub_fail_launch")
    fail.value = 1
    try:
        ad = adapters()
        assert lib.qw4cu_adapter_forward_device(C.byref(ad), AT["x"], 128, AT["slots"], None, 0, AT["y"], 96, 1, work, C.byref(err)) == abi.GPU_ERROR
    finally:
        fail.value = 0
