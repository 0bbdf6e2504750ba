"""The layer with adapters beside its router, and the pieces of a training step of the router run one behind another: logits with
adapters, routes, balance loss, its gradient, the adapters' gradients, each on the device output of the one before."""
import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
import oracle  # noqa: E402
from cases import float_layer, small_layer  # noqa: E402
from picoforge_b200 import abi, synth, tuning  # noqa: E402
from picoforge_b200.layer import MoeLayer, route  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture
def api(gpu):
    assert gpu.lib.qw4cu_set_stream(1) == 0             # the legacy default stream, which torch uses
    yield gpu
    torch.cuda.synchronize()
    assert gpu.lib.qw4cu_set_stream(None) == 0


class Setup:
    def __init__(self, api, spec, tokens, slots=3, rank=4, seed=0, strength=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed + tokens)
        self.spec, self.t, self.slots, self.rank = spec, tokens, slots, rank
        self.layer = MoeLayer(api, spec, max(tokens, 1))
        self.tune = tuning.TuneWork(api, tokens=max(tokens, 1), slots=slots, rank=rank, experts=spec.experts)
        self.x = torch.from_numpy(synth.activations(seed + 3, tokens, spec.hidden)).cuda()
        h, e = spec.hidden, spec.experts
        self.a = torch.randn(slots, rank, h, generator=gen, device="cuda") * h ** -0.5
        self.b = torch.randn(slots, e, rank, generator=gen, device="cuda") * strength
        self.scale = 0.5 + torch.rand(slots, generator=gen, device="cuda")
        slot = torch.randint(-1, slots, (tokens,), generator=gen, device="cuda")
        self.slot = slot.to(torch.int32)
        self.view = tuning.TuneWork.adapters(self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(), abi.F32, slots, rank, h, e)
        self.logits = torch.full((tokens, e), -99.0, device="cuda")
        self.ids = torch.full((tokens, spec.top_k), -1, device="cuda", dtype=torch.int32)
        self.weights = torch.full((tokens, spec.top_k), -99.0, device="cuda")
        self.y = torch.full((tokens, h), -99.0, device="cuda")

    def route(self, view="own"):
        self.tune.route(self.layer, self.view if isinstance(view, str) else view, self.x.data_ptr(), self.slot.data_ptr(), self.t,
                        self.logits.data_ptr(), self.ids.data_ptr(), self.weights.data_ptr())

    def forward(self, view="own"):
        self.tune.layer_forward(self.layer, self.view if isinstance(view, str) else view, self.x.data_ptr(), self.slot.data_ptr(), self.y.data_ptr(),
                                self.t, self.logits.data_ptr(), self.ids.data_ptr(), self.weights.data_ptr())

    def sync(self, api):
        err = abi.Qwen4Error()
        status = api.lib.qw4cu_moe_work_sync(self.layer.work, C.byref(err))
        assert status == abi.OK, err.detail
        self.tune.sync()

    def delta(self):
        """What the adapters add to the logits, in 64 bits, and the sum of the sizes of its terms."""
        out, size = (torch.zeros(self.t, self.spec.experts, dtype=torch.float64, device="cuda") for _ in range(2))
        for s in range(self.slots):
            at = torch.nonzero(self.slot == s).flatten()
            x, a, b = self.x[at].double(), self.a[s].double(), self.b[s].double()
            out[at] = self.scale[s].double() * ((x @ a.T) @ b.T)
            size[at] = self.scale[s].double() * ((x.abs() @ a.abs().T) @ b.abs().T)
        return out, size

    def close(self):
        self.layer.close()
        self.tune.close()


def layers():
    return {"Q4_K": small_layer(11), "IQ2_XXS": small_layer(12, routed=abi.IQ2_XXS, experts=32), "float": float_layer(13)}


@pytest.mark.parametrize("kind", ["Q4_K", "IQ2_XXS", "float"])
@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
def test_logits_routes_and_layer_with_adapters(api, kind, tokens):
    spec = layers()[kind]
    s = Setup(api, spec, tokens)
    s.route(None)
    s.sync(api)
    plain, plain_ids = s.logits.clone(), s.ids.clone()
    want = oracle.forward(spec, s.x.cpu().numpy())
    assert np.array_equal(plain_ids.cpu().numpy().view(np.uint32), want["ids"])
    s.route()
    s.sync(api)
    delta, size = s.delta()
    error = (s.logits.double() - plain.double() - delta).abs()
    assert (error <= 2 * U * (spec.hidden + s.rank + 16) * size + U * s.logits.double().abs() + 1e-300).all()
    # the routes are those of the logits that were handed out, bit for bit
    _, ids, weights = route(api, s.logits.cpu().numpy(), spec.top_k, spec.norm)
    assert np.array_equal(s.ids.cpu().numpy().view(np.uint32), ids) and np.array_equal(s.weights.cpu().numpy(), weights)
    kept = s.logits.clone(), s.ids.clone(), s.weights.clone()
    s.forward()
    s.sync(api)
    for p, q in zip(kept, (s.logits, s.ids, s.weights)):
        assert torch.equal(p, q)
    # every slot's tokens against an ordinary layer whose router has the adapter added to it
    for slot in range(-1, s.slots):
        at = torch.nonzero(s.slot == slot).flatten().cpu().numpy()
        if not len(at):
            continue
        merged = layers()[kind]
        w = merged.tensors[0].view(np.float32).reshape(spec.experts, spec.hidden)
        if slot >= 0:
            w += (s.scale[slot].double() * (s.b[slot].double() @ s.a[slot].double())).float().cpu().numpy()
        want = oracle.forward(merged, s.x.cpu().numpy()[at])
        same = (s.ids.cpu().numpy().view(np.uint32)[at] == want["ids"]).all(1)         # two probabilities within rounding of each other may swap
        assert same.mean() > 0.95 or len(at) < 20 and same.sum() >= len(at) - 1
        assert np.abs(s.y.cpu().numpy()[at] - want["y"])[same].max(initial=0) <= 1e-3
    # and the plain call is the plain one again
    y = torch.empty_like(s.y)
    err = abi.Qwen4Error()
    assert api.lib.qw4cu_moe_forward_device(s.layer.moe, s.x.data_ptr(), y.data_ptr(), tokens, s.ids.data_ptr(), None, s.layer.work, C.byref(err)) == abi.OK
    s.sync(api)
    assert torch.equal(s.ids, plain_ids)
    s.close()


def test_adapters_that_add_nothing(api):
    for tokens in (2, 100):
        s = Setup(api, small_layer(14), tokens)
        s.forward(None)
        s.sync(api)
        plain = [v.clone() for v in (s.logits, s.ids, s.weights, s.y)]
        s.b.zero_()
        s.forward()
        s.sync(api)
        for p, q in zip(plain, (s.logits, s.ids, s.weights, s.y)):
            assert torch.equal(p, q)
        s.close()


def test_replayed_launches_do_not_meet_adapters(api):
    """With graph mode on, a plain step that is replayed stays plain between steps with adapters, which are not."""
    s = Setup(api, small_layer(15), 80)
    api.lib.qw4cu_set_graph_mode(1)
    stream = torch.cuda.Stream()
    assert api.lib.qw4cu_set_stream(stream.cuda_stream) == 0
    try:
        err, y = abi.Qwen4Error(), torch.empty_like(s.y)
        torch.cuda.synchronize()
        kept = None
        for step in range(4):
            assert api.lib.qw4cu_moe_forward_device(s.layer.moe, s.x.data_ptr(), y.data_ptr(), s.t, s.ids.data_ptr(), None, s.layer.work, C.byref(err)) == abi.OK
            s.sync(api)
            plain = y.clone(), s.ids.clone()
            torch.cuda.synchronize()
            s.forward()
            s.sync(api)
            adapted = s.y.clone(), s.ids.clone()
            torch.cuda.synchronize()
            if kept:
                for p, q in zip(kept, plain + adapted):
                    assert torch.equal(p, q)
            kept = plain + adapted
        assert not torch.equal(kept[1], kept[3])
    finally:
        api.lib.qw4cu_set_graph_mode(0)
        assert api.lib.qw4cu_set_stream(1) == 0
        s.close()


def test_refusals(api):
    s = Setup(api, small_layer(16), 8)

    def status(**change):
        v = {"k": s.spec.hidden, "n": s.spec.experts, "t": 8, "slots": s.slot.data_ptr(), "tune": s.tune.handle} | change
        view = tuning.TuneWork.adapters(s.a.data_ptr(), s.b.data_ptr(), None, abi.F32, s.slots, s.rank, v["k"], v["n"])
        err = abi.Qwen4Error()
        return {api.lib.qw4cu_moe_forward_adapted_device(s.layer.moe, s.x.data_ptr(), s.y.data_ptr(), v["t"], C.byref(view), v["slots"], v["tune"], None,
                                                         None, None, s.layer.work, C.byref(err)),
                api.lib.qw4cu_moe_route_adapted_device(s.layer.moe, s.x.data_ptr(), v["t"], C.byref(view), v["slots"], v["tune"], None, None, None,
                                                       s.layer.work, C.byref(err))}
    assert status() == {abi.OK}
    assert status(k=s.spec.hidden // 2) == {abi.SHAPE} and status(n=s.spec.experts + 1) == {abi.SHAPE}
    assert status(t=9) == {abi.CAPACITY} and status(slots=None) == {abi.INVALID_ARGUMENT} and status(tune=None) == {abi.INVALID_ARGUMENT}
    assert status(t=0, slots=None) == {abi.OK}
    s.sync(api)
    s.slot[3] = s.slots
    assert status() == {abi.OK}
    with pytest.raises(abi.MoeError) as info:
        s.tune.sync()
    assert info.value.status == abi.RANGE and status() == {abi.BAD_STATE}
    s.close()


@pytest.mark.parametrize("tokens,norm", [(5, True), (90, True), (90, False), (700, True)])
def test_a_training_step_of_the_router(api, tokens, norm):
    """x -> logits with adapters -> routes -> balance loss -> gradient of the logits (with that of the route weights) -> gradients of the
    adapters and of x, all enqueued without a wait, against autograd in 64 bits on the logits and routes that came out."""
    spec = small_layer(17, experts=24, top_k=3)
    spec.norm = norm
    s = Setup(api, spec, tokens)
    mask = (torch.arange(tokens, device="cuda") % 5 != 4).to(torch.uint8)
    dw = torch.randn(tokens, spec.top_k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) / tokens
    config = tuning.TuneWork.router(spec.experts, spec.top_k, norm)
    counts = torch.empty(spec.experts + 1, dtype=torch.int32, device="cuda")
    sums, loss = torch.empty(spec.experts, device="cuda"), torch.empty(1, device="cuda")
    grad, dx = torch.empty_like(s.logits), torch.empty_like(s.x)
    da, db = torch.empty_like(s.a), torch.empty_like(s.b)
    s.route()
    s.tune.balance_forward(config, s.logits.data_ptr(), s.ids.data_ptr(), mask.data_ptr(), tokens, counts.data_ptr(), sums.data_ptr(), loss.data_ptr())
    s.tune.balance_backward(config, s.logits.data_ptr(), s.ids.data_ptr(), mask.data_ptr(), tokens, counts.data_ptr(), 0.3, dw.data_ptr(), grad.data_ptr())
    s.tune.adapter_backward(s.view, s.x.data_ptr(), s.slot.data_ptr(), grad.data_ptr(), None, dx.data_ptr(), da.data_ptr(), db.data_ptr(), tokens)
    s.sync(api)
    # the same in 64 bits, differentiated by torch
    a, b, x = (v.double().requires_grad_() for v in (s.a, s.b, s.x))
    delta = torch.zeros(tokens, spec.experts, dtype=torch.float64, device="cuda")
    for slot in range(s.slots):
        at = torch.nonzero(s.slot == slot).flatten()
        delta = delta.index_add(0, at, s.scale[slot].double() * ((x[at] @ a[slot].T) @ b[slot].T))
    z = (s.logits.double() - delta).detach() + delta
    p = z.softmax(1)
    keep = mask.bool()
    n, c = int(keep.sum()), torch.bincount(s.ids[keep].long().flatten(), minlength=spec.experts).double()
    value = spec.experts / n ** 2 * (c * p[keep].sum(0)).sum()
    w = p.gather(1, s.ids.long())
    if norm:
        w = w / w.sum(1, keepdim=True)
    (0.3 * value + (w * dw.double())[keep].sum()).backward()
    assert counts[:spec.experts].tolist() == c.long().tolist() and int(counts[-1]) == n
    assert abs(loss.item() - value.item()) <= 64 * U * value.item()
    # sums over a token's 24 logits and over the tokens, of terms that carry about 64 roundings each
    for got, want in ((dx, x.grad), (da, a.grad), (db, b.grad)):
        assert (got.double() - want).norm() <= 64 * U * (1 + tokens ** 0.5) * want.norm()
    s.close()
