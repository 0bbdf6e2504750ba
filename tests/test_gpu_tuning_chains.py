"""Kernels of adapters and balance loss right behind one another, each on what the one before wrote in place: the same bits as with a
wait between them."""
import pytest
import torch

from cases import small_layer
from picoforge_b200 import abi, tuning
from test_gpu_adapted_layer import Setup, api  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [5, 130, 1000])
@pytest.mark.parametrize("experts", [60, 200, 333])
def test_routes_behind_adapters_on_the_logits(api, experts, tokens):  # noqa: F811
    """Logits are adapted in place, in rows that share lines of the cache, and routed by a kernel that starts early; with the logits handed out a
    copy lies between the two."""
    s = Setup(api, small_layer(21, experts=experts), tokens)
    s.route()
    s.sync(api)
    want = s.ids.clone(), s.weights.clone()
    for _ in range(4):
        s.ids.fill_(-1)
        torch.cuda.synchronize()
        s.tune.route(s.layer, s.view, s.x.data_ptr(), s.slot.data_ptr(), tokens, None, s.ids.data_ptr(), s.weights.data_ptr())
        s.sync(api)
        assert torch.equal(s.ids, want[0]) and torch.equal(s.weights, want[1])
    s.close()


@pytest.mark.parametrize("tokens", [3, 300, 3000])
@pytest.mark.parametrize("experts", [60, 333, 1100])
def test_balance_loss_behind_adapters_in_place(api, experts, tokens):  # noqa: F811
    gen = torch.Generator(device="cuda").manual_seed(tokens + experts)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")
    hidden, rank, top = 96, 8, 4
    x, base, a, b = normal(tokens, hidden), normal(tokens, experts), normal(2, rank, hidden) / 10, normal(2, experts, rank)
    slot = torch.randint(-1, 2, (tokens,), generator=gen, device="cuda").to(torch.int32)
    ids = torch.argsort(normal(tokens, experts), 1)[:, :top].to(torch.int32).contiguous()
    config = tuning.TuneWork.router(experts, top, True)
    counts = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    sums, loss, grad = torch.empty(experts, device="cuda"), torch.empty(1, device="cuda"), torch.empty(tokens, experts, device="cuda")
    with tuning.TuneWork(api, tokens=tokens, slots=2, rank=rank, experts=experts) as work:
        view = work.adapters(a.data_ptr(), b.data_ptr(), None, 0, 2, rank, hidden, experts)

        def chain(wait):
            z = base.clone()
            for call in (lambda: work.adapter_forward(view, x.data_ptr(), slot.data_ptr(), z.data_ptr(), z.data_ptr(), tokens),
                         lambda: work.balance_forward(config, z.data_ptr(), ids.data_ptr(), None, tokens, counts.data_ptr(), sums.data_ptr(), loss.data_ptr()),
                         lambda: work.balance_backward(config, z.data_ptr(), ids.data_ptr(), None, tokens, counts.data_ptr(), 0.5, None, grad.data_ptr())):
                call()
                if wait:
                    work.sync()
            work.sync()
            return [v.clone() for v in (counts, sums, loss, grad)]
        want = chain(True)
        for _ in range(4):
            for p, q in zip(want, chain(False)):
                assert torch.equal(p, q)


def test_logits_handed_out_over_another_argument(api):  # noqa: F811
    """Refused before anything is launched, and the calls after it are as ever."""
    s = Setup(api, small_layer(22), 20)
    s.forward()
    s.sync(api)
    want = s.y.clone(), s.ids.clone(), s.logits.clone()
    api.lib.qw4cu_launch_log_begin()
    def forward(logits):
        s.tune.layer_forward(s.layer, s.view, s.x.data_ptr(), s.slot.data_ptr(), s.y.data_ptr(), s.t, logits.data_ptr(), s.ids.data_ptr(), s.weights.data_ptr())

    def route(logits):
        s.tune.route(s.layer, s.view, s.x.data_ptr(), s.slot.data_ptr(), s.t, logits.data_ptr(), s.ids.data_ptr(), s.weights.data_ptr())
    for call, others in ((forward, (s.x, s.y, s.ids, s.weights, s.slot, s.a, s.b)), (route, (s.x, s.ids, s.weights, s.slot, s.a, s.b))):
        for logits in others:
            with pytest.raises(abi.MoeError) as info:
                call(logits)
            assert info.value.status == abi.INVALID_ARGUMENT
    assert not api.launch_names()
    s.forward()
    s.sync(api)
    for p, q in zip(want, (s.y, s.ids, s.logits)):
        assert torch.equal(p, q)
    s.close()
