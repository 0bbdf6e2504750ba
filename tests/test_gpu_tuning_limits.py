"""The largest batches, projections and lists that a workspace takes."""
import pytest
import torch

from picoforge_b200 import tuning
from test_gpu_adapters import Case, api, check, close, formula, forward  # noqa: F401
from test_gpu_balance import Case as Balance
from test_gpu_balance import check as check_balance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,k,n,r,s", [(1 << 20, 16, 8, 4, 1024), (130, 1 << 20, 8, 128, 1), (130, 8, 1 << 20, 20, 2), (2, 1 << 20, 24, 128, 2), (192, 24, (1 << 20) - 3, 9, 3),
                                       (1030, 64, 64, 8, 1024)])
def test_adapters(api, t, k, n, r, s):  # noqa: F811
    check(api, Case(t, k, n, r, s, torch.bfloat16))


def test_adapters_of_one_token_each(api):  # noqa: F811
    """As many slots as tokens, every adapter in use: a tile of one row to each."""
    c = Case(1024, 96, 80, 16, 1024, torch.bfloat16)
    c.slot.copy_(torch.randperm(1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)))
    check(api, c)
    c.slot[:192].copy_(c.slot[832:].clone())
    c.t = 192
    with c.work(api) as work:                                # the few-token kernel on the last adapters of the list
        y = forward(work, c, torch.empty(192, 80, device="cuda"))
        work.sync()
    c.x, c.slot, c.by, c.dy = c.x[:192], c.slot[:192], c.by[:192], c.dy[:192]
    want, sizes = formula(c), formula(c, True)
    close(y, want[0], sizes[0], c.k + c.r, c.by)


@pytest.mark.parametrize("t,e,k", [(1 << 20, 60, 4), (20000, 4096, 8), (3, 4096, 4096), (1, 1, 1), (70000, 1024, 32)])
def test_balance(api, t, e, k):  # noqa: F811
    check_balance(api, Balance(t, e, k, True, 0.1 if t > 3 else 0.0))


def test_the_largest_workspace(api):  # noqa: F811
    with tuning.TuneWork(api, tokens=1 << 20, slots=1024, rank=128, experts=4096) as work:
        c = Case(300, 64, 48, 24, 5, torch.float32)
        y = forward(work, c)
        work.sync()
        with c.work(api) as own:
            assert torch.equal(y, forward(own, c))
            own.sync()
