"""Adapters and balance loss on columns of wider buffers, operands and results side by side: the same bits as on buffers of their own, and
what lies beside them left as it was."""
import pytest
import torch

from picoforge_b200 import tuning
from test_gpu_adapters import Case, api, backward, forward, ptr  # noqa: F401

pytestmark = pytest.mark.gpu


def side_by_side(tokens, gap, *widths):
    """Views [tokens, width] of one buffer, `gap` columns between them, and a check that the rest of it is untouched."""
    whole = torch.full((tokens, sum(widths) + gap * (len(widths) + 1)), -77.0, device="cuda")
    views, at, rest = [], gap, torch.ones(whole.shape[1], dtype=torch.bool, device="cuda")
    for width in widths:
        views.append(whole[:, at:at + width])
        rest[at:at + width] = False
        at += width + gap
    return views, lambda: bool((whole[:, rest] == -77).all())


@pytest.mark.parametrize("gap", [0, 1, 4])
@pytest.mark.parametrize("t,k,n,r", [(1, 64, 48, 8), (5, 40, 24, 5), (90, 256, 192, 16), (300, 128, 130, 24), (700, 77, 333, 64)])
def test_adapters_on_columns_of_one_buffer(api, t, k, n, r, gap):  # noqa: F811
    c = Case(t, k, n, r, 3, torch.bfloat16)
    with c.work(api) as work:
        y, (dx, da, db) = forward(work, c), backward(work, c)
        (vx, vb, vy), kept = side_by_side(t, gap, k, n, n)
        vx.copy_(c.x)
        vb.copy_(c.by)
        work.adapter_forward(c.view(), ptr(vx), c.slot.data_ptr(), ptr(vb), ptr(vy), t, *(v.stride(0) * 4 for v in (vx, vb, vy)))
        (wd, wx, wb, wx2), kept2 = side_by_side(t, gap, n, k, k, k)
        wd.copy_(c.dy)
        wx.copy_(c.x)
        wb.copy_(c.bx)
        da2, db2 = torch.empty_like(da), torch.empty_like(db)
        work.adapter_backward(c.view(), ptr(wx), c.slot.data_ptr(), ptr(wd), ptr(wb), ptr(wx2), ptr(da2), ptr(db2), t,
                              *(v.stride(0) * 4 for v in (wx, wd, wb, wx2)))
        work.sync()
    for p, q in ((vy, y), (wx2, dx), (da2, da), (db2, db)):
        assert torch.equal(p, q)
    assert kept() and kept2() and torch.equal(vx, c.x) and torch.equal(wd, c.dy)


@pytest.mark.parametrize("t,e", [(3, 64), (200, 512), (70, 1100), (33, 60)])
def test_gradient_of_the_logits_beside_them(api, t, e):  # noqa: F811
    gen = torch.Generator(device="cuda").manual_seed(t)
    logits = torch.randn(t, e, generator=gen, device="cuda")
    ids = logits.topk(4, 1).indices.to(torch.int32)
    config = tuning.TuneWork.router(e, 4, True)
    counts = torch.cat([torch.bincount(ids.flatten().long(), minlength=e), torch.tensor([t], device="cuda")]).to(torch.int32)
    (z, g), kept = side_by_side(t, 4, e, e)
    z.copy_(logits)
    want = torch.empty(t, e, device="cuda")
    with tuning.TuneWork(api, tokens=t, experts=e) as work:
        work.balance_backward(config, logits.data_ptr(), ids.data_ptr(), None, t, counts.data_ptr(), 0.5, None, want.data_ptr())
        work.balance_backward(config, ptr(z), ids.data_ptr(), None, t, counts.data_ptr(), 0.5, None, ptr(g), z.stride(0) * 4, g.stride(0) * 4)
        work.sync()
    assert torch.equal(g, want) and kept() and torch.equal(z, logits)
