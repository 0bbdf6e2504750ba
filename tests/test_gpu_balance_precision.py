"""Small probabilities keep their relative precision in the sums and in the loss.

Bound.  u = 2^-24 is half a step of FP32, d = m - z.  exp(z - m) is 2 to a product: the difference is rounded once (d u), the product once (d u, as
2^x changes by ln 2 of x's error and x is d / ln 2), log2 e is off by 0.23 u of itself, and the function by 2^-22 = 4 u.  So an exponential is off by (2.25 d + 4) u relative, the
sum of a row by the mean of that over p and by E / 32 + 5 additions, and the quotient, product and rounding of the result by 7 u; a sum over T tokens by T u more.  What is below
2^-82 of a CTA's share of a sum is rounded to the nearest multiple of it: 2^-83 for every token at most."""
import pytest
import torch

from picoforge_b200 import tuning
from test_gpu_balance import U, api  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 3, 50, 3000])
@pytest.mark.parametrize("e", [60, 512, 1024, 1500, 4096])
def test_sums_and_loss_of_unlikely_experts(api, e, tokens):  # noqa: F811
    gen = torch.Generator(device="cuda").manual_seed(e + tokens)
    # one likely expert, the others down to e^-50 of it: every expert keeps its own size in all tokens
    z = torch.linspace(0, -50, e, device="cuda") + 0.25 * torch.randn(tokens, e, generator=gen, device="cuda")
    ids = (e - 1 - torch.randint(0, e // 4, (tokens, 2), generator=gen, device="cuda")).to(torch.int32)         # among the unlikeliest
    counts, sums, loss = torch.empty(e + 1, dtype=torch.int32, device="cuda"), torch.empty(e, device="cuda"), torch.empty(1, device="cuda")
    with tuning.TuneWork(api, tokens=tokens, experts=e) as work:
        for _ in range(2):                                   # the workspace is left as it was found
            work.balance_forward(work.router(e, 2, True), z.data_ptr(), ids.data_ptr(), None, tokens, counts.data_ptr(), sums.data_ptr(), loss.data_ptr())
        work.sync()
    d = z.double().amax(1, keepdim=True) - z.double()
    p = torch.softmax(z.double(), 1)
    off = U * (2.25 * d + 2.25 * (p * d).sum(1, keepdim=True) + e / 32 + 20)
    want, room = p.sum(0), (p * off).sum(0) + U * tokens * p.sum(0) + tokens * 2.0 ** -83
    assert ((sums.double() - want).abs() <= room).all(), ((sums.double() - want).abs() / want).max().item()
    c = torch.bincount(ids.flatten().long(), minlength=e).double()
    assert counts[:e].tolist() == c.long().tolist()
    value = e / tokens ** 2 * (c * want).sum().item()
    assert abs(loss.item() - value) <= e / tokens ** 2 * (c * room).sum().item() + U * value
