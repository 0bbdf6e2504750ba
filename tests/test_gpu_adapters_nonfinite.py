"""An infinity or a NaN in any operand of the adapters reaches exactly the results that the formulas take it to; the others have the
bits that they have without it."""
import pytest
import torch

from test_gpu_adapters import Case, api, backward, formula, forward  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("r", [5, 16])
@pytest.mark.parametrize("t", [4, 200])
def test_each_operand_in_turn(api, t, r, dtype):  # noqa: F811
    c = Case(t, 256, 136, r, 2, dtype, "runs")
    c.slot[t // 2] = -1
    places = {"x": (1, 5), "dy": (1, 100), "a": (int(c.slot[1]), r - 1, 17), "b": (int(c.slot[1]), 3, r // 2), "scale": (int(c.slot[1]),), "by": (1, 7), "bx": (2, 9)}
    with c.work(api) as work:
        clean = (forward(work, c), *backward(work, c))
        for name, at in places.items():
            for bad in (float("inf"), float("-inf"), float("nan")):
                operand = getattr(c, name)
                kept = operand[at].clone()
                operand[at] = bad
                c.x[t // 2], c.dy[t // 2] = bad, bad         # a token without an adapter: reaches nothing
                got = (forward(work, c), *backward(work, c))
                work.sync()
                y, dx, da, db = formula(c)
                for g, want, before in zip(got, (c.by + y, c.bx + dx, da, db), clean):
                    assert torch.equal(torch.isfinite(g), torch.isfinite(want)), (name, bad)
                    assert torch.equal(g[torch.isfinite(g)], before[torch.isfinite(g)]), (name, bad)
                operand[at] = kept
