"""The balance loss of a router, its counts and the gradient of the logits against the definitions in 64 bits.

Bounds.  u = 2^-24 is half a step of FP32.  z - m is rounded once, so exp of it is off by |z - m| u relative, and by 4 u more for the
function itself; the sum over E experts, 32 lanes of them added in a tree, by (E / 32 + 5) u; a product or quotient by u
each.  So p is off by at most u (E / 32 + 16 + |z - m|) relative, sums over T tokens by at most T u more (and
2^-41 T where 64-bit integers of 2^-40 meet)."""
import numpy as np
import pytest
import torch

from picoforge_b200 import abi, tuning

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture
def api(gpu):
    assert gpu.lib.qw4cu_set_stream(1) == 0             # the legacy default stream, which torch uses
    yield gpu
    torch.cuda.synchronize()
    assert gpu.lib.qw4cu_set_stream(None) == 0


class Case:
    def __init__(self, t, e, k, norm=True, padded=0.0, spread=1.0, pad=0, seed=0, offset=0):
        gen = torch.Generator(device="cuda").manual_seed(1000 * seed + 31 * t + e)
        self.t, self.e, self.k, self.norm = t, e, k, norm
        store = torch.full((t * (e + pad) + offset,), float("nan"), device="cuda")
        self.z = store[offset:].view(t, e + pad)[:, :e]
        self.z.copy_(spread * torch.randn(t, e, generator=gen, device="cuda") - 0.6 * torch.log(torch.arange(e, device="cuda") + 1.0))
        self.ids = torch.argsort(torch.rand(t, e, generator=gen, device="cuda") - 0.2 * self.z, 1)[:, :k].to(torch.int32).contiguous()
        self.mask = None
        if padded:
            self.mask = (torch.rand(t, generator=gen, device="cuda") >= padded).to(torch.uint8) * 7
            self.z[self.mask == 0] = float("nan")
            self.ids[self.mask == 0] = -1
        self.dw = torch.randn(t, k, generator=gen, device="cuda") / t
        if padded:
            self.dw[self.mask == 0] = float("inf")

    def config(self):
        return tuning.TuneWork.router(self.e, self.k, self.norm)

    def work(self, api):
        return tuning.TuneWork(api, tokens=max(self.t, 1), experts=self.e)

    def valid(self):
        return torch.ones(self.t, dtype=torch.bool, device="cuda") if self.mask is None else self.mask != 0


def mask_of(c):
    return c.mask.data_ptr() if c.mask is not None else None


def forward(work, c, out=None):
    counts, sums, loss = out or (torch.full((c.e + 1,), -1, dtype=torch.int32, device="cuda"), torch.full((c.e,), -99.0, device="cuda"),
                                 torch.full((1,), -99.0, device="cuda"))
    work.balance_forward(c.config(), c.z.data_ptr(), c.ids.data_ptr(), mask_of(c), c.t, counts.data_ptr(), sums.data_ptr(), loss.data_ptr(), c.z.stride(0) * 4)
    return counts, sums, loss


def backward(work, c, counts, loss_grad=0.5, dw="own", pad=0, out=None):
    grad = torch.full((c.t, c.e + pad), -99.0, device="cuda") if out is None else out
    dw = c.dw if isinstance(dw, str) else dw
    work.balance_backward(c.config(), c.z.data_ptr(), c.ids.data_ptr(), mask_of(c), c.t, counts.data_ptr(), loss_grad, dw.data_ptr() if dw is not None else None,
                          grad.data_ptr(), c.z.stride(0) * 4, grad.stride(0) * 4)
    return grad


def softmax(z):
    e = torch.exp(z - z.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def formula_forward(c):
    valid = c.valid()
    p = softmax(c.z[valid].double())
    counts = torch.bincount(c.ids[valid].long().flatten(), minlength=c.e) if valid.any() else torch.zeros(c.e, dtype=torch.long, device="cuda")
    n = int(valid.sum())
    sums = p.sum(0)
    return counts, n, sums, c.e * (counts.double() * sums).sum().item() / n ** 2 if n else 0.0


def distance(z):
    """|z - m|, what the exponent's rounding goes with; exp is zero from 104 on, and a logit of -inf has no rounding."""
    far = (z - z.amax(1, keepdim=True)).abs()
    return torch.where(torch.isfinite(far), far, torch.zeros_like(far)).clamp(max=104)


def formula_backward(c, counts, n, loss_grad=0.5, dw="own"):
    """The gradient, and how far off it may be: the relative error of each term times its size."""
    valid = c.valid()
    grad, room = torch.zeros(c.t, c.e, dtype=torch.float64, device="cuda"), torch.zeros(c.t, c.e, dtype=torch.float64, device="cuda")
    z, ids = c.z[valid].double(), c.ids[valid].long()
    if not n:
        return grad, room
    p, far = softmax(z), distance(z)
    off = 2 * U * (c.e / 32 + c.k + 16 + far + (p * far).sum(1, keepdim=True))      # of p, and of products and sums with it
    f = counts.double()[:c.e] * (loss_grad * c.e / n ** 2)
    g = p * (f - (p * f).sum(1, keepdim=True))
    size = off * p * (f.abs() + (p * f).sum(1, keepdim=True).abs())
    dw = c.dw if isinstance(dw, str) else dw
    if dw is not None:
        d = dw[valid].double()
        if c.norm:
            chosen = z.gather(1, ids)
            w, far = softmax(chosen), distance(chosen)
            off = 2 * U * (2 * c.k + 16 + far + (w * far).sum(1, keepdim=True))
            g.scatter_add_(1, ids, w * (d - (w * d).sum(1, keepdim=True)))
            size.scatter_add_(1, ids, off * w * (d.abs() + (w * d.abs()).sum(1, keepdim=True)))
        else:
            w, off_w = p.gather(1, ids), off.gather(1, ids)
            g -= p * (w * d).sum(1, keepdim=True)
            g.scatter_add_(1, ids, w * d)
            size += p * ((off_w * w * d.abs()).sum(1, keepdim=True) + off * (w * d.abs()).sum(1, keepdim=True))
            size.scatter_add_(1, ids, off_w * w * d.abs())
    grad[valid], room[valid] = g, size
    return grad, room


def check(api, c):
    counts, n, sums, loss = formula_forward(c)
    with c.work(api) as work:
        got = forward(work, c)
        grad = backward(work, c, got[0])
        alone = backward(work, c, got[0], dw=None)
        work.sync()
    assert got[0][:c.e].tolist() == counts.tolist() and int(got[0][c.e]) == n
    far = float(distance(c.z[c.valid()].double()).max()) if n else 0.0
    relative = U * (c.e / 32 + 24 + far + c.t)
    assert ((got[1].double() - sums).abs() <= relative * sums + c.t * 2.0 ** -41 + 1e-38).all()
    assert abs(got[2].item() - loss) <= relative * loss + c.t * 2.0 ** -41
    for g, dw in ((grad, "own"), (alone, None)):
        want, room = formula_backward(c, counts, n, dw=dw)
        assert ((g.double() - want).abs() <= room + 1e-37).all(), ((g.double() - want).abs() / (room + 1e-37)).max().item()
        assert not g[~c.valid()].any()
    return got, grad


SIZES = [(1, 8, 1), (1, 512, 10), (3, 60, 4), (7, 7, 7), (33, 33, 5), (64, 512, 10), (129, 1024, 8), (40, 1500, 12), (17, 4096, 3), (5, 130, 100),
         (1000, 128, 8), (2500, 512, 10), (9000, 64, 6), (300, 1, 1), (70, 500, 40), (21, 2048, 64)]


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("padded", [0.0, 0.3])
@pytest.mark.parametrize("t,e,k", SIZES)
def test_against_the_definitions(api, t, e, k, padded, norm):
    check(api, Case(t, e, k, norm, padded))


@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 0), (0, 1), (3, 2)])
@pytest.mark.parametrize("t,e,k", [(20, 512, 10), (300, 60, 4), (11, 1200, 4)])
def test_rows_apart_and_off_the_16_byte_grid(api, t, e, k, pad, offset):
    c = Case(t, e, k, True, 0.2, pad=pad, offset=offset)
    got, grad = check(api, c)
    with c.work(api) as work:
        wide = backward(work, c, got[0], pad=3)
        work.sync()
    assert torch.equal(wide[:, :e], grad) and (wide[:, e:] == -99).all()            # what lies between the rows is left as it was


def test_sharp_and_flat_rows(api):
    for spread in (0.0, 8.0, 40.0):
        check(api, Case(200, 512, 10, True, spread=spread))


def test_experts_left_out_by_their_logits(api):
    """-inf (no probability at all), the lowest finite value, and rows of nothing but one of them."""
    for norm in (True, False):
        c = Case(50, 64, 4, norm)
        c.z[:, 10:20] = float("-inf")
        c.z[:, 30:40] = torch.finfo(torch.float32).min
        c.z[3] = torch.finfo(torch.float32).min
        c.z[4, 1:] = float("-inf")
        c.z[5] = torch.finfo(torch.float32).max
        c.ids[:] = torch.arange(4, dtype=torch.int32, device="cuda") + 40                 # among the chosen one that is left out, where the row has others
        c.ids[4] = torch.tensor([0, 3, 5, 7], dtype=torch.int32)
        c.ids[6, 0] = 12
        got, grad = check(api, c)
        assert torch.isfinite(grad).all() and not grad[torch.isinf(c.z)].any()


def test_everything_masked_and_no_tokens(api):
    c = Case(40, 32, 2, padded=0.5)
    c.mask[:] = 0
    c.z[:] = float("nan")
    for t in (40, 0):
        c.t = t
        c.z, c.ids, c.dw, c.mask = c.z[:t], c.ids[:t], c.dw[:t], c.mask[:t]
        with tuning.TuneWork(api, tokens=40, experts=32) as work:
            counts, sums, loss = forward(work, c)
            grad = backward(work, c, counts)
            work.sync()
        assert not counts.any() and not sums.any() and loss.item() == 0 and not grad.any()


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("e", [64, 512, 1100])
def test_a_row_without_a_softmax_is_reported(api, bad, e):
    c = Case(30, e, 4)
    with c.work(api) as work:
        clean = forward(work, c)
        grad = backward(work, c, clean[0])
        work.sync()
        keep = c.z.clone()
        if bad == "-inf":
            c.z[[21, 9]] = float(bad)
        else:
            c.z[21, 5] = c.z[9, e - 1] = float(bad)
        counts, sums, loss = forward(work, c)
        with pytest.raises(abi.MoeError) as info:
            work.sync()
        assert info.value.status == abi.NONFINITE and info.value.row == 9
        assert torch.equal(counts, clean[0]) and torch.isnan(sums).all() and torch.isnan(loss).all()
        with pytest.raises(abi.MoeError) as info:
            forward(work, c)
        assert info.value.status == abi.BAD_STATE
        work.reset()
        dirty = backward(work, c, clean[0])
        with pytest.raises(abi.MoeError) as info:
            work.sync()
        assert info.value.status == abi.NONFINITE and info.value.row == 9
        work.reset()
        rest = [i for i in range(30) if i not in (9, 21)]
        assert torch.equal(dirty[rest], grad[rest]) and not torch.isfinite(dirty[9]).all()
        c.z.copy_(keep)                                                                    # and the workspace is as new
        again = forward(work, c)
        work.sync()
        for p, q in zip(clean, again):
            assert torch.equal(p, q)


def test_expert_ids_out_of_range(api):
    for e, k in ((16, 4), (1100, 4), (64, 40)):
        c = Case(30, e, k)
        with c.work(api) as work:
            clean = forward(work, c)
            work.sync()
            c.ids[17, 2] = e
            counts, sums, loss = forward(work, c)
            with pytest.raises(abi.MoeError) as info:
                work.sync()
            assert info.value.status == abi.RANGE
            assert int(counts[:e].sum()) == 30 * k - 1 and torch.equal(sums, clean[1])
            work.reset()
            backward(work, c, counts)
            with pytest.raises(abi.MoeError) as info:
                work.sync()
            assert info.value.status == abi.RANGE


def test_the_same_expert_twice_in_a_token(api):
    """Routes give none, but ids are the caller's: each place counts, and each place's gradient arrives."""
    for norm in (True, False):
        c = Case(20, 64, 4, norm)
        c.ids[:, 3] = c.ids[:, 1]
        c.ids[7] = c.ids[7, 0]
        check(api, c)


def test_counts_summed_over_ranks(api):
    """The gradient for counts that other ranks' batches were added to: that of the loss over the whole job."""
    a, b = Case(40, 64, 4, seed=1), Case(60, 64, 4, seed=2)
    both = Case(100, 64, 4)
    both.z, both.ids, both.dw = torch.cat([a.z, b.z]), torch.cat([a.ids, b.ids]), torch.cat([a.dw, b.dw])
    with both.work(api) as work:
        counts = forward(work, a)[0] + forward(work, b)[0]
        parts = torch.cat([backward(work, a, counts), backward(work, b, counts)])
        whole, together = forward(work, both)[0], backward(work, both, counts)
        work.sync()
    assert torch.equal(whole, counts) and torch.equal(parts, together)


def test_the_same_bits_twice_and_in_a_graph(api):
    c, d = Case(3000, 512, 10), Case(3000, 512, 10, seed=3)
    stream = torch.cuda.Stream()
    with c.work(api) as work:
        first, second = forward(work, c), forward(work, c)
        grad, grad2 = backward(work, c, first[0]), backward(work, c, first[0])
        for p, q in zip(first + (grad,), second + (grad2,)):
            assert torch.equal(p, q)
        want = forward(work, d)
        want = [v.clone() for v in want + (backward(work, d, want[0]),)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            assert api.lib.qw4cu_set_stream(stream.cuda_stream) == 0
            with torch.cuda.graph(graph, stream=stream):
                forward(work, c, first)
                backward(work, c, first[0], out=grad)
        for name in ("z", "ids", "dw"):
            getattr(c, name).copy_(getattr(d, name))
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        del graph
        assert api.lib.qw4cu_set_stream(1) == 0
        work.sync()
        for p, q in zip(first + (grad,), want):
            assert torch.equal(p, q)


def test_two_workspaces_on_two_streams_at_once(api):
    cases = [Case(6000, 512, 10, seed=i) for i in (1, 2)]
    works = [c.work(api) for c in cases]
    want = [forward(w, c) for w, c in zip(works, cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for w, c, stream in zip(works, cases, streams):
            assert api.lib.qw4cu_set_stream(stream.cuda_stream) == 0
            with torch.cuda.stream(stream):
                got.append(forward(w, c))
    torch.cuda.synchronize()
    assert api.lib.qw4cu_set_stream(1) == 0
    for w, p, q in zip(works, want, got):
        w.sync()
        w.close()
        for u, v in zip(p, q):
            assert torch.equal(u, v)


def test_offsets_beyond_32_bits(api):
    t, e, step = 40, 64, 1 << 26
    c = Case(t, e, 4)
    far = torch.empty((t - 1) * step + e, device="cuda").as_strided((t, e), (step, 1))
    far.copy_(c.z)
    with c.work(api) as work:
        want = forward(work, c)
        grad = backward(work, c, want[0])
        c.z = far
        got = forward(work, c)
        out = torch.empty((t - 1) * step + e, device="cuda").as_strided((t, e), (step, 1))
        backward(work, c, want[0], out=out)
        work.sync()
    for p, q in zip(want + (grad,), got + (out,)):
        assert torch.equal(p, q)


def test_the_gradient_is_that_of_the_loss():
    """The formula that the kernel is held to against central differences of the loss plus <weights, dw>, in 64 bits."""
    rng = np.random.default_rng(5)
    t, e, k, lam = 4, 6, 3, 0.5
    z0, dw = rng.standard_normal((t, e)), rng.standard_normal((t, k))
    ids = np.stack([rng.permutation(e)[:k] for _ in range(t)])
    counts = np.bincount(ids.ravel(), minlength=e)
    for norm in (True, False):
        def value(z):
            p = np.exp(z - z.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            w = np.take_along_axis(p, ids, 1)
            if norm:
                w = w / w.sum(1, keepdims=True)
            return lam * e / t ** 2 * (counts * p.sum(0)).sum() + (w * dw).sum()

        class Mini:
            pass
        c = Mini()
        c.t, c.e, c.k, c.norm, c.mask = t, e, k, norm, None
        c.z, c.ids, c.dw = torch.tensor(z0, device="cuda"), torch.tensor(ids, device="cuda"), torch.tensor(dw, device="cuda")
        c.valid = lambda: torch.ones(t, dtype=torch.bool, device="cuda")
        grad, _ = formula_backward(c, torch.tensor(counts, device="cuda"), t, lam)
        for i in range(t):
            for j in range(e):
                step = np.zeros_like(z0)
                step[i, j] = 1e-5
                assert abs((value(z0 + step) - value(z0 - step)) / 2e-5 - grad[i, j].item()) < 1e-8
