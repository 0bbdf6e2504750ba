"""Low-rank adapters beside a projection and their gradients against the formulas in 64 bits.

Bounds.  u = 2^-24 is half a step of FP32.  x enters as a sum of three bf16 values that is x, and F32 adapters likewise; what is left
out of their products, beyond the second order, is below 2^-21 of them (so inside the sixteen of the bound below).  A sum of n terms in FP32 whose additions may
truncate (tensor cores) is off by at most 2 n u times the sum of the terms' sizes.  So every value is held to 2 u (n + 16) S, S the same formula on absolute
values and n the terms of both sums (`worst`), and all of them together, where errors of random sign add up like sqrt(n), to 4 u sqrt(n + 16) relative to
the norm of what the adapters give (`spread`), plus u for the one addition of base."""
import math

import pytest
import torch

from picoforge_b200 import abi, tuning

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GGUF = {torch.float32: abi.F32, torch.float16: abi.F16, torch.bfloat16: abi.BF16}
NONE = -1


def rows(t, width, pad, gen, scale=1.0):
    """[t, width] values inside rows of width + pad, so that rows need not start on a 16-byte boundary."""
    return (torch.randn(t, width + pad, generator=gen, device="cuda") * scale)[:, :width] if t else torch.zeros(0, width, device="cuda")


class Case:
    def __init__(self, t, k, n, r, slots, dtype, pattern="mixed", pad=0, seed=0, base=True):
        gen = torch.Generator(device="cuda").manual_seed(1000 * seed + t * 7 + k + n + r)
        self.t, self.k, self.n, self.r, self.s, self.dtype, self.pad = t, k, n, r, slots, dtype, pad
        self.x, self.dy = rows(t, k, pad, gen), rows(t, n, pad, gen)
        self.a = (torch.randn(slots, r, k, generator=gen, device="cuda") * k ** -0.5).to(dtype)
        self.b = torch.randn(slots, n, r, generator=gen, device="cuda").to(dtype)
        self.scale = 0.5 + torch.rand(slots, generator=gen, device="cuda")
        self.by, self.bx = (rows(t, n, pad, gen), rows(t, k, pad, gen)) if base else (None, None)
        if pattern == "mixed":
            slot = torch.randint(0, slots, (t,), generator=gen, device="cuda")
            slot[torch.rand(t, generator=gen, device="cuda") < 0.2] = NONE
        elif pattern == "runs":
            slot = (torch.arange(t, device="cuda") * slots // max(t, 1)).flip(0)
        elif pattern == "one":
            slot = torch.full((t,), slots - 1, device="cuda")
        else:
            slot = torch.full((t,), NONE, device="cuda")
        self.slot = slot.to(torch.int32)

    def view(self):
        return tuning.TuneWork.adapters(self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(), GGUF[self.dtype], self.s, self.r, self.k, self.n)

    def work(self, api):
        return tuning.TuneWork(api, tokens=max(self.t, 1), slots=self.s, rank=self.r)


def pitch(v):
    return v.stride(0) * 4 if v is not None else 0


def ptr(v):
    return v.data_ptr() if v is not None else None


def forward(work, c, y=None, base="own"):
    y = torch.full((c.t, c.n + c.pad), -99.0, device="cuda")[:, :c.n] if y is None else y
    base = c.by if isinstance(base, str) else base
    work.adapter_forward(c.view(), c.x.data_ptr(), c.slot.data_ptr(), ptr(base), y.data_ptr(), c.t, pitch(c.x), pitch(base), pitch(y))
    return y


def backward(work, c, want=("dx", "d")):
    dx = torch.full((c.t, c.k + c.pad), -99.0, device="cuda")[:, :c.k] if "dx" in want else None
    da = torch.full((c.s, c.r, c.k), -99.0, device="cuda") if "d" in want else None
    db = torch.full((c.s, c.n, c.r), -99.0, device="cuda") if "d" in want else None
    work.adapter_backward(c.view(), c.x.data_ptr(), c.slot.data_ptr(), c.dy.data_ptr(), ptr(c.bx), ptr(dx), ptr(da), ptr(db), c.t, pitch(c.x), pitch(c.dy),
                          pitch(c.bx), pitch(dx))
    return dx, da, db


def formula(c, absolute=False):
    """(y - base, dx - base, dA, dB) in 64 bits, or the same on absolute values."""
    f = (lambda v: v.double().abs()) if absolute else (lambda v: v.double())
    x, dy, a, b, scale = f(c.x), f(c.dy), f(c.a), f(c.b), f(c.scale)
    y, dx, da, db = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for s in range(c.s):
        at = torch.nonzero(c.slot == s).flatten()
        if at.numel():
            h, g = x[at] @ a[s].T, scale[s] * (dy[at] @ b[s])
            y[at], dx[at] = scale[s] * (h @ b[s].T), g @ a[s]
            da[s], db[s] = g.T @ x[at], scale[s] * (dy[at].T @ h)
    return y, dx, da, db


def close(got, want, sizes, terms, base=None):
    got, error = got.double(), None
    if base is not None:
        error = (got - (base.double() + want)).abs()
        room = U * (base.double() + want).abs()
    else:
        error, room = (got - want).abs(), 0.0
    assert (error <= 2 * U * (terms + 16) * sizes + room).all(), (error / (U * sizes + 1e-300)).max().item()
    allowed = 4 * U * math.sqrt(terms + 16) * want.norm().item() + (U * (base.double() + want).norm().item() if base is not None else 0.0)
    assert error.norm().item() <= allowed, (error.norm().item(), allowed)


def check(api, c, streams=True):
    want, sizes = formula(c), formula(c, True)
    most = int(torch.bincount(c.slot[c.slot >= 0].long(), minlength=1).max()) if c.t else 0
    with c.work(api) as work:
        y = forward(work, c)
        dx, da, db = backward(work, c)
        work.sync()
    close(y, want[0], sizes[0], c.k + c.r, c.by)
    close(dx, want[1], sizes[1], c.n + c.r, c.bx)
    close(da, want[2], sizes[2], c.n + most)
    close(db, want[3], sizes[3], c.k + most)
    return y, dx, da, db


@pytest.fixture
def api(gpu):
    assert gpu.lib.qw4cu_set_stream(1) == 0             # the legacy default stream, which torch uses
    yield gpu
    torch.cuda.synchronize()
    assert gpu.lib.qw4cu_set_stream(None) == 0


SIZES = [(1, 64, 48, 4, 1), (1, 2048, 512, 16, 4), (3, 512, 2048, 8, 2), (4, 2560, 640, 64, 3), (17, 16, 8, 1, 2), (31, 40, 24, 5, 7),
         (64, 2048, 512, 32, 48), (65, 256, 333, 20, 9), (130, 777, 65, 7, 3), (200, 1, 1, 3, 2), (257, 512, 1030, 128, 2), (333, 640, 2560, 33, 5),
         (500, 96, 160, 12, 300), (1100, 130, 70, 17, 4), (2048, 64, 128, 64, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,k,n,r,s", SIZES)
def test_against_the_formulas(api, t, k, n, r, s, dtype):
    check(api, Case(t, k, n, r, s, dtype))


@pytest.mark.parametrize("pattern", ["runs", "one", "none"])
@pytest.mark.parametrize("t,k,n,r,s", [(5, 128, 96, 16, 3), (70, 512, 320, 16, 3), (700, 256, 512, 24, 6)])
def test_where_the_tokens_of_a_slot_lie(api, t, k, n, r, s, pattern):
    c = Case(t, k, n, r, s, torch.bfloat16, pattern)
    y, dx, da, db = check(api, c)
    if pattern == "none":
        assert torch.equal(y, c.by) and torch.equal(dx, c.bx) and not da.any() and not db.any()


@pytest.mark.parametrize("t,k,n,r", [(8200, 8192, 64, 24), (1044, 19200, 19200, 16), (1030, 19200, 19200, 64), (3000, 12000, 130, 128)])
def test_sums_longer_than_an_accumulator_takes(api, t, k, n, r):
    """Runs of more than 1024 columns or tokens to a CTA: accumulators are put by and begun anew; the last of them may have a few tokens alone."""
    check(api, Case(t, k, n, r, 1, torch.bfloat16, "one"))


@pytest.mark.parametrize("pad", [1, 2, 4])
@pytest.mark.parametrize("t,k,n,r,s", [(2, 64, 48, 8, 2), (50, 128, 96, 16, 3), (400, 256, 512, 24, 2)])
def test_rows_apart_and_off_the_16_byte_grid(api, t, k, n, r, s, pad):
    c = Case(t, k, n, r, s, torch.float16, pad=pad)
    check(api, c)
    whole = torch.full((t, n + pad), -99.0, device="cuda")
    with c.work(api) as work:
        forward(work, c, whole[:, :n])
        work.sync()
    assert (whole[:, n:] == -99).all()                  # what lies between the rows is left as it was


def test_adapters_off_the_16_byte_grid(api):
    for dtype, t in ((torch.bfloat16, 3), (torch.bfloat16, 150), (torch.float32, 150)):
        c = Case(t, 128, 96, 16, 2, dtype)
        for name in ("a", "b"):
            v = getattr(c, name)
            room = torch.zeros(v.numel() + 1, dtype=dtype, device="cuda")
            room[1:] = v.flatten()
            setattr(c, name, room[1:].view(v.shape))
        check(api, c)


@pytest.mark.parametrize("t", [2, 90, 600])
def test_base_absent_in_place_or_elsewhere(api, t):
    c = Case(t, 256, 192, 16, 4, torch.bfloat16)
    with c.work(api) as work:
        apart = forward(work, c)
        alone = forward(work, c, base=None)
        y = c.by.clone()
        forward(work, c, y, base=y)
        work.sync()
    assert torch.equal(y, apart)
    assert torch.equal(alone + c.by, apart)
    assert not alone[c.slot < 0].any()


@pytest.mark.parametrize("t", [2, 90, 600])
def test_rows_of_different_pitch_and_dx_in_place(api, t):
    c = Case(t, 256, 192, 16, 4, torch.float16)
    with c.work(api) as work:
        want, (dx, da, db) = forward(work, c), backward(work, c)
        wide_base, wide_y = torch.zeros(t, 192 + 8, device="cuda"), torch.zeros(t, 192 + 12, device="cuda")
        wide_base[:, :192] = c.by
        forward(work, c, wide_y[:, :192], base=wide_base[:, :192])
        place = c.bx.clone()
        work.adapter_backward(c.view(), c.x.data_ptr(), c.slot.data_ptr(), c.dy.data_ptr(), place.data_ptr(), place.data_ptr(), None, None, t)
        work.sync()
    assert torch.equal(wide_y[:, :192], want) and not wide_y[:, 192:].any() and torch.equal(place, dx)


def test_a_smaller_call_on_a_larger_workspace(api):
    """The scratch is laid out by the call, not by the limits: other slots, ranks and token counts in turn, stale contents behind."""
    with tuning.TuneWork(api, tokens=3000, slots=40, rank=128) as work:
        for t, k, n, r, slots in ((3000, 128, 64, 128, 40), (100, 64, 96, 8, 3), (700, 96, 64, 33, 7), (1, 64, 64, 16, 1), (2999, 64, 128, 17, 40)):
            c = Case(t, k, n, r, slots, torch.bfloat16)
            y, (dx, da, db) = forward(work, c), backward(work, c)
            work.sync()
            with c.work(api) as own:
                for p, q in zip((y, dx, da, db), (forward(own, c), *backward(own, c))):
                    assert torch.equal(p, q)
                own.sync()


@pytest.mark.parametrize("t", [3, 64, 300])
def test_parts_of_the_gradient_and_the_same_bits_twice(api, t):
    c = Case(t, 256, 512, 16, 3, torch.bfloat16)
    with c.work(api) as work:
        dx, da, db = backward(work, c)
        only_x, _, _ = backward(work, c, ("dx",))
        _, only_a, only_b = backward(work, c, ("d",))
        work.sync()
        again = backward(work, c)
        y, y2 = forward(work, c), forward(work, c)
        work.sync()
    for p, q in zip((dx, da, db, dx, da, db, y), (only_x, only_a, only_b) + again + (y2,)):
        assert torch.equal(p, q)


def test_scale_absent(api):
    for t in (3, 100, 400):
        c = Case(t, 64, 64, 8, 2, torch.float32)
        c.scale = torch.ones(2, device="cuda")
        with c.work(api) as work:
            y = forward(work, c)
            view = c.view()
            view.scale = None
            z = torch.empty_like(y)
            work.adapter_forward(view, c.x.data_ptr(), c.slot.data_ptr(), c.by.data_ptr(), z.data_ptr(), c.t)
            work.sync()
        assert torch.equal(y, z)


@pytest.mark.parametrize("t", [0, 4, 80, 300])
def test_slots_out_of_range_and_no_tokens(api, t):
    c = Case(t, 64, 64, 8, 2, torch.bfloat16)
    with c.work(api) as work:
        if t:
            c.slot[t // 2] = 2
            want = formula(c)[0]
            y = forward(work, c)
            with pytest.raises(abi.MoeError) as info:
                work.sync()
            assert info.value.status == abi.RANGE
            with pytest.raises(abi.MoeError) as info:
                forward(work, c)
            assert info.value.status == abi.BAD_STATE
            work.reset()
            assert torch.equal(y[t // 2], c.by[t // 2])             # and the others are what they should be
            assert (y.double() - c.by.double() - want).abs().max().item() < 1e-4
            dx, da, db = backward(work, c)
            with pytest.raises(abi.MoeError):
                work.sync()
            work.reset()
            assert torch.equal(dx[t // 2], c.bx[t // 2])
        else:
            forward(work, c)
            _, da, db = backward(work, c)
            work.sync()
            assert not da.any() and not db.any()


def test_nonfinite_values_stay_in_their_rows(api):
    """An infinity or NaN in one token's x or dy reaches that token alone (and its own adapter's gradients)."""
    for t in (4, 200):
        c = Case(t, 256, 128, 16, 2, torch.bfloat16, "runs")
        with c.work(api) as work:
            before, clean = forward(work, c), backward(work, c)
            c.x[1, 5] = float("inf")
            c.x[2, 7] = float("nan")
            c.dy[1, 3] = float("nan")
            after, dirty = forward(work, c), backward(work, c)
            work.sync()
        keep = [i for i in range(t) if i not in (1, 2)]
        assert torch.equal(before[keep], after[keep]) and not torch.isfinite(after[1]).any() and torch.isnan(after[2]).all()
        keep = [i for i in range(t) if i != 1]
        assert torch.equal(clean[0][keep], dirty[0][keep]) and torch.isnan(dirty[0][1]).all()
        other = 1 - int(c.slot[1])
        assert torch.equal(clean[1][other], dirty[1][other]) or int(c.slot[2]) == other


def test_large_and_small_values(api):
    """Values near the ends of FP32's range, where a split into shorter numbers could overflow or vanish."""
    for scale in (1e30, 1e-25):
        for t in (3, 100):
            c = Case(t, 128, 64, 8, 2, torch.bfloat16, base=False)
            c.x *= scale
            want, sizes = formula(c)[0], formula(c, True)[0]
            with c.work(api) as work:
                y = forward(work, c)
                work.sync()
            close(y, want, sizes, c.k + c.r)


@pytest.mark.parametrize("t,step", [(40, 1 << 26), (300, 1 << 24)])
def test_offsets_beyond_32_bits(api, t, step):
    """Rows of x and y that lie more than 2^31 floats (and 2^32) apart from the first."""
    torch.cuda.empty_cache()
    c = Case(t, 256, 128, 8, 2, torch.bfloat16)
    x = torch.empty((t - 1) * step + 256, device="cuda").as_strided((t, 256), (step, 1))
    x.copy_(c.x)
    with c.work(api) as work:
        y = forward(work, c)
        g = backward(work, c)
        c.x = x
        far_y = torch.empty((t - 1) * step + 128, device="cuda").as_strided((t, 128), (step, 1))
        forward(work, c, far_y)
        far_g = backward(work, c)
        work.sync()
    assert torch.equal(y, far_y)
    for p, q in zip(g, far_g):
        assert torch.equal(p, q)


def test_captured_into_a_graph_and_replayed_on_other_values(api):
    for t in (4, 300):
        c, d = Case(t, 256, 512, 16, 3, torch.bfloat16), Case(t, 256, 512, 16, 3, torch.bfloat16, seed=5)
        stream = torch.cuda.Stream()
        with c.work(api) as work, d.work(api) as other:
            y, (dx, da, db) = forward(work, c), backward(work, c)
            want = [v.clone() for v in (forward(other, d), *backward(other, d))]
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(stream):
                assert api.lib.qw4cu_set_stream(stream.cuda_stream) == 0
                with torch.cuda.graph(graph, stream=stream):
                    forward(work, c, y)
                    work.adapter_backward(c.view(), c.x.data_ptr(), c.slot.data_ptr(), c.dy.data_ptr(), c.bx.data_ptr(), dx.data_ptr(), da.data_ptr(),
                                          db.data_ptr(), c.t)
            for name in ("x", "dy", "a", "b", "scale", "slot", "by", "bx"):
                getattr(c, name).copy_(getattr(d, name))
            torch.cuda.synchronize()
            for _ in range(2):
                with torch.cuda.stream(stream):
                    graph.replay()
            torch.cuda.synchronize()
            del graph
            assert api.lib.qw4cu_set_stream(1) == 0
            work.sync()
            for p, q in zip((y, dx, da, db), want):
                assert torch.equal(p, q)


@pytest.mark.parametrize("t,r", [(700, 16), (2500, 64), (1500, 128)])
def test_two_workspaces_on_two_streams_at_once(api, t, r):
    cases = [Case(t, 512, 512, r, 3, torch.bfloat16, seed=i) for i in (1, 2)]
    works = [c.work(api) for c in cases]
    want = [(forward(w, c), *backward(w, c)) for w, c in zip(works, cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for w, c, stream in zip(works, cases, streams):
            assert api.lib.qw4cu_set_stream(stream.cuda_stream) == 0
            with torch.cuda.stream(stream):
                got.append((forward(w, c), *backward(w, c)))
    torch.cuda.synchronize()
    assert api.lib.qw4cu_set_stream(1) == 0
    for w, p, q in zip(works, want, got):
        w.sync()
        w.close()
        for u, v in zip(p, q):
            assert torch.equal(u, v)


def test_the_gradients_are_those_of_the_forward():
    """The formulas that the kernels are held to, against central differences of the forward's, in 64 bits."""
    gen = torch.Generator().manual_seed(3)
    a, b, x, dy = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((3, 7), (5, 3), (4, 7), (4, 5)))
    scale = 0.7

    def loss(a, b, x):
        return (scale * ((x @ a.T) @ b.T) * dy).sum()

    g = scale * (dy @ b)
    for v, grad in ((a, g.T @ x), (b, scale * (dy.T @ (x @ a.T))), (x, g @ a)):
        for i in range(v.numel()):
            step = torch.zeros(v.numel(), dtype=torch.float64)
            step[i] = 1e-5
            step = step.view(v.shape)
            args = [[u + step if u is v else u for u in (a, b, x)], [u - step if u is v else u for u in (a, b, x)]]
            assert abs((loss(*args[0]) - loss(*args[1])).item() / 2e-5 - grad.flatten()[i].item()) < 1e-6


def test_kernels_that_serve_them_are_the_librarys(api):
    c = Case(100, 64, 64, 8, 2, torch.bfloat16)
    with c.work(api) as work:
        api.lib.qw4cu_launch_log_begin()
        forward(work, c)
        backward(work, c)
        names = api.launch_names()
        work.sync()
    assert names and all(n.startswith("adapter_") for n in names)
