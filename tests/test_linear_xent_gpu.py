"""Projection and loss without logits, and their gradients, against the formulas in 64 bits.

Tolerances, for each value.  z: a step of the tensor cores adds 16 products and cuts the sum off to fp32, so n steps are off by at most
n 2^-23 of S = sum |x w| (24 bits, cut off); fp32 tensors have 16 bits of each factor and no product of two low parts (3 2^-17 of S) and three times the
steps.  lse, losses: as z at worst; exponents are products in fp32 (2^-22 of the largest |z| in natural units), ex2 and the sums of at most V terms, pairwise over the tiles
(2^-21 and 2^-18).  G: relative to exp(z - lse) as far as z and lse are off, and one rounding (bf16: half of its eps, fp32: 2^-17).  dx, dw: sums of
|G| |w| and |G| |x| times that, and the steps of the sum; one rounding of what is stored.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = [torch.int64, torch.int32, torch.float32]


class Case:
    def __init__(self, M, K, V, dtype, ignored=0.2, spread=2.0, seed=0, ids=torch.int64):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + M + 3 * K + 7 * V)
        normal = lambda *s: torch.empty(*s, device="cuda").normal_(0.0, 1.0, generator=g)  # noqa: E731
        self.x, self.w = normal(M, K).to(dtype), (normal(V, K) * (spread / math.sqrt(K))).to(dtype)
        t = torch.randint(V, (M,), device="cuda", generator=g)
        gone = torch.rand(M, device="cuda", generator=g) < ignored
        self.t = torch.where(gone, torch.where(torch.rand(M, device="cuda", generator=g) < 0.5, -100, V), t)
        self.ids = self.t.to(ids)
        self.g = torch.rand(M, device="cuda", generator=g) / M
        self.dw = (normal(V, K) * 1e-3).to(dtype)
        self.M, self.K, self.V, self.dtype = M, K, V, dtype

    def formulas(self):
        x, w = self.x.double(), self.w.double()
        ok = (self.t >= 0) & (self.t < self.V)
        x = torch.where(ok[:, None], x, 0.0) if not x.isfinite().all() else x
        z, size = x @ w.T, x.abs() @ w.abs().T
        steps, bits = -(-self.K // 16), 0.0
        if self.dtype == F32:
            steps, bits = 3 * steps, 3 * 2.0 ** -17
        off = size * (steps * 2.0 ** -23 + bits)
        lse = torch.logsumexp(z, -1)
        off_lse = off.amax(-1) + z.abs().amax(-1) * 2.0 ** -22 + 2.0 ** -18 + lse.abs() * 2.0 ** -23
        at = self.t.clamp(0, self.V - 1)[:, None]
        losses = torch.where(ok, lse - z.gather(1, at)[:, 0], 0.0)
        off_losses = torch.where(ok, off_lse + off.gather(1, at)[:, 0] + losses.abs() * 2.0 ** -23, 0.0)
        return z, off, lse, off_lse, losses, off_losses, ok

    def check(self, pkg, g=None, **more):
        z, off, lse, off_lse, losses, off_losses, ok = self.formulas()
        got, got_lse = pkg.linear_xent_forward(self.x, self.w, self.ids, **more)
        assert got.dtype == got_lse.dtype == F32 and got.shape == got_lse.shape == self.t.shape
        finite = self.x.isfinite().all(-1)
        assert ((got.double() - losses).abs() <= off_losses)[finite | ~ok].all() and ((got_lse.double() - lse).abs() <= off_lse)[finite].all()
        g = self.g if g is None else g
        p = (z - lse[:, None]).exp()
        one = torch.zeros_like(p)
        one[ok, self.t[ok]] = 1.0
        factor = torch.where(ok, g.double().expand(self.M), 0.0)[:, None]
        G = (p - one) * factor
        round_g = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -16
        off_g = factor.abs() * (p * (off + off_lse[:, None] + z.abs() * 2.0 ** -22 + 2.0 ** -20) * 1.01 + one * 2.0 ** -22) + G.abs() * round_g
        held = self.dw.clone()
        dx = pkg.linear_xent_backward(g, self.x, self.w, self.ids, got_lse, self.dw, **more)
        x, w = torch.where(ok[:, None], self.x.double(), 0.0), self.w.double()
        half = torch.finfo(self.dtype).eps / 2
        terms = 1 if self.dtype == BF16 else 3
        for result, want, sizes, errors, count, before in ((dx, G @ w, G.abs() @ w.abs(), off_g @ w.abs(), self.V, 0.0),
                                                           (self.dw, G.T @ x, G.abs().T @ x.abs(), off_g.T @ x.abs(), self.M, held.double())):
            want = want + before
            tol = errors + sizes * (terms * (count // 16 + 20) * 2.0 ** -23 + (terms > 1) * 3 * 2.0 ** -17) + want.abs() * (half + 2.0 ** -22) + 1e-30
            assert result.dtype == self.dtype and ((result.double() - want).abs() <= tol).all()
        assert pkg.device_status() == 0
        # every call gives the same bits
        again, again_lse = pkg.linear_xent_forward(self.x, self.w, self.ids)
        dw = held.clone()
        assert torch.equal(pkg.linear_xent_backward(g, self.x, self.w, self.ids, got_lse, dw), dx) and torch.equal(dw, self.dw)
        assert torch.equal(again[finite | ~ok], got[finite | ~ok]) and torch.equal(again_lse[finite], got_lse[finite])
        return dx


SHAPES = [(1, 1, 1), (1, 64, 256), (2, 7, 2), (5, 24, 129), (40, 768, 5000), (127, 100, 255), (128, 64, 257), (129, 65, 511), (130, 200, 1000), (255, 8, 64), (256, 256, 512),
          (257, 264, 513), (300, 1600, 300), (513, 72, 3001), (1000, 320, 2049), (77, 33, 50257), (4100, 40, 200)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,V", SHAPES)
def test_shapes(pkg, M, K, V, dtype):
    for i, ignored in enumerate((0.0, 0.4)):
        Case(M, K, V, dtype, ignored, seed=i, ids=IDS[(M + i) % 3]).check(pkg)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,V", [(1, 64, 8000), (1, 768, 50257), (15, 40, 9001), (16, 200, 50257), (17, 72, 8192), (32, 768, 9999), (33, 136, 12001), (48, 8, 30011), (49, 264, 20000),
                                   (64, 768, 16001), (65, 64, 16001), (1, 1, 8001), (2, 33, 9000), (16, 1001, 8003), (31, 201, 8009), (47, 770, 13000), (64, 67, 16003)])
def test_few_rows(pkg, M, K, V, dtype):
    """Sizes at which the forward reads the weights into registers, and those beside them."""
    for i, ignored in enumerate((0.0, 0.4)):
        Case(M, K, V, dtype, ignored, seed=i, ids=IDS[(M + i) % 3]).check(pkg)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,V", [(1, 8, 2000), (1, 780, 50257), (3, 1100, 2001), (4, 64, 9000), (5, 2048, 3000), (8, 768, 30000), (9, 40, 2063), (16, 768, 50257), (16, 2056, 2500),
                                   (16, 4, 5000), (16, 64, 1999), (3, 40, 1), (16, 768, 9), (8, 1600, 17), (17, 64, 5000), (12, 12, 4000), (1, 1, 2000), (2, 1033, 2003), (5, 201, 9001), (7, 770, 4000), (13, 1027, 3001),
                                   (16, 3, 8001)])
def test_gradients_of_few_rows(pkg, M, K, V, dtype):
    """Sizes at which the backward works on few rows in fp32 arithmetic, and those beside them."""
    for i, ignored in enumerate((0.0, 0.4)):
        c = Case(M, K, V, dtype, ignored, seed=i, ids=IDS[(M + i) % 3])
        c.check(pkg)
        held, lse = c.dw.clone(), pkg.linear_xent_forward(c.x, c.w, c.ids)[1]
        dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, c.dw)
        assert torch.equal(pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse), dx)
        assert pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, held, want_dx=False) is None and torch.equal(held, c.dw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_rows_nan_and_infinity(pkg, dtype):
    c = Case(9, 64, 9000, dtype, 0.0)
    c.x[3, 5], c.x[4, 6] = float("nan"), float("inf")
    losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
    assert losses.isfinite().nonzero().flatten().tolist() == [0, 1, 2, 5, 6, 7, 8] and lse[3].isnan()
    c = Case(9, 64, 9000, dtype, 0.0)  # classes that no row can have: their logits are -inf
    c.w[100:9000, 0] = -float("inf")
    c.x[:, 0] = 1.0
    c.x[:, 1:], c.ids = (c.x[:, 1:].abs() + 0.1), c.ids % 100
    if dtype == BF16:
        losses, _ = pkg.linear_xent_forward(c.x, c.w, c.ids)
        want = torch.nn.functional.cross_entropy(c.x.double() @ c.w[:100].double().T, c.ids, reduction="none")
        assert ((losses - want).abs() <= 2.0 ** -14 * (1 + want)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_several_pieces_of_the_vocabulary(pkg, dtype):
    """G of the whole vocabulary is far above the size of a piece: products of one piece beside the logits of the next."""
    Case(9000, 72, 40001, dtype, 0.1).check(pkg)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_without_targets(pkg, dtype):
    c = Case(300, 64, 700, dtype, ignored=1.1)
    held = c.dw.clone()
    dx = c.check(pkg)
    assert (dx == 0).all() and torch.equal(c.dw, held)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
def test_what_rows_without_targets_hold(pkg, dtype, value):
    """Padding may hold anything: it reaches neither a loss nor a gradient."""
    for M, K, V in ((300, 96, 1000), (13, 96, 9000)):
        c = Case(M, K, V, dtype, 0.3)
        c.x[(c.t < 0) | (c.t >= c.V), ::5] = value
        dx = c.check(pkg)
        assert dx.isfinite().all() and c.dw.isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_stays_in_its_row(pkg, dtype):
    c = Case(200, 64, 600, dtype, 0.0)
    c.x[7, 3] = float("nan")
    losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
    dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, None)
    for r in (losses, lse):
        assert r.isnan().nonzero().flatten().tolist() == [7]
    assert dx[7].isnan().all() and dx.isnan().any(-1).sum() == 1


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_and_equal_logits(pkg, dtype):
    """Logits of some thousands, of which the largest takes everything; and equal ones, whose loss is log V."""
    Case(150, 64, 1000, dtype, spread=300.0).check(pkg)
    c = Case(150, 64, 1000, dtype)
    c.w[:] = c.w[0]
    c.check(pkg)
    losses, _ = pkg.linear_xent_forward(c.x, c.w, c.t.clamp(0, 999))
    assert ((losses - math.log(1000)).abs() <= 2.0 ** -17).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("apart,start", [(80, 0), (72, 8), (67, 1), (73, 4)])
def test_rows_that_lie_apart(pkg, dtype, apart, start):
    for M, V in ((140, 333), (7, 9001)):
        c = Case(M, 60, V, dtype)
        rows_apart(pkg, c, dtype, apart, start)


def rows_apart(pkg, c, dtype, apart, start):
    wide = lambda t: torch.full((t.shape[0], apart + 8), 7.0, device="cuda", dtype=dtype)  # noqa: E731
    held = {k: wide(getattr(c, k)) for k in ("x", "w", "dw")}
    for k, v in held.items():
        v[:, start:start + 60] = getattr(c, k)
        setattr(c, k, v[:, start:start + 60])
    c.check(pkg)
    assert (held["dw"][:, :start] == 7).all() and (held["dw"][:, start + 60:] == 7).all()


def test_one_factor_for_all_rows(pkg):
    for value in (1.0, -0.25, 0.0):
        Case(200, 64, 500, BF16).check(pkg, g=torch.tensor([value], device="cuda"))


def test_dx_alone_and_dw_alone(pkg):
    for dtype in (BF16, F32):
        c = Case(333, 136, 2000, dtype)
        _, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
        dw = c.dw.clone()
        dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, dw)
        assert torch.equal(pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse), dx)
        assert pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, c.dw, want_dx=False) is None and torch.equal(c.dw, dw)


def test_leading_dimensions_and_no_rows(pkg):
    c = Case(60, 64, 300, BF16)
    losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
    l3, e3 = pkg.linear_xent_forward(c.x.view(3, 20, 64), c.w, c.ids.view(3, 20))
    assert l3.shape == (3, 20) and torch.equal(l3.flatten(), losses) and torch.equal(e3.flatten(), lse)
    dx = pkg.linear_xent_backward(c.g.view(3, 20), c.x.view(3, 20, 64), c.w, c.ids.view(3, 20), e3)
    assert dx.shape == (3, 20, 64)
    held = c.dw.clone()
    losses, lse = pkg.linear_xent_forward(c.x[:0], c.w, c.ids[:0])
    dx = pkg.linear_xent_backward(torch.ones(1, device="cuda"), c.x[:0], c.w, c.ids[:0], lse, c.dw)
    assert losses.shape == (0,) and dx.shape == (0, 64) and torch.equal(c.dw, held)


def test_against_differences(pkg):
    """(f(x + e d) - f(x - e d)) / 2e with f = sum g loss, in fp32.  Along d a row's loss is a log-sum-exp of z + e u: its third derivative is at
    most (2 max |u|)^3 / 4, which e^2 / 6 of it bounds; each f is off by the losses' own bound."""
    c = Case(24, 48, 90, F32, 0.2, spread=1.0)
    e = 2.0 ** -5
    _, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
    dw = torch.zeros_like(c.w)
    dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, dw)
    d, dv = torch.randn_like(c.x), torch.randn_like(c.w) / 7
    for grad, way, u in ((dx, "x", d.double() @ c.w.double().T), (dw, "w", c.x.double() @ dv.double().T)):
        f, off = [], 0.0
        for sign in (1, -1):
            o = Case(24, 48, 90, F32, 0.2, spread=1.0)
            setattr(o, way, getattr(c, way) + sign * e * (d if way == "x" else dv))
            f.append((o.g.double() * pkg.linear_xent_forward(o.x, o.w, o.ids)[0].double()).sum())
            off = off + (o.g.double() * o.formulas()[5]).sum()
        slope = (f[0] - f[1]) / (2 * e)
        inner = (grad.double() * (d if way == "x" else dv).double()).sum()
        third = (c.g.double() * (2 * u.abs().amax(-1)) ** 3 / 4).sum()
        assert (slope - inner).abs() <= off / (2 * e) + e * e / 6 * third + 2.0 ** -14 * (grad.double() * (d if way == "x" else dv).double()).abs().sum()


def test_other_stream_and_graphs(pkg):
    for dtype in (BF16, F32):
        c = Case(700, 128, 3000, dtype)
        losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
        dw = c.dw.clone()
        dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse, dw)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        l2, e2 = pkg.linear_xent_forward(c.x, c.w, c.ids, stream=side)
        held = c.dw.clone()
        side.wait_stream(torch.cuda.current_stream())
        dx2 = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, e2, held, stream=side)
        side.synchronize()
        assert torch.equal(l2, losses) and torch.equal(dx2, dx) and torch.equal(held, dw)
        graphs, outs = [], []
        for _ in range(2):
            out = c.dw.clone()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
                l3, e3 = pkg.linear_xent_forward(c.x, c.w, c.ids)
                dx3 = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, e3, out)
            graphs.append(graph), outs.append((out, dx3))
        for graph, (out, dx3) in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, dw) and torch.equal(dx3, dx)
        c.x.copy_(torch.randn_like(c.x.float()).to(dtype))  # a new batch in the place of the captured one
        outs[0][0].copy_(c.dw)
        graphs[0].replay()
        dx = c.check(pkg)
        assert torch.equal(outs[0][1], dx) and torch.equal(outs[0][0], c.dw)


def test_two_streams_at_once(pkg):
    a, b = Case(900, 256, 4000, BF16, seed=1), Case(900, 256, 4000, F32, seed=2)
    want = []
    for c in (a, b):
        losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
        want.append((losses, pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for c, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
                got.append((losses, pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse)))
    torch.cuda.synchronize()
    for i, (losses, dx) in enumerate(got):
        assert torch.equal(losses, want[i % 2][0]) and torch.equal(dx, want[i % 2][1])
    assert pkg.device_status() == 0


def test_another_device(pkg):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    c = Case(100, 64, 300, BF16)
    losses, lse = pkg.linear_xent_forward(c.x, c.w, c.ids)
    dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, lse)
    far = [t.to("cuda:1") for t in (c.g, c.x, c.w, c.ids)]
    l2, e2 = pkg.linear_xent_forward(*far[1:])
    assert l2.device.index == 1 and torch.equal(l2.cpu(), losses.cpu()) and torch.equal(pkg.linear_xent_backward(*far, e2).cpu(), dx.cpu())


def test_refusals(pkg):
    x, w, t = torch.zeros(4, 8, device="cuda"), torch.zeros(9, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for wrong in (dict(x=x.half()), dict(x=x.bfloat16()), dict(x=x.double()), dict(x=x.T), dict(x=x[:, ::2]), dict(w=w[:, :4]), dict(w=w[:0]), dict(w=w.cpu()), dict(w=w[None]),
                  dict(targets=t[:3]), dict(targets=t.to(torch.int16)), dict(targets=t.cpu()), dict(targets=t.view(2, 2)), dict(x=x.expand(2, 4, 8)[:, :2])):
        with pytest.raises(ValueError):
            pkg.linear_xent_forward(**{**dict(x=x, w=w, targets=t), **wrong})
    one = torch.ones(1, device="cuda")
    for wrong in (dict(g=one.expand(3)), dict(g=torch.ones(2, device="cuda")), dict(g=one.double()), dict(lse=one), dict(dw=w[:8]), dict(dw=w.bfloat16()), dict(want_dx=False),
                  dict(dw=w.T.contiguous().T)):
        with pytest.raises(ValueError):
            pkg.linear_xent_backward(**{**dict(g=one, x=x, w=w, targets=t, lse=torch.zeros(4, device="cuda")), **wrong})


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,V", [(9, 1600, 9000), (40, 1600, 9000), (200, 2560, 3000)])
def test_logits_are_not_too_small(pkg, dtype, M, K, V):
    """The tensor cores cut every sum off, on average 0.28 2^-24 of it for each step of 16 products.  What is left of that is far less: a third would be the sign of
    a way that does not make up for it."""
    c = Case(M, K, V, dtype, 0.0, spread=20.0)
    z = c.x.double() @ c.w.double().T
    want = torch.logsumexp(z, -1)
    t = z.argmin(-1)
    losses, lse = pkg.linear_xent_forward(c.x, c.w, t)
    steps = K // 16 * (3 if dtype == F32 else 1)
    # the mean over the rows of roundings (2^-24 of a value each, and 2^-17 of a logit's terms, as many of either sign) is less than half of the limit
    limit = 0.28 / 3 * steps * 2.0 ** -24 + (2.0 ** -22 if dtype == F32 else 2.0 ** -23)
    at = z.gather(1, t[:, None])[:, 0]
    assert abs(((lse.double() - want) / want).mean()) < limit and abs(((lse.double() - losses.double() - at) / at).mean()) < limit


def test_fp32_gradients_are_not_too_small(pkg):
    """Segments of 192 steps take 0.25 2^-24 of a sum a step: 2.9e-6."""
    c = Case(2048, 64, 9000, F32, 0.0)
    z = c.x.double() @ c.w.double().T
    G = torch.softmax(z, -1)
    G[torch.arange(c.M), c.t] -= 1
    G *= c.g.double()[:, None]
    c.dw.zero_()
    dx = pkg.linear_xent_backward(c.g, c.x, c.w, c.ids, pkg.linear_xent_forward(c.x, c.w, c.ids)[1], c.dw)
    for got, want in ((dx, G @ c.w.double()), (c.dw, G.T @ c.x.double())):
        assert abs((got.double() * want).sum() / (want * want).sum() - 1) < 1.2e-6
