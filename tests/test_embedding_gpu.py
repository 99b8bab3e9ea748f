"""Embedding and the gradients of its tables against sums in 64 bits.

Tolerances.  Lookup: scale * row + position is one fused multiply-add, off by half a unit of fp32, and of the result's type.  Gradient: m
terms added in fp32, in whatever order, are off by at most (m + 8) 2^-24 of the sum of their sizes; then one multiply-add and one rounding.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
IDS = [torch.int64, torch.int32, torch.float32]


def half(t):
    return torch.finfo(t).eps / 2


class Batch:
    def __init__(self, shape, C, V, P, dtype=F32, grad=F32, ids=torch.int64, positions="rows", pad=0.0, out=0.0, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
        normal = lambda *s: torch.empty(*s, device="cuda").normal_(0.0, 1.0, generator=g)  # noqa: E731
        tokens = torch.randint(V, shape, device="cuda", generator=g)
        tokens = torch.where(rand(*shape) < pad, torch.full_like(tokens, V // 2), tokens)
        wrong = torch.where(rand(*shape) < 0.5, torch.full_like(tokens, -1), torch.full_like(tokens, V))
        self.tokens = torch.where(rand(*shape) < out, wrong, tokens)
        self.place = torch.arange(shape[-1], device="cuda").expand(shape)
        self.given = None
        if positions == "given":
            self.place = torch.randint(-1, P + 1, shape, device="cuda", generator=g)
            self.given = self.place.to(ids)
        self.table, self.dtable, self.dy = normal(V, C).to(dtype), normal(V, C).to(grad), normal(*shape, C).to(dtype)
        self.pos_table = self.dpos_table = None
        if positions:
            self.pos_table, self.dpos_table = normal(P, C).to(dtype), normal(P, C).to(grad)
        self.ids, self.V, self.P, self.C, self.dtype, self.grad = self.tokens.to(ids), V, P, C, dtype, grad

    def forward(self, pkg, scale, **more):
        return pkg.embedding_forward(self.ids, self.table, positions=self.given, pos_table=self.pos_table, scale=scale, **more)

    def check_forward(self, pkg, scale=1.0, **more):
        y = self.forward(pkg, scale, **more)
        by = torch.tensor(scale, dtype=F32).double().item()
        inside = ((self.tokens >= 0) & (self.tokens < self.V)).double()[..., None]
        want = self.table.double()[self.tokens.clamp(0, self.V - 1)] * by * inside
        if self.pos_table is not None:
            there = ((self.place >= 0) & (self.place < self.P)).double()[..., None]
            want = want + self.pos_table.double()[self.place.clamp(0, self.P - 1)] * there
        assert y.shape == want.shape and y.dtype == self.dtype
        assert ((y.double() - want).abs() <= (half(self.dtype) + half(F32) * (self.dtype != F32)) * (1 + 2.0 ** -20) * want.abs()).all()

    def expected(self, held, index, rows, scale):
        index, d = index.reshape(-1), self.dy.double().view(-1, self.C)
        ok = (index >= 0) & (index < rows)
        index, d = index[ok], d[ok]
        by = torch.tensor(scale, dtype=F32).double().item()
        zeros = torch.zeros(rows, self.C, dtype=torch.float64, device="cuda")
        total, size = zeros.index_add(0, index, d), zeros.index_add(0, index, d.abs())
        count = torch.bincount(index, minlength=rows).double()[:, None]
        want = held.double() + by * total
        tol = abs(by) * size * (count + 8) * 2.0 ** -24 + want.abs() * (half(F32) + half(self.grad) * (self.grad != F32)) * (1 + 2.0 ** -7) + 1e-40
        return want, torch.where(count > 0, tol, 0.0)

    def check_backward(self, pkg, scale=1.0, **more):
        want = self.expected(self.dtable, self.tokens, self.V, scale)
        want_pos = self.dpos_table is not None and self.expected(self.dpos_table, self.place, self.P, 1.0)
        again = [None if t is None else t.clone() for t in (self.dtable, self.dpos_table)]
        pkg.embedding_backward(self.dy, self.ids, self.dtable, positions=self.given, dpos_table=self.dpos_table, scale=scale, **more)
        assert ((self.dtable.double() - want[0]).abs() <= want[1]).all()
        if want_pos:
            assert ((self.dpos_table.double() - want_pos[0]).abs() <= want_pos[1]).all()
        pkg.embedding_backward(self.dy, self.ids, again[0], positions=self.given, dpos_table=again[1], scale=scale)
        assert torch.equal(again[0], self.dtable) and (again[1] is None or torch.equal(again[1], self.dpos_table))
        assert pkg.device_status() == 0


SHAPES = [((1,), 8, 5, 3), ((1, 1), 1, 1, 1), ((3, 7), 12, 5, 9), ((130,), 768, 50257, 1024), ((2, 129), 200, 40, 130), ((5, 33), 37, 1000, 20), ((8, 1000), 64, 50257, 1024),
          ((2, 3, 50), 96, 511, 50), ((1, 2049), 4, 512, 4000), ((40, 1), 1600, 513, 1)]


@pytest.mark.parametrize("dtype,grad", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("shape,C,V,P", SHAPES)
def test_shapes_and_types(pkg, shape, C, V, P, dtype, grad):
    for i, (positions, pad, out) in enumerate([("rows", 0.0, 0.0), (None, 0.5, 0.2), ("given", 0.9, 0.1)]):
        b = Batch(shape, C, V, P, dtype, grad, IDS[i], positions, pad, out, seed=i)
        b.check_forward(pkg, scale=[1.0, 3.5, -0.1][i])
        b.check_backward(pkg, scale=[1.0, 3.5, -0.1][i])


@pytest.mark.parametrize("n,V", [(1, 1), (7, 2), (31, 3), (4, 1 << 20), (1000, 1), (2047, 70000), (2049, 255), (16385, 256), (40000, 65536), (66000, 300000), (70000, 1), (150000, 128), (150000, 1 << 17)])
def test_runs_of_equal_tokens(pkg, n, V):
    """Lists on both sides of where ranges change their length, buckets that are compared, that take one pass and two, runs over many ranges."""
    for pad in (0.0, 0.7):
        Batch((n,), 8, V, 1, pad=pad, positions=None, out=0.05, seed=n).check_backward(pkg, 2.0)


def test_tokens_all_outside(pkg):
    b = Batch((3, 50), 16, 10, 50, out=1.0)
    held = b.dtable.clone()
    b.check_forward(pkg)
    b.check_backward(pkg)
    assert torch.equal(b.dtable, held)
    y = pkg.embedding_forward(b.ids, b.table)
    assert (y == 0).all()


def test_one_token_everywhere(pkg):
    b = Batch((6, 1000), 40, 30, 1000, pad=1.0)
    b.check_backward(pkg)


def test_what_no_token_names_is_left_alone(pkg):
    """Not even read: other rows may hold what a sum would carry along."""
    b = Batch((4, 100), 64, 1000, 200, positions="rows")
    b.dtable[700:] = float("nan")
    b.dpos_table[100:] = float("inf")
    b.tokens.clamp_(max=699)
    b.ids = b.tokens.clone()
    kept = b.dtable[700:].clone(), b.dpos_table[100:].clone()
    pkg.embedding_backward(b.dy, b.ids, b.dtable, dpos_table=b.dpos_table)
    assert b.dtable[:700].isfinite().all() and b.dpos_table[:100].isfinite().all()
    assert torch.equal(b.dtable[700:].isnan(), kept[0].isnan()) and torch.equal(b.dpos_table[100:], kept[1])


def test_nan_stays_in_its_row(pkg):
    b = Batch((2, 64), 32, 500, 64)
    b.tokens = torch.arange(128, device="cuda").view(2, 64)
    b.ids = b.tokens
    b.dy[0, 5, 3] = float("nan")
    pkg.embedding_backward(b.dy, b.ids, b.dtable, dpos_table=b.dpos_table)
    assert b.dtable.isnan().nonzero().tolist() == [[5, 3]] and b.dpos_table.isnan().nonzero().tolist() == [[5, 3]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("apart,start", [(64, 0), (72, 8), (67, 1), (65, 0), (68, 2)])
def test_rows_that_lie_apart(pkg, dtype, apart, start):
    """Views of wider tensors, on any boundary; what stands between the rows stays."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    wide = lambda n: torch.empty(n, apart + 8, device="cuda").normal_(0.0, 1.0, generator=g).to(dtype)  # noqa: E731
    b = Batch((3, 41), 60, 70, 41, dtype, dtype)
    held = {k: wide(n) for k, n in (("table", 70), ("pos_table", 41), ("dtable", 70), ("dpos_table", 41), ("dy", 123))}
    before = {k: v.clone() for k, v in held.items()}
    for k, v in held.items():
        setattr(b, k, v[:, start:start + 60])
    b.tokens, b.ids, b.given, b.place = b.tokens.view(-1), b.ids.view(-1), b.place.reshape(-1).contiguous(), b.place.reshape(-1)
    b.check_forward(pkg, 1.5)
    want, want_pos = b.expected(b.dtable, b.tokens, 70, 1.5), b.expected(b.dpos_table, b.place, 41, 1.0)
    pkg.embedding_backward(b.dy, b.ids, b.dtable, positions=b.given, dpos_table=b.dpos_table, scale=1.5)
    assert ((b.dtable.double() - want[0]).abs() <= want[1]).all() and ((b.dpos_table.double() - want_pos[0]).abs() <= want_pos[1]).all()
    for k in ("dtable", "dpos_table"):
        assert torch.equal(held[k][:, :start], before[k][:, :start]) and torch.equal(held[k][:, start + 60:], before[k][:, start + 60:])


def test_position_alone_and_table_alone(pkg):
    b = Batch((4, 30), 24, 9, 40, positions="given")
    want, want_pos = b.expected(b.dtable, b.tokens, 9, 1.0), b.expected(b.dpos_table, b.place, 40, 1.0)
    pkg.embedding_backward(b.dy, b.ids, b.dtable)
    pkg.embedding_backward(b.dy, b.ids, None, positions=b.given, dpos_table=b.dpos_table)
    assert ((b.dtable.double() - want[0]).abs() <= want[1]).all() and ((b.dpos_table.double() - want_pos[0]).abs() <= want_pos[1]).all()
    c = Batch((4, 30), 24, 9, 25, positions="rows")  # the last positions have no row
    want_pos = c.expected(c.dpos_table, c.place, 25, 1.0)
    pkg.embedding_backward(c.dy, c.ids, None, dpos_table=c.dpos_table)
    assert ((c.dpos_table.double() - want_pos[0]).abs() <= want_pos[1]).all()


def test_no_tokens(pkg):
    b = Batch((0, 5), 8, 9, 5)
    held = b.dtable.clone()
    assert b.forward(pkg, 1.0).shape == (0, 5, 8)
    pkg.embedding_backward(b.dy, b.ids, b.dtable, dpos_table=b.dpos_table)
    torch.cuda.synchronize()
    assert torch.equal(b.dtable, held)


def test_gradient_against_differences(pkg):
    """<dy, y(table + d) - y(table)> is <dtable, d>: the lookup is linear in its tables, so this is off by roundings alone: 2^-22 of the sizes."""
    b = Batch((3, 20), 16, 7, 20)
    b.dtable.zero_(), b.dpos_table.zero_()
    pkg.embedding_backward(b.dy, b.ids, b.dtable, dpos_table=b.dpos_table, scale=2.5)
    d, dp = torch.randn_like(b.table), torch.randn_like(b.pos_table)
    y0 = b.forward(pkg, 2.5).double()
    b.table, b.pos_table = b.table + d, b.pos_table + dp
    y1 = b.forward(pkg, 2.5).double()
    left, right = (b.dy.double() * (y1 - y0)).sum(), (b.dtable.double() * d.double()).sum() + (b.dpos_table.double() * dp.double()).sum()
    sizes = (b.dy.double().abs() * (y1.abs() + y0.abs())).sum()
    assert (left - right).abs() <= 2.0 ** -21 * sizes


def test_other_stream_and_graph(pkg):
    b = Batch((8, 300), 128, 5000, 300, pad=0.3)
    want, want_pos = b.dtable.clone(), b.dpos_table.clone()
    y = b.forward(pkg, 1.0)
    pkg.embedding_backward(b.dy, b.ids, want, dpos_table=want_pos)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    held = b.dtable.clone(), b.dpos_table.clone()
    side.wait_stream(torch.cuda.current_stream())
    y2 = b.forward(pkg, 1.0, stream=side)
    pkg.embedding_backward(b.dy, b.ids, held[0], dpos_table=held[1], stream=side)
    side.synchronize()
    assert torch.equal(y2, y) and torch.equal(held[0], want) and torch.equal(held[1], want_pos)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same pool, replayed one behind the other
        graph, out = torch.cuda.CUDAGraph(), (b.dtable.clone(), b.dpos_table.clone())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            y3 = b.forward(pkg, 1.0)
            pkg.embedding_backward(b.dy, b.ids, out[0], dpos_table=out[1])
        graphs.append(graph), outs.append((y3, *out))
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[1], want) and torch.equal(o[2], want_pos)
    assert torch.equal(outs[1][0], y)
    b.tokens = torch.randint(5000, (8, 300), device="cuda")  # new tokens in the place of the captured ones
    b.ids.copy_(b.tokens)
    for o in outs:
        o[1].copy_(b.dtable), o[2].copy_(b.dpos_table)
    graphs[0].replay()
    b.check_backward(pkg)
    assert torch.equal(outs[0][1], b.dtable)


def test_another_device(pkg):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    b = Batch((2, 30), 16, 9, 30)
    for name in ("tokens", "ids", "place", "table", "pos_table", "dy", "dtable", "dpos_table"):
        setattr(b, name, getattr(b, name).to("cuda:1"))
    y = b.forward(pkg, 1.0)
    assert y.device.index == 1 and torch.equal(y, b.table[b.tokens] + b.pos_table[b.place])


def test_refusals(pkg):
    t, x = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, 8, device="cuda")
    for wrong in (dict(tokens=t.to(torch.int16)), dict(table=x.half()), dict(table=x[None]), dict(table=x.T), dict(pos_table=x[:, :4]), dict(pos_table=x.bfloat16()),
                  dict(positions=t), dict(positions=t[:2], pos_table=x), dict(positions=t.int(), pos_table=x), dict(table=x[:0]), dict(table=x.cpu()),
                  dict(tokens=torch.zeros(8, dtype=torch.int64, device="cuda")[::2])):
        with pytest.raises(ValueError):
            pkg.embedding_forward(**{**dict(tokens=t, table=x), **wrong})
    for wrong in (dict(dy=x[:3]), dict(dy=x.half()), dict(dy=x.T), dict(dtable=x[:, :4]), dict(dtable=None), dict(dpos_table=x.bfloat16()), dict(positions=t), dict(tokens=t.cpu()),
                  dict(dtable=x.expand(4, 8)[:1].expand(4, 8))):
        with pytest.raises(ValueError):
            pkg.embedding_backward(**{**dict(dy=x, tokens=t, dtable=torch.zeros_like(x)), **wrong})
    same = torch.zeros(8, 8, device="cuda")
    for wrong in (dict(dtable=same, dpos_table=same), dict(dtable=same, dpos_table=same[2:]), dict(dtable=x)):
        with pytest.raises(pkg.AttnError):
            pkg.embedding_backward(**{**dict(dy=x, tokens=t), **wrong})
