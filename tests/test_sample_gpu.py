"""The draw of a class from rows of logits (xent_sm100_sample) against the definition in 64 bits.

The classes are whole numbers and have to be equal.  The kernel's weights are rounded to 2^-44 of the largest, those here to 2^-53 of
themselves, so a draw whose border lies within C 2^-44 of u may differ: with C = 50257 classes that is one row in about 10^5 at worst
(2 C borders of that width, over a sum of at least 1), and the rows below are seeded.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def plain(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, in 64 bits on the host."""
    x = x.double().cpu()
    if bool(x.isnan().any()) or bool((x == -INF).all()):
        return -1
    if not temperature > 0:
        return int((x == x.max()).nonzero()[0])
    w = torch.where(x == x.max(), 1.0, ((x - x.max()) / temperature).exp().nan_to_num(0.0))
    w[x == -INF] = 0.0
    order = torch.sort(x, descending=True, stable=True).indices
    z = w[order]
    n = top_k if 1 <= top_k < len(x) else len(x)
    if top_p < 1.0:
        before = z[:n].cumsum(0) - z[:n]
        n = max(1, int((before < top_p * z[:n].sum()).sum()))
    kept = torch.zeros_like(w)
    kept[order[:n]] = 1.0
    if min_p > 0:
        kept[w < min(min_p, 1.0)] = 0.0
    total = (w * kept).cumsum(0)
    u = min(max(u, 0.0), 1 - 2.0 ** -53)
    return int((total > u * total[-1]).nonzero()[0])


def check(pkg, x, u, temperature=None, top_k=None, top_p=None, min_p=None, **more):
    rows = x.shape[0]
    column = lambda v, t: None if v is None else torch.tensor(v if isinstance(v, list) else [v] * rows, dtype=t, device="cuda")  # noqa: E731
    args = [column(temperature, torch.float32), column(top_k, torch.int32), column(top_p, torch.float32), column(min_p, torch.float32)]
    got = pkg.sample(x, u, *args, **more)
    assert got.dtype == torch.int32 and got.shape == (rows,)
    host = [None if a is None else a.cpu() for a in args]
    names = ("temperature", "top_k", "top_p", "min_p")
    want = [plain(x[r], u[r].item(), **{n: a[r].item() for n, a in zip(names, host) if a is not None}) for r in range(rows)]
    assert got.tolist() == want
    assert pkg.device_status() == 0
    return got


def rows_of(rows, C, spread=2.5, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + C)
    return torch.empty(rows, C, device="cuda").normal_(0.0, spread, generator=g), torch.rand(rows, device="cuda", generator=g)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=100, top_p=0.95, min_p=0.01),
            dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0), dict(top_k=7, top_p=0.3), dict(temperature=0.05, top_p=0.999),
            dict(temperature=50.0, top_p=0.8), dict(top_k=3000, min_p=0.002)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 2), (2, 33), (5, 1000), (3, 1025), (9, 50257), (2, 128256)])
def test_against_the_definition(pkg, rows, C, settings):
    check(pkg, *rows_of(rows, C), **settings)


@pytest.mark.parametrize("rows", [1, 2, 20, 40, 80, 150, 300, 700])
def test_every_number_of_rows(pkg, rows):
    """Settings of their own in each row."""
    x, u = rows_of(rows, 3001, 2.0, rows)
    r = range(rows)
    check(pkg, x, u, [0.0 if i % 7 == 3 else 0.5 + i % 5 * 0.3 for i in r], [[0, 1, 5, 300, 3000, 3001, 9999, -4][i % 8] for i in r],
          [[1.0, 0.9, 0.5, 2.0, 0.0, -1.0][i % 6] for i in r], [[0.0, 0.1, 0.001, -1.0, 0.9][i % 5] for i in r])


@pytest.mark.parametrize("C", [425984, 300001, 65536])
def test_longest_rows(pkg, C):
    check(pkg, *rows_of(2, C), temperature=0.9, top_k=50000, top_p=0.97)
    check(pkg, *rows_of(2, C, 1.0), top_p=0.5)


@pytest.mark.parametrize("C", [10, 4096, 50257])
@pytest.mark.parametrize("kinds", [1, 2, 9])
def test_ties(pkg, C, kinds):
    """Few different logits: which of the equal ones are kept goes by the index."""
    x, u = rows_of(8, C)
    x = (x.abs() * 10).long().remainder(kinds).float() / 4
    for settings in (dict(), dict(top_k=5), dict(top_k=C // 2), dict(top_k=C - 1), dict(top_p=0.5), dict(top_p=0.3, top_k=C // 3 + 1), dict(min_p=0.9), dict(temperature=0.0),
                     dict(top_p=0.75, min_p=0.8)):
        check(pkg, x, u, **settings)
    x[:, ::2] *= -1  # -0 and 0 are one value
    x[x == 0] *= -1
    check(pkg, x, u, top_k=max(1, C // 4))


def test_borders(pkg):
    """u on and next to the borders between classes of equal weight, where every number is exact."""
    x = torch.zeros(9, 8, device="cuda")
    u = torch.tensor([0.0, 0.125, 0.125 - 2.0 ** -26, 0.5, 0.5 - 2.0 ** -25, 0.875, 1 - 2.0 ** -24, 1.0, -3.0], device="cuda")
    assert check(pkg, x, u).tolist() == [0, 1, 0, 4, 3, 7, 7, 7, 0]
    assert check(pkg, x, u, top_p=0.5).tolist() == [0, 0, 0, 2, 1, 3, 3, 3, 0]
    assert check(pkg, x, u, top_k=6).tolist() == [0, 0, 0, 3, 2, 5, 5, 5, 0]
    assert pkg.sample(x[:1], torch.full((1,), NAN, device="cuda")).item() == 0


@pytest.mark.parametrize("C", [5, 1500, 50257])
def test_infinities_and_nan(pkg, C):
    """-inf has no weight, +inf all of it; a row with a NaN or of -inf alone draws nothing, and keeps that to itself."""
    x, u = rows_of(13, C)
    x[12, : C // 2] = torch.finfo(torch.float32).min
    x[0, : C - 2] = -INF
    x[1] = -INF
    x[2, C // 2] = NAN
    x[3, 0], x[4, C - 1] = INF, INF
    x[5, 1] = x[5, 3] = INF
    x[6, 1:] = -INF
    x[7, 0], x[7, 1] = NAN, INF
    x[8, 2:] = -1e30
    x[9] = -3e38
    x[9, 4] = 3e38
    x[10, : C - 1] = -INF
    x[11] = torch.finfo(torch.float32).min
    for settings in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_k=C - 1, top_p=0.9), dict(top_k=3), dict(top_k=C // 2 + 1), dict(min_p=0.5), dict(temperature=1e-30), dict(temperature=1e30),
                     dict(temperature=INF), dict(temperature=INF, top_p=0.5), dict(temperature=NAN), dict(top_p=NAN), dict(min_p=NAN), dict(top_p=1e-38)):
        if settings.get("temperature") == INF:  # infinite logits over an infinite temperature
            keep = [r for r in range(13) if r not in (3, 4, 5, 7)]
            check(pkg, x[keep], u[keep], **settings)
        else:
            check(pkg, x, u, **settings)


def test_far_outliers(pkg):
    """Logits that a bias has put far below or above the others."""
    x, u = rows_of(6, 50257)
    x[:, 1000:30000] -= 1e9
    x[2:4, 100] += 1e4
    x[4:, :40000] = -65504.0
    for settings in (dict(), dict(top_k=50), dict(top_k=25000), dict(top_k=45000), dict(top_p=0.9), dict(temperature=1e8, top_p=0.7), dict(temperature=1e5, top_k=30000)):
        check(pkg, x, u, **settings)


def test_rows_that_lie_apart(pkg):
    """The last token's logits of each sequence, as a view; rows on odd addresses."""
    x, _ = rows_of(12, 5003)
    u = torch.rand(4, device="cuda")
    check(pkg, x.view(4, 3, 5003)[:, -1], u, top_k=9, temperature=0.8)
    check(pkg, x[:4, 3:5000], u, top_p=0.9)
    check(pkg, x[:4, 1:2], u, top_p=0.9)


def test_streams_graphs_and_the_same_answer(pkg):
    x, u = rows_of(30, 50257)
    want = check(pkg, x, u, top_p=0.9, temperature=0.8)
    t, p = torch.full((30,), 0.8, device="cuda"), torch.full((30,), 0.9, device="cuda")
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [pkg.sample(x, u, t, None, p, None, stream=other if i % 2 else None) for i in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.sample(x, u, t, None, p, None)
    x2, u2 = rows_of(30, 50257, seed=9)
    x.copy_(x2), u.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, check(pkg, x2, u2, top_p=0.9, temperature=0.8))


def test_refusals(pkg):
    x, u = rows_of(4, 50)
    one = torch.ones(4, device="cuda")
    for args in ((x.double(), u), (x[0], u), (x.cpu(), u), (x.t(), u), (x, u[:3]), (x, u.double()), (x, u.cpu()), (x, u, one.double()), (x, u, one[:2]), (x, u, None, one),
                 (x, u, None, one.long()), (x, u, None, None, one.view(4, 1)), (x, u, None, None, None, one.cpu()), (x[:, :0], u), (x[:, ::2], u)):
        with pytest.raises(ValueError):
            pkg.sample(*args)
    assert pkg.sample(x[:0], u[:0]).shape == (0,)
    with pytest.raises(pkg.AttnError):
        pkg.sample(torch.zeros(1, 425985, device="cuda"), u[:1])
