"""What bf16 gradients of the projection with its loss are rounded to.

x and w have no feature in common, so every logit is 0, every probability 1 / V, a power of two that bf16 holds, and a target's entry, 1 / V - 1, becomes -1: G is off by
1 / V at the target and by nothing that matters elsewhere (exponentials are within 2^-18 of their power of two), if the factor of all rows is not rounded with it.  Weights come
in pairs +w, -w, rows of x too, so the gradients are -g w[target] and -g x, to which a call adds at most g / V of |w|, n / 16 + 20 steps of the tensor cores, each off by
2^-23 of the sum of sizes, 2^-20 for the factor's own products, and one rounding of the result: half a unit of its last place.  With -g rounded to bf16 first (g = 1 / 3001: 1.7e-3 off)
a third of the values are one unit off.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
G = 1.0 / 3001


def half_unit(want):
    return torch.ldexp(torch.ones_like(want), torch.frexp(want)[1] - 9)


class Case:
    def __init__(self, M, V, apart=64, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + M + V)

        def pairs(n):  # rows i and i + n / 2 are opposite, whole numbers of 64 to 127
            a = torch.randint(64, 128, (n // 2, 32), device="cuda", generator=g) * (2 * torch.randint(2, (n // 2, 32), device="cuda", generator=g) - 1)
            return torch.cat([a, -a]).to(BF16)

        def wide(n):
            return torch.zeros(n, apart, device="cuda", dtype=BF16)[:, :64]

        self.x, self.w, self.dw = wide(M), wide(V), wide(V)
        self.x[:, :32], self.w[:, 32:] = pairs(M), pairs(V)
        self.t = torch.randperm(V, device="cuda", generator=g).repeat(M // V + 1)[:M]
        gone = (torch.rand(M // 2, device="cuda", generator=g) < 0.3).repeat(2)
        self.t[gone] = -100
        self.ok = ~gone
        self.held = (torch.randn(V, 64, device="cuda", generator=g) * 0.05).to(BF16)
        self.M, self.V = M, V

    def run(self, pkg, g):
        self.dw.copy_(self.held)
        _, lse = pkg.linear_xent_forward(self.x, self.w, self.t)
        dx = pkg.linear_xent_backward(g, self.x, self.w, self.t, lse, self.dw)
        assert pkg.device_status() == 0
        return dx

    def check(self, pkg, g, dw=True):
        dx = self.run(pkg, g)
        by = torch.where(self.ok, g.double().expand(self.M), 0.0)[:, None]
        one = torch.zeros(self.M, self.V, device="cuda", dtype=torch.float64)
        one[self.ok, self.t[self.ok]] = 1.0
        p = torch.full_like(one, 1.0 / self.V)
        x, w = self.x.double(), self.w.double()
        for got, parts, before, n in ((dx, (by * (p - one), one * by.abs(), (p + one) * by.abs(), w), 0.0, self.V),
                                      (self.dw, ((by * (p - one)).T, (one * by.abs()).T, ((p + one) * by.abs()).T, x), self.held.double(), self.M)):
            exact, targets, sizes, other = parts
            if not dw and got is self.dw:
                continue
            want = before + exact @ other
            # what is rounded is want + e, |e| <= off: below |want| + off, whose unit is the larger one where a power of two lies between
            off = targets @ other.abs() / self.V + sizes @ other.abs() * (n // 16 + 20) * 2.0 ** -23 + want.abs() * 2.0 ** -20
            assert ((got.double() - want).abs() <= half_unit(want.abs() + off) + off).all()


@pytest.mark.parametrize("M,V,apart", [(6, 4096, 64), (10, 4096, 64), (40, 1024, 72), (300, 4096, 64), (6, 4096, 67), (300, 4096, 67), (1000, 2048, 64), (9000, 16384, 64)])
def test_a_factor_that_all_rows_share_is_not_rounded(pkg, M, V, apart):
    c = Case(M, V, apart)
    for g in (torch.tensor([G], device="cuda"), torch.tensor([-G * 2.0 ** 40], device="cuda"), torch.full((M,), G, device="cuda")):
        c.check(pkg, g)


@pytest.mark.parametrize("M", [20, 700])
def test_factors_that_differ_by_powers_of_two(pkg, M):
    """2^-100 to 2^20: none leaves the range that G has."""
    c = Case(M, 4096)
    k = torch.randint(-100, 21, (M,), device="cuda")
    c.check(pkg, torch.ldexp(torch.full((M,), G, device="cuda"), k), dw=False)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), 3e38])
def test_factors_of_rows_without_targets(pkg, value):
    c = Case(300, 4096)
    g = torch.where(c.ok, G, 0.0).float()
    dx, dw = c.run(pkg, g), c.dw.clone()
    assert torch.equal(c.run(pkg, torch.where(c.ok, g, value)), dx) and torch.equal(c.dw, dw)


def test_factors_that_are_no_normal_numbers(pkg):
    """0, infinity, NaN and less than 2^-126: as far as products of them go."""
    c = Case(100, 1024)
    for value in (0.0, 2.0 ** -130):
        dx = c.run(pkg, torch.tensor([value], device="cuda"))
        assert (dx.abs() <= value * 255).all() and torch.equal(c.dw, c.held)
    for value in (float("inf"), float("nan")):
        assert not c.run(pkg, torch.tensor([value], device="cuda"))[c.ok, 32:].isfinite().any()
