"""That the attention over a paged cache takes its operands in full: queries and weights with 24 bits, keys and values of fp32 pages too.
The bound of test_paged_gpu.py holds for the worst sum of roundings and is some hundred times what they come to, so it says
nothing about a term of eight bits that is lost; the norm of the error does.

With e = 2^-24 and entries of variance one, roundings to nearest as independent errors of at most e relative, e / sqrt(3) on the root mean square:
  scores   D additions of partial sums that grow as sqrt(d / D) of a score's size: e sqrt(D / 6) at most where they run one behind the other,
           4.6 e at D = 128; the tensor cores add 16 products at a time, cutting off, (0.18 D / 16 + 0.5) e, 2 e at D = 128
  weights  the difference to the maximum, up to 10 of them, in 2^x: e log(2) 10 / sqrt(3) = 4 e; the exponential itself 2 e
  sums     over n keys, by 32 threads or in steps of 64 keys: e sqrt(n / 64 / 6), 1.6 e at n = 1000
  The squares of these add up to (6.7 e)^2 at most, relative to the output's norm, since errors of one key's weight do
  not know those of another's.  The limit is 16 e, 9.5e-7.
A term of eight bits that is missing leaves values too small by up to 2^-15 of them, 2^-17 on average (7.6e-6): of weights, keys and values that
is what the result is off by, of queries it is times the scores' size.  What that makes of the norm is tested here on the host.
"""
import pytest

torch = pytest.importorskip("torch")

E = 2.0 ** -24
LIMIT = 16 * E


def cut(x, terms):
    """The first `terms` pieces of eight bits of fp32 values, in 64 bits."""
    total, rest = torch.zeros_like(x, dtype=torch.float64), x.float()
    for _ in range(terms):
        piece = (rest.view(torch.int32) & -65536).view(torch.float32)
        total, rest = total + piece.double(), rest - piece
    return total


def off(got, want):
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize("D,n", [(64, 20), (64, 700), (128, 1000), (200, 300)])
def test_a_lost_term_shows(D, n):
    g = torch.Generator().manual_seed(D + n)
    q, k, v = (torch.randn(rows, D, generator=g) for rows in (64, n, n))
    x = q * (D ** -0.5 * 1.4426950408889634)
    want = torch.softmax(x.double() @ k.double().T * 0.6931471805599453, -1) @ v.double()

    def attention(tq=3, tp=3, tk=3, tv=3):
        z = cut(x, tq) @ cut(k, tk).T
        p = torch.exp2(z - z.amax(-1, keepdim=True)).float()
        return cut(p, tp) @ cut(v, tv) / p.double().sum(-1, keepdim=True)

    assert off(attention(), want) < LIMIT / 16
    for lost in ("tq", "tp", "tk", "tv"):
        assert off(attention(**{lost: 2}), want) > 2 * LIMIT, lost


# new tokens, positions before, query heads, key/value heads, head size, page size: both widths of the kernels for one, two, up to eight
# and many rows, by tensor maps and without, one CTA a unit and clusters
FORMS = [([1] * 3, [900, 30, 257], 2, 2, 64, 16), ([1] * 110, [i * 9 for i in range(110)], 12, 12, 64, 16), ([1] * 40, [i * 20 for i in range(40)], 12, 12, 128, 16),
         ([2, 2], [900, 31], 2, 2, 64, 16), ([1, 1], [500, 77], 4, 2, 128, 16), ([3], [800], 1, 1, 64, 16), ([4, 1], [700, 40], 2, 2, 64, 16), ([4], [600], 2, 1, 128, 16),
         ([8], [300], 1, 1, 40, 16), ([300], [700], 2, 2, 64, 16), ([300], [700], 2, 1, 64, 7), ([250, 40], [300, 900], 3, 1, 128, 16), ([250], [300], 2, 2, 96, 7),
         ([700], [300], 25, 25, 64, 16), ([1], [900], 2, 2, 200, 16), ([2, 2], [300, 40], 2, 2, 256, 16), ([30], [300], 2, 1, 136, 16), ([1], [60], 2, 2, 8, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads,kv,D,page", FORMS, ids=[f"{len(f[0])}x{max(f[0])}-{f[2]}over{f[3]}-D{f[4]}-page{f[5]}" for f in FORMS])
def test_no_term_is_lost(pkg, new, past, heads, kv, D, page, dtype):
    from test_paged_gpu import Step

    st = Step(new, past, heads, kv, D, page, dtype, seed=len(new) + D)
    st.fill()
    q = st.normal(st.tokens, heads * D)
    n = st.starts[-1]
    got = pkg.paged_attention(q, *st.args(), max_new=max(new))[:n].double()
    assert off(got, st.want(q)[0]) < LIMIT
    assert pkg.device_status() == 0
