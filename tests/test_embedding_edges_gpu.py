"""Gradients of embedding tables at the ends of what the calls allow: the longest tables, the shortest sequences."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("grad", [BF16, F32])
@pytest.mark.parametrize("rows", [1 << 30, (1 << 30) - 1])
def test_as_many_rows_as_there_may_be(pkg, rows, grad):
    """Whole numbers, whose sums fp32 and bf16 hold.  Places without a token stand between those of token 0, whose digits above
    the bucket's wrap to the same number where that has too few bits."""
    n = 1000  # of which 320 have the lowest digits of token 0 or none: few enough to be compared each with each
    tokens = torch.full((n,), 5, device="cuda")
    tokens[::5], tokens[2::10], tokens[1::50], tokens[3::50] = 0, -1, rows - 1, 128
    dy = torch.ones(n, 1, device="cuda", dtype=grad)
    for positions in (False, True):
        table = torch.zeros(rows, 1, device="cuda", dtype=grad)
        if positions:
            pkg.embedding_backward(dy, tokens, None, positions=tokens, dpos_table=table)
        else:
            pkg.embedding_backward(dy, tokens, table)
        got = {i: table[i].item() for i in (0, 1, 5, 128, rows - 1)}
        table[[0, 5, 128, rows - 1]] = 0
        assert got == {0: 200.0, 1: 0.0, 5: 660.0, 128: 20.0, rows - 1: 20.0} and not table.any() and pkg.device_status() == 0
        del table


@pytest.mark.parametrize("dtype,grad", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("n,T,C", [(1 << 20, 1, 8), (1 << 20, 3, 40), (1 << 18, 16, 768), (70001, 1, 37), (70001, 2, 264), (8192, 1, 768), (8191, 8, 65), (5000, 1, 1), (512, 1, 768), (511, 7, 72)])
def test_many_short_sequences(pkg, n, T, C, dtype, grad):
    """A row of the position table gets a term from each of n / T sequences, nearly all of one size here, so that a sum of one behind the other would be cut off again and again.  Terms are
    added eight at a time, those by threads that have at most a 64th of the sequences each, and theirs in pairs: (8 + sequences / 512 + 10) roundings, and 8 of the last steps."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n + T)
    n -= n % T
    dy = (0.1 + 1e-3 * torch.rand(n // T, T, C, device="cuda", generator=g)).to(dtype)
    held = (torch.randn(T + 1, C, device="cuda", generator=g)).to(grad)
    dpos, both = held.clone(), held.clone()
    tokens = torch.randint(50, (n // T, T), device="cuda", generator=g)
    pkg.embedding_backward(dy, tokens, None, dpos_table=dpos)
    pkg.embedding_backward(dy, tokens, torch.zeros(50, C, device="cuda", dtype=grad), dpos_table=both)
    want = held.double()
    want[:T] += dy.double().sum(0)
    size = torch.zeros_like(want)
    size[:T] = dy.double().sum(0)
    half = torch.finfo(grad).eps / 2 * (grad == BF16) * (1 + 2.0 ** -7)
    assert ((dpos.double() - want).abs() <= size * (n // T / 512 + 26) * 2.0 ** -24 + want.abs() * (half + 2.0 ** -24)).all()
    assert torch.equal(dpos, both) and torch.equal(dpos[T:], held[T:]) and pkg.device_status() == 0
