"""Gradients of embedding tables where the plan changes: the longest tables.

Values are whole numbers whose sums, and the steps to them, fp32 holds, and bf16 as well: results have to be equal.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("grad", [BF16, F32])
@pytest.mark.parametrize("rows", [1 << 30, (1 << 30) - 1])
def test_as_many_rows_as_there_may_be(pkg, rows, grad):
    """Places without a token between those of token 0, whose digits above the bucket's wrap to the same number where that has too few bits."""
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
