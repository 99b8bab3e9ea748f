"""The gradients of embedding tables at every way to the order of tokens and on both sides of its limits: 512 places (no list), 8192 (buckets, ranges of 8 places; above,
a cluster, 16), 16384 (32); with positions that are a token's place (added up beside the sort) or given (two lists), or alone; in all types, and rows that start anywhere.

Against sums in 64 bits, with the bounds of test_embedding_gpu.py: m terms added in fp32 are off by (m + 8) 2^-24 of the sum of their sizes, then one multiply-add and one rounding.
"""
import pytest

torch = pytest.importorskip("torch")

from test_embedding_gpu import Batch  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)]


def check(pkg, b, scale, table=True):
    if table:
        return b.check_backward(pkg, scale)
    want, tol = b.expected(b.dpos_table, b.place, b.P, 1.0)
    again = b.dpos_table.clone()
    pkg.embedding_backward(b.dy, b.ids, None, positions=b.given, dpos_table=b.dpos_table)
    assert ((b.dpos_table.double() - want).abs() <= tol).all() and pkg.device_status() == 0
    pkg.embedding_backward(b.dy, b.ids, None, positions=b.given, dpos_table=again)
    assert torch.equal(again, b.dpos_table)


@pytest.mark.parametrize("n", [512, 513, 8192, 8193, 12001, 16384, 16385, 70001])
@pytest.mark.parametrize("dtype,grad", TYPES)
@pytest.mark.parametrize("C", [48, 37])
def test_both_sides_of_every_limit(pkg, n, dtype, grad, C):
    for i, (positions, T, P, pad, table) in enumerate([(None, n, 1, 0.5, True), ("rows", n, n - 3, 0.3, True), ("given", n, 700, 0.6, True), ("rows", n, 3000, 0.0, False),
                                                       ("given", n, 40, 0.0, False)]):
        b = Batch((n,), C, 9000, P, dtype, grad, [torch.int64, torch.int32, torch.float32][(n + i) % 3], positions, pad, 0.05, seed=n + i)
        check(pkg, b, [1.0, -0.5, 3.0][i % 3], table)


@pytest.mark.parametrize("dtype,grad", TYPES)
@pytest.mark.parametrize("shape,C", [((9, 1000), 1600), ((16, 1024), 768), ((48, 1024), 264), ((24, 700), 1)])
def test_batches_of_sequences(pkg, shape, C, dtype, grad):
    for i, positions in enumerate(("rows", "given")):
        check(pkg, Batch(shape, C, 5001, shape[1], dtype, grad, positions=positions, pad=0.5, out=0.1, seed=i), 2.0)


@pytest.mark.parametrize("n", [8193, 16385])
def test_rows_that_lie_apart_in_long_lists(pkg, n):
    """Views of wider tensors; what stands between the rows stays."""
    for dtype, grad, start in ((BF16, BF16, 3), (F32, F32, 1), (BF16, F32, 8)):
        b = Batch((n,), 40, 300, 900, dtype, grad, positions="given", pad=0.2)
        held = {k: torch.full((getattr(b, k).shape[0], 61), 7.0, device="cuda", dtype=getattr(b, k).dtype) for k in ("dy", "dtable", "dpos_table")}
        for k, v in held.items():
            v[:, start:start + 40] = getattr(b, k)
            setattr(b, k, v[:, start:start + 40])
        want, want_pos = b.expected(b.dtable, b.tokens, 300, 1.5), b.expected(b.dpos_table, b.place, 900, 1.0)
        pkg.embedding_backward(b.dy, b.ids, b.dtable, positions=b.given, dpos_table=b.dpos_table, scale=1.5)
        assert ((b.dtable.double() - want[0]).abs() <= want[1]).all() and ((b.dpos_table.double() - want_pos[0]).abs() <= want_pos[1]).all()
        for k in ("dtable", "dpos_table"):
            assert (held[k][:, :start] == 7).all() and (held[k][:, start + 40:] == 7).all()


def test_captured_and_on_another_stream(pkg):
    """A list sorted by a cluster, replayed on new tokens, and with another call beside it."""
    b = Batch((20, 1000), 96, 4000, 1000, pad=0.4, seed=3)
    out = b.dtable.clone(), b.dpos_table.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.embedding_backward(b.dy, b.ids, out[0], dpos_table=out[1])
    for seed in (4, 5):
        c = Batch((20, 1000), 96, 4000, 1000, pad=0.7, seed=seed)
        b.ids.copy_(c.ids), b.dy.copy_(c.dy), out[0].copy_(c.dtable), out[1].copy_(c.dpos_table)
        other, side = c.dtable.clone(), torch.cuda.Stream()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            pkg.embedding_backward(c.dy, c.ids, other)
        torch.cuda.synchronize()
        c.check_backward(pkg)
        assert torch.equal(out[0], c.dtable) and torch.equal(out[1], c.dpos_table) and torch.equal(other, c.dtable)
