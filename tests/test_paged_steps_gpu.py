"""Steps as a serving program makes them: page tables with room for the longest context there may be, and single tokens
beside pieces of prompts where that takes two launches, one behind the other."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def widen(st, positions):
    """The same step with a table for contexts of `positions`; what stands behind a sequence's last page is not read."""
    room = torch.full((st.table.shape[0], -(-positions // st.P)), 1 << 30, dtype=torch.int32, device="cuda")
    room[:, :st.table.shape[1]] = st.table
    st.table = room
    return st


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("positions", [2049, 8193, 32768, 131072])
@pytest.mark.parametrize("new,past,heads,kv,D", [([1] * 110, [(i * 37) % 700 for i in range(110)], 12, 12, 64), ([1] * 3, [0, 600, 31], 2, 2, 128), ([1, 2, 0, 1], [700, 3, 50, 64], 8, 2, 64),
                                                 ([1] * 10 + [200], [80 * i for i in range(11)], 4, 1, 128), ([300, 20], [600, 64], 3, 3, 64), ([1, 3], [900, 5], 2, 1, 136)])
def test_tables_wider_than_the_contexts(pkg, new, past, heads, kv, D, positions, dtype):
    from test_paged_gpu import Step

    st = widen(Step(new, past, heads, kv, D, 16, dtype), positions)
    st.fill()
    st.check(pkg, max_new=max(new))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("seqs,positions", [(40, 0), (20, 8200)])  # more units than the tile kernel takes in about two rounds, or room for long contexts
def test_single_tokens_and_pieces_in_two_launches(pkg, seqs, positions, dtype):
    """The kernels behind them may start early, and do so again and again: every result is that of the first call."""
    from test_paged_gpu import Step

    st = Step([1] * seqs + [200, 300], [(i * 61) % 700 for i in range(seqs + 2)], 12, 12, 64, 16, dtype)
    if positions:
        widen(st, positions)
    st.fill()
    q = st.normal(st.tokens, 768)
    out = st.check(pkg, q, max_new=300)
    n = st.starts[-1]
    weights = st.normal(64, 768)
    torch.cuda.synchronize()
    want = pkg.linear_forward(out[:n].contiguous(), weights)
    torch.cuda.synchronize()
    for i in range(30):
        buf = torch.full_like(out, float(i))
        assert torch.equal(pkg.linear_forward(pkg.paged_attention(q, *st.args(), max_new=300, out=buf)[:n], weights), want)
    # appends in front of them, over and over on one cache
    qkv = st.normal(st.tokens, 3 * 768)
    pkg.paged_append(qkv, *st.args())
    torch.cuda.synchronize()
    want = pkg.paged_attention(qkv[:, :768], *st.args(), max_new=300).clone()
    torch.cuda.synchronize()
    for i in range(20):
        other = qkv + 1.0 + i
        pkg.paged_attention(pkg.paged_append(other, *st.args()), *st.args(), max_new=300)
        assert torch.equal(pkg.paged_attention(pkg.paged_append(qkv, *st.args()), *st.args(), max_new=300)[:n], want[:n])
    assert pkg.device_status() == 0
