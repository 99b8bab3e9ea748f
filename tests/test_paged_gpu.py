"""The paged key/value cache and its attention (include/attn_sm100.h) against plain arithmetic in 64 bits.

Tolerances, with e = 2^-24 (half a step of fp32):
  stored values   fp32 as they came; bf16 rounded once, which torch's own conversion does too: equal bits
  rotated values  a cos - b sin in fp32, two products and a sum: 3 e (|a cos| + |b sin|), and half a step of bf16 (2^-8
                  relative) where pages are bf16
  attention       a score is a sum of D products, its relative error at most (D + 3) e of the sum of their sizes A; the weight
                  exp2(score - maximum) has besides the rounding of a difference (e times its size, which A bounds twice) and the error
                  of the exponential (4 e); numerator and sum each add up n such terms (n e), and what they are weighted with
                  is the size of the values: |error| <= 2 (A (D + 5) + n + 8) e sum_j p_j |v_j|
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Step:
    """A step's lengths over pages in no order; every row of the pages that no sequence has filled holds NaN."""

    def __init__(self, new, past, heads, kv, D, page, dtype, seed=0, spare=3, tail=2, interleaved=False):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.new, self.past, self.heads, self.kv, self.D, self.P = new, past, heads, kv, D, page
        need = [-(-(a + b) // page) for a, b in zip(new, past)]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(1, max(need))
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [1 << 30] * (width - n))  # entries behind the last position are not read
            at += n
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.starts, self.tokens = cu, cu[-1] + tail  # rows behind the last sequence
        self.table, self.cu, self.before = ints(rows), ints(cu), ints(past)
        shape = (self.pages, kv, page, D)
        if interleaved:  # keys and values of a page side by side
            both = torch.full((self.pages, 2, kv, page, D), float("nan"), device="cuda", dtype=TYPES[dtype])
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = (torch.full(shape, float("nan"), device="cuda", dtype=TYPES[dtype]) for _ in range(2))

    def normal(self, *shape):
        return torch.empty(shape, device="cuda").normal_(0.0, 1.0, generator=self.g)

    def args(self):
        return self.k, self.v, self.table, self.cu, self.before

    def where(self, s, p):
        return int(self.table[s, p // self.P]), p % self.P

    def fill(self, counts=None):
        """Keys and values of every position that the sequences hold (after the step)."""
        for s, n in enumerate(counts or [a + b for a, b in zip(self.new, self.past)]):
            p = torch.arange(n, device="cuda")
            page, row = self.table[s].long()[p // self.P], p % self.P
            for t in (self.k, self.v):
                t[page, :, row] = self.normal(n, self.kv, self.D).to(t.dtype)

    def context(self, s):
        """Keys and values of sequence s, [kv, positions, D] in 64 bits."""
        p = torch.arange(self.new[s] + self.past[s], device="cuda")
        page, row = self.table[s].long()[p // self.P], p % self.P
        return tuple(t[page, :, row].double().transpose(0, 1) for t in (self.k, self.v))

    def want(self, q, scale=None):
        """The attention of the new tokens and how far fp32 arithmetic may be from it, [tokens, heads * D] both."""
        scale = self.D ** -0.5 if scale is None else scale
        out, tol = torch.zeros(2, self.starts[-1], self.heads, self.D, device="cuda", dtype=torch.float64)
        G = self.heads // self.kv
        for s, n in enumerate(self.new):
            if not n:
                continue
            k, v = self.context(s)
            k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
            x = q[self.starts[s]:self.starts[s] + n].double().view(n, self.heads, self.D).transpose(0, 1)
            seen = torch.arange(k.shape[1], device="cuda") <= self.past[s] + torch.arange(n, device="cuda")[:, None]
            z = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
            size = (x.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(z.isneginf(), 0.0).amax(-1, keepdim=True)
            p = torch.softmax(z, -1)
            rows = slice(self.starts[s], self.starts[s] + n)
            out[rows] = (p @ v).transpose(0, 1)
            tol[rows] = (2 * (size * (self.D + 5) + k.shape[1] + 8) * E * (p @ v.abs())).transpose(0, 1)
        return out.flatten(1), tol.flatten(1)

    def check(self, pkg, q=None, scale=None, **more):
        q = self.normal(self.tokens, self.heads * self.D) if q is None else q
        out = torch.full((self.tokens, self.heads * self.D), 7.0, device="cuda")
        got = pkg.paged_attention(q, *self.args(), scale=scale, out=out, **more)
        assert got is out
        want, tol = self.want(q, scale)
        n = self.starts[-1]
        assert bool((out[n:] == 7.0).all()), "rows of no sequence were written"
        off = (out[:n].double() - want).abs()
        assert bool((off <= tol).all()), f"off by {off.max().item():.3e}, {(off / tol).max().item():.2f} of what rounding explains"
        assert pkg.device_status() == 0
        return out


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
LENGTHS = [([1], [0]), ([1, 1, 1], [0, 15, 16]), ([5, 0, 33, 1], [0, 7, 100, 31]), ([70], [3])]
SHAPES = [(2, 2, 64, 16), (4, 2, 8, 1), (6, 2, 40, 7), (3, 3, 256, 32), (5, 1, 128, 24)]


def rotated(x, table, pairs):
    """x [tokens, heads, D] by table [tokens, R], and the size of what is rounded."""
    R = table.shape[1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if pairs else (x[..., :R // 2], x[..., R // 2:R])
    c, s = table[:, None, :R // 2], table[:, None, R // 2:]
    y, size = x.clone(), torch.zeros_like(x)
    for out, (first, second) in ((y, (a * c - b * s, b * c + a * s)), (size, ((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()))):
        if pairs:
            out[..., 0:R:2], out[..., 1:R:2] = first, second
        else:
            out[..., :R // 2], out[..., R // 2:R] = first, second
    return y, size


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,kv,D,page", SHAPES)
@pytest.mark.parametrize("new,past", LENGTHS)
@pytest.mark.parametrize("rotary,pairs", [(0, False), ("all", False), ("all", True), ("eights", False), ("eights", True), ("part", False), ("part", True)])
def test_append(pkg, new, past, heads, kv, D, page, dtype, rotary, pairs):
    st = Step(new, past, heads, kv, D, page, dtype)
    W = (heads + 2 * kv) * D
    wide = st.normal(st.tokens, W + 12)  # rows that lie apart
    wide[st.starts[-1]:] = float("nan")
    qkv = wide[:, :W]
    R = {0: 0, "all": D, "eights": max(8, D // 16 * 8), "part": D // 4 * 2 - (2 if D > 8 else 0)}[rotary]
    table = pkg.rotary_table(max(a + b for a, b in zip(new, past)), R) if R else None
    k0, v0 = st.k.clone(), st.v.clone()
    q = pkg.paged_append(qkv, *st.args(), rotary=table, rotary_pairs=pairs)
    n = st.starts[-1]
    x = qkv[:n].double().view(n, heads + 2 * kv, D)
    size = torch.zeros_like(x)
    if R:
        at = torch.cat([torch.arange(b, a + b) for a, b in zip(new, past)]).cuda()
        y, sizes = rotated(x[:, :heads + kv], table[at].double(), pairs)
        x, size = torch.cat([y, x[:, heads + kv:]], 1), torch.cat([sizes, size[:, heads + kv:]], 1)
    else:
        assert q.data_ptr() == qkv.data_ptr()
    assert q.shape == (st.tokens, heads * D)
    assert bool(((q[:n].double().view(n, heads, D) - x[:, :heads]).abs() <= 3 * E * size[:, :heads]).all())
    for got, start, first in ((st.k, k0, heads), (st.v, v0, heads + kv)):
        touched = torch.zeros(st.pages, page, dtype=torch.bool, device="cuda")
        for s, count in enumerate(new):
            for i in range(count):
                where, t = st.where(s, past[s] + i), st.starts[s] + i
                touched[where] = True
                want, slack = x[t, first:first + kv], 3 * E * size[t, first:first + kv]
                have = got[where[0], :, where[1]]
                if dtype == "bf16" and not bool(slack.any()):
                    assert torch.equal(have, want.float().bfloat16())
                else:
                    half = 2.0 ** -8 * (want.abs() + slack) if dtype == "bf16" else 0.0
                    assert bool(((have.double() - want).abs() <= slack + half).all())
        rest = ~touched[:, None, :, None].expand(st.pages, kv, page, D)
        assert bool((got[rest].isnan() == start[rest].isnan()).all()), "rows of other positions were written"
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_append_many_sequences(pkg, dtype):
    """More sequences than one look at their beginnings covers, empty ones among them."""
    new = [(i * 7) % 4 for i in range(1500)]
    past = [(i * 13) % 50 for i in range(1500)]
    st = Step(new, past, 2, 1, 16, 8, dtype, tail=5)
    qkv = st.normal(st.tokens, 4 * 16)
    pkg.paged_append(qkv, *st.args())
    p = torch.cat([torch.arange(b, a + b) for a, b in zip(new, past)]).cuda()
    s = torch.repeat_interleave(torch.arange(1500), torch.tensor(new)).cuda()
    page = st.table[s, p // 8].long()
    assert torch.equal(st.k[page, :, p % 8], qkv[:st.starts[-1], None, 32:48].to(st.k.dtype))
    assert torch.equal(st.v[page, :, p % 8], qkv[:st.starts[-1], None, 48:64].to(st.k.dtype))
    assert int((~st.k.isnan()).sum()) == sum(new) * 16
    assert pkg.device_status() == 0


def test_append_leaves_out_positions_without_a_page(pkg):
    """A page number out of range, a position behind the table or behind the angles: nothing is stored, the status says so."""
    st = Step([3, 3, 2, 2], [6, 0, 14, 1], 1, 1, 8, 8, "fp32")
    st.table[0, 1] = st.pages  # positions 8 and on of sequence 0
    st.table[1, 0] = -1
    st.before[3] = -2
    qkv = st.normal(st.tokens, 24)
    pkg.paged_append(qkv, *st.args())
    assert pkg.device_status() == 2001
    assert torch.equal(st.k[st.table[0, 0], 0, 6:8], qkv[0:2, 8:16])  # what has a page is stored
    assert torch.equal(st.k[st.table[2, 1], 0, 6:8], qkv[6:8, 8:16])
    assert int((~st.k.isnan()).sum()) == 4 * 8
    st = Step([4], [6], 1, 1, 8, 8, "fp32")
    pkg.paged_append(st.normal(st.tokens, 24), *st.args(), rotary=pkg.rotary_table(8, 8))
    assert pkg.device_status() == 2001
    assert int((~st.k.isnan()).sum()) == 2 * 8
    st = Step([4], [6], 1, 1, 8, 8, "fp32")
    pkg.paged_append(st.normal(st.tokens, 24), st.k, st.v, st.table[:, :1].contiguous(), st.cu, st.before)
    assert pkg.device_status() == 2001
    assert int((~st.k.isnan()).sum()) == 2 * 8


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,kv,D,page", [(2, 2, 64, 16), (3, 3, 8, 1), (2, 1, 24, 5), (6, 2, 40, 24), (4, 4, 128, 32), (8, 1, 64, 16), (2, 2, 136, 16),
                                             (3, 1, 256, 8), (10, 2, 96, 100)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1, 1], [0, 15, 16, 700]), ([2, 0, 1, 2], [63, 9, 127, 0]), ([4, 3], [0, 300])])
def test_few_new_tokens(pkg, new, past, heads, kv, D, page, dtype):
    st = Step(new, past, heads, kv, D, page, dtype, seed=len(new) + D)
    st.fill()
    st.check(pkg, max_new=max(new))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,kv,D,page", [(2, 2, 64, 16), (3, 1, 64, 7), (6, 2, 128, 32), (2, 2, 40, 24), (5, 5, 16, 128), (2, 2, 96, 16), (2, 1, 200, 16)])
@pytest.mark.parametrize("new,past", [([17], [0]), ([128, 127, 129], [0, 1, 128]), ([1, 200, 0, 64, 1], [300, 511, 5, 0, 64]), ([9, 30], [1000, 63])])
def test_many_new_tokens(pkg, new, past, heads, kv, D, page, dtype):
    st = Step(new, past, heads, kv, D, page, dtype, seed=len(new) + D)
    st.fill()
    st.check(pkg, max_new=max(new))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads,kv,D", [([1] * 20 + [40], [17 * i for i in range(21)], 2, 2, 64), ([1, 30], [9000, 10], 4, 2, 64),
                                                 ([1, 3, 0, 200] + [1] * 34, [5 + 11 * i for i in range(38)], 12, 12, 64),
                                                 ([1, 100, 1], [200, 0, 64], 4, 1, 128), ([2, 60, 1], [63, 128, 700], 5, 5, 40)])
@pytest.mark.parametrize("known", [False, True])
def test_single_tokens_beside_pieces(pkg, known, new, past, heads, kv, D, dtype):
    """One kernel or two, by the number of sequences, their lengths and the rows they have on average."""
    st = Step(new, past, heads, kv, D, 16, dtype)
    st.fill()
    st.check(pkg, max_new=max(new) if known else 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads,kv,D", [([1], [30011], 4, 1, 64), ([1, 1], [9000, 17], 2, 2, 128), ([40], [9001], 3, 1, 64), ([3, 150], [5000, 2500], 2, 1, 128)])
def test_long_contexts(pkg, new, past, heads, kv, D, dtype):
    st = Step(new, past, heads, kv, D, 64, dtype)
    st.fill()
    st.check(pkg, max_new=max(new))


@pytest.mark.parametrize("max_new", [0, 20, 1000])
def test_max_new_is_a_bound(pkg, max_new):
    st = Step([1, 20, 7], [40, 3, 150], 2, 1, 64, 16, "bf16")
    st.fill()
    st.check(pkg, max_new=max_new)


def test_strides(pkg):
    """Queries inside the rows of the fused projection, keys and values of a page side by side, a scale of the caller's."""
    for dtype in TYPES:
        st = Step([40, 1, 3], [100, 77, 0], 4, 2, 64, 16, dtype, interleaved=True)
        st.fill()
        st.check(pkg, q=st.normal(st.tokens, 8 * 64)[:, :4 * 64], scale=0.3, max_new=40)
        st.check(pkg, q=st.normal(st.tokens, 8 * 64)[:, 64:5 * 64], scale=-0.1)
        st.check(pkg, scale=0.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past", [([4], [10]), ([60, 3], [100, 2]), ([130], [0])])
def test_what_a_row_does_not_see_does_not_reach_it(pkg, new, past, dtype):
    """NaN and infinities in keys and values of later tokens of the same sequence."""
    st = Step(new, past, 2, 1, 64, 16, dtype)
    st.fill()
    q = st.normal(st.tokens, 128)
    clean = st.check(pkg, q, max_new=max(new)).clone()
    kept = st.k.clone(), st.v.clone()
    for s, n in enumerate(new):
        page, row = st.where(s, past[s] + n - 1)
        st.k[page, :, row], st.v[page, :, row] = float("nan"), float("inf")
        page, row = st.where(s, past[s] + n - 2)
        st.v[page, :, row, ::2] = float("nan")
    out = pkg.paged_attention(q, *st.args(), max_new=max(new))
    st.k[:], st.v[:] = kept
    tol = st.want(q)[1]
    for s, n in enumerate(new):
        a, b = st.starts[s], st.starts[s] + n
        assert bool(((out[a:b - 2] - clean[a:b - 2]).abs() <= 2 * tol[a:b - 2]).all())
        assert bool(out[b - 2].isnan().view(2, 64)[:, ::2].all()) and bool(out[b - 2].isfinite().view(2, 64)[:, 1::2].all())
        assert bool(out[b - 1].isnan().all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_scores_of_infinity(pkg, n, dtype):
    """A key whose score is -inf has no weight; a row of such keys alone is 0."""
    st = Step([n, n], [50, 0], 1, 1, 64, 16, dtype)
    st.fill()
    q = st.normal(st.tokens, 64)
    q[:, 0] = 1.0
    for s, p in ((0, 3), (0, 20)):
        page, row = st.where(s, p)
        st.k[page, :, row, 0] = float("-inf")
    st.check(pkg, q, max_new=n)
    for p in range(n):
        page, row = st.where(1, p)
        st.k[page, :, row, 0] = float("-inf")
    out = pkg.paged_attention(q, *st.args(), max_new=n)
    assert bool((out[st.starts[1]:st.starts[2]] == 0).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 40, 150])
def test_large_scores(pkg, n, dtype):
    """One key far above the others, and scores that rise along the context: the maximum moves again and again."""
    st = Step([n, n], [300, 513], 2, 2, 64, 16, dtype)
    st.fill()
    q = st.normal(st.tokens, 128)
    for s in range(2):
        for p in range(st.past[s] + n):
            page, row = st.where(s, p)
            st.k[page, :, row] *= 1 + p / 60 if s else (40 if p == 211 else 1)
    st.check(pkg, q, max_new=n)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_pages_that_are_not_there(pkg, n):
    """Their keys have no weight, the status says so; more new tokens than max_new: the sequence's rows stay as they were."""
    st = Step([n], [50], 1, 1, 64, 16, "bf16")
    st.fill()
    q = st.normal(st.tokens, 64)
    lost = st.table.clone()
    lost[0, 1] = st.pages
    out = pkg.paged_attention(q, st.k, st.v, lost, st.cu, st.before, max_new=n)
    assert pkg.device_status() == 2002
    k, v = st.context(0)
    z = q[:n].double() @ k[0].T / 8
    z[:, 16:32] = float("-inf")
    z.masked_fill_(torch.arange(50 + n, device="cuda") > 50 + torch.arange(n, device="cuda")[:, None], float("-inf"))
    size = (q[:n].double().abs() @ k[0].abs().T / 8).max()
    assert (out[:n].double() - torch.softmax(z, -1) @ v[0]).abs().max() <= 2 * (size * 69 + 50 + n + 8) * E * v.abs().max()
    if n > 1:
        out = torch.full_like(q, 7.0)
        pkg.paged_attention(q, *st.args(), max_new=n - 1, out=out)
        assert pkg.device_status() == 2002 and bool((out == 7.0).all())
    out = torch.full_like(q, 7.0)
    pkg.paged_attention(q, st.k, st.v, st.table, st.cu, ints([-5]), max_new=n, out=out)
    assert pkg.device_status() == 2002 and bool((out == 7.0).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,D", [(1, 64), (3, 64), (40, 64), (300, 64), (3, 136)])
@pytest.mark.parametrize("past", [2 ** 31 - 1, 2 ** 31 - 20, 2 ** 30, 81])
def test_positions_behind_the_table(pkg, past, n, D, dtype):
    """Every new token lies behind the page table: none is stored, each sees the keys that the table has room for."""
    st = Step([n], [80], 2, 1, D, 16, dtype, tail=0)
    st.table = st.table[:, :5].contiguous()  # room for 80 positions
    st.fill([80])
    q = st.normal(n, 2 * D)
    before = ints([past])
    k, v = st.k.clone(), st.v.clone()
    pkg.paged_append(st.normal(n, 4 * D), st.k, st.v, st.table, st.cu, before)
    assert pkg.device_status() == 2001
    assert torch.equal(st.k.nan_to_num(), k.nan_to_num()) and torch.equal(st.v.nan_to_num(), v.nan_to_num())
    got = pkg.paged_attention(q, st.k, st.v, st.table, st.cu, before, max_new=n)
    assert pkg.device_status() == 2002
    st.new, st.past, st.starts = [1] * n, [79] * n, list(range(n + 1))  # the same as n sequences that share those pages
    st.table = st.table.repeat(n, 1)
    want, tol = st.want(q)
    assert bool(((got.double() - want).abs() <= tol).all())


def test_under_inference_mode(pkg):
    """As a program that generates would call them, with tensors made there."""
    with torch.inference_mode():
        st = Step([1, 9], [30, 2], 2, 2, 64, 16, "bf16", tail=0)
        st.fill([30, 2])
        qkv = st.normal(st.tokens, 3 * 128)
        q = pkg.paged_append(qkv, *st.args())
        assert torch.equal(q, qkv[:, :128]) and q.data_ptr() == qkv.data_ptr()
        st.check(pkg, q, max_new=9)
        logits = st.normal(3, 1000)
        assert torch.equal(pkg.sample(logits, torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")), logits.argmax(1).int())


@pytest.mark.parametrize("n", [1, 40])
def test_offsets_beyond_32_bits(pkg, n):
    """Pages of a cache of more than 2^32 bytes and 2^31 elements, of which only the last ones are used."""
    pages = 2 ** 31 // (64 * 64) + 40
    k, v = (torch.empty(pages, 1, 64, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    st = Step([n], [100], 1, 1, 64, 64, "bf16", spare=0)
    st.fill()
    far = st.table + (pages - st.pages)
    k[pages - st.pages:], v[pages - st.pages:] = st.k, st.v
    q = st.normal(st.tokens, 64)
    assert torch.equal(pkg.paged_attention(q, k, v, far, st.cu, st.before, max_new=n)[:n], st.check(pkg, q, max_new=n)[:n])
    qkv = st.normal(st.tokens, 192)
    pkg.paged_append(qkv, k, v, far, st.cu, st.before)
    pkg.paged_append(qkv, *st.args())
    assert torch.equal(k[pages - st.pages:].nan_to_num(5.0), st.k.nan_to_num(5.0)) and torch.equal(v[pages - st.pages:].nan_to_num(5.0), st.v.nan_to_num(5.0))


@pytest.mark.parametrize("shape", [([1, 1, 1], [30, 200, 999]), ([50, 1, 200], [30, 200, 600])])
def test_the_same_bits_every_time(pkg, shape):
    st = Step(*shape, 4, 2, 64, 16, "bf16")
    st.fill()
    q = st.normal(st.tokens, 256)
    first = st.check(pkg, q, max_new=max(shape[0]))
    for _ in range(20):
        out = torch.full_like(first, 7.0)
        assert torch.equal(pkg.paged_attention(q, *st.args(), max_new=max(shape[0]), out=out), first)


def test_two_streams_and_a_graph(pkg):
    """Calls at once on two streams, and one captured and replayed with other lengths, pages and values in its tensors."""
    a, b = Step([1, 60], [100, 30], 2, 2, 64, 16, "bf16", seed=1), Step([7, 60], [10, 300], 2, 2, 64, 16, "bf16", seed=2)
    a.fill(), b.fill()
    qa, qb = a.normal(a.tokens, 128), b.normal(b.tokens, 128)
    wa, wb = a.check(pkg, qa, max_new=60), b.check(pkg, qb, max_new=60)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (st, q, stream) in enumerate(((a, qa, sa), (b, qb, sb))):
            got[i].append(pkg.paged_attention(q, *st.args(), max_new=60, stream=stream))
    torch.cuda.synchronize()
    for have, want, n in ((got[0], wa, 61), (got[1], wb, 67)):
        assert all(torch.equal(x[:n], want[:n]) for x in have)

    # one step of append and attention, captured over tensors that hold one set of lengths, replayed over another
    st = Step([1, 1], [40, 110], 2, 2, 64, 16, "bf16", tail=0)
    st.fill()
    st.before.copy_(ints([15, 100]))
    qkv = st.normal(2, 3 * 128)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        out = pkg.paged_attention(pkg.paged_append(qkv, *st.args()), *st.args(), max_new=1)
    for past in ([15, 100], [16, 101], [3, 40]):
        st.past = past
        st.before.copy_(ints(past))
        qkv.copy_(st.normal(2, 3 * 128))
        graph.replay()
        torch.cuda.synchronize()
        want, tol = st.want(qkv[:, :128])
        assert bool(((out.double() - want).abs() <= tol).all())
        for s in range(2):
            page, row = st.where(s, past[s])
            assert torch.equal(st.k[page, :, row].flatten(), qkv[s, 128:256].bfloat16())
    assert pkg.device_status() == 0


def test_a_device_that_is_not_current(pkg):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    st = Step([1, 9], [30, 2], 2, 2, 64, 16, "fp32")
    st.fill()
    q = st.normal(st.tokens, 128)
    want = st.check(pkg, q)
    there = [t.to("cuda:1") for t in (q, *st.args())]
    assert torch.equal(pkg.paged_attention(*there)[:10].cpu(), want[:10].cpu())
    with pytest.raises(ValueError):
        pkg.paged_attention(q, *there[1:])


def test_refusals(pkg):
    st = Step([2, 3], [4, 5], 2, 2, 64, 16, "bf16", tail=0)
    q, qkv, a = st.normal(5, 128), st.normal(5, 384), st.args()

    def with_(i, t):
        return tuple(t if j == i else x for j, x in enumerate(a))

    wrong = [with_(0, st.k.half()), with_(0, st.k.float()), with_(1, st.v[:-1]), with_(0, st.k.transpose(1, 2)), with_(1, st.v[..., :32]), with_(0, st.k[0]),
             with_(2, st.table.long()), with_(2, st.table[:1]), with_(2, st.table[0]), with_(3, st.cu[:2]), with_(3, st.cu.long()), with_(4, st.before[:1]),
             with_(4, st.before.float()), with_(2, st.table.cpu()), with_(0, st.k.cpu()), with_(0, st.k[:, :0])]
    for w in wrong:
        with pytest.raises(ValueError):
            pkg.paged_attention(q, *w)
        with pytest.raises(ValueError):
            pkg.paged_append(qkv, *w)
    for bad in (q.double(), q[:, :100], q.view(5, 2, 64), q.t(), q.cpu(), q[:, ::2]):
        with pytest.raises(ValueError):
            pkg.paged_attention(bad, *a)
    wide = st.normal(5, 384)
    with pytest.raises(ValueError):  # out inside the rows of q
        pkg.paged_attention(wide[:, 128:256], *a, out=wide.view(-1)[:640].view(5, 128))
    with pytest.raises(ValueError):
        pkg.paged_attention(q, *a, out=q)
    for more in ({"max_new": -1}, {"out": q[:4]}, {"out": q.double()}, {"out": torch.empty(128, 5, device="cuda").t()}):
        with pytest.raises(ValueError):
            pkg.paged_attention(q, *a, **more)
    with pytest.raises(pkg.AttnError):
        pkg.paged_attention(q, *a, scale=float("nan"))
    for bad in (qkv.double(), qkv[:, :256], qkv[:, :300], qkv.t()):
        with pytest.raises(ValueError):
            pkg.paged_append(bad, *a)
    for rotary in (torch.zeros(9, 63, device="cuda"), torch.zeros(9, 66, device="cuda"), torch.zeros(9, 64), torch.zeros(64, 9, device="cuda").t(),
                   torch.zeros(9, 64, device="cuda").double()):
        with pytest.raises(ValueError):
            pkg.paged_append(qkv, *a, rotary=rotary)
    with pytest.raises(pkg.AttnError):  # rows that do not begin on 16 bytes
        pkg.paged_attention(st.normal(5, 130)[:, 1:129], *a)
    assert pkg.paged_attention(q[:0], *a).shape == (0, 128)  # no rows: nothing to do
    assert pkg.paged_append(qkv[:0], *a).shape == (0, 128)
    assert pkg.device_status() == 0


# ---------------------------------------------------------------------------------------------
# what decides between the kernels and their forms, each with its neighbours
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("page", [1, 4, 8, 48, 64, 100, 128, 192])
@pytest.mark.parametrize("D", [64, 72, 128])
def test_page_sizes(pkg, D, page, dtype):
    st = Step([150, 1, 20], [70, 131, 64], 2, 1, D, page, dtype, seed=page)
    st.fill()
    st.check(pkg, max_new=150)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("D", [64, 96])
def test_every_small_number_of_rows(pkg, rows, D, dtype):
    """As new tokens, and as query heads of one key/value head."""
    for new, heads in ((rows, 1), (1, rows)):
        st = Step([new, 1, new], [200, 40, 0], heads, 1, D, 16, dtype, seed=rows)
        st.fill()
        st.check(pkg, max_new=new)
        st.check(pkg)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("seqs,heads,kv,D,new", [(110, 12, 12, 64, 1), (40, 12, 12, 128, 1), (110, 24, 12, 64, 1), (110, 12, 12, 48, 2), (45, 24, 12, 96, 1),
                                                 (300, 4, 4, 64, 1), (1100, 1, 1, 64, 1)])
def test_many_sequences(pkg, seqs, heads, kv, D, new, dtype):
    """Enough of them for a warp each; none, one or `new` tokens, from no context to some pages."""
    counts = [(0, 1, new, new)[i % 4] for i in range(seqs)]
    st = Step(counts, [(i * 37) % 150 for i in range(seqs)], heads, kv, D, 16, dtype)
    st.fill()
    st.check(pkg, max_new=new)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_many_ragged_pieces(pkg, D, dtype):
    """More sequences than the order of their lengths is looked at for, and pieces among single tokens."""
    new = [(i * 53) % 140 + 1 if i % 3 else 1 for i in range(70)]
    st = Step(new, [(i * 91) % 400 for i in range(70)], 4, 2, D, 32, dtype)
    st.fill()
    st.check(pkg, max_new=max(new))
    st.check(pkg)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads", [([700], [500], 25), ([400, 300, 130], [64, 1000, 3], 25), ([128] * 12, [0] * 12, 13)])
def test_more_units_than_sms(pkg, new, past, heads, dtype):
    """Whole rounds of the SMs, and a rest of them that is cut into pieces."""
    st = Step(new, past, heads, heads, 64, 16, dtype)
    st.fill()
    st.check(pkg, max_new=max(new))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("page,D", [(8, 64), (16, 128), (64, 64), (100, 64), (32, 40)])
@pytest.mark.parametrize("n", [1, 6, 70])
def test_holes(pkg, n, page, D, dtype):
    """Pages that are not there at the beginning, inside and at the end of a context."""
    st = Step([n, n], [330, 200], 2, 2, D, page, dtype)
    st.fill()
    q = st.normal(st.tokens, 2 * D)
    lost = st.table.clone()
    for where in ((0, 0), (0, 150 // page), (1, (200 + n - 1) // page)):
        lost[where] = -7
    out = pkg.paged_attention(q, st.k, st.v, lost, st.cu, st.before, max_new=n)
    assert pkg.device_status() == 2002
    for s in range(2):
        k, v = st.context(s)
        there = torch.tensor([0 <= int(lost[s, p // page]) < st.pages for p in range(k.shape[1])], device="cuda")
        x = q[st.starts[s]:st.starts[s + 1]].double().view(n, 2, D).transpose(0, 1)
        seen = (torch.arange(k.shape[1], device="cuda") <= st.past[s] + torch.arange(n, device="cuda")[:, None]) & there
        z = (x @ k.transpose(1, 2) * D ** -0.5).masked_fill(~seen, float("-inf"))
        size = (x.abs() @ k.abs().transpose(1, 2) * D ** -0.5).amax(-1, keepdim=True)
        want = torch.softmax(z, -1) @ v
        tol = 2 * (size * (D + 5) + k.shape[1] + 8) * E * (torch.softmax(z, -1) @ v.abs())
        got = out[st.starts[s]:st.starts[s + 1]].double().view(n, 2, D).transpose(0, 1)
        assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [2, 4, 6, 100])
def test_a_bad_query_stays_by_itself(pkg, n, dtype):
    st = Step([n, n], [150, 3], 2, 1, 64, 16, dtype)
    st.fill()
    q = st.normal(st.tokens, 128)
    clean = st.check(pkg, q, max_new=n).clone()
    q[1, 5], q[n, 70] = float("nan"), float("inf")
    out = pkg.paged_attention(q, *st.args(), max_new=n)
    for t in range(2 * n):
        for h in range(2):
            got, had = out[t, 64 * h:64 * h + 64], clean[t, 64 * h:64 * h + 64]
            if (t, h) in ((1, 0), (n, 1)):
                assert bool(got.isnan().all())
            else:
                assert torch.equal(got, had)


@pytest.mark.parametrize("n", [1, 5, 100])
def test_large_finite_values(pkg, n):
    """fp32 keys and values as large as sums of them in fp32 allow: a weight is at most 1, so n of them times values below the largest
    number over n stay below it.  Their terms are finite, too."""
    st = Step([n], [70], 1, 1, 64, 16, "fp32")
    st.fill()
    q = st.normal(st.tokens, 64) * 1e-30  # times the scale above 2^-102: its terms are normal numbers
    for p in range(70 + n):
        page, row = st.where(0, p)
        st.k[page, :, row] *= 1e29
        st.v[page, :, row] = st.v[page, :, row].clamp(-1, 1) * (3.4e38 / (71 + n))
    st.check(pkg, q, max_new=n)


def test_rows_of_no_sequence_alone(pkg):
    """A captured step of which nothing is left: no new token in any sequence, rows in the buffers all the same."""
    for dtype in TYPES:
        st = Step([0, 0, 0], [5, 0, 40], 2, 2, 64, 16, dtype, tail=7)
        st.fill()
        k0 = st.k.clone()
        for max_new in (0, 1, 7):
            st.check(pkg, max_new=max_new)
        pkg.paged_append(st.normal(7, 384), *st.args())
        assert torch.equal(st.k.nan_to_num(3.0), k0.nan_to_num(3.0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_what_follows_a_call_waits_for_all_of_it(pkg, dtype):
    """Calls of two launches side by side (single tokens and pieces; whole rounds and a rest), and kernels behind them that may start early."""
    st = Step([1] * 20 + [200, 300], [500] * 22, 12, 12, 64, 16, dtype)
    big = Step([700], [900], 25, 25, 64, 16, dtype)
    w = st.normal(64, 12 * 64)
    w2 = st.normal(64, 25 * 64)
    for s, weights, m in ((st, w, 300), (big, w2, 700)):
        s.fill()
        q = s.normal(s.tokens, s.heads * 64)
        out = s.check(pkg, q, max_new=m)
        n = s.starts[-1]
        torch.cuda.synchronize()
        want = pkg.linear_forward(out[:n].contiguous(), weights)
        torch.cuda.synchronize()
        for i in range(30):
            buf = torch.full_like(out, float(i))
            got = pkg.linear_forward(pkg.paged_attention(q, *s.args(), max_new=m, out=buf)[:n], weights)
            assert torch.equal(got, want)
    # and the append that the next step's attention reads, over and over on one cache
    qkv = st.normal(st.tokens, 3 * 12 * 64)
    pkg.paged_append(qkv, *st.args())
    torch.cuda.synchronize()
    want = pkg.paged_attention(qkv[:, :768], *st.args(), max_new=300).clone()
    n = st.starts[-1]
    for i in range(20):
        other = qkv + 1.0 + i
        pkg.paged_attention(pkg.paged_append(other, *st.args()), *st.args(), max_new=300)
        got = pkg.paged_attention(pkg.paged_append(qkv, *st.args()), *st.args(), max_new=300)
        assert torch.equal(got[:n], want[:n])


@pytest.mark.parametrize("stride", [2 ** 33, 2 ** 34])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_pages_very_far_apart(pkg, n, stride):
    """The last page begins 2^33 or 2^34 elements behind the first: either side of what 32-bit places reach."""
    if torch.cuda.mem_get_info()[0] < 50 << 30:
        pytest.skip("needs 36 GB")
    store = torch.empty(stride + 4 * 2 * 64 * 64, dtype=torch.bfloat16, device="cuda")
    k = store.as_strided((2, 2, 64, 64), (stride, 64 * 64, 64, 1))
    v = store.as_strided((2, 2, 64, 64), (stride, 64 * 64, 64, 1), 2 * 64 * 64)
    st = Step([n], [80], 2, 2, 64, 64, "bf16", spare=0)
    st.fill()
    st.k.nan_to_num_(0.5), st.v.nan_to_num_(0.5)
    k.copy_(st.k), v.copy_(st.v)
    q = st.normal(st.tokens, 128)
    want, tol = st.want(q)
    got = pkg.paged_attention(q, k, v, st.table, st.cu, st.before, max_new=n)[:n]
    assert bool(((got.double() - want).abs() <= tol).all())
    qkv = st.normal(st.tokens, 384)
    pkg.paged_append(qkv, k, v, st.table, st.cu, st.before)
    pkg.paged_append(qkv, *st.args())
    assert torch.equal(k, st.k) and torch.equal(v, st.v)
    assert pkg.device_status() == 0


SCRIPT = """
import sys
import torch
import __graft_entry__ as entry

pkg = entry.load_package()
pkg.lib()
n, bf16 = int(sys.argv[1]), sys.argv[2] == "bf16"
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
qkv = torch.randn(n, 384, device="cuda")
k, v = (torch.randn(4, 2, 64, 64, device="cuda", dtype=torch.bfloat16 if bf16 else torch.float32) for _ in range(2))
args = (k, v, ints([[2, 0, 1]]), ints([0, n]), ints([50]))
logits, u, top_k = torch.randn(3, 50257, device="cuda"), torch.rand(3, device="cuda"), ints([5, 500, 5000])
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = pkg.paged_attention(pkg.paged_append(qkv, *args), *args, max_new=n)
    drawn = pkg.sample(logits, u, None, top_k)
graph.replay()
torch.cuda.synchronize()
again = pkg.paged_attention(pkg.paged_append(qkv, *args), *args, max_new=n)
assert torch.equal(out, again) and torch.equal(drawn, pkg.sample(logits, u, None, top_k)) and bool(out.isfinite().all())
assert pkg.device_status() == 0
"""


@pytest.mark.parametrize("n,dtype", [(1, "bf16"), (1, "fp32"), (5, "bf16"), (100, "bf16"), (100, "fp32")])
def test_first_call_under_capture(n, dtype):
    """The first call of a process may be one that a stream captures."""
    import os
    import subprocess
    import sys

    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    r = subprocess.run([sys.executable, "-c", SCRIPT, str(n), dtype], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
