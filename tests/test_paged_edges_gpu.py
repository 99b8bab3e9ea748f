"""Calls of the paged cache that its description allows and test_paged_gpu.py does not make; its tolerances."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

# new tokens, positions before, query heads, key/value heads, head size: the kernels for one and two rows, up to eight, many rows
FORMS = [([1, 1], [700, 40], 2, 2, 64), ([1], [300], 2, 2, 128), ([2], [300], 2, 2, 64), ([1], [90], 2, 1, 128), ([3, 4], [500, 7], 1, 1, 64), ([2], [130], 4, 1, 96),
         ([7], [200], 1, 1, 64), ([40], [300], 2, 1, 64), ([30, 1], [90, 200], 2, 2, 128), ([1], [60], 1, 1, 8), ([2], [60], 3, 1, 16), ([1, 3], [200, 50], 2, 1, 136),
         ([1], [400], 3, 3, 256)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads,kv,D", FORMS)
def test_values_of_keys_without_weight_do_not_count(pkg, new, past, heads, kv, D, dtype):
    """A key whose score is -inf has no weight, whatever its value is."""
    from test_paged_gpu import Step

    st = Step(new, past, heads, kv, D, 16, dtype, seed=D)
    st.fill()
    q = st.normal(st.tokens, heads * D)
    q.view(-1, heads, D)[:, :, 0] = 1.0
    where = [st.where(s, p) for s, n in enumerate(past) for p in (0, 3, 20, n - 1, n) if p < n + new[s]]
    for page, row in where:
        st.k[page, :, row, 0] = float("-inf")
    want, tol = st.want(q)
    for i, (page, row) in enumerate(where):
        st.v[page, :, row] = (float("nan"), float("inf"), float("-inf"))[i % 3]
    out = pkg.paged_attention(q, *st.args(), max_new=max(new))[:st.starts[-1]]
    assert bool(((out.double() - want).abs() <= tol).all())
    assert pkg.device_status() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("new,past,heads,kv,D", FORMS)
def test_infinite_values_of_small_weight_count(pkg, new, past, heads, kv, D, dtype):
    """A key that a row sees has a weight, also where that is too small for fp32: an infinite value of it leaves no finite result."""
    from test_paged_gpu import Step

    st = Step(new, past, heads, kv, D, 16, dtype, seed=D)
    st.fill()
    q = st.normal(st.tokens, heads * D)
    q.view(-1, heads, D)[:, :, 0] = 40.0
    for s, n in enumerate(past):
        page, row = st.where(s, n)  # the first new token: 40 * 100 / sqrt(D), 230 and more above the other scores
        st.k[page, :, row, 0] = 100.0
        page, row = st.where(s, 5)
        st.v[page, :, row, 3] = float("inf")
    out = pkg.paged_attention(q, *st.args(), max_new=max(new))[:st.starts[-1]].view(-1, heads, D)
    assert not bool(out[:, :, 3].isfinite().any())
    assert bool(out[:, :, 4:].isfinite().all()) and bool(out[:, :, :3].isfinite().all())


@pytest.mark.parametrize("rotary", [0, 64])
def test_queries_are_cut_off_from_autograd(pkg, rotary):
    """No call of generation is differentiable, with and without rotation: no gradient reaches the queries alone."""
    from test_paged_gpu import Step

    st = Step([2, 5], [30, 0], 2, 2, 64, 16, "bf16", tail=0)
    qkv = st.normal(st.tokens, 3 * 128).requires_grad_()
    q = pkg.paged_append(qkv, *st.args(), rotary=pkg.rotary_table(40, rotary) if rotary else None)
    assert not q.requires_grad and q.grad_fn is None
    if not rotary:
        assert q.data_ptr() == qkv.data_ptr() and torch.equal(q, qkv.detach()[:, :128])
    st.fill()
    out = pkg.paged_attention(st.normal(st.tokens, 128).requires_grad_(), *st.args(), max_new=5)
    assert not out.requires_grad
