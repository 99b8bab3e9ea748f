"""What the entry points at both ends of a training step (embedding, projection with its loss) refuse: nothing here reaches a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

NULL, ARGUMENT, UNSUPPORTED, ALIGN = -1, -8, -3, -4


def at(n):
    return ctypes.c_void_p(n)


P, ODD = at(1 << 20), at((1 << 20) + 1)

EMBED = dict(tokens=P, table=P, positions=None, pos_table=P, y=P, n=5, ld=64, pos_ld=64, scale=1.0, type=0, ids=1, T=5, C=64, V=100, Pn=9, stream=None)
EMBED_GRAD = dict(dy=P, tokens=P, dtable=at(1 << 24), positions=None, dpos=at(1 << 25), scratch=at(1 << 26), n=5, ld_dy=64, ld=64, pos_ld=64, scale=1.0, type=0, grad=0,
                  ids=1, T=5, C=64, V=100, Pn=9, stream=None)
LOSS = dict(x=P, w=P, targets=P, losses=P, lse=P, scratch=P, ldx=64, ldw=64, type=1, ids=1, rows=5, V=100, K=64, stream=None)
LOSS_GRAD = dict(g=P, x=P, w=P, targets=P, lse=P, dx=at(1 << 21), dw=at(1 << 22), scratch=P, ldx=64, ldw=64, lddw=64, one=0, type=1, ids=1, rows=5, V=100, K=64, stream=None)


@pytest.mark.parametrize("wrong,code", [
    (dict(tokens=None), NULL), (dict(table=None), NULL), (dict(y=None), NULL), (dict(n=-1), ARGUMENT), (dict(C=0), ARGUMENT), (dict(V=0), ARGUMENT),
    (dict(ld=63), ARGUMENT), (dict(pos_ld=63), ARGUMENT), (dict(Pn=0), ARGUMENT), (dict(T=0), ARGUMENT), (dict(type=2), ARGUMENT), (dict(ids=3), ARGUMENT),
    (dict(ids=-1), ARGUMENT), (dict(table=ODD), ALIGN), (dict(y=ODD), ALIGN), (dict(pos_table=ODD), ALIGN), (dict(tokens=at((1 << 20) + 4)), ALIGN),
    (dict(ids=0, tokens=at((1 << 20) + 2)), ALIGN), (dict(positions=at((1 << 20) + 4)), ALIGN)])
def test_embedding_forward_refuses(pkg, wrong, code):
    assert pkg.lib().tensor_sm100_embedding_forward(*{**EMBED, **wrong}.values()) == code


@pytest.mark.parametrize("wrong,code", [
    (dict(dy=None), NULL), (dict(tokens=None), NULL), (dict(dtable=None, dpos=None), NULL), (dict(scratch=None), NULL), (dict(n=-1), ARGUMENT), (dict(C=0), ARGUMENT),
    (dict(V=0), ARGUMENT), (dict(Pn=0), ARGUMENT), (dict(T=0), ARGUMENT), (dict(ld_dy=63), ARGUMENT), (dict(ld=63), ARGUMENT), (dict(pos_ld=63), ARGUMENT),
    (dict(type=2), ARGUMENT), (dict(grad=2), ARGUMENT), (dict(ids=3), ARGUMENT), (dict(dy=ODD), ALIGN), (dict(dtable=ODD), ALIGN), (dict(dpos=ODD), ALIGN),
    (dict(scratch=at((1 << 26) + 128)), ALIGN), (dict(tokens=at((1 << 20) + 4)), ALIGN), (dict(n=(1 << 30) + 1), UNSUPPORTED),
    (dict(C=(1 << 20) + 1, ld=1 << 21, ld_dy=1 << 21, pos_ld=1 << 21), UNSUPPORTED),
    (dict(dpos=at((1 << 24) + 4 * 64 * 50)), ARGUMENT), (dict(dpos=at((1 << 24) - 4)), ARGUMENT), (dict(dy=at((1 << 24) + 4 * 64 * 99)), ARGUMENT),
    (dict(dy=at((1 << 25) + 64)), ARGUMENT)])
def test_embedding_backward_refuses(pkg, wrong, code):
    assert pkg.lib().tensor_sm100_embedding_backward(*{**EMBED_GRAD, **wrong}.values()) == code


HEAD_WRONG = [(dict(x=None), NULL), (dict(w=None), NULL), (dict(targets=None), NULL), (dict(lse=None), NULL), (dict(scratch=None), NULL), (dict(rows=-1), ARGUMENT),
              (dict(V=0), ARGUMENT), (dict(K=0), ARGUMENT), (dict(ldx=63), ARGUMENT), (dict(ldw=63), ARGUMENT), (dict(type=2), ARGUMENT), (dict(type=-1), ARGUMENT),
              (dict(ids=3), ARGUMENT), (dict(x=ODD), ALIGN), (dict(w=ODD), ALIGN), (dict(scratch=at((1 << 20) + 128)), ALIGN), (dict(lse=at((1 << 20) + 2)), ALIGN),
              (dict(targets=at((1 << 20) + 4)), ALIGN), (dict(rows=(1 << 30) + 1), UNSUPPORTED), (dict(V=(1 << 30) + 1), UNSUPPORTED),
              (dict(rows=1 << 30, V=1 << 30), UNSUPPORTED), (dict(K=(1 << 24) + 1, ldx=1 << 25, ldw=1 << 25, lddw=1 << 25), UNSUPPORTED)]


def without(d, *names):
    return {k: v for k, v in d.items() if k not in names}


@pytest.mark.parametrize("wrong,code", HEAD_WRONG + [(dict(losses=None), NULL), (dict(losses=at((1 << 20) + 2)), ALIGN)])
def test_linear_xent_forward_refuses(pkg, wrong, code):
    assert pkg.lib().xent_sm100_linear_forward(*{**LOSS, **without(wrong, "lddw")}.values()) == code


@pytest.mark.parametrize("wrong,code", HEAD_WRONG + [(dict(g=None), NULL), (dict(dx=None, dw=None), NULL), (dict(lddw=63), ARGUMENT), (dict(dx=ODD), ALIGN), (dict(dw=ODD), ALIGN),
                                                     (dict(g=at((1 << 20) + 2)), ALIGN), (dict(rows=(1 << 20) + 1), UNSUPPORTED), (dict(dx=at(1 << 22)), ARGUMENT),
                                                     (dict(dx=P), ARGUMENT), (dict(dw=P), ARGUMENT), (dict(dw=at((1 << 20) + 4 * 128)), ARGUMENT),
                                                     (dict(w=at((1 << 22) + 99 * 128 + 62)), ARGUMENT), (dict(lse=at((1 << 21) + 16)), ARGUMENT)])
def test_linear_xent_backward_refuses(pkg, wrong, code):
    assert pkg.lib().xent_sm100_linear_backward(*{**LOSS_GRAD, **wrong}.values()) == code


def test_scratch_sizes(pkg):
    L = pkg.lib()
    forward, backward, embed = L.xent_sm100_linear_forward_scratch_bytes, L.xent_sm100_linear_backward_scratch_bytes, L.tensor_sm100_embedding_backward_scratch_bytes
    for bad in [(0, 10, 8), (5, 0, 8), (5, 10, 0), (-1, 10, 8)]:
        rows, V, K = bad
        assert backward(P, P, 8, 8, 1, rows, V, K) == 0 and forward(P, P, 8, 8, 1, rows, V, K) == 0
    for rows in (1, 16, 17, 300):
        for V in (1, 2, 5000):
            for K in (1, 2, 3, 7, 1600):
                for type in (0, 1):
                    assert forward(P, P, K, K, type, rows, V, K) > 0 and backward(P, P, K, K, type, rows, V, K) >= rows * K * 4
    assert forward(P, P, 8, 8, 2, 5, 10, 8) == 0 and backward(P, P, 7, 8, 1, 5, 10, 8) == 0
    # bf16 tensors on 16-byte boundaries are read where they are; others are copied, and fp32 ones become two planes
    direct, moved, strided, fp32 = forward(P, P, 768, 768, 1, 100, 50257, 768), forward(P, at((1 << 20) + 2), 768, 768, 1, 100, 50257, 768), forward(P, P, 768, 770, 1, 100, 50257, 768), \
        forward(P, P, 768, 768, 0, 100, 50257, 768)
    assert direct < 1 << 20 and moved == strided
    assert 50257 * 768 * 2 <= moved - direct < 50257 * 768 * 2 + 512 and fp32 - direct >= (50257 + 100) * 768 * 4
    # G is there for a piece of the vocabulary at a time: twice 128 MB and the sums, where the logits take 1.6 GB
    assert backward(P, P, 768, 768, 1, 8192, 50257, 768) < 512 << 20
    assert embed(0, 64, 10, 0) == 0 and embed(10, 64, 0, 0) == 0 and 0 < embed(10, 64, 10, 0) < embed(10, 64, 10, 10)


def test_tensors_that_are_not_on_a_gpu(pkg):
    """There is no CPU path: a tensor in host memory is an error, not a pointer that a kernel would follow."""
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: pkg.embedding_forward(t, x), lambda: pkg.embedding_backward(x, t, x), lambda: pkg.linear_xent_forward(x, x, t),
                 lambda: pkg.linear_xent_backward(torch.ones(1), x, x, t, torch.zeros(4))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        pkg.embedding_forward([1, 2], x)
    with pytest.raises(TypeError):
        pkg.linear_xent_forward(x, x, None)
