"""What the entry points of generation (paged cache, draw of a token) refuse: nothing here reaches a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

NULL, ARGUMENT, UNSUPPORTED, ALIGN = -1, -8, -3, -4
P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 4)

APPEND = dict(qkv=P, q_out=P, k=P, v=P, table=P, cu=P, past=P, rotary=None, ld=3 * 128, page_stride=2 * 16 * 64, type=1, tokens=5, seqs=2, heads=2, kv=2, D=64,
              page=16, pages=8, width=4, positions=0, dim=0, pairs=0, stream=None)
FORWARD = dict(q=P, k=P, v=P, table=P, cu=P, past=P, out=P, ld=128, page_stride=2 * 16 * 64, type=1, tokens=5, seqs=2, heads=2, kv=2, D=64, page=16, pages=8, width=4,
               max_new=3, scale=0.125, stream=None)
SAMPLE = dict(logits=P, u=P, t=None, k=None, p=None, m=None, tokens=P, ld=100, rows=3, C=100, stream=None)

CACHE_WRONG = [(dict(k=None), NULL), (dict(v=None), NULL), (dict(table=None), NULL), (dict(cu=None), NULL), (dict(past=None), NULL),
               (dict(tokens=-1), ARGUMENT), (dict(seqs=0), ARGUMENT), (dict(heads=0), ARGUMENT), (dict(kv=0), ARGUMENT), (dict(heads=3), ARGUMENT),
               (dict(D=0), ARGUMENT), (dict(page=0), ARGUMENT), (dict(pages=0), ARGUMENT), (dict(width=0), ARGUMENT), (dict(type=2), ARGUMENT), (dict(type=-1), ARGUMENT),
               (dict(D=60), UNSUPPORTED), (dict(D=264, ld=1 << 14, page_stride=1 << 20), UNSUPPORTED), (dict(page=(1 << 20) + 1, page_stride=1 << 40), UNSUPPORTED),
               (dict(width=1 << 27, page=16), UNSUPPORTED), (dict(page_stride=2 * 16 * 64 - 8), ARGUMENT), (dict(page_stride=2 * 16 * 64 + 4), ALIGN),
               (dict(k=ODD), ALIGN), (dict(v=ODD), ALIGN)]


@pytest.mark.parametrize("wrong,code", CACHE_WRONG + [
    (dict(qkv=None), NULL), (dict(rotary=P, q_out=None, positions=9, dim=64), NULL), (dict(rotary=P, positions=9, dim=63), ARGUMENT),
    (dict(rotary=P, positions=9, dim=66), ARGUMENT), (dict(rotary=P, positions=0, dim=64), ARGUMENT), (dict(rotary=P, positions=9, dim=0), ARGUMENT),
    (dict(ld=380), ARGUMENT), (dict(ld=386), ALIGN), (dict(qkv=ODD), ALIGN), (dict(q_out=ODD), ALIGN)])
def test_append_refuses(pkg, wrong, code):
    assert pkg.lib().attn_sm100_paged_append(*{**APPEND, **wrong}.values()) == code


@pytest.mark.parametrize("wrong,code", CACHE_WRONG + [
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(ld=124), ARGUMENT), (dict(ld=130), ALIGN), (dict(max_new=-1), ARGUMENT),
    (dict(scale=float("nan")), ARGUMENT), (dict(q=ODD), ALIGN), (dict(out=ODD), ALIGN)])
def test_forward_refuses(pkg, wrong, code):
    assert pkg.lib().attn_sm100_paged_forward(*{**FORWARD, **wrong}.values()) == code


@pytest.mark.parametrize("wrong,code", [(dict(logits=None), NULL), (dict(u=None), NULL), (dict(tokens=None), NULL), (dict(rows=-1), ARGUMENT), (dict(C=0), ARGUMENT),
                                        (dict(ld=99), ARGUMENT), (dict(C=425985, ld=1 << 20), UNSUPPORTED)])
def test_sample_refuses(pkg, wrong, code):
    assert pkg.lib().xent_sm100_sample(*{**SAMPLE, **wrong}.values()) == code


def test_the_code_has_a_text(pkg):
    assert len(pkg.lib().attn_sm100_strerror(ARGUMENT)) > 8 and pkg.lib().attn_sm100_strerror(ARGUMENT) != b"unknown error"


def test_tensors_that_are_not_on_a_gpu(pkg):
    """There is no CPU path: a tensor in host memory is an error, not a pointer that a kernel would follow."""
    ints = torch.zeros(2, dtype=torch.int32)
    pages = torch.zeros(2, 1, 8, 8)
    with pytest.raises(ValueError):
        pkg.paged_append(torch.zeros(1, 24), pages, pages, ints.view(1, 2), ints, ints[:1])
    with pytest.raises(ValueError):
        pkg.paged_attention(torch.zeros(1, 8), pages, pages, ints.view(1, 2), ints, ints[:1])
    with pytest.raises(ValueError):
        pkg.sample(torch.zeros(1, 8), torch.zeros(1))
    with pytest.raises(TypeError):
        pkg.sample([1.0], torch.zeros(1))


def test_rotary_table(pkg):
    """Cosines, then sines, of angles in 64 bits: a far position keeps its phase (2^-24 a value: one rounding)."""
    t = pkg.rotary_table(100001, 6, base=500.0, device="cpu")
    assert t.shape == (100001, 6) and t.dtype == torch.float32
    i = torch.arange(3, dtype=torch.float64)
    angle = 100000.0 * 500.0 ** (-2 * i / 6)
    assert (t[100000].double() - torch.cat([angle.cos(), angle.sin()])).abs().max() <= 2.0 ** -24
    for wrong in ((0, 4), (4, 3), (4, 0)):
        with pytest.raises(ValueError):
            pkg.rotary_table(*wrong, device="cpu")
