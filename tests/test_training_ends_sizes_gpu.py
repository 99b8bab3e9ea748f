"""Sizes that the Python calls at both ends of a training step do not take: the error says so."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
UNSUPPORTED = -3


def test_more_features_than_there_may_be(pkg):
    one, t = torch.ones(1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    wide, long = torch.zeros(1, (1 << 20) + 1, device="cuda"), torch.zeros(1, (1 << 24) + 1, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: pkg.embedding_forward(t, wide), lambda: pkg.embedding_backward(wide, t, torch.zeros_like(wide)), lambda: pkg.linear_xent_forward(long, long.clone(), t),
                 lambda: pkg.linear_xent_backward(one, long, long.clone(), t, torch.zeros(1, device="cuda"), torch.zeros_like(long))):
        with pytest.raises(pkg.AttnError) as e:
            call()
        assert e.value.code == UNSUPPORTED


def test_more_rows_than_the_gradients_take(pkg):
    n = (1 << 20) + 1
    x, w, t = torch.zeros(n, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(n, dtype=torch.int32, device="cuda")
    losses, lse = pkg.linear_xent_forward(x, w, t)
    with pytest.raises(pkg.AttnError) as e:
        pkg.linear_xent_backward(torch.ones(1, device="cuda"), x, w, t, lse)
    assert e.value.code == UNSUPPORTED
