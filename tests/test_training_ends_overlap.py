"""Results of the entry points at both ends of a training step that overlap what the call reads: refused, nothing here reaches a GPU."""
import pytest

torch = pytest.importorskip("torch")

from test_training_ends import EMBED, EMBED_GRAD, LOSS, at  # noqa: E402

ARGUMENT = -8
LOOKUP = {**EMBED, "tokens": at(1 << 20), "table": at(1 << 21), "pos_table": at(1 << 22), "y": at(1 << 23), "ld": 72}
ROWS = 5 * 64 * 4  # bytes of y, and of dy


@pytest.mark.parametrize("y", [1 << 21, (1 << 21) - ROWS + 4, (1 << 21) + (99 * 72 + 63) * 4, (1 << 22) + (8 * 64 + 63) * 4, (1 << 22) - 4, (1 << 20) + 4 * 8 + 4, (1 << 20) - ROWS + 4])
def test_embedding_forward(pkg, y):
    call = pkg.lib().tensor_sm100_embedding_forward
    assert call(*{**LOOKUP, "y": at(y)}.values()) == ARGUMENT
    assert call(*{**LOOKUP, "n": 0, "y": at(y)}.values()) != ARGUMENT  # nothing is written


@pytest.mark.parametrize("wrong", [dict(tokens=at(1 << 24)), dict(tokens=at((1 << 25) + 9 * 64 * 4 - 8)), dict(positions=at((1 << 24) + 99 * 64 * 4)), dict(positions=at((1 << 25) - 8))])
def test_embedding_backward(pkg, wrong):
    call = pkg.lib().tensor_sm100_embedding_backward
    assert call(*{**EMBED_GRAD, **wrong}.values()) == ARGUMENT


SCORE = {**LOSS, "x": at(1 << 20), "w": at(1 << 21), "targets": at(1 << 22), "losses": at(1 << 23), "lse": at(1 << 24)}


@pytest.mark.parametrize("result", ["losses", "lse"])
@pytest.mark.parametrize("place", [1 << 20, (1 << 20) + 5 * 128 - 4, (1 << 20) - 16, (1 << 21) + 100 * 128 - 4, (1 << 22) + 4 * 8 + 4, (1 << 22) - 4])
def test_linear_xent_forward(pkg, result, place):
    call = pkg.lib().xent_sm100_linear_forward
    assert call(*{**SCORE, result: at(place)}.values()) == ARGUMENT
    assert call(*{**SCORE, "lse": at((1 << 23) + 16)}.values()) == ARGUMENT
    assert call(*{**SCORE, "rows": 0, result: at(place)}.values()) != ARGUMENT  # nothing is written
