"""Sizes that the entry points at both ends of a training step do not take: their scratch size is 0, and what the call says is that the size is not supported, with or without a
scratch buffer.  Nothing here reaches a GPU.
"""
import pytest

torch = pytest.importorskip("torch")

from test_training_ends import EMBED_GRAD, LOSS, LOSS_GRAD, NULL, UNSUPPORTED, P, without  # noqa: E402

WIDE = dict(C=(1 << 20) + 1, ld=1 << 21, ld_dy=1 << 21, pos_ld=1 << 21)


@pytest.mark.parametrize("wrong", [dict(n=(1 << 30) + 1), WIDE, dict(V=(1 << 30) + 1), dict(Pn=(1 << 30) + 1, positions=P)])
def test_embedding_backward(pkg, wrong):
    a = {**EMBED_GRAD, **wrong}
    assert pkg.lib().tensor_sm100_embedding_backward_scratch_bytes(a["n"], a["C"], a["V"], a["Pn"] if a["positions"] else 0) == 0
    for scratch in (a["scratch"], None):
        assert pkg.lib().tensor_sm100_embedding_backward(*{**a, "scratch": scratch}.values()) == UNSUPPORTED
    assert pkg.lib().tensor_sm100_embedding_backward(*{**EMBED_GRAD, "scratch": None}.values()) == NULL
