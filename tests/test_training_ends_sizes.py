"""Sizes that the entry points at both ends of a training step do not take: their scratch size is 0, and what the call says is that the size is not supported, with or without a
scratch buffer.  Nothing here reaches a GPU.
"""
import pytest

torch = pytest.importorskip("torch")

from test_training_ends import EMBED_GRAD, LOSS, LOSS_GRAD, NULL, UNSUPPORTED, P  # noqa: E402

WIDE = dict(C=(1 << 20) + 1, ld=1 << 21, ld_dy=1 << 21, pos_ld=1 << 21)


@pytest.mark.parametrize("wrong", [dict(n=(1 << 30) + 1), WIDE, dict(V=(1 << 30) + 1), dict(Pn=(1 << 30) + 1, positions=P)])
def test_embedding_backward(pkg, wrong):
    a = {**EMBED_GRAD, **wrong}
    assert pkg.lib().tensor_sm100_embedding_backward_scratch_bytes(a["n"], a["C"], a["V"], a["Pn"] if a["positions"] else 0) == 0
    for scratch in (a["scratch"], None):
        assert pkg.lib().tensor_sm100_embedding_backward(*{**a, "scratch": scratch}.values()) == UNSUPPORTED
    assert pkg.lib().tensor_sm100_embedding_backward(*{**EMBED_GRAD, "scratch": None}.values()) == NULL


LONG = dict(K=(1 << 24) + 1, ldx=1 << 25, ldw=1 << 25)
HEAD = [dict(rows=(1 << 30) + 1), dict(V=(1 << 30) + 1), LONG, dict(ldx=(1 << 34) + 8), dict(ldw=(1 << 34) + 8), dict(rows=1 << 30, V=1 << 30)]


@pytest.mark.parametrize("wrong", HEAD)
def test_linear_xent_forward(pkg, wrong):
    a = {**LOSS, **wrong}
    assert pkg.lib().xent_sm100_linear_forward_scratch_bytes(*(a[k] for k in ("x", "w", "ldx", "ldw", "type", "rows", "V", "K"))) == 0
    for scratch in (P, None):
        assert pkg.lib().xent_sm100_linear_forward(*{**a, "scratch": scratch}.values()) == UNSUPPORTED
    assert pkg.lib().xent_sm100_linear_forward(*{**LOSS, "scratch": None}.values()) == NULL


@pytest.mark.parametrize("wrong", HEAD + [dict(rows=(1 << 20) + 1)])
def test_linear_xent_backward(pkg, wrong):
    a = {**LOSS_GRAD, **wrong, "lddw": 1 << 25}
    assert pkg.lib().xent_sm100_linear_backward_scratch_bytes(*(a[k] for k in ("x", "w", "ldx", "ldw", "type", "rows", "V", "K"))) == 0
    for scratch in (P, None):
        assert pkg.lib().xent_sm100_linear_backward(*{**a, "scratch": scratch}.values()) == UNSUPPORTED
    assert pkg.lib().xent_sm100_linear_backward(*{**LOSS_GRAD, "scratch": None}.values()) == NULL
