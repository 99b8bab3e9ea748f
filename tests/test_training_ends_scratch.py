"""The scratch buffer of the projection's gradients against what its header says it holds."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

P = ctypes.c_void_p(1 << 20)


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("rows,V,K", [(8192, 50257, 768), (4096, 50257, 768), (16384, 50257, 768), (32768, 50257, 768), (3001, 50257, 1600), (1 << 17, 50257, 768), (8192, 128000, 64)])
def test_linear_xent_backward(pkg, rows, V, K, type):
    """G of two pieces of the vocabulary, each of 256 MB, or 16384 bytes a row (fp32 32768) where that is more; x as bf16 planes, w too if fp32; dx in fp32.  (8192 x 50257 bf16: two
    pieces of 210 MB, where the logits take 823 MB.)"""
    planes = 2 if type == 0 else 1
    G = 2 * max(256 << 20, 16384 * planes * rows)
    held = rows * K * 2 * planes + rows * K * 4 + (V * K * 2 * planes if type == 0 else 0)
    got = pkg.lib().xent_sm100_linear_backward_scratch_bytes(P, P, K, K, type, rows, V, K)
    assert held < got <= G + held + 4096
    if (rows, V, K, type) == (8192, 50257, 768, 1):
        assert abs(got - held - 2 * rows * 50 * 256 * 2) < 4096
