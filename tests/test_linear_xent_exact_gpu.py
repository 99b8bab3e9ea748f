"""Logits of which the tensor cores cut nothing off: whole numbers, one feature that is not zero, rows filled up with zeros.

Logits are multiplied by 1 + 0.28 2^-24 for each step of 16 features (three steps for fp32 tensors), which is what other data loses on average.  Here it is the error: |z| of the largest logit times that, and
two roundings of it and of its exponent (2^-22 in all).  Sums of exponentials add 2^-18, losses are off by the target's logit as well, and results are rounded to 2^-24.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def check(pkg, x, w, t, dtype, kept=0.0):
    """kept: what is cut off for each |x| |w|, besides."""
    M, K = x.shape
    z, size = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    want = torch.logsumexp(z, -1)
    at = z.gather(1, t[:, None])[:, 0]
    losses, lse = pkg.linear_xent_forward(x, w, t)
    steps = -(-K // 16) * (3 if dtype == F32 else 1)
    off = (z.abs() * (0.28 * steps * 2.0 ** -24 + 2.0 ** -22) + size * kept).amax(-1) + 2.0 ** -18
    assert ((lse.double() - want).abs() <= off + want.abs() * 2.0 ** -24).all()
    assert ((losses.double() - (want - at)).abs() <= 2 * off + (want - at).abs() * 2.0 ** -24).all() and pkg.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,V", [(1, 768, 5000), (16, 1600, 3000), (40, 768, 5000), (60, 4096, 1000), (300, 768, 2000), (520, 4096, 1000), (130, 1001, 999)])
def test_nothing_is_cut_off(pkg, dtype, M, K, V):
    g = torch.Generator(device="cuda")
    g.manual_seed(M + K)
    t = torch.randint(V, (M,), device="cuda", generator=g)

    def whole(rows, most):
        return torch.randint(-most, most + 1, (rows, K), device="cuda", generator=g).to(dtype)

    check(pkg, whole(M, 3), whole(V, 3), t, dtype)  # sums below 2^16
    one = torch.zeros(M, K, device="cuda", dtype=dtype)
    one[torch.arange(M), torch.randint(K, (M,), device="cuda", generator=g)] = 5.0
    check(pkg, one, whole(V, 120), t, dtype)
    filled = torch.zeros(M, K, device="cuda")  # 48 features of 24 bits: at most nine steps cut something off, and fp32 factors have 16 bits
    filled[:, :48] = torch.randn(M, 48, device="cuda", generator=g) * 10
    w = torch.randn(V, K, device="cuda", generator=g)
    check(pkg, filled.to(dtype), w.to(dtype), t, dtype, kept=3 * 2.0 ** -23 if dtype == BF16 else 9 * 2.0 ** -23 + 3 * 2.0 ** -17)
