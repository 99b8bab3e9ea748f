"""The projection with its loss when operands never arrive: its waits end, the call says so, and the next one is right."""
import time

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("loaded", [0, 1, 170])  # tiles, of 430: 148 CTAs have two or three each
def test_tiles_that_never_arrive(pkg, dtype, loaded):
    L = pkg.lib()
    M, K, V = 2500, 200, 7500
    x, w, t = torch.randn(M, K, device="cuda").to(dtype), torch.randn(V, K, device="cuda").to(dtype), torch.zeros(M, dtype=torch.int64, device="cuda")
    kind = int(dtype == torch.bfloat16)
    want, want_lse = pkg.linear_xent_forward(x, w, t)
    losses, lse = torch.empty_like(want), torch.empty_like(want)
    sizes = (K, K, kind, 1, M, V, K)
    scratch = torch.zeros(L.xent_sm100_linear_forward_scratch_bytes(x.data_ptr(), w.data_ptr(), K, K, kind, M, V, K), dtype=torch.uint8, device="cuda")
    assert pkg.device_status() == 0
    t0 = time.perf_counter()
    stream = torch.cuda.current_stream().cuda_stream
    args = [p.data_ptr() for p in (x, w, t, losses, lse, scratch)]
    assert L.xent_sm100_selftest_linear_wait_limit(*args, *sizes, loaded, stream) == 0
    assert pkg.device_status(clear=True) in (1302, 1304)
    assert 0.5 < time.perf_counter() - t0 < 3.0
    losses, lse = pkg.linear_xent_forward(x, w, t)  # the context, and tensor memory, are as before
    assert torch.equal(losses, want) and torch.equal(lse, want_lse) and pkg.device_status() == 0
    assert L.xent_sm100_selftest_linear_wait_limit(*args, *sizes, 1 << 30, stream) == 0  # everything is loaded
    assert pkg.device_status() == 0


def test_argument_range(pkg):
    L = pkg.lib()
    x = torch.zeros(100, 8, device="cuda")
    held = [torch.zeros(1 << 18, device="cuda") for _ in range(4)]  # targets, losses, lse, scratch
    args = (x.data_ptr(), x.data_ptr(), *(h.data_ptr() for h in held))
    assert L.xent_sm100_selftest_linear_wait_limit(*args, 8, 8, 0, 1, 100, 100, 8, -1, None) == -2
    assert L.xent_sm100_selftest_linear_wait_limit(*args, 8, 8, 0, 1, 16, 100, 8, 0, None) == -2  # rows that go another way
