"""Both ends of a training step together, with the weights of the projection tied to the token table as GPT-2 has them: lookup, LayerNorm, projection
with loss, and back, both gradients of the table added into one tensor.

Tolerances are for the 2-norm of the difference, relative.  fp32: products have 16 bits of each factor (3 2^-17 at most), the gradients pass through two of
them (G holds the logits' error again, at most that of z in absolute size: |z| < 16 gives 2^-12), everything else is 2^-20: 2^-11.  bf16:
x, G, dx and what is stored are rounded to 2^-8 each, five of them on the way back: 2^-5.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def off(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("B,T,C,V", [(2, 33, 64, 500), (4, 256, 128, 5001), (1, 1, 32, 50)])
def test_tied_table_fp32(pkg, B, T, C, V):
    g = torch.Generator(device="cuda")
    g.manual_seed(B * T)
    normal = lambda *s: torch.empty(*s, device="cuda").normal_(0.0, 1.0, generator=g)  # noqa: E731
    wte, wpe, gain, shift = normal(V, C) / math.sqrt(C), normal(T, C) / math.sqrt(C), 1 + 0.1 * normal(C), 0.1 * normal(C)
    tokens = torch.randint(V, (B, T), device="cuda", generator=g)
    targets = torch.roll(tokens, -1, 1)
    targets[:, -1] = -1 if T > 1 else 0
    count = (targets >= 0).sum()

    x = pkg.embedding_forward(tokens, wte, pos_table=wpe)
    y, mean, rstd = pkg.layernorm_forward(x, gain, shift)
    losses, lse = pkg.linear_xent_forward(y, wte, targets)
    dwte, dwpe, dgain, dshift, dx = (torch.zeros_like(t) for t in (wte, wpe, gain, shift, x))
    dy = pkg.linear_xent_backward((1.0 / count).float().view(1), y, wte, targets, lse, dwte)
    pkg.layernorm_backward(dy, x, mean, rstd, gain, dgain, dshift, dx)
    pkg.embedding_backward(dx, tokens, dwte, dpos_table=dwpe)

    p = [t.double().requires_grad_() for t in (wte, wpe, gain, shift)]
    h = torch.nn.functional.layer_norm(p[0][tokens] + p[1][:T], (C,), p[2], p[3], 1e-5)
    loss = torch.nn.functional.cross_entropy((h @ p[0].T).view(-1, V), targets.view(-1), ignore_index=-1)
    loss.backward()
    assert abs(losses.double().sum().item() / count.item() - loss.item()) <= 2.0 ** -11 * loss.item()
    for got, want in zip((dwte, dwpe, dgain, dshift), p):
        assert off(got, want.grad) <= 2.0 ** -11
    assert pkg.device_status() == 0


def test_tied_table_bf16(pkg):
    B, T, C, V = 3, 100, 128, 3000
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    wte = (torch.empty(V, C, device="cuda").normal_(0.0, 1.0, generator=g) / 4).bfloat16()
    tokens = torch.randint(V, (B, T), device="cuda", generator=g, dtype=torch.int32)
    x = pkg.embedding_forward(tokens, wte, scale=math.sqrt(C) / 4)
    losses, lse = pkg.linear_xent_forward(x, wte, tokens)
    dwte = torch.zeros_like(wte)
    dx = pkg.linear_xent_backward(torch.full((1,), 1.0 / (B * T), device="cuda"), x, wte, tokens, lse, dwte)
    pkg.embedding_backward(dx, tokens, dwte, scale=math.sqrt(C) / 4)
    w = wte.double().requires_grad_()
    y = w[tokens.long()] * (math.sqrt(C) / 4)
    loss = torch.nn.functional.cross_entropy((y @ w.T).view(-1, V), tokens.long().view(-1))
    loss.backward()
    assert off(dwte, w.grad) <= 2.0 ** -5


def test_steps_in_a_graph(pkg):
    """A whole step captured once and replayed on new tokens, as a training loop would."""
    B, T, C, V = 4, 64, 64, 1000
    wte = torch.randn(V, C, device="cuda") / 8
    tokens = torch.randint(V, (B, T), device="cuda")
    g = torch.ones(1, device="cuda")

    def step(dw):
        x = pkg.embedding_forward(tokens, wte)
        losses, lse = pkg.linear_xent_forward(x, wte, tokens)
        dw.zero_()
        pkg.embedding_backward(pkg.linear_xent_backward(g, x, wte, tokens, lse, dw), tokens, dw)
        return losses

    dw, other = torch.empty_like(wte), torch.empty_like(wte)
    step(dw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        losses = step(dw)
    for i in range(20):
        tokens.copy_(torch.randint(V, (B, T), device="cuda"))
        graph.replay()
        assert torch.equal(step(other), losses) and torch.equal(other, dw)
    assert pkg.device_status() == 0
