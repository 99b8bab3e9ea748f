"""A run of the generation operators together, as a program uses them: prompts of different lengths, one of them prefilled in pieces, decoding steps
of all sequences at once, each token drawn from the logits.

Every attention of every layer and step is compared with the 64-bit attention over all rows that the layer's projection has
given for the sequence so far (rounded to the cache's type), within the tolerance of test_paged_gpu.py; the drawn tokens are
those of the definition on the step's logits.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
C, H, V, LAYERS, BLOCK = 128, 2, 500, 2, 64
E = 2.0 ** -24


class Model:
    """A GPT of this library's entry points, its residual and head left to torch.  `seen`: what each layer's projection gave and
    what its attention made of it, in the last step."""

    def __init__(self, pkg, dtype):
        g = torch.Generator(device="cuda")
        g.manual_seed(5)
        make = lambda *shape: torch.empty(shape, device="cuda").normal_(0.0, 0.1, generator=g)  # noqa: E731
        self.pkg, self.wte, self.wpe = pkg, make(V, C), make(BLOCK, C)
        self.layers = [dict(qkv=make(3 * C, C), proj=make(C, C), ln=1 + make(C)) for _ in range(LAYERS)]
        self.k, self.v = ([torch.zeros(40, H, 8, C // H, device="cuda", dtype=dtype) for _ in range(LAYERS)] for _ in range(2))

    def step(self, tokens, table, cu, past, positions, max_new):
        x, self.seen = self.wte[tokens] + self.wpe[positions], []
        for n, w in enumerate(self.layers):
            h, _, _ = self.pkg.layernorm_forward(x, w["ln"])
            cache = (self.k[n], self.v[n], table, cu, past)
            qkv = self.pkg.linear_forward(h, w["qkv"])
            out = self.pkg.paged_attention(self.pkg.paged_append(qkv, *cache), *cache, max_new=max_new)
            self.seen.append((qkv, out))
            x = x + self.pkg.linear_forward(out, w["proj"])
        return x @ self.wte.T


def attention(rows, count, dtype):
    """The last `count` rows' attention over all rows [positions, 3C] of a sequence, in 64 bits, and what fp32 may be off by."""
    D = C // H
    q, k, v = (t.view(-1, H, D).transpose(0, 1) for t in rows.split(C, 1))
    q, k, v = q[:, -count:].double(), k.to(dtype).double(), v.to(dtype).double()
    seen = torch.ones(count, k.shape[1], dtype=torch.bool, device="cuda").tril(k.shape[1] - count)
    z = (q @ k.transpose(1, 2) * D ** -0.5).masked_fill(~seen, float("-inf"))
    size = (q.abs() @ k.abs().transpose(1, 2) * D ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    p = torch.softmax(z, -1)
    return tuple(t.transpose(0, 1).reshape(count, C) for t in (p @ v, 2 * (size * (D + 5) + k.shape[1] + 8) * E * (p @ v.abs())))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_generation(pkg, dtype):
    from test_sample_gpu import plain

    model = Model(pkg, dtype)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(V, (n,), generator=g).tolist() for n in (1, 9, 30)]
    table = ints(torch.randperm(40, generator=g)[:24].view(3, 8).tolist())
    done = [0, 0, 0]
    history = [[torch.empty(0, 3 * C, device="cuda") for _ in texts] for _ in range(LAYERS)]
    settings = dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)
    for _ in range(24):
        # the prompt of 30 comes in pieces of 13, next to the sequences that already decode
        new = [min(13, len(t) - d) for t, d in zip(texts, done)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        tokens = torch.tensor([x for t, d, n in zip(texts, done, new) for x in t[d:d + n]], device="cuda")
        positions = torch.tensor([d + i for d, n in zip(done, new) for i in range(n)], device="cuda")
        logits = model.step(tokens, table, ints(cu), ints(done), positions, max(new))
        for past, (qkv, out) in zip(history, model.seen):
            for s, n in enumerate(new):
                past[s] = torch.cat([past[s], qkv[cu[s]:cu[s + 1]]])
                want, tol = attention(past[s], n, dtype)
                assert bool(((out[cu[s]:cu[s + 1]].double() - want).abs() <= tol).all())
        last = logits[torch.tensor(cu[1:], device="cuda") - 1]
        u = torch.rand(3, generator=g).cuda()
        per_row = lambda name, t: torch.full((3,), settings[name], dtype=t, device="cuda")  # noqa: E731
        drawn = pkg.sample(last, u, per_row("temperature", torch.float32), per_row("top_k", torch.int32), per_row("top_p", torch.float32),
                           per_row("min_p", torch.float32)).tolist()
        rounded = {n: torch.tensor(v, dtype=torch.float32).item() if n != "top_k" else v for n, v in settings.items()}
        assert drawn == [plain(last[s], u[s].item(), **rounded) for s in range(3)]
        for s in range(3):
            done[s] += new[s]
            if done[s] == len(texts[s]):
                texts[s].append(drawn[s])
    assert all(len(t) > 20 for t in texts)
    assert pkg.device_status() == 0
