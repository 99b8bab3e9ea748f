"""Generation with a paged key/value cache, and the draw of the next token: what is measured of these operators.

A case is a dict of plain values, ``kind`` first:

  append   the keys and values of a step's new tokens, rotated by their positions where the model rotates, into the
           pages of their sequences (pkg.paged_append)
  attend   attention of a step's new tokens over their sequences' pages (pkg.paged_attention): one token of each
           sequence in a decoding step, a piece of a prompt in a prefill step, both in a mixed one
  sample   the next token of each row of logits, by temperature, top-k, top-p and min-p, from given random numbers
           (pkg.sample)

``prepare`` makes what a program holds before the call, ``run`` makes the call and returns everything that it produces.
Lengths and page tables are part of a case and do not depend on the seed.
"""
import importlib.util
import os
import random
import sys

import torch

own = False
VOCAB = 50257  # classes of the GPT-2 tokenizer


def package():
    """The package directory has a dot in its name, so it is loaded by path (from the working folder)."""
    if "gptc_b200" not in sys.modules:
        here = os.path.join(os.getcwd(), "gpt.c_b200")
        spec = importlib.util.spec_from_file_location("gptc_b200", os.path.join(here, "__init__.py"),
                                                      submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["gptc_b200"] = mod
        spec.loader.exec_module(mod)
        mod.init()
    return sys.modules["gptc_b200"]


def _cache(kind, name, **more):
    c = {"name": name, "kind": kind, "seqs": 1, "singles": 0, "new": [1, 1], "past": [0, 0], "heads": 12, "kv_heads": 12, "D": 64, "page": 16,
         "dtype": "bf16", "rotary": 0, "pairs": False}
    c.update(more)
    for key in ("new", "past"):
        c[key + "_lo"], c[key + "_hi"] = c.pop(key)
    return c


def listed():
    return [
        # one decoding step of a batch of GPT-2 124M sequences: nothing but latency
        _cache("append", "append_decode", seqs=24, past=[10, 1000]),
        # pieces of prompts of a model that rotates its positions, heads shared by four queries
        _cache("append", "append_prefill_rotary", seqs=7, new=[300, 2000], past=[0, 3000], heads=20, kv_heads=5, D=128, page=32, rotary=128),
        # GPT-2 XL width in fp32, part of each head rotated in pairs of neighbours, pages of an odd size
        _cache("append", "append_fp32_pairs", seqs=5, new=[100, 1200], heads=25, kv_heads=25, page=24, dtype="fp32", rotary=32, pairs=True),
        # infer_gpt's single sequence near the end of the GPT-2 block of 1024, in fp32 throughout: the smallest call
        _cache("attend", "decode_one_fp32", past=[1000, 1000], dtype="fp32"),
        # a decoding step of a full batch within GPT-2's block size
        _cache("attend", "decode_batch", seqs=96, past=[30, 1022]),
        # long contexts of few sequences, heads shared by four queries
        _cache("attend", "decode_long_shared", seqs=6, past=[9000, 40000], heads=20, kv_heads=5, D=128, page=64),
        # pieces of long prompts over what is already cached: the largest call
        _cache("attend", "prefill_long", seqs=4, new=[700, 1024], past=[3500, 7000], page=32),
        # short prompts from their start, GPT-2 XL heads, fp32 pages
        _cache("attend", "prefill_fp32", seqs=6, new=[60, 500], past=[0, 100], heads=25, kv_heads=25, dtype="fp32"),
        # a serving step: most sequences decode, two bring pieces of their prompts
        _cache("attend", "mixed_step", seqs=34, singles=32, new=[200, 500], past=[100, 2000], heads=20, kv_heads=5, D=128),
        # one sequence, as infer_gpt draws: temperature alone, and here top-k
        {"name": "sample_one", "kind": "sample", "rows": 1, "V": VOCAB, "t": True, "k": 40, "p": 0.0, "m": 0.0, "spread": 2.5},
        # a decoding step's rows, nucleus and smallest probability
        {"name": "sample_batch", "kind": "sample", "rows": 96, "V": VOCAB, "t": True, "k": 0, "p": 0.92, "m": 0.02, "spread": 2.5},
        # many rows, every restriction at once
        {"name": "sample_many", "kind": "sample", "rows": 500, "V": VOCAB, "t": True, "k": 1000, "p": 0.95, "m": 0.001, "spread": 2.0},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "mixed", "sample", "sample"])
    if kind == "sample":
        return {"kind": "sample", "rows": _log(rng, 1, 500), "V": rng.choice([VOCAB, VOCAB, 50304, _log(rng, 20, 120000)]) if rng.random() < 0.8 else 32000,
                "t": rng.random() < 0.8, "k": rng.choice([0, 1, 40, _log(rng, 1, 5000)]), "p": rng.choice([0.0, 0.5, 0.9, 0.99]),
                "m": rng.choice([0.0, 0.0, 0.05, 0.3]), "spread": round(rng.uniform(0.5, 4.0), 2)}
    kv = rng.choice([1, 2, 5, 8, 12, 12, 20, 25])
    heads = kv * (1 if kv >= 12 else rng.choice([1, 2, 3, 4, 8]))
    D = rng.choice([64, 64, 64, 128, 128, 32, 40, 80, 96])
    c = {"heads": heads, "kv_heads": kv, "D": D, "page": rng.choice([8, 16, 16, 24, 32, 64, 100, 128]), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    c.update({"rotary": 0, "pairs": False, "singles": 0, "new_lo": 1, "new_hi": 1, "past_lo": 0})
    if kind == "append":
        c.update(seqs=_log(rng, 1, 64), new_hi=_log(rng, 1, 2000), past_hi=rng.randint(0, 3000), rotary=rng.choice([0, D, D // 4 * 2]), pairs=rng.random() < 0.3)
        while c["seqs"] * c["new_hi"] * (heads + 2 * kv) * D > 30e6:
            c["seqs"] -= c["seqs"] // 8 + (c["seqs"] > 1)
            c["new_hi"] -= c["new_hi"] // 8
    elif kind == "decode":
        c.update(seqs=_log(rng, 1, 128), past_hi=_log(rng, 1, 40000))
        c["new_hi"] = rng.choice([1, 1, 1, 2, 4])
        while c["seqs"] * c["past_hi"] * kv * D > 130e6 or c["seqs"] * c["past_hi"] * heads * c["new_hi"] > 6e7:
            c["seqs"] -= c["seqs"] // 8 + (c["seqs"] > 1)
            c["past_hi"] -= c["past_hi"] // 8
    else:
        c.update(seqs=_log(rng, 1, 16), new_hi=_log(rng, 8, 1024), past_hi=_log(rng, 1, 7000))
        if kind == "mixed":
            c["seqs"] = max(2, c["seqs"])
            c["singles"] = c["seqs"] - 1 - rng.randint(0, c["seqs"] // 2 - 1)
        else:
            c["new_lo"] = c["new_hi"] // 2 + 1
        while c["seqs"] * heads * c["new_hi"] * (c["past_hi"] + c["new_hi"]) * max(D, 64) > (1.2e10 if c["dtype"] == "bf16" else 4e9):
            c["past_hi"] -= c["past_hi"] // 8
            c["new_hi"] -= c["new_hi"] // 8
            c["new_lo"] = min(c["new_lo"], c["new_hi"])
    return {"kind": "append" if kind == "append" else "attend", **c}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """New tokens and cached tokens of each sequence: whole ranges, the largest of both among them."""
    r = random.Random(case["seqs"] * 1009 + case["past_hi"] * 31 + case["new_hi"])
    new = [1 if s < case["singles"] else r.randint(case["new_lo"], case["new_hi"]) for s in range(case["seqs"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    new[-1], past[-1] = case["new_hi"], case["past_hi"]
    return new, past


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_cache(case, seed):
    g = _generator(seed)
    new, past = _lengths(case)
    P, H, KV, D = case["page"], case["heads"], case["kv_heads"], case["D"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    need = [(a + b + P - 1) // P for a, b in zip(new, past)]
    pages = sum(need) + 3
    order = list(range(pages))
    random.Random(pages).shuffle(order)  # pages are handed out as they come free
    width, table, at = max(need), [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"kind": case["kind"], "H": H, "KV": KV, "D": D, "max_new": max(new), "longest": max(a + b for a, b in zip(new, past)),
         "table": _ints(table), "cu": _ints(cu), "past": _ints(past)}
    for name in ("k_pages", "v_pages"):  # keys and values as projections give them: about a standard deviation of 1
        s[name] = torch.empty((pages, KV, P, D), device="cuda", dtype=dtype).normal_(0.0, 1.0, generator=g)
    if case["kind"] == "attend":
        s["q"] = torch.empty((cu[-1], H * D), device="cuda").normal_(0.0, 1.0, generator=g)
        return s
    s["qkv"] = torch.empty((cu[-1], (H + 2 * KV) * D), device="cuda").normal_(0.0, 1.0, generator=g)
    s["rotary"], s["pairs"] = None, case["pairs"]
    if case["rotary"]:
        R = case["rotary"]
        angle = torch.arange(s["longest"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        s["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return s


def _prepare_sample(case, seed):
    g = _generator(seed)
    rows, V = case["rows"], case["V"]
    s = {"kind": "sample", "logits": torch.empty((rows, V), device="cuda").normal_(0.0, case["spread"], generator=g),
         "u": torch.rand(rows, device="cuda", generator=g), "temperature": None, "top_k": None, "top_p": None, "min_p": None}
    near = torch.rand(rows, device="cuda", generator=g)  # rows of one batch come from requests with settings of their own
    if case["t"]:
        s["temperature"] = 0.6 + 0.6 * near
    if case["k"]:
        s["top_k"] = (case["k"] * (0.5 + near)).round().clamp(min=1).int()
    if case["p"]:
        s["top_p"] = case["p"] * (0.9 + 0.1 * near)
    if case["m"]:
        s["min_p"] = case["m"] * (0.5 + near)
    return s


def prepare(case, seed):
    return (_prepare_sample if case["kind"] == "sample" else _prepare_cache)(case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _tokens(s, count):
    """The sequence and the position of each new token."""
    t = torch.arange(count, device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    return seq, t - s["cu"].long()[seq], s["past"].long()[seq] + t - s["cu"].long()[seq]


def _rotate(x, table, pairs):
    """x [tokens, heads, D], table [tokens, R]: the first R columns of each head, by the angle of their token."""
    R = table.shape[1]
    cos, sin = table[:, None, :R // 2], table[:, None, R // 2:]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if pairs else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1), x[..., R:]], -1)


def _plain_append(s):
    qkv, H, KV, D, P = s["qkv"], s["H"], s["KV"], s["D"], s["k_pages"].shape[2]
    seq, _, at = _tokens(s, qkv.shape[0])
    q, k, v = qkv.view(-1, H + 2 * KV, D).split([H, KV, KV], 1)
    if s["rotary"] is not None:
        q, k = _rotate(q, s["rotary"][at], s["pairs"]), _rotate(k, s["rotary"][at], s["pairs"])
    page, row = s["table"].long()[seq, at // P], at % P
    s["k_pages"][page, :, row] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, :, row] = v.to(s["v_pages"].dtype)
    return q.reshape(-1, H * D), s["k_pages"], s["v_pages"]


def _plain_attend(s):
    H, KV, D, P, S = s["H"], s["KV"], s["D"], s["k_pages"].shape[2], s["past"].shape[0]
    count = s["q"].shape[0]
    cu, past = s["cu"].long(), s["past"].long()
    i, j = torch.arange(s["max_new"], device="cuda"), torch.arange(s["longest"], device="cuda")
    page = s["table"].long()[:, j // P]
    k, v = (s[name][page, :, j % P].float() for name in ("k_pages", "v_pages"))  # [S, keys, KV, D]
    q = s["q"].view(count, KV, H // KV, D)[(cu[:-1, None] + i).clamp(max=count - 1)]
    scores = torch.einsum("sihgd,sjhd->shgij", q, k) * D ** -0.5
    seen = (j <= past[:, None, None] + i[:, None])[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    out = torch.einsum("shgij,sjhd->sihgd", p / p.sum(-1, keepdim=True), v)
    seq, new, _ = _tokens(s, count)
    return out[seq, new].reshape(count, H * D)


def _plain_sample(s):
    x = s["logits"].double()
    rows, V = x.shape
    one = lambda v, other: torch.full((rows, 1), other, device="cuda", dtype=torch.float64) if v is None else v.double()[:, None]  # noqa: E731
    w = ((x - x.amax(-1, keepdim=True)) / one(s["temperature"], 1.0)).exp()  # 64 bits: the draw's borders are as near as 1e-9
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(V, device="cuda")
    kept = rank < one(s["top_k"], V)
    below = torch.where(kept, sorted_w, 0.0).cumsum(-1)
    kept = kept & ((below - sorted_w < one(s["top_p"], 2.0) * below[:, -1:]) | (rank == 0)) & (sorted_w >= one(s["min_p"], 0.0))
    w = w * torch.zeros_like(w).scatter_(1, order, kept.double())
    total = w.cumsum(-1)
    return (total <= s["u"].double()[:, None] * total[:, -1:]).sum(-1).int()


def run(s):
    if own:
        pkg = package()
        if s["kind"] == "append":
            q = pkg.paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["past"], rotary=s["rotary"], rotary_pairs=s["pairs"])
            return q, s["k_pages"], s["v_pages"]
        if s["kind"] == "attend":
            return pkg.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["past"], max_new=s["max_new"])
        return pkg.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["V"]
        return {"bytes": 4 * n + 8 * case["rows"], "flops": 3 * n}
    new, past = _lengths(case)
    H, KV, D, each = case["heads"], case["kv_heads"], case["D"], 2 if case["dtype"] == "bf16" else 4
    tokens = sum(new)
    if case["kind"] == "append":
        moved = tokens * 2 * KV * D * (4 + each)
        if case["rotary"]:
            moved += tokens * H * D * 8 + 4 * case["rotary"] * tokens
        return {"bytes": moved, "flops": 3 * tokens * (H + KV) * case["rotary"]}
    cached = sum(a + b for a, b in zip(new, past))
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, past))
    return {"bytes": cached * 2 * KV * D * each + tokens * H * D * 8, "flops": 4 * seen * H * D}


def _exact_cache(case, seed):
    s = _prepare_cache(case, seed)
    new, past = _lengths(case)
    P, H, KV, D = case["page"], case["heads"], case["kv_heads"], case["D"]
    table = s["table"].tolist()
    at, outs = 0, []
    if case["kind"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        q = s["qkv"].double()[:, :H * D].reshape(-1, H, D).clone()
        k = s["qkv"].double()[:, H * D:(H + KV) * D].reshape(-1, KV, D).clone()
        v = s["qkv"].double()[:, (H + KV) * D:].reshape(-1, KV, D)
        where = torch.tensor([table[n][p // P] * P + p % P for n in range(len(new)) for p in range(past[n], past[n] + new[n])], device="cuda")
        where_at = torch.tensor([p for n in range(len(new)) for p in range(past[n], past[n] + new[n])], device="cuda")
        if case["rotary"]:
            R = case["rotary"]
            c, d = s["rotary"].double()[where_at, :R // 2], s["rotary"].double()[where_at, R // 2:]
            for x in (q, k):
                turned = torch.view_as_complex(torch.stack([c, d], -1))[:, None]
                first = x[..., :R].reshape(*x.shape[:2], R // 2, 2) if case["pairs"] else x[..., :R].reshape(*x.shape[:2], 2, R // 2).transpose(-1, -2)
                y = torch.view_as_real(torch.view_as_complex(first.contiguous()) * turned)
                x[..., :R] = (y if case["pairs"] else y.transpose(-1, -2)).reshape(*x.shape[:2], R)
        for pages, rows in ((k_pages, k), (v_pages, v)):
            pages.transpose(1, 2)[where // P, where % P] = rows
        return q.reshape(-1, H * D), k_pages, v_pages
    if 4 * H * D * sum(a * (a + b) for a, b in zip(new, past)) > 1e12:
        return None
    for n in range(len(new)):
        ctx = past[n] + new[n]
        used = s["table"][n, :(ctx + P - 1) // P].long()
        k, v = (s[name][used].double().transpose(0, 1).reshape(KV, -1, D)[:, :ctx].repeat_interleave(H // KV, 0) for name in ("k_pages", "v_pages"))
        q = s["q"][at:at + new[n]].double().view(new[n], H, D).transpose(0, 1)
        z = torch.matmul(q, k.transpose(1, 2)) / D ** 0.5
        z = z + torch.full((new[n], ctx), float("-inf"), device="cuda", dtype=torch.float64).triu(past[n] + 1)
        outs.append(torch.matmul(torch.exp(z - torch.logsumexp(z, -1, keepdim=True)), v).transpose(0, 1).reshape(new[n], H * D))
        at += new[n]
    return torch.cat(outs)


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    found = []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        if s["temperature"] is not None:
            x = x / s["temperature"][r].double()
        z, order = torch.sort(torch.softmax(x, -1), descending=True, stable=True)
        n = case["V"] if s["top_k"] is None else min(case["V"], int(s["top_k"][r]))
        z, order = z[:n], order[:n]
        if s["top_p"] is not None:
            before = torch.cumsum(z, 0) - z
            n = max(1, int((before < s["top_p"][r].double() * z.sum()).sum()))
        if s["min_p"] is not None:
            n = min(n, int((z[:n] >= s["min_p"][r].double() * z[0]).sum()))
        by_index = torch.argsort(order[:n])
        c = torch.cumsum(z[:n][by_index], 0)
        found.append(order[:n][by_index][int(torch.searchsorted(c, s["u"][r].double() * c[-1], right=True).clamp(max=n - 1))])
    return torch.stack(found).int()


def exact(case, seed):
    return (_exact_sample if case["kind"] == "sample" else _exact_cache)(case, seed)
