"""Both ends of a language model in training and scoring: what is measured of the embedding and of the loss that keeps no logits.

A case is a dict of plain values, ``kind`` first:

  embed        rows of the token table, scaled, and of the position table, added (pkg.embedding_forward)
  embed_grad   the gradients of both tables, added to what they hold (pkg.embedding_backward)
  loss         vocabulary projection and cross-entropy of each row, without its logits in memory (pkg.linear_xent_forward)
  loss_grad    the same with the gradients of its input and of the weights, as a training step makes both calls
               (pkg.linear_xent_forward, pkg.linear_xent_backward)

``prepare`` makes what a program holds before the call, ``run`` makes the call and returns everything that it produces.
"""
import importlib.util
import math
import os
import sys

import torch

own = False
VOCAB = 50257  # classes of the GPT-2 tokenizer
IGNORED = -100  # the target of a row that has none


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


def _embed(kind, name, **more):
    """B sequences of T tokens; positions: "none", "rows" (a token's place in its sequence) or "given" (one number a token);
    pad: share of the tokens that are the padding token; grad: type of the tables' gradients."""
    c = {"name": name, "kind": kind, "B": 1, "T": 1024, "V": VOCAB, "C": 768, "P": 1024, "dtype": "fp32", "grad": "fp32", "ids": "int64",
         "positions": "rows", "scale": 1.0, "pad": 0.0}
    return {**c, **more}


def _loss(kind, name, **more):
    """rows of K features against V classes; spread: standard deviation of a row's logits; ignored: share of the rows without a
    target; weights: a factor for each row instead of one for all."""
    c = {"name": name, "kind": kind, "rows": 8192, "K": 768, "V": VOCAB, "dtype": "bf16", "ids": "int64", "spread": 2.0, "ignored": 0.0, "weights": False}
    return {**c, **more}


def listed():
    return [
        # one decoding step of a batch of GPT-2 124M sequences, each at a position of its own: nothing but latency
        _embed("embed", "embed_decode", B=24, T=1, positions="given", dtype="bf16"),
        # the training batch of GPT-2 124M as train_gpt runs it
        _embed("embed", "embed_gpt2", B=8),
        # packed sequences at GPT-2 XL width, a table that is scaled by the root of its width, no positions
        _embed("embed", "embed_wide_scaled", B=64, C=1600, dtype="bf16", positions="none", scale=40.0, ids="int32"),
        # a short fine-tuning batch: one sequence
        _embed("embed_grad", "embed_grad_one", T=130),
        # the training batch of GPT-2 124M
        _embed("embed_grad", "embed_grad_gpt2", B=8),
        # a large batch of bf16 gradients at XL width, half of it padding: one row of the table takes half of the batch
        _embed("embed_grad", "embed_grad_padded", B=48, C=1600, dtype="bf16", grad="bf16", pad=0.5, positions="rows", scale=40.0, ids="int32"),
        # scoring one short text: the weights have to be read, little else
        _loss("loss", "loss_short", rows=40),
        # evaluation of a validation batch
        _loss("loss", "loss_eval", rows=8192),
        # the same in fp32, as train_gpt holds its tensors
        _loss("loss", "loss_eval_fp32", rows=2048, dtype="fp32", ids="int32"),
        # training step of GPT-2 124M, bf16 activations and weights
        _loss("loss_grad", "train_gpt2"),
        # the same in fp32; a tenth of the rows are prompts without a target, rows have weights of their own
        _loss("loss_grad", "train_gpt2_fp32", rows=4096, dtype="fp32", ignored=0.1, weights=True),
        # XL width, odd numbers of rows
        _loss("loss_grad", "train_xl_odd", rows=3001, K=1600, ignored=0.2),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "loss", "loss_grad", "loss_grad"])
    dtype = rng.choice(["bf16", "fp32"])
    ids = rng.choice(["int64", "int32"])
    V = rng.choice([VOCAB, VOCAB, 50304, _log(rng, 2, 128000)])
    if kind in ("embed", "embed_grad"):
        T = _log(rng, 1, 1024)
        B = _log(rng, 1, 64)
        C = rng.choice([768, 768, 1024, 1600, _log(rng, 8, 2048)])
        positions = rng.choice(["none", "rows", "rows", "given"])
        return {"kind": kind, "B": B, "T": T, "V": V, "C": C, "P": max(T, rng.choice([1, 1024])), "dtype": dtype, "grad": rng.choice(["fp32", dtype]), "ids": ids,
                "positions": positions, "scale": rng.choice([1.0, round(math.sqrt(C), 4)]), "pad": rng.choice([0.0, 0.0, 0.3, 0.9])}
    rows = _log(rng, 1, 8192)
    K = rng.choice([768, 768, 1024, 1600, _log(rng, 8, 1600)])
    most = (3.0e11 if dtype == "bf16" else 1.5e11) * (1.0 if kind == "loss_grad" else 1.05)
    while rows * K * V > most:
        rows -= rows // 8
    return {"kind": kind, "rows": rows, "K": K, "V": V, "dtype": dtype, "ids": ids, "spread": round(rng.uniform(0.3, 4.0), 2),
            "ignored": rng.choice([0.0, 0.0, 0.1, 0.7]), "weights": rng.random() < 0.4}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int32": torch.int32, "int64": torch.int64}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, std, dtype, g):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(TYPES[dtype])


def _words(count, V, g):
    """Tokens as text has them: the n-th most frequent one about as often as 1 / (n + 3), frequent ones anywhere in the table."""
    u = torch.rand(count, device="cuda", dtype=torch.float64, generator=g)
    rank = (3.0 * ((V + 3.0) / 3.0) ** u - 3.0).long().clamp(0, V - 1)
    return torch.randperm(V, device="cuda", generator=g)[rank]


def _prepare_embed(case, seed):
    g = _generator(seed)
    B, T, V, C, P = (case[k] for k in ("B", "T", "V", "C", "P"))
    ids = TYPES[case["ids"]]
    tokens = _words(B * T, V, g)
    padding = torch.rand(B * T, device="cuda", generator=g) < case["pad"]
    tokens = torch.where(padding, torch.full_like(tokens, V - 1), tokens).view(B, T).to(ids)
    s = {"kind": case["kind"], "tokens": tokens, "scale": case["scale"], "positions": None, "place": case["positions"] != "none"}
    if case["positions"] == "given":
        s["positions"] = torch.randint(P, (B, T), device="cuda", generator=g).to(ids)
    if case["kind"] == "embed":
        s["table"] = _normal((V, C), 0.02, case["dtype"], g)
        s["pos_table"] = _normal((P, C), 0.02, case["dtype"], g) if s["place"] else None
    else:
        s["dy"] = _normal((B, T, C), 1e-3, case["dtype"], g)
        s["dtable"] = _normal((V, C), 1e-3, case["grad"], g)  # what the projection or an earlier batch has left there
        s["dpos_table"] = _normal((P, C), 1e-3, case["grad"], g) if s["place"] else None
    return s


def _prepare_loss(case, seed):
    g = _generator(seed)
    rows, K, V = case["rows"], case["K"], case["V"]
    targets = _words(rows, V, g)
    targets = torch.where(torch.rand(rows, device="cuda", generator=g) < case["ignored"], torch.full_like(targets, IGNORED), targets).to(TYPES[case["ids"]])
    s = {"kind": case["kind"], "targets": targets, "x": _normal((rows, K), 1.0, case["dtype"], g),  # a LayerNorm's output
         "w": _normal((V, K), case["spread"] / math.sqrt(K), case["dtype"], g)}
    if case["kind"] == "loss_grad":
        s["dw"] = _normal((V, K), 1e-3 / math.sqrt(K), case["dtype"], g)  # of an earlier part of the batch
        s["g"] = torch.full((1,), 1.0 / rows, device="cuda")
        if case["weights"]:
            s["g"] = (0.5 + torch.rand(rows, device="cuda", generator=g)) / rows
    return s


def prepare(case, seed):
    return (_prepare_embed if case["kind"].startswith("embed") else _prepare_loss)(case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _places(s):
    B, T = s["tokens"].shape
    return torch.arange(T, device="cuda").expand(B, T) if s["positions"] is None else s["positions"].long()


def _plain_embed(s):
    y = s["table"][s["tokens"].long()].float() * s["scale"]
    if s["place"]:
        y = y + s["pos_table"][_places(s)].float()
    return y.to(s["table"].dtype)


def _added(held, index, rows):
    """`rows` of 32 bits added to the rows of `held` that `index` names; sums in 64 bits, since a row may take half of them."""
    total = torch.zeros(held.shape, device="cuda", dtype=torch.float64).index_add_(0, index.reshape(-1), rows.reshape(-1, rows.shape[-1]).double())
    held.copy_((held.double() + total).to(held.dtype))


def _plain_embed_grad(s):
    dy = s["dy"].float()
    _added(s["dtable"], s["tokens"].long(), dy * s["scale"])
    if s["place"]:
        _added(s["dpos_table"], _places(s), dy)
    return s["dtable"], s["dpos_table"]


def _plain_loss(s, logits):
    target = s["targets"].long()
    counts = target >= 0
    top = logits.amax(-1, keepdim=True)
    lse = ((logits - top).exp().sum(-1, keepdim=True).log() + top)[:, 0]
    return torch.where(counts, lse - logits.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0), lse


def _plain_loss_grad(s):
    x, w, target = s["x"].float(), s["w"].float(), s["targets"].long()
    logits = x @ w.t()
    losses, lse = _plain_loss(s, logits)
    d = (logits - lse[:, None]).exp()
    d[torch.arange(d.shape[0], device="cuda"), target.clamp(min=0)] -= 1.0
    d = d * torch.where(target >= 0, s["g"], 0.0)[:, None]
    s["dw"].copy_((s["dw"].float() + d.t() @ x).to(s["dw"].dtype))
    return losses, lse, (d @ w).to(s["x"].dtype), s["dw"]


def run(s):
    if own:
        pkg = package()
        if s["kind"] == "embed":
            return pkg.embedding_forward(s["tokens"], s["table"], positions=s["positions"], pos_table=s["pos_table"], scale=s["scale"])
        if s["kind"] == "embed_grad":
            pkg.embedding_backward(s["dy"], s["tokens"], s["dtable"], positions=s["positions"], dpos_table=s["dpos_table"], scale=s["scale"])
            return s["dtable"], s["dpos_table"]
        losses, lse = pkg.linear_xent_forward(s["x"], s["w"], s["targets"])
        if s["kind"] == "loss":
            return losses, lse
        return losses, lse, pkg.linear_xent_backward(s["g"], s["x"], s["w"], s["targets"], lse, s["dw"]), s["dw"]
    if s["kind"] == "loss":
        return _plain_loss(s, s["x"].float() @ s["w"].float().t())
    return {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "loss_grad": _plain_loss_grad}[s["kind"]](s)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ---------------------------------------------------------------------------------------------
def work(case):
    each = 2 if case["dtype"] == "bf16" else 4
    if case["kind"].startswith("loss"):
        rows, K, V = case["rows"], case["K"], case["V"]
        moved = (rows + V) * K * each + 16 * rows
        if case["kind"] == "loss":
            return {"bytes": moved, "flops": 2.0 * rows * K * V}
        return {"bytes": moved + (rows + 2 * V) * K * each, "flops": 6.0 * rows * K * V}
    n, C, place = case["B"] * case["T"], case["C"], case["positions"] != "none"
    # rows of the tables that the tokens name, each once: the expected number of different words
    words = sum(1.0 - math.exp(-n * (1.0 - case["pad"]) * math.log((r + 4.0) / (r + 3.0)) / math.log((case["V"] + 3.0) / 3.0)) for r in range(case["V"]))
    places = 0 if not place else min(case["P"], n) if case["positions"] == "given" else case["T"]
    if case["kind"] == "embed":
        return {"bytes": (n + words + places) * C * each + 8 * n, "flops": 2 * n * C}
    return {"bytes": n * C * each + 2 * (words + places) * C * (2 if case["grad"] == "bf16" else 4) + 8 * n, "flops": (1 + place) * n * C}


def _exact_embed(case, seed):
    s = _prepare_embed(case, seed)
    at = s["tokens"].flatten().long()
    n = torch.arange(at.numel(), device="cuda")
    where = n % case["T"] if s["positions"] is None else s["positions"].flatten().long()
    if case["kind"] == "embed":
        y = torch.nn.functional.embedding(at, s["table"].double()) * case["scale"]
        if s["place"]:
            y += torch.nn.functional.embedding(where, s["pos_table"].double())
        return y.view(case["B"], case["T"], -1)

    def summed(held, index, factor):
        # by sorted index: runs of equal ones, and the differences of running sums at their ends
        order = torch.argsort(index, stable=True)
        ends = torch.searchsorted(index[order], torch.arange(held.shape[0], device="cuda"), right=True)
        run = torch.cat([torch.zeros(1, case["C"], device="cuda", dtype=torch.float64), s["dy"].view(-1, case["C"]).double()[order].cumsum(0)])
        return held.double() + factor * (run[ends] - run[torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])])

    return summed(s["dtable"], at, case["scale"]), summed(s["dpos_table"], where, 1.0) if s["place"] else None


def _exact_loss(case, seed):
    s = _prepare_loss(case, seed)
    x, w = s["x"].double(), s["w"].double()
    losses, lses, dx = [], [], []
    dw = s["dw"].double() if case["kind"] == "loss_grad" else None
    for r in range(0, case["rows"], 1024):  # in pieces of the rows
        part, target = x[r:r + 1024], s["targets"][r:r + 1024].long()
        logp = torch.log_softmax(part @ w.T, -1)
        lses.append(torch.logsumexp(part @ w.T, -1))
        losses.append(torch.nn.functional.nll_loss(logp, target, ignore_index=IGNORED, reduction="none"))
        if dw is None:
            continue
        kept = target != IGNORED
        factor = s["g"].double().expand(case["rows"])[r:r + 1024] * kept
        d = (logp.exp() - torch.nn.functional.one_hot(target * kept, case["V"])) * factor[:, None]
        dx.append(d @ w)
        dw += d.T @ part
    if dw is None:
        return torch.cat(losses), torch.cat(lses)
    return torch.cat(losses), torch.cat(lses), torch.cat(dx), dw


def exact(case, seed):
    return (_exact_embed if case["kind"].startswith("embed") else _exact_loss)(case, seed)
