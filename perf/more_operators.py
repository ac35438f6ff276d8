"""Operators at the two dense ends of a compressed model whose speed is watched: the embedding table and the head.

  embed       rows of the table for token ids, times a factor (``embed``)
  embed_grad  its gradient: the rows of the incoming gradient added up by token (``embed_grad``)
  loss        softmax cross entropy of hidden states against the rows of the head, token by token, without keeping the logits
              (``head_loss``): what scoring a text costs
  tune        the mean loss and its gradients with respect to the hidden states and the head: a training step of the head

An id or a target outside the vocabulary (-1: padding, or a prompt's tokens that are not trained on) reads zeros, has no loss and no
gradient.  Shapes are those of a Mistral-7B model (vocabulary 32000, hidden 4096) and a Gemma-3-27B model (262144, 5376, embeddings times
bf16(sqrt(5376)) = 73.5), and a small model of odd sizes.  All data is synthetic and seeded.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SKIP = -1                                                              # the id or target of a token that does not count


# ----------------------------------------------------------------------------- the cases
def _table(name, op, tokens, vocab, hidden, scale=1.0, type="bf16", skip=0.0):
    return {"name": name, "op": op, "tokens": tokens, "vocab": vocab, "hidden": hidden, "scale": scale, "type": type, "skip": skip}


def _head(name, op, tokens, vocab, hidden, skip=0.0):
    """``skip``: the share of tokens without a target."""
    return {"name": name, "op": op, "tokens": tokens, "vocab": vocab, "hidden": hidden, "skip": skip}


def listed():
    return [
        # a chat's decode step: the smallest call, latency alone
        _table("embed_1tok", "embed", 1, 32000, 4096),
        # a batch of prompts of a 27B model
        _table("embed_27b_8x1024", "embed", 8 * 1024, 262144, 5376, scale=73.5),
        # one sequence of a 7B model
        _table("embed_grad_2047", "embed_grad", 2047, 32000, 4096),
        # sixteen padded sequences of a 27B model: the largest table
        _table("embed_grad_27b_16x1024", "embed_grad", 16 * 1024, 262144, 5376, scale=73.5, skip=0.2),
        # a small model's table in fp32, sizes that are no multiple of anything
        _table("embed_grad_odd_fp32", "embed_grad", 777, 10007, 1001, type="fp32"),
        # the log-likelihood of one token: latency, and the head read once
        _head("loss_1tok", "loss", 1, 32000, 4096),
        # the perplexity of a 2048-token window of a 7B model
        _head("loss_2047", "loss", 2047, 32000, 4096),
        # a 27B model's answer after a prompt that does not count
        _head("loss_27b_1000", "loss", 1000, 262144, 5376, skip=0.3),
        # a step on a handful of tokens: reading the head and writing its gradient
        _head("tune_16tok", "tune", 16, 32000, 4096),
        # a small model, odd vocabulary, ragged tokens
        _head("tune_odd", "tune", 333, 10007, 1000),
        # two sequences of question and answer of a 7B model
        _head("tune_2x2048", "tune", 2 * 2048, 32000, 4096, skip=0.4),
        # a sequence of a 27B model: the largest step
        _head("tune_27b_2048", "tune", 2048, 262144, 5376),
    ]


def _log_int(rng, lo, hi):
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "loss", "tune"])
    skip = rng.choice([0.0, 0.0, rng.uniform(0.05, 0.9)])
    vocab = _log_int(rng, 100, 262144)
    if op in ("embed", "embed_grad"):
        type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        hidden = rng.choice([8 * _log_int(rng, 8, 672), 8 * _log_int(rng, 8, 672), _log_int(rng, 60, 5376)])
        case = _table("", op, _log_int(rng, 1, 16384 if op == "embed_grad" else 8192), vocab, hidden,
                      rng.choice([1.0, round(math.sqrt(hidden), 2)]), type, skip)
    else:
        hidden = 8 * _log_int(rng, 8, 672)
        tokens = _log_int(rng, 1, 4096)
        while tokens * vocab * hidden > 2048 * 262144 * 5376:
            tokens = tokens // 2
        case = _head("", op, tokens, vocab, hidden, skip)
    del case["name"]
    return case


def _counted(case):
    """How many tokens count (those that do not are spread over the sequence)."""
    return case["tokens"] - int(case["tokens"] * case["skip"])


def work(case):
    n, V, H = case["tokens"], case["vocab"], case["hidden"]
    live = _counted(case)
    if case["op"] in ("embed", "embed_grad"):
        size = TYPES[case["type"]].itemsize
        if case["op"] == "embed":
            return {"bytes": live * H * size + n * H * size + 8 * n, "flops": live * H}
        return {"bytes": live * H * size + V * H * size + 8 * n, "flops": live * H}
    if case["op"] == "loss":
        return {"bytes": 2 * H * (V + live) + 12 * n, "flops": 2 * live * V * H}
    return {"bytes": 2 * H * (V + live) + 2 * H * (V + n) + 8 * n + 4, "flops": 8 * live * V * H}


# ----------------------------------------------------------------------------- preparation
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (seed % 1_000_003) + 29)


def _tokens(g, case):
    """Token ids as text has them (a few of them most of the time), with the share ``skip`` of them left out."""
    n, V = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    out = torch.randperm(n, generator=g, device=DEV)[:n - _counted(case)]
    ids[out] = SKIP
    return ids


def prepare(case, seed):
    g = _gen(seed)
    n, V, H = case["tokens"], case["vocab"], case["hidden"]
    state = {"op": case["op"], "vocab": V, "ids": _tokens(g, case)}
    if case["op"] in ("embed", "embed_grad"):
        type, state["scale"] = TYPES[case["type"]], case["scale"]
        if case["op"] == "embed":
            state["table"] = torch.randn(V, H, generator=g, device=DEV, dtype=type).mul_(0.02)
        else:
            state["grad"] = torch.randn(n, H, generator=g, device=DEV, dtype=type).mul_(0.01)
        return state
    w = torch.randn(V, H, generator=g, device=DEV, dtype=torch.bfloat16).mul_(0.02)
    # normalised hidden states that lean towards the row of their target, some much, some not at all
    x = torch.randn(n, H, generator=g, device=DEV)
    lean = 6.0 * torch.rand(n, 1, generator=g, device=DEV)
    x += lean * w[state["ids"].clamp_min(0)].float() / (0.02 * math.sqrt(H))
    x = (x / x.square().mean(-1, keepdim=True).sqrt()).bfloat16()
    state["x"], state["w"] = (x.requires_grad_(), w.requires_grad_()) if case["op"] == "tune" else (x, w)
    return state


# ----------------------------------------------------------------------------- one pass
def _run_own(st):
    import cobalt_b200 as cb
    if st["op"] == "embed":
        return cb.embed(st["ids"], st["table"], st["scale"])
    if st["op"] == "embed_grad":
        return cb.embed_grad(st["grad"], st["ids"], st["vocab"], st["scale"])
    if st["op"] == "loss":
        return cb.head_loss(st["x"], st["w"], st["ids"], reduction="none")
    loss = cb.head_loss(st["x"], st["w"], st["ids"], reduction="mean")
    return (loss.detach(), *torch.autograd.grad(loss, (st["x"], st["w"])))


@torch.no_grad()
def run(st):
    if own:
        with torch.enable_grad():
            return _run_own(st)
    ids, V = st["ids"], st["vocab"]
    live = (ids >= 0) & (ids < V)
    if st["op"] == "embed":
        rows = st["table"][torch.where(live, ids, 0)].float() * st["scale"]
        return torch.where(live[:, None], rows, 0.0).to(st["table"].dtype)
    if st["op"] == "embed_grad":
        grad = st["grad"]
        total = torch.zeros(V, grad.shape[1], device=grad.device)
        total.index_add_(0, ids[live], grad[live].float())
        return (total * st["scale"]).to(grad.dtype)
    x, w = st["x"].float(), st["w"].float()
    t = torch.where(live, ids, 0)[:, None]
    logits = x @ w.T
    top = logits.amax(-1, keepdim=True)
    at = logits.gather(1, t)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    loss = torch.where(live, (top - at + torch.log(total))[:, 0], 0.0)
    if st["op"] == "loss":
        return loss
    n = live.sum().clamp_min(1)
    d = e.div_(total)
    d.scatter_add_(1, t, torch.full_like(at, -1.0))
    d.mul_(torch.where(live, 1.0 / n, 0.0)[:, None])
    return loss.sum() / n, (d @ w).bfloat16(), (d.T @ x).bfloat16()


# ----------------------------------------------------------------------------- the definition in 64 bits
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    ids, V = st["ids"], case["vocab"]
    kept = torch.nonzero((ids != SKIP)).flatten()                       # ids are inside the vocabulary otherwise
    tokens = ids[kept]
    n, H = case["tokens"], case["hidden"]
    if case["op"] == "embed":
        out = torch.zeros(n, H, dtype=torch.float64, device=DEV)
        out[kept] = case["scale"] * st["table"].index_select(0, tokens).double()
        return out
    if case["op"] == "embed_grad":
        out = torch.zeros(V, H, dtype=torch.float64, device=DEV)
        out.index_put_((tokens,), case["scale"] * st["grad"][kept].double(), accumulate=True)
        return out
    x, piece = st["x"][kept].double(), 16384
    lse = torch.full((len(kept),), -math.inf, dtype=torch.float64, device=DEV)
    for v0 in range(0, V, piece):
        lse = torch.logaddexp(lse, torch.logsumexp(torch.mm(x, st["w"][v0:v0 + piece].double().t()), 1))
    at = torch.cat([(x[i:i + 256] * st["w"][tokens[i:i + 256]].double()).sum(1) for i in range(0, len(kept), 256)])
    loss = torch.zeros(n, dtype=torch.float64, device=DEV)
    loss[kept] = lse - at
    if case["op"] == "loss":
        return loss
    dx = torch.zeros(n, H, dtype=torch.float64, device=DEV)
    dw = torch.empty(V, H, dtype=torch.float64, device=DEV)
    part = torch.zeros_like(x)
    for v0 in range(0, V, piece):
        w = st["w"][v0:v0 + piece].double()
        d = torch.exp(torch.mm(x, w.t()) - lse[:, None])
        here = torch.nonzero((tokens >= v0) & (tokens < v0 + piece)).flatten()
        d[here, tokens[here] - v0] -= 1.0
        d /= len(kept)
        part += torch.mm(d, w)
        dw[v0:v0 + piece] = torch.mm(d.t(), x)
    dx[kept] = part
    return loss.sum() / len(kept), dx, dw
