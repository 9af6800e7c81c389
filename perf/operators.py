"""The operators on the two ends of the decoder's vocabulary, as cases to be measured: the log-probabilities of given
tokens with entropy and top alternatives (``custom_ops.token_logprobs``), and the scaled embedding lookup with its
gradient (``custom_ops.token_embedding``).  ``run`` computes them in elementary torch operations, or, where ``own`` is
set, with the framework's entry points."""
import math

import torch

own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one graph node's answer: the latency of a single token at the vocabulary of the translation benchmark
        {"name": "logprobs one node", "op": "logprobs", "rows": 1, "vocab": 40000, "type": "float16", "top": 5, "tokens": False,
         "train": False, "left_out": 0.0, "width": 40000},
        # the graph of one sentence (25 source tokens, four nodes each) at batch 1
        {"name": "logprobs one sentence", "op": "logprobs", "rows": 100, "vocab": 40000, "type": "float16", "top": 8, "tokens": True,
         "train": False, "left_out": 0.0, "width": 40000},
        # a decoding batch of 64 sentences of 100 nodes, with an n-best list per node
        {"name": "logprobs decoding batch", "op": "logprobs", "rows": 6400, "vocab": 40000, "type": "float16", "top": 20, "tokens": True,
         "train": False, "left_out": 0.0, "width": 40000},
        # a training batch of 40 graphs of 128 nodes: log-probability and entropy with their gradient; the nodes behind the
        # sentences' ends, a third of the batch, are left out
        {"name": "logprobs training batch", "op": "logprobs", "rows": 5120, "vocab": 40000, "type": "float16", "top": 0, "tokens": True,
         "train": True, "left_out": 0.33, "width": 40000},
        # an odd vocabulary inside a wider projection, bfloat16, the alternatives trained too
        {"name": "logprobs training odd", "op": "logprobs", "rows": 1001, "vocab": 50021, "type": "bfloat16", "top": 4, "tokens": True,
         "train": True, "left_out": 0.1, "width": 50048},
        # few rows of a very large vocabulary in float32, the longest list
        {"name": "logprobs large vocabulary", "op": "logprobs", "rows": 64, "vocab": 250007, "type": "float32", "top": 64, "tokens": True,
         "train": False, "left_out": 0.0, "width": 250007},
        # the embedding of one emitted token
        {"name": "embedding one token", "op": "embedding", "count": 1, "vocab": 40000, "dim": 512, "type": "float16", "train": False,
         "common": 0.0, "left_out": 0.0},
        # the decoder input of a training batch, forward alone
        {"name": "embedding batch", "op": "embedding", "count": 5120, "vocab": 40000, "dim": 512, "type": "float16", "train": False,
         "common": 0.6, "left_out": 0.33},
        # the same with its gradient: most nodes of a glanced graph hold one and the same token
        {"name": "embedding training batch", "op": "embedding", "count": 5120, "vocab": 40000, "dim": 512, "type": "float16",
         "train": True, "common": 0.6, "left_out": 0.33},
        # a large batch of text: token frequencies fall off with their rank
        {"name": "embedding training large", "op": "embedding", "count": 32768, "vocab": 64000, "dim": 2048, "type": "bfloat16",
         "train": True, "common": 0.0, "left_out": 0.0},
        # odd sizes in float32
        {"name": "embedding training odd", "op": "embedding", "count": 3001, "vocab": 10007, "dim": 333, "type": "float32", "train": True,
         "common": 0.2, "left_out": 0.1},
        # a long prompt batch, forward alone
        {"name": "embedding prompts", "op": "embedding", "count": 131072, "vocab": 128000, "dim": 1024, "type": "bfloat16",
         "train": False, "common": 0.0, "left_out": 0.0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["float16", "bfloat16", "float32"])
    size = 4 if kind == "float32" else 2
    if rng.random() < 0.5:
        train = rng.random() < 0.5
        vocab = _spread(rng, 200, 262144)
        rows = _spread(rng, 1, max(1, min(16384, 380000000 // (vocab * size))))
        return {"op": "logprobs", "rows": rows, "vocab": vocab, "type": kind, "top": rng.choice([0, 1, 5, 13, 20, 64]), "tokens": True,
                "train": train, "left_out": rng.choice([0.0, 0.1, 0.33]), "width": vocab + rng.choice([0, 0, 1, 24])}
    vocab = _spread(rng, 200, 262144)
    dim = _spread(rng, 16, 4096)
    while vocab * dim * size > 280000000:
        dim = max(16, dim // 2 - dim % 3)
    count = _spread(rng, 1, max(1, min(131072, 120000000 // (dim * size))))
    return {"op": "embedding", "count": count, "vocab": vocab, "dim": dim, "type": kind, "train": rng.random() < 0.6,
            "common": rng.choice([0.0, 0.2, 0.6]), "left_out": rng.choice([0.0, 0.1, 0.33])}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = _TYPES[case["type"]]
    state = {"case": dict(case)}
    if case["op"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        buffer = torch.empty((rows, case["width"]), dtype=kind, device=dev)
        step = max(1, (1 << 27) // case["width"])
        for at in range(0, rows, step):  # in pieces: the numbers are drawn in 32 bits
            part = buffer[at:at + step]
            part.copy_(torch.randn(part.shape, generator=gen, device=dev) * 3.0)
        state["logits"] = buffer[:, :vocab]
        state["tokens"] = None
        if case["tokens"]:
            tokens = torch.randint(0, vocab, (rows,), generator=gen, device=dev)
            state["tokens"] = tokens.masked_fill(torch.rand((rows,), generator=gen, device=dev) < case["left_out"], -1)
        if case["train"]:
            state["logits"].requires_grad_(True)
            # gradients of a mean over the batch, scaled as half-precision training scales its loss
            scale = 1024.0 / rows
            state["up_logprob"] = torch.randn((rows,), generator=gen, device=dev) * scale
            state["up_entropy"] = torch.randn((rows,), generator=gen, device=dev) * (0.1 * scale)
            state["up_top"] = torch.randn((rows, top), generator=gen, device=dev) * scale if top else None
        return state
    count, vocab, dim = case["count"], case["vocab"], case["dim"]
    weight = torch.empty((vocab, dim), dtype=kind, device=dev)
    weight.copy_(torch.randn((vocab, dim), generator=gen, device=dev) * dim ** -0.5)
    # ranks whose frequency falls off as 1 / rank; one token (the third) common besides; pads behind the sentences' ends
    tokens = (torch.exp(torch.rand((count,), generator=gen, device=dev, dtype=torch.float64) * math.log(vocab)).long() - 1).clamp(0, vocab - 1)
    tokens.masked_fill_(torch.rand((count,), generator=gen, device=dev) < case["common"], 3)
    tokens.masked_fill_(torch.rand((count,), generator=gen, device=dev) < case["left_out"], 1)
    state.update(weight=weight, tokens=tokens, scale=dim ** 0.5, pad=1)
    if case["train"]:
        weight.requires_grad_(True)
        up = torch.empty((count, dim), dtype=kind, device=dev)
        up.copy_(torch.randn((count, dim), generator=gen, device=dev))
        state["up"] = up
    return state


def run(state):
    case = state["case"]
    if own:
        return _own_logprobs(case, state) if case["op"] == "logprobs" else _own_embedding(case, state)
    with torch.no_grad():
        return _plain_logprobs(case, state) if case["op"] == "logprobs" else _plain_embedding(case, state)


def _own_logprobs(case, state):
    from pcfg_nat_amd import custom_ops
    logits, top = state["logits"], case["top"]
    got = custom_ops.token_logprobs(logits, state["tokens"], top=top, entropy=True)
    outs = [t for t in got if t is not None]
    if case["train"]:
        ends, ups = [got.logprobs, got.entropy], [state["up_logprob"], state["up_entropy"]]
        if top:
            ends.append(got.top_logprobs)
            ups.append(state["up_top"])
        outs += torch.autograd.grad(ends, logits, ups)
    return tuple(t.detach() for t in outs)


def _own_embedding(case, state):
    from pcfg_nat_amd import custom_ops
    out = custom_ops.token_embedding(state["weight"], state["tokens"], scale=state["scale"], padding_idx=state["pad"])
    if not case["train"]:
        return (out,)
    grad, = torch.autograd.grad(out, state["weight"], state["up"])
    return out.detach(), grad


def _plain_logprobs(case, state):
    logits, tokens, top = state["logits"], state["tokens"], case["top"]
    vocab = logits.shape[1]
    x = logits.float()
    shifted = x - x.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    probs = e / total
    lp = shifted - torch.log(total)
    entropy = -(probs * lp).sum(1)
    out = tokens < 0 if tokens is not None else torch.zeros_like(entropy, dtype=torch.bool)
    outs = []
    if tokens is not None:
        outs.append(lp.gather(1, tokens.clamp(min=0).unsqueeze(1)).squeeze(1).masked_fill(out, 0.0))
    outs.append(entropy.masked_fill(out, 0.0))
    if top:
        # one whole number per entry, ordered by value first and by index, the lowest first, behind it
        bits = (x + 0.0).view(torch.int32).long()
        ordered = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        keys = (ordered << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
        ids = vocab - 1 - (torch.topk(keys, top, dim=1).values & 0xFFFFFFFF)
        outs.append(lp.gather(1, ids).masked_fill(out.unsqueeze(1), float("-inf")))
        outs.append(ids.masked_fill(out.unsqueeze(1), -1))
    if case["train"]:
        up, up_entropy = state["up_logprob"].unsqueeze(1), state["up_entropy"].unsqueeze(1)
        over = up + (state["up_top"].sum(1, keepdim=True) if top else 0.0)
        grad = -probs * (over + up_entropy * (lp + entropy.unsqueeze(1)))
        grad.scatter_add_(1, tokens.clamp(min=0).unsqueeze(1), up)
        if top:
            grad.scatter_add_(1, ids, state["up_top"])
        outs.append(grad.masked_fill_(out.unsqueeze(1), 0.0).to(logits.dtype))
    return tuple(outs)


def _plain_embedding(case, state):
    weight, tokens, scale = state["weight"], state["tokens"], state["scale"]
    out = (weight[tokens].float() * scale).to(weight.dtype)
    if not case["train"]:
        return (out,)
    up = state["up"].float().masked_fill(tokens.eq(state["pad"]).unsqueeze(1), 0.0)
    grad = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device).index_add_(0, tokens, up)
    return out, (grad * scale).to(weight.dtype)


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "logprobs":
        live = case["rows"] * (1.0 - case["left_out"])
        numbers = live * case["vocab"]
        written = case["rows"] * (4 + 4 + 12 * case["top"])
        if case["train"]:
            return {"bytes": int(numbers * size + case["rows"] * case["vocab"] * size + written + case["rows"] * (8 + 8 + 4 * case["top"])),
                    "flops": int(10 * numbers)}
        return {"bytes": int(numbers * size + written + case["rows"] * 8), "flops": int(5 * numbers)}
    count, dim, vocab = case["count"], case["dim"], case["vocab"]
    met = min(count, vocab)  # rows of the weight that are read, at the most
    moved = (met + count) * dim * size + 8 * count
    if case["train"]:
        moved += (count + vocab) * dim * size
    return {"bytes": int(moved), "flops": int((2 if case["train"] else 1) * count * dim)}


def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        return _exact_logprobs(case, state) if case["op"] == "logprobs" else _exact_embedding(case, state)


def _exact_logprobs(case, state):
    logits, tokens, top = state["logits"].detach(), state["tokens"], case["top"]
    rows, vocab = logits.shape
    parts = []
    step = max(1, (1 << 26) // vocab)
    for at in range(0, rows, step):
        x = logits[at:at + step].double()
        n = x.shape[0]
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        p = lp.exp()
        entropy = torch.special.entr(p).sum(1)
        t = tokens[at:at + step] if tokens is not None else torch.zeros((n,), dtype=torch.long, device=x.device)
        live = t >= 0
        line = torch.arange(n, device=x.device)
        piece = []
        if tokens is not None:
            piece.append(torch.where(live, lp[line, t.clamp(min=0)], torch.zeros_like(entropy)))
        piece.append(torch.where(live, entropy, torch.zeros_like(entropy)))
        if top:
            order = x.sort(dim=1, descending=True, stable=True).indices[:, :top]
            best = lp.gather(1, order)
            best[~live] = float("-inf")
            piece.append(best)
        if case["train"]:
            # the gradient as a difference of what arrives at an entry and its share of what arrives at the row
            arrives = -state["up_entropy"][at:at + step].double().unsqueeze(1) * p * (lp + 1.0)
            arrives[line, t.clamp(min=0)] += state["up_logprob"][at:at + step].double()
            if top:
                for k in range(top):
                    arrives[line, order[:, k]] += state["up_top"][at:at + step, k].double()
            # (d entropy / d log-probability is -p (lp + 1); the log-softmax takes a p-weighted share of the sum off)
            grad = arrives - p * arrives.sum(1, keepdim=True)
            grad[~live] = 0.0
            piece.append(grad)
        parts.append(piece)
    whole = [torch.cat([p[k] for p in parts]) for k in range(len(parts[0]))]
    if top:
        whole.insert(2 if tokens is None else 3, None)  # the alternatives' indexes
    return tuple(whole)


def _exact_embedding(case, state):
    weight, tokens, scale = state["weight"].detach(), state["tokens"], state["scale"]
    out = weight.double()[tokens] * scale
    if not case["train"]:
        return (out,)
    keep = tokens != state["pad"]
    grad = torch.zeros(weight.shape, dtype=torch.float64, device=weight.device)
    grad.index_put_((tokens[keep],), state["up"].double()[keep] * scale, accumulate=True)
    return out, grad
