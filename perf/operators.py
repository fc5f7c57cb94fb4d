"""The operators between the simulator and a policy network, as measured cases.

What an environment returns is a grid of categorical cells (and a mission text); what it takes is one action of a few.
Between them stand four operators: the embedding of cells or of text tokens with its gradient, the adjustment of a
policy's logits (penalties for what was answered before, biases, masks of what may be answered), the draw of an answer,
and the log-probabilities and entropies that a policy gradient trains on.

``own = False`` computes them in elementary torch operations, ``own = True`` through ``multigrid_amd.policy``.
"""
import math

import torch

own = False

CELL_FIELDS = (11, 6, 7)  # types, colours and states of a cell: the rows that a one-hot cell has
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IDS = {"uint8": torch.uint8, "int32": torch.int32, "int64": torch.int64}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "uint8": 1, "int32": 4, "int64": 8}
KINDS = ("cells", "cells_train", "tokens", "tokens_train", "adjust", "adjust_train", "draw", "logprob_train")


def listed():
    return [
        # the observation of one environment of two agents, as an evaluation loop embeds it: latency
        dict(name="cells-one-env", op="cells", n=98, dim=32, dtype="fp32", ids="uint8"),
        # a training step of the first layer on 4096 environments of two agents, in full precision
        dict(name="cells-train-4096-envs", op="cells_train", n=4096 * 98, dim=64, dtype="fp32", ids="uint8"),
        # the same in bfloat16 on 65536 environments, the largest two-agent batch of the simulator's own benchmark
        dict(name="cells-train-65536-envs", op="cells_train", n=65536 * 98, dim=32, dtype="bf16", ids="uint8"),
        # mission texts of a batch, tokenised: the lookup alone, wide rows
        dict(name="tokens-lookup", op="tokens", n=16384, rows=32000, dim=2048, dtype="bf16", ids="int64"),
        # the same in training: an odd number of tokens over a vocabulary of no round size, padded
        dict(name="tokens-train", op="tokens_train", n=8190, rows=30011, dim=1024, dtype="bf16", ids="int64"),
        # one answer of a policy that answers in words: one row, latency
        dict(name="adjust-one-row", op="adjust", n=1, k=32000, t=512, dtype="bf16", ids="int64", mask="bits"),
        # a batch of answers under one grammar each
        dict(name="adjust-256-rows", op="adjust", n=256, k=128000, t=2048, dtype="bf16", ids="int32", mask="bits"),
        # 131072 environments of eight agents, seven actions, the last sixteen actions remembered: a training step
        dict(name="adjust-train-actions", op="adjust_train", n=131072 * 8, k=7, t=16, dtype="fp32", ids="uint8", mask="bool"),
        # the actions of the same batch
        dict(name="draw-actions", op="draw", n=131072 * 8, k=7, dtype="fp32"),
        # words for 64 rows, a vocabulary of odd size
        dict(name="draw-64-rows", op="draw", n=64, k=128003, dtype="fp16"),
        # log-probabilities and entropies of the actions taken, with the gradient
        dict(name="logprob-train-actions", op="logprob_train", n=131072 * 8, k=7, dtype="fp32"),
        # the same for words, an odd vocabulary
        dict(name="logprob-train-tokens", op="logprob_train", n=4095, k=30011, dtype="bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(KINDS)
    dtype, ids = rng.choice(sorted(DTYPES)), rng.choice(sorted(IDS))
    if op.startswith("cells"):
        dim = rng.choice((_log(rng, 4, 128), 16, 32, 64))
        n = _log(rng, 1, 65536 * 98 * 131 // (3 * BYTES[ids] + 2 * dim * BYTES[dtype]))
        return dict(op=op, n=n, dim=dim, dtype=dtype, ids=ids)
    if op.startswith("tokens"):
        dim = rng.choice((_log(rng, 8, 4096), 256, 512, 1024))
        rows = _log(rng, 30, min(131072, 1 << 25 >> (dim - 1).bit_length()) if op == "tokens_train" else 131072)
        ids = "int32" if ids == "uint8" and rows > 255 else ids
        return dict(op=op, n=_log(rng, 1, (1 << 24) // dim), rows=rows, dim=dim, dtype=dtype, ids=ids)
    if rng.random() < 0.4:  # actions
        k, n, t = rng.randint(2, 40), 0, rng.randint(1, 32)
        n = _log(rng, 1, 7 * 131072 * 8 // k)
    else:  # words
        k, t = _log(rng, 64, 131072), _log(rng, 1, 2048)
        n = _log(rng, 1, min(8192, (1 << 25) // k))
        ids = "int32" if ids == "uint8" else ids
    case = dict(op=op, n=n, k=k, dtype=dtype)
    if op.startswith("adjust"):
        case.update(t=t, ids=ids, mask=rng.choice(("bits", "bool", "none")))
    return case


def _zipf(n, rows, gen):
    """Tokens as texts have them: the frequency of a token falls with its rank, and ranks lie anywhere in the table."""
    rank = torch.exp(torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * math.log(rows + 1)).long() - 1
    return rank.clamp_(0, rows - 1) * 7919 % rows if rows % 7919 else rank.clamp_(0, rows - 1)


def _cells(n, gen):
    """Cells as views show them: unseen, empty and wall for the most part, an object here and there."""
    u = torch.rand((n, 3), generator=gen, device="cuda")
    kind = torch.where(u[:, 0] < 0.3, 0, torch.where(u[:, 0] < 0.75, 1, torch.where(u[:, 0] < 0.92, 2, 3 + (u[:, 1] * 8).int().clamp_(max=7))))
    colour = torch.where(kind == 2, 5, torch.where(kind > 2, (u[:, 2] * 6).int().clamp_(max=5), 0))
    state = torch.where(kind > 2, (u[:, 1] * 8 % 1 * 7).int().clamp_(max=6), 0)
    return torch.stack((kind, colour, state), dim=-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    dtype, n, op = DTYPES[case["dtype"]], case["n"], case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    s = {"op": op, "case": case}
    train = op.endswith("train")
    if op.startswith(("cells", "tokens")):
        dim, rows = case["dim"], case.get("rows", sum(CELL_FIELDS))
        if op.startswith("cells"):
            s["fields"], s["ids"], s["scale"] = CELL_FIELDS, _cells(n, gen).to(IDS[case["ids"]]), 1.0
        else:
            ids = _zipf(n, rows, gen)
            if case["ids"] != "uint8":  # padding behind the shorter texts
                ids = torch.where(uniform(n) < 0.1, -1, ids)
            s["fields"], s["ids"], s["scale"] = None, ids.to(IDS[case["ids"]]), math.sqrt(dim)
        s["table"] = (normal(rows, dim) * dim ** -0.5).to(dtype).requires_grad_(train)
        if train:
            s["grad"] = normal(n, dim).to(dtype)
        return s
    k = case["k"]
    s["logits"] = (normal(n, k) * (1.0 if k <= 64 else 2.5)).to(dtype)
    s["temperature"] = 1.0 if k <= 64 else 0.8
    if op.startswith("adjust"):
        t = case["t"]
        s["history"] = _zipf(n * t, k, gen).view(n, t).to(IDS[case["ids"]])
        s["lengths"] = (uniform(n) * (t + 1)).int().clamp_(max=t)
        s["repetition"], s["presence"], s["frequency"] = 1.0 + 0.3 * uniform(n), 0.5 * uniform(n), 0.1 * uniform(n)
        s["bias"] = normal(k) * 0.5
        s["mask"] = None
        if case["mask"] == "bool":
            s["mask"] = uniform(n, k) < 0.8
        elif case["mask"] == "bits":
            words = torch.randint(-(1 << 31), 1 << 31, (2, n, (k + 31) // 32), generator=gen, device="cuda")
            s["mask"] = (words[0] | words[1]).int()
        if train:
            s["grad"] = normal(n, k).to(dtype)
    elif op == "draw":
        s["uniforms"] = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    else:  # as they come from the adjustment: some places masked, never all of a row
        hidden = uniform(n, k) < 0.15
        hidden[torch.arange(n, device="cuda"), (uniform(n) * k).long().clamp_(max=k - 1)] = False
        s["logits"].masked_fill_(hidden, -math.inf)
        s["tokens"] = torch.multinomial(torch.softmax(s["logits"].float(), -1), 1, generator=gen)[:, 0]
        s["grad"], s["grad_entropy"] = normal(n) / n, torch.full((n,), -0.01 / n, device="cuda")
    s["logits"].requires_grad_(train)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _rows_of(ids, fields, rows):
    """Rows of the table that each token reads, [n, fields], and whether it reads one at all."""
    sizes = fields or (rows,)
    ids = ids.long().view(len(ids), len(sizes))
    size = torch.tensor(sizes, device=ids.device)
    reads = (ids >= 0) & (ids < size)
    return torch.where(reads, ids + (size.cumsum(0) - size), 0), reads


def _embed(s):
    table = s["table"].detach()
    at, reads = _rows_of(s["ids"], s["fields"], len(table))
    x = (table.float()[at] * reads[..., None]).sum(1) * s["scale"]
    return x.to(table.dtype)


def _embed_grad(s):
    rows, dim = s["table"].shape
    at, reads = _rows_of(s["ids"], s["fields"], rows)
    g = s["grad"].float()
    if rows <= 64:  # a product with the rows' indicator, 4096 tokens at a time
        pieces = -(-len(g) // 4096)
        hot = torch.zeros((pieces * 4096, rows), device=g.device).index_put_(
            (torch.arange(len(g), device=g.device)[:, None].expand_as(at), at), reads.float(), accumulate=True)
        g = torch.cat((g, g.new_zeros((pieces * 4096 - len(g), dim))))
        d = torch.bmm(hot.view(pieces, 4096, rows).transpose(1, 2), g.view(pieces, 4096, dim)).sum(0)
    else:
        d = torch.zeros((rows, dim), device=g.device).index_add_(0, at[:, 0], g * reads)
    return (d * s["scale"]).to(s["table"].dtype)


def _counts(s):
    n, k = s["logits"].shape
    h = s["history"].long()
    counted = (torch.arange(h.shape[1], device=h.device) < s["lengths"][:, None]) & (h >= 0) & (h < k)
    return torch.zeros((n, k), device=h.device).scatter_add_(1, torch.where(counted, h, 0), counted.float())


def _allowed(s):
    n, k = s["logits"].shape
    if s["mask"] is None or s["mask"].dtype == torch.bool:
        return s["mask"]
    bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    return bits.view(n, -1)[:, :k] != 0


def _adjust(s):
    x, c, r = s["logits"].detach().float(), _counts(s), s["repetition"][:, None]
    x = torch.where(c > 0, torch.where(x > 0, x / r, x * r) - s["presence"][:, None], x)
    x = x - s["frequency"][:, None] * c + s["bias"]
    allowed = _allowed(s)
    return (x if allowed is None else torch.where(allowed, x, -math.inf)).to(s["logits"].dtype)


def _adjust_grad(s):
    x, c, r = s["logits"].detach().float(), _counts(s), s["repetition"][:, None]
    g = s["grad"].float()
    g = torch.where(c > 0, torch.where(x > 0, g / r, g * r), g)
    allowed = _allowed(s)
    return (g if allowed is None else torch.where(allowed, g, 0.0)).to(s["logits"].dtype)


def _draw(s):
    z = s["logits"].detach().double()  # next to a border of two tokens 32 bits are too few
    z = (z - z.amax(1, keepdim=True)) / s["temperature"]
    p = torch.exp(z)
    upto = p.cumsum(1)
    token = (upto <= s["uniforms"][:, None] * upto[:, -1:]).sum(1).clamp_(max=z.shape[1] - 1)
    return token, (z.gather(1, token[:, None])[:, 0] - torch.log(upto[:, -1])).float()


def _logprob_parts(s):
    z = s["logits"].detach().float()
    z = (z - z.amax(1, keepdim=True)) / s["temperature"]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logp, p = z - torch.log(total), e / total
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    return logp, p, entropy


def _logprob_train(s):
    logp, p, entropy = _logprob_parts(s)
    taken = s["tokens"][:, None]
    g, ge = s["grad"][:, None], s["grad_entropy"][:, None]
    d = -g * p - ge * torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
    d = d.scatter_add(1, taken, g)
    return logp.gather(1, taken)[:, 0], entropy, (d / s["temperature"]).to(s["logits"].dtype)


def _plain(s):
    op = s["op"]
    if op in ("cells", "tokens"):
        return _embed(s)
    if op in ("cells_train", "tokens_train"):
        return _embed(s), _embed_grad(s)
    if op == "adjust":
        return _adjust(s)
    if op == "adjust_train":
        return _adjust(s), _adjust_grad(s)
    return _draw(s) if op == "draw" else _logprob_train(s)


# ---- the framework's operators -------------------------------------------------------------------------------------


def _own(s):
    from multigrid_amd import policy

    op = s["op"]
    if op.startswith(("cells", "tokens")):
        out = policy.embed(s["ids"], s["table"], fields=s["fields"], scale=s["scale"])
        if op in ("cells", "tokens"):
            return out
        return out, torch.autograd.grad(out, s["table"], s["grad"])[0]
    if op.startswith("adjust"):
        out = policy.adjust_logits(s["logits"], history=s["history"], lengths=s["lengths"], repetition=s["repetition"],
                                   presence=s["presence"], frequency=s["frequency"], bias=s["bias"], mask=s["mask"])
        if op == "adjust":
            return out
        return out, torch.autograd.grad(out, s["logits"], s["grad"])[0]
    if op == "draw":
        return policy.draw(s["logits"], s["uniforms"], temperature=s["temperature"])
    logprob, entropy = policy.token_logprobs(s["logits"], s["tokens"], temperature=s["temperature"])
    return logprob, entropy, torch.autograd.grad((logprob, entropy), s["logits"], (s["grad"], s["grad_entropy"]))[0]


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- what a pass cannot do without, and what it computes -----------------------------------------------------------


def work(case):
    n, op, e = case["n"], case["op"], BYTES[case["dtype"]]
    if op.startswith(("cells", "tokens")):
        fields, rows, dim = (3, sum(CELL_FIELDS), case["dim"]) if op.startswith("cells") else (1, case["rows"], case["dim"])
        moved = n * fields * BYTES[case["ids"]] + min(n * fields, rows) * dim * e + n * dim * e
        if op.endswith("train"):
            moved += n * dim * e + rows * dim * e
        return {"bytes": moved, "flops": n * fields * dim * (2 if op.endswith("train") else 1)}
    k = case["k"]
    if op.startswith("adjust"):
        moved = 2 * n * k * e + n * case["t"] * BYTES[case["ids"]] + 16 * n + 4 * k
        moved += {"none": 0, "bool": n * k, "bits": n * ((k + 31) // 32) * 4}[case["mask"]]
        return {"bytes": moved + (2 * n * k * e if op.endswith("train") else 0), "flops": 5 * n * k}
    if op == "draw":
        return {"bytes": n * k * e + n * (8 + 8 + 4), "flops": 6 * n * k}
    return {"bytes": 2 * n * k * e + n * (8 + 4 * 4), "flops": 14 * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op.startswith(("cells", "tokens")):
        table, sizes = s["table"].detach().double(), s["fields"] or (len(s["table"]),)
        ids = s["ids"].long().view(case["n"], len(sizes))
        out, grads = torch.zeros((case["n"], case["dim"]), device="cuda", dtype=torch.float64), []
        for f, part in enumerate(table.split(list(sizes))):
            i, found = ids[:, f], (ids[:, f] >= 0) & (ids[:, f] < sizes[f])
            out[found] += part[i[found]]
            if op.endswith("train"):
                g = s["grad"].double()
                if sizes[f] <= 64:
                    grads += [g[i == r].sum(0) for r in range(sizes[f])]
                else:
                    order = torch.argsort(i, stable=True)
                    many = torch.bincount(i[found], minlength=sizes[f]).cpu()
                    pieces = g[order][int((i < 0).sum()):][:int(many.sum())].split(many.tolist())
                    grads += [p.sum(0) for p in pieces]
        if not op.endswith("train"):
            return out * s["scale"]
        return out * s["scale"], torch.stack(grads) * s["scale"]
    x, (n, k) = s["logits"].detach().double(), s["logits"].shape
    if op.startswith("adjust"):
        h = s["history"].long()
        row = torch.arange(n, device="cuda")[:, None].expand_as(h)
        live = torch.arange(h.shape[1], device="cuda")[None] < s["lengths"][:, None]
        live &= (h >= 0) & (h < k)
        c = torch.bincount((row * k + h)[live], minlength=n * k).view(n, k)
        rep = torch.where(x > 0, 1.0 / s["repetition"].double()[:, None], s["repetition"].double()[:, None])
        factor = torch.where(c > 0, rep, 1.0)
        y = x * factor - (c > 0) * s["presence"].double()[:, None] - c * s["frequency"].double()[:, None] + s["bias"].double()
        if s["mask"] is not None:
            if s["mask"].dtype == torch.bool:
                barred = ~s["mask"]
            else:
                at = torch.arange(k, device="cuda")
                barred = (s["mask"].long()[:, at // 32] >> (at % 32)) % 2 == 0
            y[barred], factor[barred] = -math.inf, 0.0
        return (y, factor * s["grad"].double()) if op.endswith("train") else y
    z = x / s["temperature"]
    lse = torch.logsumexp(z, 1)
    if op == "draw":
        border = s["uniforms"] * torch.exp(z - z.amax(1, keepdim=True)).sum(1)
        token = torch.searchsorted(torch.exp(z - z.amax(1, keepdim=True)).cumsum(1), border[:, None], right=True)[:, 0].clamp_(max=k - 1)
        return token, z[torch.arange(n, device="cuda"), token] - lse
    logp = z - lse[:, None]
    p = torch.exp(logp)
    entropy = -(p * logp.clamp(min=-1e300)).sum(1)
    hot = torch.zeros_like(p)
    hot[torch.arange(n, device="cuda"), s["tokens"]] = 1.0
    d = s["grad"].double()[:, None] * (hot - p) - s["grad_entropy"].double()[:, None] * p * (logp.clamp(min=-1e300) + entropy[:, None])
    return logp[torch.arange(n, device="cuda"), s["tokens"]], entropy, d / s["temperature"]
