"""The operators behind several continuations of one prompt, each in its plain form and, with `own`, as
the calls a user makes of this library's kernels.

`copy`       blocks of the cache's pools, or rows of per-sequence state, copied to other places of the
             pools or into other pools: the partly filled last block of a forked sequence, the blocks of
             a cache that is given another size.
`attention`  one new token a sequence over the paged cache, where sequences list the same blocks for
             what they share.
`logprobs`   log-probabilities of given tokens under the output head, without keeping the logits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 64          # positions of a cache block


# -- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # one sequence forked into eight at the 1.5B widths: its last block, 37 positions filled, in 28 layers
        {"name": "fork 8, last block", "op": "copy", "entries": 28, "pool": 256, "heads": 2, "dim": 128,
         "copies": 7, "rows": 37, "from_one": True, "fresh": False, "dtype": "bfloat16"},
        # a cache of 19,200 positions of the same model moved into a pool of another size
        {"name": "resize, 300 blocks", "op": "copy", "entries": 28, "pool": 400, "heads": 2, "dim": 128,
         "copies": 300, "rows": 64, "from_one": False, "fresh": True, "dtype": "bfloat16"},
        # recurrent states of 16 heads of 64 x 64 in six layers, one sequence forked into 32
        {"name": "fork 32, fp32 states", "op": "copy", "entries": 6, "pool": 64, "heads": 16, "dim": 64,
         "copies": 31, "rows": 64, "from_one": True, "fresh": False, "dtype": "float32"},
        # a step of four samples of a short prompt
        {"name": "4 samples of 1000", "op": "attention", "heads": 12, "kv_heads": 2, "dim": 128, "layers": 2,
         "prompts": 1, "samples": 4, "shared": 1000, "tail": 60, "tree": False},
        # the benchmark's decode length, sixteen samples
        {"name": "16 samples of 2048", "op": "attention", "heads": 12, "kv_heads": 2, "dim": 128, "layers": 2,
         "prompts": 1, "samples": 16, "shared": 2048, "tail": 200, "tree": False},
        # five prompts of unequal lengths with nine samples each, half of which were forked once more
        {"name": "5 prompts x 9, forked twice", "op": "attention", "heads": 8, "kv_heads": 4, "dim": 64,
         "layers": 2, "prompts": 5, "samples": 9, "shared": 3000, "tail": 333, "tree": True},
        # a long document and as many samples as a batch takes
        {"name": "64 samples of 32000", "op": "attention", "heads": 12, "kv_heads": 2, "dim": 128, "layers": 2,
         "prompts": 1, "samples": 64, "shared": 32000, "tail": 500, "tree": False},
        # the tokens of one short continuation, at the 1.5B output head
        {"name": "5 tokens, bf16", "op": "logprobs", "rows": 5, "hidden": 1536, "vocab": 151936,
         "dtype": "bfloat16", "bias": False, "scale": 1.0, "softcap": 0.0},
        # four choices of some eighty tokens; a vocabulary that is no multiple of anything, a bias, a cap
        {"name": "333 tokens, capped", "op": "logprobs", "rows": 333, "hidden": 2048, "vocab": 50257,
         "dtype": "bfloat16", "bias": True, "scale": 0.5, "softcap": 30.0},
        # a document's perplexity
        {"name": "2047 tokens, bf16", "op": "logprobs", "rows": 2047, "hidden": 1536, "vocab": 151936,
         "dtype": "bfloat16", "bias": False, "scale": 1.0, "softcap": 0.0},
        # the true 32-bit mode
        {"name": "64 tokens, fp32", "op": "logprobs", "rows": 64, "hidden": 1024, "vocab": 32768,
         "dtype": "float32", "bias": False, "scale": 1.0, "softcap": 0.0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["copy", "attention", "attention", "logprobs"])
    if op == "copy":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        c = {"op": op, "entries": rng.randint(1, 32), "heads": rng.choice([1, 2, 3, 4, 8]),
             "dim": rng.choice([16, 48, 64, 128, 256]), "copies": _log_uniform(rng, 1, 400),
             "rows": rng.choice([64, 64, rng.randint(1, 63)]), "from_one": rng.random() < 0.4,
             "fresh": rng.random() < 0.5, "dtype": dtype}
        per = c["entries"] * c["heads"] * BLOCK * c["dim"] * (4 if dtype == "float32" else 2)
        c["copies"] = max(1, min(c["copies"], (250 << 20) // per))
        c["pool"] = 2 * c["copies"] + rng.randint(1, 40)
        return c
    if op == "attention":
        heads, kv_heads = rng.choice([(12, 2), (28, 4), (40, 8), (8, 8), (16, 1), (8, 4)])
        c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128]),
             "layers": rng.randint(1, 3), "prompts": _log_uniform(rng, 1, 8),
             "samples": _log_uniform(rng, 1, 64), "shared": _log_uniform(rng, 1, 32000),
             "tail": _log_uniform(rng, 1, 600), "tree": rng.random() < 0.4}
        while c["prompts"] * c["samples"] > 64:
            c["prompts"] = max(1, c["prompts"] // 2)
            c["samples"] = min(c["samples"], 64)
        most = 64 * 32500 * 2 * 128 * 2                  # what the largest listed case reads and holds
        per = c["layers"] * c["prompts"] * c["samples"] * kv_heads * c["dim"]
        c["shared"] = max(1, min(c["shared"], most // per - c["tail"]))
        return c
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    c = {"op": op, "rows": _log_uniform(rng, 1, 2047), "hidden": 8 * _log_uniform(rng, 8, 448),
         "vocab": _log_uniform(rng, 300, 152064), "dtype": dtype, "bias": rng.random() < 0.3,
         "scale": rng.choice([1.0, 1.0, 0.25]), "softcap": rng.choice([0.0, 0.0, 20.0])}
    most = 2047 * 1536 * 151936 // (16 if dtype == "float32" else 1)
    c["rows"] = max(1, min(c["rows"], most // (c["hidden"] * c["vocab"])))
    return c


# -- sizes that follow from a case alone -----------------------------------------------------

def _lengths(case):
    """Per prompt: (shared positions, [(positions of a second common piece, tail) per sample])."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    prompts = []
    for p in range(case["prompts"]):
        shared = case["shared"] if p == 0 else rng.randint(max(1, case["shared"] // 2), case["shared"])
        branch = case["tail"] // 2 + BLOCK if case["tree"] else 0
        rows = []
        for s in range(case["samples"]):
            again = branch if s % 2 else 0
            rows.append((again, rng.randint(1, case["tail"])))
        prompts.append((shared, rows))
    return prompts


def _tables(case):
    """The block lists as a cache makes them when a sequence is forked: whole blocks are listed by every
    sequence, the block that is partly filled where they part is each sequence's own. Returns (lists of
    blocks, lengths, blocks in all), blocks numbered as they were taken."""
    lists, lengths, taken = [], [], 0

    def take(n):
        nonlocal taken
        taken += n
        return list(range(taken - n, taken))

    for shared, rows in _lengths(case):
        common = take(shared // BLOCK)
        branch = None
        for again, tail in rows:
            at, mine = shared, list(common)
            if again:
                at += again
                if branch is None:
                    branch = take(at // BLOCK - shared // BLOCK)
                mine += branch
            n = at + tail
            mine += take(-(-n // BLOCK) - len(mine))
            lists.append(mine)
            lengths.append(n)
    return lists, lengths, taken


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, dtype, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


# -- the inputs ------------------------------------------------------------------------------

def prepare(case, seed):
    g = _generator(seed)
    rng = random.Random(seed)
    if case["op"] == "copy":
        dtype = getattr(torch, case["dtype"])
        shape = (case["entries"], case["pool"], case["heads"], BLOCK, case["dim"])
        tensors = [torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(2)]
        places = rng.sample(range(case["pool"]), case["copies"] + (1 if case["from_one"] else case["copies"])
                            if not case["fresh"] else case["copies"])
        dst = places[:case["copies"]]
        if case["fresh"]:                        # the blocks held, wherever they lie, one behind the other
            src, dst = dst, list(range(case["copies"]))
        else:
            src = places[case["copies"]:]
        if case["from_one"]:
            src = [src[0]] * case["copies"]
        into = [torch.zeros((case["entries"], case["copies"] + 16) + shape[2:], device="cuda", dtype=dtype)
                for _ in tensors] if case["fresh"] else None
        index = [torch.tensor(x, device="cuda") for x in (src, dst)]
        return {"case": case, "tensors": tensors, "into": into, "src": src, "dst": dst, "index": index}
    if case["op"] == "attention":
        lists, lengths, blocks = _tables(case)
        order = list(range(blocks + 3))          # blocks lie anywhere in the pool
        rng.shuffle(order)
        width = max(len(x) for x in lists)
        tables = [[order[b] for b in x] + [-1] * (width - len(x)) for x in lists]
        h, kv, d, layers = case["heads"], case["kv_heads"], case["dim"], case["layers"]
        q = _normal((layers, len(lists), h * d), g, torch.bfloat16, 2.0)
        keys = _normal((layers, blocks + 3, kv, BLOCK, d), g, torch.bfloat16)
        values = _normal((layers, blocks + 3, kv, BLOCK, d), g, torch.bfloat16)
        state = {"case": case, "q": q, "keys": keys, "values": values, "scale": d ** -0.5,
                 "tables": torch.tensor(tables, dtype=torch.int32, device="cuda"),
                 "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
        if own:        # (made when a sequence is forked or ends, used by every layer of the steps between)
            from semantic_aware_adaptive_kv_cache_precision_b200 import ops
            state["plan"] = ops.plan_shared(tables, lengths, h, kv, device="cuda")
        return state
    dtype = getattr(torch, case["dtype"])
    x = _normal((case["rows"], case["hidden"]), g, dtype)
    head = _normal((case["vocab"], case["hidden"]), g, dtype, 2.0 / math.sqrt(case["hidden"]))
    bias = _normal((case["vocab"],), g, dtype) if case["bias"] else None
    targets = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
    return {"case": case, "x": x, "head": head, "bias": bias, "targets": targets}


# -- one pass --------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _call(state, case)
    if case["op"] == "copy":
        return _plain_copy(state, case)
    if case["op"] == "attention":
        return _plain_attention(state, case)
    return _plain_logprobs(state, case)


def _call(state, case):
    from semantic_aware_adaptive_kv_cache_precision_b200 import ops
    if case["op"] == "copy":
        ops.copy_blocks(state["tensors"], state["src"], state["dst"], into=state["into"], rows=case["rows"])
        return state["into"] or state["tensors"]
    if case["op"] == "attention":
        return [ops.shared_decode_attention(state["q"][i], state["keys"][i], state["values"][i],
                                            state["lengths"], state["tables"], state["plan"], case["heads"],
                                            case["kv_heads"], case["dim"], state["scale"])
                for i in range(case["layers"])]
    return list(ops.token_logprobs(state["x"], state["head"], state["targets"], state["bias"],
                                   scale=case["scale"], softcap=case["softcap"]))


def _plain_copy(state, case):
    src, dst = state["index"]
    rows = case["rows"]
    into = state["into"] or state["tensors"]
    a, b = state["tensors"]
    into[0][:, dst, :, :rows] = a[:, src, :, :rows]
    into[1][:, dst, :, :rows] = b[:, src, :, :rows]
    return into


def _plain_attention(state, case):
    layers, kv, d = case["layers"], case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    tables = state["tables"].long().clamp(min=0)
    b, width = tables.shape

    def positions(pool):             # [layers, b, kv, positions, d] in 32 bits
        return pool[:, tables].permute(0, 1, 3, 2, 4, 5).reshape(layers, b, kv, width * BLOCK, d).float()

    q = state["q"].float().view(layers, b, kv, group, d) * state["scale"]
    scores = q @ positions(state["keys"]).transpose(-1, -2)
    seen = torch.arange(width * BLOCK, device=q.device) < state["lengths"].view(1, b, 1, 1, 1)
    scores = scores.masked_fill_(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p @ positions(state["values"])) / p.sum(-1, keepdim=True)
    return list(out.to(torch.bfloat16).view(layers, b, kv * group * d).unbind(0))


def _plain_logprobs(state, case):
    z = state["x"].float() @ state["head"].float().t()
    if state["bias"] is not None:
        z += state["bias"].float()
    z *= case["scale"]
    if case["softcap"]:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    top = z.amax(-1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))).squeeze(-1)
    mine = z.gather(1, state["targets"].long().unsqueeze(1)).squeeze(1)
    return [mine - lse, lse]


# -- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"] == "copy":
        size = 4 if case["dtype"] == "float32" else 2
        one = 2 * case["entries"] * case["heads"] * case["rows"] * case["dim"] * size
        return {"bytes": one * (case["copies"] + (1 if case["from_one"] else case["copies"])), "flops": 0}
    if case["op"] == "attention":
        lists, lengths, _ = _tables(case)
        filled = {}                                # positions in use of every distinct block
        for blocks, n in zip(lists, lengths):
            for i, block in enumerate(blocks):
                filled[block] = min(BLOCK, n - i * BLOCK)
        row = case["kv_heads"] * case["dim"]
        return {"bytes": case["layers"] * (4 * row * sum(filled.values()) + 4 * len(lists) * case["heads"] * case["dim"]),
                "flops": case["layers"] * 4 * case["heads"] * case["dim"] * sum(lengths)}
    size = 4 if case["dtype"] == "float32" else 2
    t, k, v = case["rows"], case["hidden"], case["vocab"]
    return {"bytes": size * (t * k + v * k + (v if case["bias"] else 0)) + 12 * t, "flops": 2 * t * k * v}


# -- the same from the definitions, in 64 bits ------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "copy":
        return None                                # nothing is computed: every element is one that was there
    if case["op"] == "attention":
        q, group = state["q"].double(), case["heads"] // case["kv_heads"]
        d = case["dim"]
        out = [torch.empty(q.shape[1:], dtype=torch.float64, device=q.device) for _ in range(case["layers"])]
        for i in range(case["layers"]):
            for b, n in enumerate(state["lengths"].tolist()):
                blocks = state["tables"][b, :-(-n // BLOCK)].long()
                for h in range(case["kv_heads"]):
                    k = state["keys"][i, blocks, h].reshape(-1, d)[:n].double()
                    v = state["values"][i, blocks, h].reshape(-1, d)[:n].double()
                    mine = q[i, b].view(-1, d)[h * group:(h + 1) * group]
                    weights = torch.softmax(torch.einsum("gd,nd->gn", mine, k) / math.sqrt(d), dim=1)
                    out[i][b].view(-1, d)[h * group:(h + 1) * group] = torch.einsum("gn,nd->gd", weights, v)
        return out
    w, logprob, lse = state["head"].double(), [], []
    for x, t in zip(state["x"].split(128), state["targets"].split(128)):
        z = torch.einsum("tk,vk->tv", x.double(), w)
        if state["bias"] is not None:
            z = z + state["bias"].double()
        z = z * case["scale"]
        if case["softcap"]:
            z = torch.tanh(z / case["softcap"]) * case["softcap"]
        lse.append(torch.logsumexp(z, 1))
        logprob.append(torch.log_softmax(z, 1)[torch.arange(len(t), device=t.device), t.long()])
    return [torch.cat(logprob), torch.cat(lse)]
