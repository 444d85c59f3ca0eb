"""What is measured of the operators around a batch of token sequences: embedding rows looked up and their
gradient, a paged cache's block tables grown on the GPU, and the slots that a pass's new tokens take.

``run`` computes each in its plain form (elementary torch operations); where ``own`` is true it makes the calls
a user makes of :mod:`eagle_b200` instead. A case is a dict of plain values, its ``"op"`` one of ``lookup``,
``gradient``, ``tables`` and ``slots``.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "int32": torch.int32,
          "int64": torch.int64}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int32": 4, "int64": 8}


def listed():
    return [
        # one decode step of a served batch: a token per sequence; what counts is the latency of the call
        dict(name="lookup_decode", op="lookup", batch=64, seq=1, rows=32768, dim=1024, table="bf16", out="bf16",
             ids="int32", scale=1.0, pad=0.0),
        # a packed prompt batch of odd length and an odd width, padded places among it, rows scaled by sqrt(dim)
        dict(name="lookup_odd", op="lookup", batch=1, seq=10007, rows=50021, dim=1001, table="fp16", out="fp16",
             ids="int64", scale=math.sqrt(1001.0), pad=0.05),
        # a training microbatch: a master table in 32 bits, activations in 16
        dict(name="lookup_train", op="lookup", batch=16, seq=4096, rows=131072, dim=4096, table="fp32", out="bf16",
             ids="int64", scale=64.0, pad=0.0),
        # fine-tuning on one short ragged sequence: latency of the sort and the sums
        dict(name="gradient_short", op="gradient", batch=1, seq=301, rows=8209, dim=520, grad="fp16", out="fp32",
             ids="int32", scale=1.0, pad=0.1),
        # a microbatch into a 32-bit gradient
        dict(name="gradient_train", op="gradient", batch=8, seq=2048, rows=65536, dim=2048, grad="bf16", out="fp32",
             ids="int64", scale=math.sqrt(2048.0), pad=0.02),
        # the largest microbatch, its gradient in 16 bits
        dict(name="gradient_large", op="gradient", batch=32, seq=4096, rows=131072, dim=4096, grad="bf16", out="bf16",
             ids="int64", scale=1.0, pad=0.0),
        # a decode step: every sequence grows by one token, one in block takes a new block, some have ended
        dict(name="tables_decode", op="tables", requests=192, width=256, block=16, blocks=32768, cached=4000, grow=1,
             done=0.05, lengths="int32"),
        # prompts admitted: most blocks are taken now, and the last requests do not fit any more
        dict(name="tables_prompts", op="tables", requests=1024, width=1024, block=16, blocks=550000, cached=1024,
             grow=15000, done=0.02, lengths="int32"),
        # a large pool over many sequences, lengths in 64 bits
        dict(name="tables_large", op="tables", requests=8191, width=2048, block=32, blocks=6000000, cached=20000,
             grow=24000, done=0.02, lengths="int64"),
        # a decode step's slots, padded to the width that its graph was captured for
        dict(name="slots_decode", op="slots", requests=192, capacity=256, width=256, block=16, fresh="one", start=4000,
             done=0.05, lengths="int32", slots="int64"),
        # a few prompts of unequal length packed, blocks of no power of two
        dict(name="slots_prompts", op="slots", requests=61, capacity=16381, width=512, block=24, fresh="ragged",
             start=2000, done=0.0, lengths="int64", slots="int64"),
        # chunks of many prompts at once
        dict(name="slots_large", op="slots", requests=4096, capacity=1 << 20, width=1024, block=64, fresh="ragged",
             start=30000, done=0.02, lengths="int32", slots="int32"),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("lookup", "gradient", "tables", "slots"))
    if op in ("lookup", "gradient"):
        n = _log(rng, 1, 65536 if op == "lookup" else 131072)
        batch = min(n, rng.choice((1, 1, 2, 8, 32)))
        dim = rng.choice((1, 2, 8, 8, 8)) * _log(rng, 16, 512)
        case = dict(op=op, batch=batch, seq=max(1, n // batch), rows=_log(rng, 100, 131072), dim=dim,
                    out=rng.choice(("bf16", "fp16", "fp32")), ids=rng.choice(("int32", "int64")),
                    scale=rng.choice((1.0, math.sqrt(dim))), pad=rng.choice((0.0, 0.02, 0.3)))
        case["table" if op == "lookup" else "grad"] = rng.choice(("bf16", "fp16", "fp32"))
        return case
    requests, block = _log(rng, 1, 8191 if op == "tables" else 4096), rng.choice((1, 8, 16, 16, 24, 32, 64, 128))
    done, lengths = rng.choice((0.0, 0.02, 0.3)), rng.choice(("int32", "int64"))
    if op == "tables":
        width = _log(rng, 16, 2048)
        cached, grow = rng.randint(0, width * block // 2), rng.choice((1, 1, rng.randint(1, width * block // 2)))
        blocks = max(8, int(requests * (cached + grow) / (2 * block) * rng.uniform(0.9, 1.5)))
        return dict(op=op, requests=requests, width=width, block=block, blocks=blocks, cached=cached, grow=grow,
                    done=done, lengths=lengths)
    fresh = rng.choice(("one", "ragged"))
    capacity = requests + rng.randint(0, requests) if fresh == "one" else _log(rng, max(256, 4 * requests), 1 << 20)
    width = _log(rng, 16, 2048)
    return dict(op=op, requests=requests, capacity=capacity, width=width, block=block, fresh=fresh,
                start=rng.randint(0, width * block // 2), done=done, lengths=lengths,
                slots=rng.choice(("int32", "int64")))


# ------------------------------------------------------------------------- inputs

def _tokens(case, gen):
    """Token ids as text has them: the r-th most frequent about 1/r as often as the first, in no order of id,
    and -1 in padded places."""
    n, rows = case["batch"] * case["seq"], case["rows"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(rows)).long() - 1).clamp_(0, rows - 1)
    ids = torch.randperm(rows, generator=gen, device="cuda")[rank]
    padded = torch.rand(n, generator=gen, device="cuda") < case["pad"]
    return torch.where(padded, -1, ids).view(case["batch"], case["seq"]).to(DTYPES[case["ids"]])


def _whole(gen, low, high, n):
    """``n`` whole numbers of [low, high]."""
    return torch.randint(low, high + 1, (n,), generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "lookup":
        state["tokens"] = _tokens(case, gen)
        state["table"] = torch.randn(case["rows"], case["dim"], generator=gen, device="cuda",
                                     dtype=DTYPES[case["table"]])
    elif case["op"] == "gradient":
        state["tokens"] = _tokens(case, gen)
        state["grad"] = torch.randn(case["batch"], case["seq"], case["dim"], generator=gen, device="cuda",
                                    dtype=DTYPES[case["grad"]])
    elif case["op"] == "tables":
        r, w, b, p = case["requests"], case["width"], case["block"], case["blocks"]
        cached = _whole(gen, 0, case["cached"], r).clamp_(max=w * b)
        held = (cached + b - 1) // b
        held = torch.where(torch.cumsum(held, 0) <= p, held, 0)  # what the pool could give them
        cached = torch.minimum(cached, held * b)
        first = torch.cumsum(held, 0) - held
        owner = torch.randperm(p, generator=gen, device="cuda")
        column = torch.arange(w, device="cuda")
        at = (first[:, None] + column).clamp_(max=p - 1)
        state["table"] = torch.where(column < held[:, None], owner[at], -1).to(torch.int32)
        state["used"] = torch.zeros(p, dtype=torch.bool, device="cuda")
        state["used"][owner[:int(held.sum())]] = True
        free = torch.nonzero(~state["used"]).flatten()
        state["pool"] = torch.zeros(p, dtype=torch.int32, device="cuda")
        state["pool"][:free.numel()] = free
        state["count"] = torch.tensor([free.numel()], dtype=torch.int32, device="cuda")
        grown = cached + (_whole(gen, 0, case["grow"], r) if case["grow"] > 1 else 1)
        state["lengths"] = grown.clamp_(max=w * b).to(DTYPES[case["lengths"]])
        state["held"] = held.to(torch.int32)
        state["terminated"] = torch.rand(r, generator=gen, device="cuda") < case["done"]
    else:
        r, w, b, t = case["requests"], case["width"], case["block"], case["capacity"]
        if case["fresh"] == "one":
            fresh = torch.ones(r, dtype=torch.int64, device="cuda")
        else:
            weight = _whole(gen, 1, 1000, r) ** 2
            fresh = 1 + weight * (t - t // 64 - r) // weight.sum()
        start = _whole(gen, 0, case["start"], r)
        state["fresh"] = torch.minimum(fresh, w * b - start).to(DTYPES[case["lengths"]])
        state["start"] = start.to(DTYPES[case["lengths"]])
        most = 2**31 // b - 1 if case["slots"] == "int32" else 2**31 - 1
        state["table"] = _whole(gen, 0, min(most, r * w), r * w).view(r, w).to(torch.int32)
        state["terminated"] = torch.rand(r, generator=gen, device="cuda") < case["done"]
    if own:  # the prepared call, with its workspace, that a program keeps from step to step
        state["call"] = _prepared(state)
    return state


def _prepared(s):
    import eagle_b200 as eb

    if s["op"] == "lookup":
        return eb.Embedding(s["table"], s["tokens"], scale=s["scale"], dtype=DTYPES[s["out"]])
    if s["op"] == "gradient":
        return eb.EmbeddingGrad(s["grad"], s["tokens"], s["rows"], scale=s["scale"], dtype=DTYPES[s["out"]])
    if s["op"] == "tables":
        return eb.BlockTables(s["lengths"], s["held"], s["table"], s["pool"], s["count"], block=s["block"],
                              used=s["used"], terminated=s["terminated"])
    return eb.SlotMap(s["table"], s["start"], s["fresh"], s["capacity"], block=s["block"],
                      terminated=s["terminated"], dtype=DTYPES[s["slots"]])


# ------------------------------------------------------------------------- the operators

def run(state):
    op = state["op"]
    if own:
        out = state["call"]()
        if op == "tables":
            blocks, cells = out
            return {"table": state["table"], "used": state["used"], "blocks": blocks, "cells": cells}
        if op == "slots":
            slots, positions, requests, offsets = out
            return {"slots": slots, "positions": positions, "requests": requests, "offsets": offsets}
        return out
    return {"lookup": _lookup, "gradient": _gradient, "tables": _tables, "slots": _slots}[op](state)


def _lookup(s):
    tokens, table = s["tokens"], s["table"]
    known = (tokens >= 0) & (tokens < s["rows"])
    rows = table[torch.where(known, tokens, 0).long()].float() * s["scale"]
    return torch.where(known[..., None], rows, 0.0).to(DTYPES[s["out"]])


def _gradient(s):
    tokens, grad = s["tokens"].flatten(), s["grad"].flatten(0, 1)
    # a frequent token's row is a long sum, so it is taken in 64 bits; padded places fall on a row behind the last
    total = torch.zeros(s["rows"] + 1, s["dim"], dtype=torch.float64, device=grad.device)
    total.index_add_(0, torch.where(tokens < 0, s["rows"], tokens).long(), grad.double())
    return (total[:s["rows"]] * s["scale"]).to(DTYPES[s["out"]])


def _tables(s):
    block, width, pool, table = s["block"], s["width"], s["pool"].long(), s["table"]
    held = s["held"].long()
    need = torch.where(s["terminated"], 0, (s["lengths"].long() + block - 1) // block)
    fresh = torch.where(need > width, 0, (need - held).clamp(min=0))
    upto = torch.cumsum(fresh, 0)
    fits = (need <= width) & ((fresh == 0) | (upto <= s["count"]))
    column = torch.arange(width, device=table.device)
    j = column - held[:, None]
    at = (upto - fresh)[:, None] + j
    now = fits[:, None] & (j >= 0) & (j < fresh[:, None])
    grown = torch.where(now, pool[at.clamp(0, pool.numel() - 1)].to(torch.int32), table)
    taken = torch.where(fits & (fresh > 0), upto, 0).max()
    given = s["terminated"][:, None] & (j < 0)
    used = torch.cat((s["used"], s["used"][:1]))  # a place behind the last block for what is no release
    used[torch.where(given, table.long(), s["blocks"])] = False
    used[torch.where(torch.arange(pool.numel(), device=table.device) < taken, pool, s["blocks"])] = True
    blocks = torch.where(s["terminated"], 0, torch.where(fits, torch.maximum(need, held), held)).to(torch.int32)
    return {"table": grown, "used": used[:-1], "blocks": blocks,
            "cells": torch.stack((taken, (~fits).sum())).to(torch.int32)}


def _slots(s):
    block, table, device = s["block"], s["table"], s["table"].device
    fresh = torch.where(s["terminated"], 0, s["fresh"].long())
    upto = torch.cumsum(fresh, 0)
    q = torch.arange(s["capacity"], device=device)
    request = torch.searchsorted(upto, q, right=True)
    real = request < s["requests"]
    r = torch.where(real, request, 0)
    position = s["start"].long()[r] + q - (upto - fresh)[r]
    slot = table[r, torch.where(real, position // block, 0)].long() * block + position % block
    return {"slots": torch.where(real, slot, -1).to(DTYPES[s["slots"]]),
            "positions": torch.where(real, position, 0).to(DTYPES[s["lengths"]]),
            "requests": torch.where(real, request, -1).to(torch.int32),
            "offsets": torch.cat((upto.new_zeros(1), upto)).to(torch.int32)}


# ------------------------------------------------------------------------- what a pass cannot do without

def _distinct(case):
    """The rows of the table that the case's tokens are expected to name."""
    n, rows = case["batch"] * case["seq"] * (1.0 - case["pad"]), case["rows"]
    rank = np.arange(1, rows + 1, dtype=np.float64)
    share = np.log1p(1.0 / rank) / math.log(rows + 1)
    return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(share, 1.0 - 1e-12)))))


def work(case):
    if case["op"] in ("lookup", "gradient"):
        n, dim = case["batch"] * case["seq"], case["dim"]
        ids, real = n * BYTES[case["ids"]], n * (1.0 - case["pad"])
        if case["op"] == "lookup":
            return {"bytes": ids + _distinct(case) * dim * BYTES[case["table"]] + n * dim * BYTES[case["out"]],
                    "flops": real * dim}
        return {"bytes": ids + real * dim * BYTES[case["grad"]] + case["rows"] * dim * BYTES[case["out"]],
                "flops": real * dim + case["rows"] * dim}
    r, length = case["requests"], BYTES[case["lengths"]]
    if case["op"] == "tables":
        wanted = r * (1 - case["done"]) * (case["grow"] / 2 / case["block"] if case["grow"] > 1 else 1 / case["block"])
        taken = min(wanted, case["blocks"])
        returned = r * case["done"] * min(case["cached"] / 2 / case["block"], case["width"])
        # lengths, held, mask and new counts of each request; an id read, an id and a used byte written for each
        # block taken; an id read and a used byte written for each block given back
        return {"bytes": r * (length + 4 + 1 + 4) + taken * 9 + returned * 5 + 12, "flops": 0}
    t = case["capacity"]
    real = r * (1 - case["done"]) if case["fresh"] == "one" else t - t // 64
    return {"bytes": r * (2 * length + 1 + 4) + 4 + real / case["block"] * 4
            + t * (BYTES[case["slots"]] + length + 4), "flops": 0}


def exact(case, seed):
    """The computed rows in 64 bits, on the host; the index operators have whole numbers only."""
    if case["op"] not in ("lookup", "gradient"):
        return None
    n, dim, rows = case["batch"] * case["seq"], case["dim"], case["rows"]
    if n * dim > 1 << 26 or rows * dim > 1 << 28:
        return None
    state = prepare(case, seed)
    ids = state["tokens"].cpu().numpy().reshape(-1).astype(np.int64)
    if case["op"] == "lookup":
        # the rows that are named, taken apart once, in order of their id
        named, place = np.unique(ids, return_inverse=True)
        values = state["table"][torch.from_numpy(np.maximum(named, 0)).cuda()].cpu().double().numpy()
        values *= case["scale"]
        values[named < 0] = 0.0
        return torch.from_numpy(values[place].reshape(case["batch"], case["seq"], dim))
    order = np.argsort(ids, kind="stable")
    order = order[ids[order] >= 0]
    result = np.zeros((rows, dim))
    if order.size:
        named, first = np.unique(ids[order], return_index=True)
        grad = state["grad"].reshape(n, dim).cpu().double().numpy()
        result[named] = np.add.reduceat(grad[order], first, axis=0) * case["scale"]
    return torch.from_numpy(result)
