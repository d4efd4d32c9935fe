"""What the paged key-value cache's operators compute and what it costs.

Each case is one call as a serving program makes it: tokens written to a paged
cache, one new token's attention over it, the attention weight that a prompt
puts on each of its keys, and the eviction of a cache to a budget.  `run` gives
the plain form of the operator in elementary torch operations, or, where `own`
is true, the framework's own call.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One decoding step of GPT-2 small for eight users: the cache write is all latency.
        {"name": "append-token", "op": "append", "dtype": "bf16", "b": 8, "hkv": 12, "d": 64, "page": 16,
         "tokens": 1, "start": 500, "ragged": False},
        # Prompts of a 32-head model written to the cache after their prefill, padded to the longest.
        {"name": "append-prompt", "op": "append", "dtype": "bf16", "b": 4, "hkv": 32, "d": 128, "page": 16,
         "tokens": 4096, "start": 0, "ragged": True},
        # One user of GPT-2 small in mid conversation: the shortest step.
        {"name": "decode-one", "op": "decode", "dtype": "bf16", "b": 1, "h": 12, "hkv": 12, "d": 64, "page": 16,
         "len": 300, "ragged": False, "weights": False},
        # A full batch of a 32-head model, conversations of every length up to 4096.
        {"name": "decode-batch", "op": "decode", "dtype": "bf16", "b": 32, "h": 32, "hkv": 32, "d": 128, "page": 16,
         "len": 4096, "ragged": True, "weights": False},
        # One very long document, four query heads to a cached head.
        {"name": "decode-long", "op": "decode", "dtype": "f16", "b": 1, "h": 32, "hkv": 8, "d": 128, "page": 64,
         "len": 131072, "ragged": False, "weights": False},
        # A batch whose cache is kept to a budget: the step also adds up each key's weight.
        {"name": "decode-weights", "op": "decode", "dtype": "bf16", "b": 16, "h": 32, "hkv": 8, "d": 128, "page": 16,
         "len": 8191, "ragged": True, "weights": True},
        # The exact fp32 path at the widest head, pages of an odd size.
        {"name": "decode-f32", "op": "decode", "dtype": "f32", "b": 5, "h": 8, "hkv": 4, "d": 256, "page": 24,
         "len": 2047, "ragged": True, "weights": True},
        # The weight that two short prompts put on their keys.
        {"name": "keys-short", "op": "keys", "dtype": "bf16", "b": 2, "h": 12, "hkv": 12, "d": 64, "nq": 1000,
         "nkv": 1000, "causal": True},
        # A whole long prompt.
        {"name": "keys-long", "op": "keys", "dtype": "bf16", "b": 1, "h": 16, "hkv": 16, "d": 128, "nq": 8192,
         "nkv": 8192, "causal": True},
        # The last window of a very long prompt against all of its keys, grouped heads.
        {"name": "keys-window", "op": "keys", "dtype": "f16", "b": 1, "h": 32, "hkv": 8, "d": 128, "nq": 200,
         "nkv": 32768, "causal": True},
        # GPT-2 small's cache halved.
        {"name": "evict-short", "op": "evict", "dtype": "bf16", "b": 2, "hkv": 12, "d": 64, "page": 16, "len": 1024,
         "ragged": False, "keep": 512, "recent": 64},
        # Long conversations brought back to their budget.
        {"name": "evict-long", "op": "evict", "dtype": "bf16", "b": 4, "hkv": 8, "d": 128, "page": 16, "len": 50000,
         "ragged": True, "keep": 8192, "recent": 1024},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "keys", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d = rng.choice([64, 64, 128, 128, 128, 96, 256])
    page = rng.choice([16, 16, 32, 64, 24, 1, 128, 7])
    if op == "append":
        hkv, b = rng.choice([1, 2, 8, 12, 16, 32]), _spread(rng, 1, 32)
        tokens = rng.choice([1, _spread(rng, 1, max(1, 4096 * 4 * 32 * 128 // (b * hkv * d * 2)))])
        tokens = min(tokens, 8192)
        return {"op": op, "dtype": dtype, "b": b, "hkv": hkv, "d": d, "page": page, "tokens": tokens,
                "start": rng.randrange(0, 700), "ragged": rng.random() < 0.7}
    if op == "decode":
        hkv = rng.choice([1, 2, 4, 8, 12, 16, 32])
        group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
        h = hkv * min(group, 64 // hkv)
        b = _spread(rng, 1, 48)
        top = min(131072, 60_000_000 // (b * hkv * d))
        weights = rng.random() < 0.4
        if weights:
            top = min(top, 30_000_000 // (b * h))
        return {"op": op, "dtype": dtype, "b": b, "h": h, "hkv": hkv, "d": d, "page": page,
                "len": _spread(rng, 1, max(1, top)), "ragged": rng.random() < 0.7, "weights": weights}
    if op == "keys":
        d = rng.choice([64, 128])
        hkv = rng.choice([1, 2, 4, 8, 12])
        h = hkv * rng.choice([1, 1, 2, 4])
        b = rng.choice([1, 1, 2, 3])
        nkv = _spread(rng, 1, min(32768, int(math.sqrt(500_000_000 / (b * h)))))
        nq = nkv if rng.random() < 0.6 else _spread(rng, 1, nkv)
        return {"op": op, "dtype": rng.choice(["bf16", "f16"]), "b": b, "h": h, "hkv": hkv, "d": d, "nq": nq,
                "nkv": nkv, "causal": rng.random() < 0.8}
    hkv, b = rng.choice([1, 2, 8, 12, 32]), _spread(rng, 1, 16)
    length = _spread(rng, 2, min(131072, 40_000_000 // (b * hkv * d)))
    keep = _spread(rng, 1, length)
    return {"op": op, "dtype": dtype, "b": b, "hkv": hkv, "d": d, "page": page, "len": length,
            "ragged": rng.random() < 0.6, "keep": keep, "recent": rng.randrange(0, keep + 1) // 2}


def _lens(case, top):
    """Every sequence's length: all alike, or spread over [1, top] in a shuffled order."""
    b = case["b"]
    if not case["ragged"]:
        return [top] * b
    return [1 + (top - 1) * (i * 7 % b + 1) // b for i in range(b)]


def _paged(case, top, g):
    """Pools as a server keeps them: one allocation, other users' pages between this batch's."""
    page, b = case["page"], case["b"]
    per = (top + page - 1) // page
    pages = b * per + 8
    table = torch.randperm(pages, device="cuda", generator=g)[: b * per].to(torch.int32).view(b, per)
    shape, dt = (pages, case["hkv"], page, case["d"]), DTYPES[case["dtype"]]
    k = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dt)
    v = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dt)
    return k, v, table.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, b, d, dt = case["op"], case["b"], case["d"], DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": case}
    if op == "append":
        n = _lens(case, case["tokens"])
        s["k"], s["v"], s["table"] = _paged(case, case["start"] + case["tokens"], g)
        # The new rows as a layer has them: views of one packed projection [B, T, 2, Hkv, D].
        kv = randn(b, case["tokens"], 2, case["hkv"], d).to(dt)
        s["k_new"], s["v_new"] = (kv[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
        s["start"], s["counts"] = ints([case["start"]] * b), ints(n)
    elif op == "decode":
        s["k"], s["v"], s["table"] = _paged(case, case["len"], g)
        s["q"] = randn(b, case["h"], d).to(dt)
        s["lens"] = ints(_lens(case, case["len"]))
        if case["weights"]:
            cap = s["table"].shape[1] * case["page"]
            s["weights"] = torch.rand(b, case["hkv"], cap, device="cuda", generator=g)
            s["weights_out"] = s["weights"].clone()
    elif op == "keys":
        n = case["nkv"]
        s["q"], s["k"] = randn(b, case["h"], case["nq"], d).to(dt), randn(b, case["hkv"], n, d).to(dt)
        # The log-sum-exp that the prompt's forward pass left behind.
        s["lse"] = torch.empty(b, case["h"], case["nq"], device="cuda")
        for i in range(b):
            for h in range(case["h"]):
                x = s["q"][i, h].float() @ s["k"][i, h * case["hkv"] // case["h"]].float().T / math.sqrt(d)
                if case["causal"]:
                    row = torch.arange(n - case["nq"], n, device="cuda")[:, None]
                    x.masked_fill_(torch.arange(n, device="cuda")[None] > row, -math.inf)
                s["lse"][i, h] = torch.logsumexp(x, -1)
    else:
        s["k"], s["v"], table = _paged(case, case["len"] + case["keep"] + case["page"], g)
        per = (case["len"] + case["page"] - 1) // case["page"]
        s["table"] = table[:, :per].contiguous()
        s["dst"] = table[:, per: per + (case["keep"] + case["page"] - 1) // case["page"]].contiguous()
        s["lens"] = ints(_lens(case, case["len"]))
        # Accumulated weight is small for most keys and large for a few.
        s["weights"] = torch.rand(b, case["hkv"], case["len"], device="cuda", generator=g) ** 8
    return s


def _gae():
    return importlib.import_module("geodesic-attention-engine-gae-_b200")


def _gather(pages, table):
    """The cached rows in order: [B, Hkv, M * page, D]."""
    x = pages[table.long()]
    b, m, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, m * p, d)


def _append(s):
    page = s["case"]["page"]
    b, h, t, d = s["k_new"].shape
    at = torch.arange(t, device="cuda")[None]
    at = torch.where(at < s["counts"][:, None], at, 0)  # padding writes its sequence's first token again
    to = s["start"].long()[:, None] + at
    pg, slot = s["table"].long().gather(1, to // page), to % page
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        pool[pg, :, slot] = new.permute(0, 2, 1, 3).gather(1, at[:, :, None, None].expand(b, t, h, d))
    return {"k": s["k"], "v": s["v"]}


def _decode(s):
    q, lens = s["q"].float(), s["lens"]
    b, h, d = q.shape
    k, v = _gather(s["k"], s["table"]).float(), _gather(s["v"], s["table"]).float()
    hkv, n = k.shape[1], k.shape[2]
    x = (q.view(b, hkv, h // hkv, d) @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    seen = (torch.arange(n, device="cuda")[None] < lens[:, None])[:, None, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    r = {"out": (p @ v).view(b, h, d).to(s["q"].dtype), "lse": (top + torch.log(total)).view(b, h)}
    if "weights" in s:
        r["weights"] = s["weights"] + p.sum(2)
    return r


def _keys(s):
    q, k, c = s["q"].float(), s["k"].float(), s["case"]
    b, h, nq, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    x = (q.view(b, hkv, h // hkv * nq, d) @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    w = torch.exp(x - s["lse"].view(b, hkv, h // hkv * nq, 1))
    if c["causal"]:
        row = torch.arange(n - nq, n, device="cuda").repeat(h // hkv)[:, None]
        w = torch.where(torch.arange(n, device="cuda")[None] <= row, w, 0.0)
    return w.sum(2)


def _evict(s):
    keep, recent, page = s["case"]["keep"], s["case"]["recent"], s["case"]["page"]
    w, lens = s["weights"], s["lens"].long()
    b, h, n = w.shape
    at = torch.arange(n, device="cuda")[None, None]
    x = torch.where(at >= (lens - recent)[:, None, None], math.inf, w)
    x = torch.where(at < lens[:, None, None], x, -math.inf)
    kept = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :keep]
    left = torch.clamp(lens, max=keep)
    there = torch.arange(keep, device="cuda")[None, None] < left[:, None, None]
    kept = torch.sort(torch.where(there, kept, n), dim=-1).values
    pos = torch.where(there, kept, kept[..., :1])  # an unused place takes its row's first key again
    pg = s["table"].long()[:, None].expand(b, h, -1).gather(2, pos // page)
    to = torch.where(there, torch.arange(keep, device="cuda")[None, None], 0)
    to_pg = s["dst"].long()[:, None].expand(b, h, -1).gather(2, to // page)
    hh = torch.arange(h, device="cuda")[None, :, None].expand(b, h, keep)
    for pool in (s["k"], s["v"]):
        pool[to_pg, hh, to % page] = pool[pg, hh, pos % page]
    return {"k": s["k"], "v": s["v"], "lens": left.to(torch.int32), "kept": torch.where(there, kept, -1).to(torch.int32),
            "weights": torch.where(there, w.gather(2, pos), 0.0)}


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _append, "decode": _decode, "keys": _keys, "evict": _evict}[op](s)
    gae = _gae()
    if op == "append":
        gae.paged_append(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["start"], counts=s["counts"])
        return {"k": s["k"], "v": s["v"]}
    if op == "decode":
        if "weights" not in s:
            out, lse = gae.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], return_lse=True)
            return {"out": out, "lse": lse}
        out, lse = gae.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], return_lse=True,
                                       weights=s["weights"], weights_out=s["weights_out"])
        return {"out": out, "lse": lse, "weights": s["weights_out"]}
    if op == "keys":
        c = s["case"]
        return gae.attention_key_weights(s["q"], s["k"], s["lse"], causal=c["causal"], q_offset=c["nkv"] - c["nq"])
    lens, kept, weights = gae.paged_evict(s["k"], s["v"], s["table"], s["lens"], s["weights"], s["dst"],
                                          keep=s["case"]["keep"], recent=s["case"]["recent"])
    return {"k": s["k"], "v": s["v"], "lens": lens, "kept": kept, "weights": weights}


def work(case):
    e, d, b = DTYPES[case["dtype"]].itemsize, case["d"], case["b"]
    if case["op"] == "append":
        n = sum(_lens(case, case["tokens"]))
        return {"bytes": 4 * n * case["hkv"] * d * e, "flops": 0}
    if case["op"] == "decode":
        n = sum(_lens(case, case["len"]))
        more = 8 * n * case["hkv"] if case["weights"] else 0
        return {"bytes": 2 * n * case["hkv"] * d * e + 2 * b * case["h"] * d * e + 4 * b * case["h"] + more,
                "flops": 4 * n * case["h"] * d}
    if case["op"] == "keys":
        nq, n = case["nq"], case["nkv"]
        pairs = nq * (n - nq) + nq * (nq + 1) // 2 if case["causal"] else nq * n
        return {"bytes": b * (case["h"] * nq + case["hkv"] * n) * d * e + 4 * b * (case["h"] * nq + case["hkv"] * n),
                "flops": 2 * b * case["h"] * pairs * d}
    lens = _lens(case, case["len"])
    kept = sum(min(x, case["keep"]) for x in lens) * case["hkv"]
    return {"bytes": 4 * sum(lens) * case["hkv"] + kept * (4 * d * e + 8), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    op, d, b = case["op"], case["d"], case["b"]
    if op == "append":
        page = case["page"]
        k, v = s["k"].double(), s["v"].double()
        for i, (n, start) in enumerate(zip(s["counts"].tolist(), s["start"].tolist())):
            pos = torch.arange(start, start + n, device="cuda")
            pg = s["table"][i, pos // page].long()
            k[pg, :, pos % page] = s["k_new"][i, :, :n].transpose(0, 1).double()
            v[pg, :, pos % page] = s["v_new"][i, :, :n].transpose(0, 1).double()
        return {"k": k, "v": v}
    if op == "decode":
        h, hkv = case["h"], case["hkv"]
        out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
        lse = torch.empty(b, h, dtype=torch.float64, device="cuda")
        r = {"out": out, "lse": lse}
        if case["weights"]:
            r["weights"] = s["weights"].double()
        for i, n in enumerate(s["lens"].tolist()):
            pg = s["table"][i].long()
            for j in range(hkv):
                kj = s["k"][pg, j].reshape(-1, d)[:n].double()
                vj = s["v"][pg, j].reshape(-1, d)[:n].double()
                heads = slice(j * (h // hkv), (j + 1) * (h // hkv))
                x = s["q"][i, heads].double() @ kj.T / math.sqrt(d)
                lse[i, heads] = torch.logsumexp(x, 1)
                p = torch.softmax(x, 1)
                out[i, heads] = p @ vj
                if case["weights"]:
                    r["weights"][i, j, :n] += p.sum(0)
        return r
    if op == "keys":
        h, hkv, nq, n = case["h"], case["hkv"], case["nq"], case["nkv"]
        w = torch.zeros(b, hkv, n, dtype=torch.float64, device="cuda")
        for i in range(b):
            for j in range(h):
                kj = s["k"][i, j // (h // hkv)].double()
                for at in range(0, nq, 2048):
                    x = s["q"][i, j, at: at + 2048].double() @ kj.T / math.sqrt(d) - s["lse"][i, j, at: at + 2048, None].double()
                    if case["causal"]:
                        x = x + torch.full_like(x, -math.inf).triu(n - nq + at + 1)
                    w[i, j // (h // hkv)] += torch.exp(x).sum(0)
        return w
    page, keep = case["page"], case["keep"]
    k, v = s["k"].double(), s["v"].double()
    kept = torch.full((b, case["hkv"], keep), -1, dtype=torch.int32, device="cuda")
    weights = torch.zeros(b, case["hkv"], keep, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    for i, n in enumerate(lens):
        for j in range(case["hkv"]):
            w, m = s["weights"][i, j, :n].double(), min(n, keep)
            tail = min(case["recent"], n)
            # ascending by (weight, latest first): the last of the list are kept
            order = torch.flip(torch.argsort(torch.flip(w[: n - tail], (0,)), stable=True), (0,))
            pos = torch.cat([(n - tail - 1) - order[: m - min(tail, m)], torch.arange(n - tail, n, device="cuda")]).sort().values
            kept[i, j, :m], weights[i, j, :m] = pos.to(torch.int32), w[pos]
            at = torch.arange(m, device="cuda")
            src, dst = s["table"][i, pos // page].long(), s["dst"][i, at // page].long()
            k[dst, j, at % page], v[dst, j, at % page] = k[src, j, pos % page], v[src, j, pos % page]
    return {"k": k, "v": v, "lens": torch.tensor([min(x, keep) for x in lens], dtype=torch.int32, device="cuda"),
            "kept": kept, "weights": weights}
