"""Operators around a paged KV cache, as cases that can be timed and compared: what is run, over which sizes, and what it must give.

  op       "decode"   attention of one new token of every context over its pages
           "packed"   causal attention of prompts of different lengths, one behind the other, over their pages
           "copy"     pages copied within a pool, in every layer of it
           "logprobs" log probabilities of given tokens, entropy and the largest alternatives of rows of logits
  dtype    "f16" | "bf16" | "f32": of the cache and the queries, or of the logits
  heads, kv_heads, size   of the attention; page: tokens of a page
  batch    contexts or sequences
  lo, hi   keys of a context (decode) or new tokens of a sequence (packed), spread evenly between the two
  past     keys that each sequence has in its pages in front of its new tokens, at most (packed; spread evenly from 0)
  layers, pages, pairs, row   layers of the pool, its pages a layer, pages copied, elements of a token's row (copy)
  rows, vocab, top            rows of logits, their width, alternatives asked for (logprobs)
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 32000
# query heads, kv heads, head size: those of the stage configurations, and odd ones
HEADS = [(64, 8, 128), (32, 32, 128), (40, 40, 128), (6, 6, 48), (12, 12, 64), (16, 2, 128), (12, 3, 128), (10, 5, 80), (32, 1, 64), (7, 1, 128), (8, 4, 36), (4, 2, 160)]
MOST_BYTES = 1.0e9      # of a drawn decode's cache
MOST_FLOPS = 2.7e11     # of a drawn packed call


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    def decode(name, heads, dtype, batch, lo, hi, page=16):
        return dict(name=name, op="decode", dtype=dtype, heads=heads[0], kv_heads=heads[1], size=heads[2], page=page, batch=batch, lo=lo, hi=hi)

    def packed(name, heads, dtype, batch, lo, hi, past=0, page=16):
        return dict(decode(name, heads, dtype, batch, lo, hi, page), op="packed", past=past)

    return [
        # one user's next token behind a short prompt: nothing but latency
        decode("decode-b1", (64, 8, 128), "f16", 1, 301, 301),
        # a full batch whose contexts have come to very different lengths
        decode("decode-b64-ragged", (64, 8, 128), "f16", 64, 57, 4096),
        # few users with long documents: the keys of a context have to be shared out
        decode("decode-b3-long", (32, 32, 128), "bf16", 3, 20011, 32768, page=64),
        # a small fp32 model's users
        decode("decode-f32-b16", (12, 12, 64), "f32", 16, 33, 1023),
        # one short prompt
        packed("packed-1x77", (64, 8, 128), "f16", 1, 77, 77),
        # a step of a server: prompts of many lengths, some of them the next part of one that has begun
        packed("packed-9-ragged", (32, 32, 128), "bf16", 9, 1, 1023, past=1500, page=32),
        # one long prompt
        packed("packed-1x4096", (64, 8, 128), "f16", 1, 4096, 4096),
        # prompts of a small fp32 model
        packed("packed-f32-5", (12, 12, 64), "f32", 5, 100, 900),
        # contexts that were forked write on: their last pages are copied, in every layer of a stage
        dict(name="copy-fork", op="copy", dtype="f16", layers=10, pages=256, page=16, row=2048, pairs=5),
        # a pool's pages moved to its front
        dict(name="copy-compact", op="copy", dtype="f16", layers=4, pages=6000, page=16, row=2048, pairs=1999),
        # the sampled tokens of a decode step
        dict(name="logprobs-b7", op="logprobs", dtype="f32", rows=7, vocab=VOCAB, top=5),
        # a prompt that is scored
        dict(name="logprobs-prompt", op="logprobs", dtype="f16", rows=2047, vocab=VOCAB, top=20),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["decode", "decode", "packed", "packed", "copy", "logprobs"])
    dtype = rng.choice(["f16", "f16", "bf16", "f32"])
    wide = 4 if dtype == "f32" else 2
    page = rng.choice([16, 32, 64, 128])
    if op == "copy":
        layers, row = rng.choice([1, 2, 5, 10]), 2 * rng.choice([1024, 4096, 768, 288])
        pairs = log(1, 2000)
        pairs = max(1, min(pairs, int(5.0e8 / (layers * page * row * wide))))
        return dict(op=op, dtype=dtype, layers=layers, pages=3 * pairs + rng.randrange(1, 50), page=page, row=row, pairs=pairs)
    if op == "logprobs":
        vocab = rng.choice([VOCAB, VOCAB, 32001, log(300, 130000)])
        return dict(op=op, dtype=dtype, rows=min(log(1, 2000), 65000000 // vocab), vocab=vocab, top=rng.choice([1, 3, 5, 10, 20, 32]))
    heads, kv_heads, size = rng.choice(HEADS)
    case = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, size=size, page=page)
    if op == "decode":
        batch, hi = log(1, 100), log(2, 40000)
        hi = max(2, min(hi, int(MOST_BYTES / (batch * 2 * kv_heads * size * wide))))
        return dict(case, batch=batch, lo=rng.randint(1, hi), hi=hi)
    batch, hi, past = log(1, 24), log(2, 4096), rng.choice([0, 0, log(10, 8000)])
    while batch * heads * hi * (hi + past) * max(16, size) * 4 > MOST_FLOPS or batch * heads * hi * (hi + past) > 1.1e9:    # (scores of the plain form)
        hi, past = max(2, hi * 3 // 4), past * 3 // 4
    return dict(case, batch=batch, lo=rng.randint(1, hi), hi=hi, past=past)


def spread(lo, hi, n):
    """n whole numbers, evenly from lo to hi."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def sequences(case):
    """(new tokens, keys in front of them) of every sequence; the past of a sequence goes the other way than its length"""
    return list(zip(spread(case["lo"], case["hi"], case["batch"]), reversed(spread(0, case["past"], case["batch"]) if case["batch"] > 1 else [case["past"]])))


# ---- what a program has in hand -------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if dt == torch.float32 else torch.float16).to(dt)

    if case["op"] == "logprobs":
        logits = normal(case["rows"], case["vocab"]).mul_(3.0)
        return dict(case, logits=logits, tokens=torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32))
    if case["op"] == "copy":
        pool = normal(case["layers"], case["pages"], case["page"], case["row"])
        order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        return dict(case, pool=pool, pairs=torch.stack([order[:case["pairs"]], order[-case["pairs"]:]], dim=1).contiguous())     # (source, destination)

    kv = case["kv_heads"] * case["size"]
    if case["op"] == "decode":
        tokens, keys = [1] * case["batch"], spread(case["lo"], case["hi"], case["batch"])
    else:
        tokens, keys = [n for n, _ in sequences(case)], [n + past for n, past in sequences(case)]
    most = (max(keys) + case["page"] - 1) // case["page"]
    used = [(k + case["page"] - 1) // case["page"] for k in keys]
    pool = normal(sum(used) + 3, case["page"], 2 * kv)
    order = torch.randperm(sum(used) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["batch"], most), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    first = [0]
    for n in tokens:
        first.append(first[-1] + n)

    def numbers(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    return dict(case, pool=pool, table=table, lengths=numbers(keys), first=numbers(first), start=numbers([k - n for k, n in zip(keys, tokens)]),
                q=normal(sum(tokens), case["heads"] * case["size"]), most_keys=max(keys), most_tokens=max(tokens), tokens=sum(tokens))


def run(s):
    return {"decode": run_decode, "packed": run_packed, "copy": run_copy, "logprobs": run_logprobs}[s["op"]](s)


# ---- with the framework's kernels -------------------------------------------------------------------
def handles(s):
    """What a program makes once: the description of its pages and shape, the workspace, the array that receives the outputs."""
    if "handles" not in s:
        from glinthawk_amd import ops
        from glinthawk_amd._lib import Shape

        ops.init(0)
        shape = Shape(dim=s["heads"] * s["size"], n_layers=1, n_heads=s["heads"], n_kv_heads=s["kv_heads"], hidden_dim=8, seq_len=s["most_keys"])
        pages = ops.pages(s["pool"], s["table"])
        if s["op"] == "decode":
            room = ops.attn_decode_paged_workspace(s["batch"], s["most_keys"], shape, s["q"].dtype)
        else:
            room = ops.attn_packed_workspace(s["batch"], s["tokens"], s["most_keys"], shape, s["q"].dtype)
        s["handles"] = ops, shape, pages, torch.empty(max(room, 16), dtype=torch.uint8, device="cuda"), torch.zeros_like(s["q"])
    return s["handles"]


def run_decode(s):
    if own:
        ops, shape, pages, workspace, out = handles(s)
        ops.attn_decode_paged(s["q"], pages, s["lengths"], out, s["most_keys"], shape, workspace)
        return out
    k, v = keys_and_values(s)
    kv_heads, group = s["kv_heads"], s["heads"] // s["kv_heads"]
    q = s["q"].float().reshape(s["batch"], kv_heads, group, s["size"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(s["size"])
    hidden = torch.arange(scores.shape[-1], device="cuda")[None, :] >= s["lengths"][:, None]
    scores = scores.masked_fill_(hidden[:, None, None, :], -math.inf)
    return torch.matmul(softmax(scores), v).reshape(s["batch"], -1).to(s["q"].dtype)


def run_packed(s):
    if own:
        ops, shape, pages, workspace, out = handles(s)
        ops.attn_packed(s["q"], pages, s["first"], s["start"], out, s["most_keys"], shape, workspace)
        return out
    k, v = keys_and_values(s)
    batch, kv_heads, group, size, t = s["batch"], s["kv_heads"], s["heads"] // s["kv_heads"], s["size"], s["most_tokens"]
    token = torch.arange(t, device="cuda")
    rows = (s["first"][:-1, None] + token[None, :]).clamp(max=s["tokens"] - 1)                       # (batch, t): the sequences side by side
    q = s["q"].float()[rows].reshape(batch, t, kv_heads, group, size).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * t, size)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).div_(math.sqrt(size)).reshape(batch, kv_heads, group, t, -1)
    hidden = torch.arange(scores.shape[-1], device="cuda")[None, None, :] > (s["start"][:, None] + token[None, :])[:, :, None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    out = torch.matmul(softmax(scores).reshape(batch, kv_heads, group * t, -1), v)
    out = out.reshape(batch, kv_heads, group, t, size).permute(0, 3, 1, 2, 4).reshape(batch, t, -1)
    there = token[None, :] < (s["first"][1:] - s["first"][:-1])[:, None]
    return out[there].to(s["q"].dtype)


def run_copy(s):
    if own:
        from glinthawk_amd import ops

        ops.copy_pages(s["pool"], s["pairs"])
        return s["pool"]
    pairs = s["pairs"].long()
    s["pool"][:, pairs[:, 1]] = s["pool"][:, pairs[:, 0]]
    return s["pool"]


def run_logprobs(s):
    if own:
        from glinthawk_amd import ops

        if "workspace" not in s:
            ops.init(0)
            s["workspace"] = torch.empty(max(16, ops.token_logprobs_workspace(s["rows"], s["vocab"], s["top"])), dtype=torch.uint8, device="cuda")
        return ops.token_logprobs(s["logits"], s["tokens"], s["top"], s["workspace"])
    x = s["logits"].float()
    x = x - x.amax(dim=1, keepdim=True)
    e = x.exp()
    z = e.sum(dim=1)
    log_z = z.log()
    entropy = log_z - (e * x).sum(dim=1) / z
    given = x.gather(1, s["tokens"].long()[:, None])[:, 0] - log_z
    # largest first, ties by the lower index: whole numbers in the order of the values (logits are finite), the index below
    bits = (s["logits"].float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits) * (1 << 32) + ((1 << 32) - 1 - torch.arange(s["vocab"], device="cuda"))[None, :]
    best = (1 << 32) - 1 - (order.topk(s["top"], dim=1).values & ((1 << 32) - 1))
    return given, entropy, best.to(torch.int32), x.gather(1, best) - log_z[:, None]


# ---- the plain forms' parts -------------------------------------------------------------------------
def keys_and_values(s):
    """(batch, kv_heads, keys, size) each, in 32 bits; behind a context's keys whatever its first page holds"""
    rows = s["pool"][s["table"].long()].reshape(s["batch"], -1, 2, s["kv_heads"], s["size"])[:, :s["most_keys"]].float().permute(2, 0, 3, 1, 4)
    return rows[0].contiguous(), rows[1].contiguous()


def softmax(scores):
    e = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    return e.div_(e.sum(dim=-1, keepdim=True))


# ---- from the definition, in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        want = s["pool"].double()
        for source, destination in s["pairs"].tolist():
            want[:, destination] = s["pool"][:, source].double()
        return want
    if case["op"] == "logprobs":
        given, entropy, best = [], [], []
        for row, token in zip(s["logits"], s["tokens"].tolist()):
            p = torch.log_softmax(row.double(), dim=0)
            given.append(p[token])
            entropy.append(-(p.exp() * p).sum())
            best.append(p.sort(descending=True, stable=True).values[:case["top"]])
        return torch.stack(given), torch.stack(entropy), None, torch.stack(best)
    size, group = case["size"], case["heads"] // case["kv_heads"]
    firsts, starts, lengths, out = s["first"].tolist(), s["start"].tolist(), s["lengths"].tolist(), torch.zeros_like(s["q"], dtype=torch.float64)
    for i in range(case["batch"]):
        n = firsts[i + 1] - firsts[i]
        rows = torch.cat([s["pool"][p] for p in s["table"][i, :(lengths[i] + case["page"] - 1) // case["page"]].tolist()])[:lengths[i]].double()
        where = torch.arange(lengths[i], device="cuda")[None, :] <= starts[i] + torch.arange(n, device="cuda")[:, None]
        for h in range(case["heads"]):
            c = h // group * size
            k, v = rows[:, c:c + size], rows[:, case["kv_heads"] * size + c:case["kv_heads"] * size + c + size]
            score = s["q"][firsts[i]:firsts[i + 1], h * size:(h + 1) * size].double() @ k.t().contiguous() * size ** -0.5
            weight = torch.softmax(torch.where(where, score, -math.inf), dim=1)
            out[firsts[i]:firsts[i + 1], h * size:(h + 1) * size] = weight @ v
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    wide = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["page"] * case["row"] * wide + 8 * case["pairs"], "flops": 0}
    if case["op"] == "logprobs":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * wide + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * values}
    if case["op"] == "decode":
        pairs = keys = sum(spread(case["lo"], case["hi"], case["batch"]))
        tokens = case["batch"]
    else:
        pairs = sum(n * past + n * (n + 1) // 2 for n, past in sequences(case))
        keys, tokens = sum(n + past for n, past in sequences(case)), sum(n for n, _ in sequences(case))
    pages = sum(-(-n // case["page"]) for n in (spread(case["lo"], case["hi"], case["batch"]) if case["op"] == "decode" else [n + p for n, p in sequences(case)]))
    return {"bytes": (2 * keys * case["kv_heads"] + 2 * tokens * case["heads"]) * case["size"] * wide + 4 * pages + 12 * case["batch"],
            "flops": 4 * pairs * case["heads"] * case["size"]}
