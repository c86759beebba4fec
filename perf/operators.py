"""What is measured of the serving operators: appending to a paged KV cache, attention over it, and sampling.

A user's step is one run of the three: the projections of a step's new tokens are normed, rotated and appended to the
paged cache (q4kb200.paged_append), every new token attends to its sequence's pages (q4kb200.paged_attention), and the
logits of the last rows are sampled (q4kb200.sample). Each case is one call of one of them. Sequence lengths of a case
come from its own "lens" number, so that its work is known; every value comes from the seed.

With `own` false, `run` computes the same in elementary torch operations; `exact` does so in 64 bits."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
ROPE_BASE = 1e6
VOCAB = 151936
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat session decoding: one new token over a short context, fp32 activations over the engine's fp16 cache
        attention("decode 1x500", 1, (1, 1), (500, 500), "f32", page=16),
        # the batched decode workload: 64 sessions with ragged contexts of 512 to 4096
        attention("decode 64x512-4096", 64, (1, 1), (512, 4096), "f32", page=64),
        # two long documents on one rank of a tensor-parallel job (2 KV heads of it), 16-bit activations
        attention("decode 2x131071", 2, (1, 1), (131071, 131071), "bf16", heads=8, kv_heads=2, page=128),
        # a few draft tokens verified per sequence, sliding window, one KV head per query head
        attention("draft 16x5 window", 16, (5, 5), (3000, 9000), "f16", heads=16, kv_heads=16, head_dim=64, page=32, window=2048),
        # one prefill pass of a long prompt: 512 new tokens after 3584 cached ones
        attention("chunk 512 at 4096", 1, (512, 512), (4096, 4096), "f32", page=16),
        # continuous batching: decoding sequences and prompt chunks of odd sizes in one call, rows of padding behind them
        attention("mixed 12x1-1000", 12, (1, 1000), (1000, 8000), "bf16", page=16, pad=37),
        # a whole long prompt at once
        attention("prefill 8192", 1, (8192, 8192), (8192, 8192), "bf16", page=128),
        # one token of each of 64 sessions: queries and keys normed and rotated, keys and values appended
        append("append 64x1", 64, (1, 1), (512, 4096), "f32", page=64),
        # a prompt's pass over many tokens, 16-bit
        append("append 8192", 3, (2000, 3500), (2000, 30000), "bf16", page=16, pad=5),
        # one session's next token, the usual chat settings
        sampling("sample 1", 1, VOCAB, "f32", "all"),
        # the batched decode workload's rows with settings of their own, 16-bit logits with their many ties
        sampling("sample 64 bf16", 64, VOCAB, "bf16", "mixed"),
        # many rows of a best-of-n job, nucleus sampling alone
        sampling("sample 257 top-p", 257, VOCAB, "f32", "top_p"),
    ]


def attention(name, sequences, new, ctx, type, heads=32, kv_heads=8, head_dim=128, page=16, window=0, pad=0, lens=7):
    return {"name": name, "op": "attention", "sequences": sequences, "new_min": new[0], "new_max": new[1], "ctx_min": ctx[0], "ctx_max": ctx[1],
            "type": type, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "window": window, "pad": pad, "lens": lens}


def append(name, sequences, new, ctx, type, heads=32, kv_heads=8, head_dim=128, page=16, pad=0, lens=7):
    return {**attention(name, sequences, new, ctx, type, heads, kv_heads, head_dim, page, 0, pad, lens), "op": "append"}


def sampling(name, rows, vocab, type, filters):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "type": type, "filters": filters}


def spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "sample"))
    if op == "sample":
        c = sampling("", spread(rng, 1, 256), rng.choice((VOCAB, spread(rng, 1000, 200000))), rng.choice(("f32", "bf16", "f16")),
                     rng.choice(("all", "mixed", "top_p", "top_k", "min_p", "none")))
    else:
        kv_heads, group, head_dim = rng.choice((1, 2, 4, 8, 8)), rng.choice((1, 2, 4, 4, 5, 8)), rng.choice((64, 128, 128))
        shape = {"heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice((16, 32, 64, 128, 256)),
                 "type": rng.choice(("f32", "f16", "bf16")), "pad": rng.choice((0, 0, 3, 29)), "lens": rng.randrange(1 << 20)}
        if op == "append":
            sequences = spread(rng, 1, 128)
            new = spread(rng, 1, max(1, 8192 // sequences))
            c = append("", sequences, (rng.choice((1, new)), new), (new, new + spread(rng, 16, 8192)), **shape)
        else:
            kind = rng.choice(("decode", "draft", "chunk"))
            most = 60000 // kv_heads if kind == "decode" else 16000
            sequences = spread(rng, 1, 96 if kind == "decode" else 24)
            new = 1 if kind == "decode" else rng.randint(2, 8) if kind == "draft" else spread(rng, 9, 2048)
            # the plain form's scores, padded to the longest, stay below 2^30 values
            most = min(most, (1 << 30) // (sequences * kv_heads * group * new), (1 << 22) // sequences * 8 // kv_heads)
            ctx = spread(rng, max(new, 40), max(new, 40, most))
            c = attention("", sequences, (new if kind == "draft" else 1, new), (max(1, ctx // rng.randint(1, 6)), ctx), window=rng.choice((0, 0, 0, 300, 1024)), **shape)
    del c["name"]
    return c


def lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["sequences"])]
    return new, [max(n, rng.randint(case["ctx_min"], case["ctx_max"])) for n in new]


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 10 * n}  # one exponential and the sums of each value
    new, ctx = lengths(case)
    heads, kv, d, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    tokens, table = sum(new), sum(-(-c // case["page"]) for c in ctx) * 4
    if case["op"] == "append":
        rows = tokens * d
        return {"bytes": rows * size * (2 * heads + 2 * kv) + rows * 2 * 2 * kv + table, "flops": 10 * rows * (heads + kv)}
    pairs = kept = 0
    for n, c in zip(new, ctx):
        first = c - n + 1  # keys of the first new token
        if window:
            pairs += sum(min(first + i, window) for i in range(n))
            kept += min(c, window + n - 1)
        else:
            pairs += n * first + n * (n - 1) // 2
            kept += c
    return {"bytes": 2 * tokens * heads * d * size + 4 * tokens * heads + kept * kv * d * 2 * 2 + table, "flops": 4 * d * heads * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    dtype = TYPES[case["type"]]
    if case["op"] == "sample":
        rows, vocab, f = case["rows"], case["vocab"], case["filters"]
        # a bulk of unlikely tokens and a few likely ones, flatter and more peaked rows
        logits = randn(rows, vocab) * (1.0 + 2.0 * rand(rows, 1)) + 8.0 * (rand(rows, vocab) > 0.9997)
        on = lambda name: rand(rows) > (1.0 if f not in (name, "all", "mixed") else 0.3 if f == "mixed" else -1.0)  # noqa: E731
        zero = torch.zeros(rows, device="cuda")
        return {"logits": logits.to(dtype), "uniform": rand(rows),
                "temperature": (0.6 + 0.6 * rand(rows)) * (1.0 if f != "mixed" else (rand(rows) > 0.1).float()),
                "top_k": torch.where(on("top_k"), (1.0 + 99.0 * rand(rows)).int(), zero.int()),
                "top_p": torch.where(on("top_p"), 0.8 + 0.19 * rand(rows), zero + 1.0),
                "min_p": torch.where(on("min_p"), 0.02 + 0.08 * rand(rows), zero)}
    new, ctx = lengths(case)
    heads, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    need = [-(-c // page) for c in ctx]
    order = torch.randperm(sum(need) + 7, generator=g, device="cuda").int()
    table = torch.zeros(len(ctx), max(need), dtype=torch.int32)
    host, at = order.cpu(), 0
    for i, n in enumerate(need):
        table[i, :n] = host[at:at + n]
        at += n
    tokens, cached = sum(new) + case["pad"], torch.float16 if case["type"] != "bf16" else torch.bfloat16
    state = {"q_start": torch.tensor([0] + new).cumsum(0).int().cuda(), "kv_len": torch.tensor(ctx).int().cuda(), "table": table.cuda(),
             "max_new": max(new), "max_kv": max(ctx), "window": case["window"],
             "out": torch.zeros(tokens, heads, d, device="cuda", dtype=dtype)}
    if case["op"] == "append":
        # the rows of one fused projection
        state["qkv"] = randn(tokens, heads + 2 * kv, d).to(dtype)
        state["gamma_q"], state["gamma_k"] = 1.0 + 0.1 * randn(d), 1.0 + 0.1 * randn(d)
        state["k"] = torch.zeros(sum(need) + 7, kv, page, d, device="cuda", dtype=cached)
        state["v"] = torch.zeros_like(state["k"])
    else:
        # normed and rotated queries and keys; some heads look more sharply than others
        state["q"] = (randn(tokens, heads, d) * (0.5 + 2.0 * rand(1, heads, 1))).to(dtype)
        state["k"] = randn(sum(need) + 7, kv, page, d, dtype=cached)
        state["v"] = randn(sum(need) + 7, kv, page, d, dtype=cached)
        state["lse"] = torch.zeros(tokens, heads, device="cuda")
    return state


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return run_own(s)
    if "logits" in s:
        return plain_sample(s)
    return plain_append(s) if "qkv" in s else plain_attention(s)


def binding():
    if "q4kb200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-4b-q4_k_m-inference-engine_b200", "python"))
    import q4kb200

    return q4kb200


def run_own(s):
    q = binding()
    if "logits" in s:
        tokens, logprob = q.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprob": logprob}
    cache = q.PagedKV(s["k"], s["v"])
    batch = q.PagedBatch(s["q_start"], s["kv_len"], s["table"], max_new=s["max_new"])
    if "qkv" in s:
        heads, kv = s["out"].shape[1], s["k"].shape[1]
        query, key, value = s["qkv"].split((heads, kv, kv), dim=1)
        q.paged_append(cache, batch, key, value, q=query, q_out=s["out"], q_gamma=s["gamma_q"], k_gamma=s["gamma_k"], epsilon=EPS, rope_base=ROPE_BASE)
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    q.paged_attention(cache, batch, s["q"], out=s["out"], lse=s["lse"], window=s["window"])
    return {"out": s["out"], "lse": s["lse"]}


def places(s, tokens):
    """Of each of the batch's tokens: its sequence and its position there (rows behind the last sequence are not among them)."""
    at = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["q_start"][1:], at, right=True).clamp(max=len(s["kv_len"]) - 1)
    return seq, at - s["q_start"][seq + 1] + s["kv_len"][seq], at < s["q_start"][-1]


def plain_append(s):
    tokens, heads, d = s["out"].shape
    pages, kv, page, _ = s["k"].shape
    seq, position, real = places(s, tokens)
    x = s["qkv"].float()
    query, key, value = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    angle = position.double()[:, None] * ROPE_BASE ** (-torch.arange(0, d, 2, device="cuda").double() / d)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def normed_rotated(t, gamma):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * gamma
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    out = torch.where(real[:, None, None], normed_rotated(query, s["gamma_q"]).to(s["out"].dtype), s["out"])
    keep = real.nonzero()[:, 0]
    where = (s["table"][seq, position // page].long()[keep], slice(None), (position % page)[keep])
    s["k"][where] = normed_rotated(key, s["gamma_k"])[keep].to(s["k"].dtype)
    s["v"][where] = value[keep].to(s["v"].dtype)
    return {"q": out, "k": s["k"], "v": s["v"]}


def plain_attention(s):
    tokens, heads, d = s["out"].shape
    _, kv, page, _ = s["k"].shape
    n, new, ctx = len(s["kv_len"]), s["max_new"], s["max_kv"]
    # every sequence's pages, padded to the longest: [n][kv][ctx][d]
    rows = lambda t: t[s["table"].long()].permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)[:, :, :ctx].float()  # noqa: E731
    key = torch.arange(ctx, device="cuda")
    at = (s["q_start"][:-1, None] + torch.arange(new, device="cuda")).clamp(max=tokens - 1)
    last = s["kv_len"][:, None] - (s["q_start"][1:] - s["q_start"][:-1])[:, None] + torch.arange(new, device="cuda")  # [n][new]
    seen = (key <= last[..., None]) & (key < s["kv_len"][:, None, None])
    if s["window"]:
        seen &= key > last[..., None] - s["window"]
    query = s["q"][at].float().reshape(n, new, kv, heads // kv, d).permute(0, 2, 3, 1, 4)  # [n][kv][group][new][d]
    score = query.reshape(n, kv, -1, d) @ rows(s["k"]).transpose(-1, -2)
    score = score.mul_(d ** -0.5).view(n, kv, heads // kv, new, ctx).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(n, kv, -1, ctx) @ rows(s["v"])).view(n, kv, heads // kv, new, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, new, heads, d)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(n, new, heads)
    seq, _, real = places(s, tokens)
    turn = (torch.arange(tokens, device="cuda") - s["q_start"][seq]).clamp(max=new - 1)
    return {"out": torch.where(real[:, None, None], out[seq, turn], 0.0).to(s["out"].dtype), "lse": torch.where(real[:, None], lse[seq, turn], 0.0)}


def plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    weight = ((x - x.amax(-1, keepdim=True)) / heat).exp()
    weight = weight * ~greedy[:, None] + (torch.arange(vocab, device="cuda") == x.argmax(-1, keepdim=True)) * greedy[:, None]
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices  # ties: the lowest index first
    sorted_ = weight.gather(-1, order)
    top_k = torch.where(s["top_k"] > 0, s["top_k"].long(), vocab)[:, None]
    sorted_ = sorted_ * (torch.arange(vocab, device="cuda") < top_k)
    sums = sorted_.cumsum(-1)
    top_p = torch.where(s["top_p"] < 1, s["top_p"].double(), math.inf)[:, None]
    sorted_ = sorted_ * (sums - sorted_ < top_p * sums[:, -1:]) * (sorted_ >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(weight).scatter_(-1, order, sorted_)
    sums = kept.cumsum(-1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(-1, keepdim=True).clamp(max=vocab - 1)
    logprob = (kept.gather(-1, token) / sums[:, -1:]).log()
    return {"tokens": token[:, 0].int(), "logprob": logprob[:, 0].float()}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return exact_sample({k: v.double().cpu().numpy() for k, v in s.items()})
    new, ctx = lengths(case)
    return exact_append(s, new, ctx) if case["op"] == "append" else exact_attention(s, new, ctx, case["window"])


def exact_sample(s):
    logprob = np.zeros(len(s["uniform"]))
    for r, x in enumerate(s["logits"]):
        if s["temperature"][r] <= 0:
            continue  # the likeliest token alone: its probability is 1
        order = np.argsort(-x, kind="stable")
        if s["top_k"][r] > 0:
            order = order[:int(s["top_k"][r])]
        w = np.exp((x[order] - x[order[0]]) / s["temperature"][r])
        if s["top_p"][r] < 1:
            n = int(np.searchsorted(np.cumsum(w), s["top_p"][r] * w.sum())) + 1
            order, w = order[:n], w[:n]
        keep = w >= s["min_p"][r]
        order, w = order[keep], w[keep]
        by = np.argsort(order)
        sums = np.cumsum(w[by])
        at = min(int(np.searchsorted(sums, s["uniform"][r] * sums[-1], side="right")), len(by) - 1)
        logprob[r] = np.log(w[by[at]] / sums[-1])
    return {"tokens": None, "logprob": logprob}


def exact_append(s, new, ctx):
    _, heads, d = s["out"].shape
    kv, page = s["k"].shape[1:3]
    q, k, v = s["out"].double(), s["k"].double(), s["v"].double()
    theta = torch.tensor([ROPE_BASE ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        x = s["qkv"][start:start + n].double()
        position = torch.arange(c - n, c, device="cuda")
        turn = torch.polar(torch.ones(n, d // 2, dtype=torch.float64, device="cuda"), position.double()[:, None] * theta)[:, None]
        rotated = []
        for part, gamma in ((x[:, :heads], s["gamma_q"]), (x[:, heads:heads + kv], s["gamma_k"])):
            y = part / (part.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * gamma.double()
            z = torch.complex(y[..., :d // 2], y[..., d // 2:].contiguous()) * turn
            rotated.append(torch.cat((z.real, z.imag), -1))
        q[start:start + n] = rotated[0]
        pages = s["table"][i, position // page].long()
        k[pages, :, position % page] = rotated[1]
        v[pages, :, position % page] = x[:, heads + kv:]
        start += n
    return {"q": q, "k": k, "v": v}


def exact_attention(s, new, ctx, window):
    _, heads, d = s["out"].shape
    kv, page = s["k"].shape[1:3]
    out, lse = torch.zeros_like(s["out"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
    start = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        pages = s["table"][i, :-(-c // page)].long()
        for h in range(heads):
            k, v = (t[pages, h * kv // heads].reshape(-1, d)[:c].double() for t in (s["k"], s["v"]))
            for at in range(0, n, 2048):
                rows = slice(start + at, start + min(n, at + 2048))
                score = s["q"][rows, h].double() @ k.T / math.sqrt(d)
                last = torch.arange(c - n + at, c - n + min(n, at + 2048), device="cuda")[:, None]
                key = torch.arange(c, device="cuda")
                hidden = key > last
                if window:
                    hidden = hidden | (key <= last - window)
                score.masked_fill_(hidden, -math.inf)
                lse[rows, h] = torch.logsumexp(score, -1)
                out[rows, h] = torch.softmax(score, -1) @ v
        start += n
    return {"out": out, "lse": lse}
