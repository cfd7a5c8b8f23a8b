"""What the operators for sampled and bounded serving are measured on: the pick of a token by chance,
attention of a batch over one shared prefix, attention over a sliding window with sinks.

Architecture of the cases: the benchmark's attention heads (32 query / 8 kv heads of 128, bf16 pages
of 64 tokens) and vocabulary (151936), and generic ones beside them. The pages of a sequence lie
anywhere in the pool, as they do once a server has freed and reused some.

Where `own` is false run() computes an operator from elementary torch operations in 32 bits (the
sampler in 64: its sums decide between whole numbers), where it is true through the framework.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
HEAD, PAGE = 128, 64
SCALE = HEAD ** -0.5


def listed():
    return [
        # The smallest call: one user's token, the filters that chat servers set by default.
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "dtype": "bf16", "filters": "k-p"},
        # A served batch with nucleus sampling only: nothing bounds the set but its mass.
        {"name": "sample_32_top_p", "kind": "sample", "rows": 32, "vocab": 151936, "dtype": "bf16", "filters": "p"},
        # The decode step's largest batch, 32-bit logits, every request with settings of its own.
        {"name": "sample_64_mixed_f32", "kind": "sample", "rows": 64, "vocab": 151936, "dtype": "f32",
         "filters": "mixed"},
        # A small vocabulary of odd size, plain temperature: the whole distribution is drawn from.
        {"name": "sample_7_plain_odd", "kind": "sample", "rows": 7, "vocab": 32003, "dtype": "f32", "filters": "none"},
        # One user far into a conversation, bounded to a window of 1024 with four first tokens kept.
        {"name": "window_1x8192", "kind": "window", "batch": 1, "tokens": 1, "context": 8192, "window": 1024,
         "sinks": 4, "q_heads": 32, "kv_heads": 8},
        # A served batch of long contexts at uneven positions.
        {"name": "window_32x8192", "kind": "window", "batch": 32, "tokens": 1, "context": 8192, "window": 2048,
         "sinks": 4, "q_heads": 32, "kv_heads": 8},
        # Speculative decoding under a window: four candidates a sequence, odd window, seven heads to a kv head.
        {"name": "window_6x4x3001", "kind": "window", "batch": 6, "tokens": 4, "context": 3001, "window": 701,
         "sinks": 17, "q_heads": 28, "kv_heads": 4},
        # The prompt pass of one long document under a window: the largest piece of work for the plain form.
        {"name": "window_prompt_1x7000", "kind": "window_prompt", "batch": 1, "tokens": 7000, "before": 0,
         "window": 1024, "sinks": 4, "q_heads": 32, "kv_heads": 8},
        # Three requests' second chunk of a prompt, behind 1000 tokens that are in the pages already.
        {"name": "window_prompt_3x701", "kind": "window_prompt", "batch": 3, "tokens": 701, "before": 1000,
         "window": 512, "sinks": 64, "q_heads": 32, "kv_heads": 8},
        # A few continuations of one chat prompt.
        {"name": "shared_4x2048", "kind": "shared", "batch": 4, "tokens": 1, "prefix": 2048, "own_keys": 100,
         "q_heads": 32, "kv_heads": 8},
        # A served batch behind one long system prompt or document.
        {"name": "shared_32x16384", "kind": "shared", "batch": 32, "tokens": 1, "prefix": 16384, "own_keys": 256,
         "q_heads": 32, "kv_heads": 8},
        # Many samples of one long document, two tokens verified at a time: the largest batch of query rows.
        {"name": "shared_64x2x30001", "kind": "shared", "batch": 64, "tokens": 2, "prefix": 30001, "own_keys": 300,
         "q_heads": 32, "kv_heads": 8},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


_HEADS = [(32, 8), (32, 8), (16, 8), (8, 8), (28, 4), (6, 2), (8, 1), (40, 8)]


def draw(rng):
    kind = rng.choice(["sample", "sample", "window", "window", "window_prompt", "shared", "shared"])
    if kind == "sample":
        return {"kind": kind, "rows": _spread(rng, 1, 64), "vocab": _spread(rng, 1000, 151936),
                "dtype": rng.choice(["bf16", "f32"]), "filters": rng.choice(["none", "k", "p", "min", "k-p", "mixed"])}
    q_heads, kv_heads = rng.choice(_HEADS)
    if kind == "window_prompt":
        tokens = _spread(rng, 16, 6000)
        return {"kind": kind, "batch": _spread(rng, 1, max(1, min(16, 6000 // tokens))), "tokens": tokens,
                "before": rng.choice([0, 0, _spread(rng, 1, 1500)]), "window": _spread(rng, 1, 4096),
                "sinks": rng.choice([0, 1, 4, _spread(rng, 1, 300)]), "q_heads": q_heads, "kv_heads": kv_heads}
    tokens = rng.choice([1, 1, 1, rng.randint(1, min(8, 32 * kv_heads // q_heads))])
    if kind == "window":
        batch = _spread(rng, 1, 64)
        context = _spread(rng, 2 * tokens, min(30000, 262144 // batch))
        return {"kind": kind, "batch": batch, "tokens": tokens, "context": context, "window": _spread(rng, 1, 8192),
                "sinks": rng.choice([0, 1, 4, _spread(rng, 1, 300)]), "q_heads": q_heads, "kv_heads": kv_heads}
    return {"kind": kind, "batch": _spread(rng, 1, 64 // min(2, tokens)), "tokens": tokens,
            "prefix": _spread(rng, 1, 30000), "own_keys": _spread(rng, 8, 300), "q_heads": q_heads,
            "kv_heads": kv_heads}


# ---- inputs ---------------------------------------------------------------------------------------

def _logits(case, gen):
    """Rows from nearly certain to nearly undecided: Zipf's law with an exponent of its own for each row over a
    random order of the vocabulary, noise on top, and the first 50 ids (reserved ones) banned."""
    rows, vocab = case["rows"], case["vocab"]
    sharp = 0.9 + 1.6 * torch.rand((rows, 1), generator=gen, device=DEVICE)
    rank = torch.rand((rows, vocab), generator=gen, device=DEVICE).argsort(dim=1).float() + 1.0
    x = 12.0 - sharp * rank.log() + 0.3 * torch.randn((rows, vocab), generator=gen, device=DEVICE)
    x[:, :50] = -math.inf
    return x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)


def _filters(case, gen):
    """One setting for all rows as numbers, or one for each row as tensors."""
    kind, rows = case["filters"], case["rows"]
    if kind == "mixed":
        def u():
            return torch.rand(rows, generator=gen, device=DEVICE)
        off = torch.arange(rows, device=DEVICE) % 3
        return {"temperature": 0.5 + u(), "top_k": torch.where(off == 0, 0, 1 + (200 * u()).int()).int(),
                "top_p": torch.where(off == 1, 1.0, 0.8 + 0.2 * u()), "min_p": torch.where(off == 2, 0.0, 0.1 * u())}
    return {"temperature": 0.8, "top_k": 50 if "k" in kind else 0, "top_p": 0.9 if "p" in kind.split("-") else 1.0,
            "min_p": 0.05 if kind == "min" else 0.0}


def _pool(sequences, pages, kv_heads, gen):
    """Pages of random rows and a block table that hands them out in random order."""
    shape = (sequences * pages, kv_heads, PAGE, HEAD)
    k = torch.empty(shape, dtype=torch.bfloat16, device=DEVICE).normal_(generator=gen)
    v = torch.empty(shape, dtype=torch.bfloat16, device=DEVICE).normal_(generator=gen)
    order = torch.randperm(sequences * pages, generator=gen, device=DEVICE).to(torch.int32)
    return k, v, order.view(sequences, pages)


def _positions(batch, last, spread, gen):
    """int32 [batch]: `last` for the first sequence, up to `spread` earlier for the others."""
    back = (torch.rand(batch, generator=gen, device=DEVICE) * (spread + 1)).to(torch.int32)
    back[0] = 0
    return (last - back).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    if kind == "sample":
        return {"case": case, "logits": _logits(case, gen), **_filters(case, gen),
                "uniform": torch.rand(case["rows"], generator=gen, device=DEVICE)}
    batch, tokens, kv = case["batch"], case["tokens"], case["kv_heads"]
    state = {"case": case}
    if kind == "window_prompt":
        keys = case["before"] + tokens
        state["position"] = torch.full((batch,), case["before"], dtype=torch.int32, device=DEVICE)
    elif kind == "window":
        keys = case["context"]
        state["position"] = _positions(batch, keys - tokens, (keys - tokens) // 2, gen)
    else:
        keys = case["own_keys"]
        state["position"] = _positions(batch, keys - tokens, (keys - tokens) // 2, gen)
        state["prefix_pool"] = _pool(1, -(-case["prefix"] // PAGE), kv, gen)
        state["prefix_length"] = torch.tensor([case["prefix"]], dtype=torch.int32, device=DEVICE)
    state["keys"] = keys
    state["pool"] = _pool(batch, -(-keys // PAGE), kv, gen)
    state["query"] = torch.empty((batch * tokens, case["q_heads"], HEAD), dtype=torch.bfloat16,
                                 device=DEVICE).normal_(generator=gen)
    return state


# ---- the plain forms --------------------------------------------------------------------------------

def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape

    def column(v):
        return (v if isinstance(v, torch.Tensor) else torch.full((rows,), v, device=x.device)).double()[:, None]

    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    z = (value - value[:, :1]) / column(s["temperature"])
    weight = z.exp()
    place = torch.arange(vocab, device=x.device)[None]
    top_k = column(s["top_k"])
    kept = (place < top_k) | (top_k <= 0)
    kept &= z >= column(s["min_p"]).log()
    weight = weight * kept
    sums = weight.cumsum(1)
    top_p = column(s["top_p"])
    # a token is kept while the sum of those before it is short of the share
    kept &= (sums - weight < top_p * sums[:, -1:]) | (top_p >= 1)
    weight = weight * kept
    by_id = torch.zeros_like(weight).scatter_(1, index, weight)
    sums = by_id.cumsum(1)
    total = sums[:, -1:]
    token = (sums > s["uniform"].double()[:, None] * total).int().argmax(1)
    picked = by_id.gather(1, token[:, None])
    return token, (picked / total).log()[:, 0].float()


def _unpaged(pool, table):
    """[sequences, kv heads, tokens, HEAD] in 32 bits: the 16-byte chunks of row r of a page are exchanged by r & 7."""
    pages = pool[table.long()]
    row = torch.arange(PAGE, device=pool.device)
    chunk = torch.arange(16, device=pool.device)[None] ^ (row[:, None] & 7)
    pages = pages.view(*pages.shape[:-1], 16, 8)[..., row[:, None], chunk, :]
    pages = pages.reshape(*table.shape, pool.shape[1], PAGE, HEAD).transpose(1, 2)
    return pages.reshape(table.shape[0], pool.shape[1], -1, HEAD).float()


def _softmax(scores):
    top = scores.amax(-1, keepdim=True)
    weight = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    return weight / weight.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_attention(s):
    case = s["case"]
    batch, tokens, kv, heads = case["batch"], case["tokens"], case["kv_heads"], case["q_heads"]
    group = heads // kv
    k, v = (_unpaged(p, s["pool"][2]) for p in s["pool"][:2])
    q = s["query"].view(batch, tokens, kv, group, HEAD).permute(0, 2, 1, 3, 4).reshape(batch, kv, tokens * group, HEAD)
    q = q.float() * SCALE
    place = torch.arange(k.shape[2], device=k.device)[None, None]
    at = s["position"].long()[:, None, None] + torch.arange(tokens, device=k.device)[None, :, None]
    visible = place <= at
    if case["kind"] != "shared":
        visible = visible & ((place > at - case["window"]) | (place < case["sinks"]))
    visible = visible.repeat_interleave(group, 1)[:, None]
    scores = (q @ k.transpose(2, 3)).masked_fill_(~visible, -math.inf)
    if case["kind"] != "shared":
        out = _softmax(scores) @ v
    else:
        pk, pv = (_unpaged(p, s["prefix_pool"][2])[0, :, :case["prefix"]] for p in s["prefix_pool"][:2])
        far = q.transpose(0, 1).reshape(kv, -1, HEAD) @ pk.transpose(1, 2)
        far = far.view(kv, batch, tokens * group, -1).transpose(0, 1)
        weight = _softmax(torch.cat([far, scores], -1))
        far = weight[..., :case["prefix"]].transpose(0, 1).reshape(kv, batch * tokens * group, -1) @ pv
        out = weight[..., case["prefix"]:] @ v + far.view(kv, batch, tokens * group, HEAD).transpose(0, 1)
    out = out.view(batch, kv, tokens, group, HEAD).transpose(1, 2)
    return out.reshape(batch * tokens, heads * HEAD).to(torch.bfloat16)


# ---- the framework's calls --------------------------------------------------------------------------

def _handles(s):
    """What a program sets up once for its cache: the view of its pages and the attention over them."""
    from starter_b200 import ops
    case = s["case"]
    batch, tokens, kv, heads = case["batch"], case["tokens"], case["kv_heads"], case["q_heads"]
    cache = ops.PagedKV(batch, kv, s["keys"], DEVICE, block_table=s["pool"][2], pools=s["pool"][:2])
    if case["kind"] == "window":
        attention = ops.WindowAttention(batch, heads, kv, s["keys"], DEVICE, case["window"], case["sinks"], tokens)
        return cache, attention
    if case["kind"] == "window_prompt":
        return cache, None
    prefix = ops.PagedKV(1, kv, case["prefix"], DEVICE, block_table=s["prefix_pool"][2], pools=s["prefix_pool"][:2])
    attention = ops.SharedPrefixAttention(batch, heads, kv, case["prefix"], s["keys"], DEVICE, tokens)
    return cache, attention, prefix


def _own(s):
    from starter_b200 import ops
    case = s["case"]
    if case["kind"] == "sample":
        return ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                 top_p=s["top_p"], min_p=s["min_p"])
    if "handles" not in s:
        s["handles"] = _handles(s)
    cache, attention = s["handles"][:2]
    if case["kind"] == "window_prompt":
        return ops.window_prompt_attention(s["query"], cache, s["position"], case["tokens"], SCALE, case["window"],
                                           case["sinks"])
    if case["kind"] == "window":
        return attention.run(s["query"], cache, s["position"], SCALE)
    return attention.run(s["query"], s["handles"][2], s["prefix_length"], cache, s["position"], SCALE)


def run(state):
    if own:
        return _own(state)
    return _plain_sample(state) if state["case"]["kind"] == "sample" else _plain_attention(state)


def work(case):
    kind = case["kind"]
    if kind == "sample":
        entries = case["rows"] * case["vocab"]
        return {"bytes": entries * (2 if case["dtype"] == "bf16" else 4) + case["rows"] * 16, "flops": 2 * entries}
    batch, tokens, kv, heads = case["batch"], case["tokens"], case["kv_heads"], case["q_heads"]
    key_bytes, io = 2 * 2 * HEAD * kv, 2 * 2 * HEAD * heads * batch * tokens
    if kind == "shared":
        # the sequences' own positions are spread over the second half of their pages
        mine = batch * (case["own_keys"] - (case["own_keys"] - tokens) // 4)
        return {"bytes": (case["prefix"] + mine) * key_bytes + io,
                "flops": 4 * HEAD * heads * tokens * (batch * case["prefix"] + mine)}
    if kind == "window":
        first, spread = case["context"] - tokens, (case["context"] - tokens) // 2
        firsts = [first - round(i * spread / 8) for i in range(9)]
        share = batch / 9
    else:
        firsts, share = [case["before"]], batch

    def seen(at):
        """Keys that the row at this position sees."""
        near = max(0, at - case["window"] + 1)
        return at + 1 - near + min(near, case["sinks"])

    def seen_by_any(at):
        near = max(0, at - case["window"] + 1)
        return at + tokens - near + min(near, case["sinks"])

    return {"bytes": share * sum(seen_by_any(a) for a in firsts) * key_bytes + io,
            "flops": 4 * HEAD * heads * share * sum(seen(a + t) for a in firsts for t in range(tokens))}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _exact_sample(s):
    import numpy as np
    tokens, chances = [], []
    x = s["logits"].double().cpu().numpy()
    for row in range(x.shape[0]):
        def setting(name):
            v = s[name]
            return float(v[row]) if isinstance(v, torch.Tensor) else float(torch.tensor(v, dtype=torch.float32))
        ids = np.lexsort((np.arange(x.shape[1]), -x[row]))          # largest first, equal ones by their index
        z = (x[row][ids] - x[row][ids[0]]) / setting("temperature")
        k = int(setting("top_k"))
        n = k if 0 < k < len(ids) else len(ids)
        n = min(n, int(np.count_nonzero(np.exp(z) >= setting("min_p")))) if setting("min_p") > 0 else n
        w = np.exp(z[:n])
        if setting("top_p") < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), setting("top_p") * np.sum(w))))
        ids, w = ids[:n], w[:n]
        order = np.argsort(ids)
        ids, w = ids[order], w[order]
        at = int(np.searchsorted(np.cumsum(w), float(s["uniform"][row]) * np.sum(w), side="right"))
        at = min(at, n - 1)
        tokens.append(int(ids[at]))
        chances.append(math.log(w[at] / np.sum(w)))
    return torch.tensor(tokens, dtype=torch.int64), torch.tensor(chances, dtype=torch.float64)


def _key_rows(pool, table, head, places):
    """Rows of one head at the given places of one sequence, in 64 bits."""
    r = places % PAGE
    flat = pool[table[places // PAGE].long(), head, r].double().view(-1, 16, 8)
    return flat.gather(1, (torch.arange(16, device=pool.device)[None] ^ (r[:, None] & 7))[..., None].expand(-1, -1, 8)).reshape(-1, HEAD)


def _exact_attention(s):
    case = s["case"]
    batch, tokens, kv, heads = case["batch"], case["tokens"], case["kv_heads"], case["q_heads"]
    group = heads // kv
    q = s["query"].view(batch, tokens, heads, HEAD)
    out = torch.zeros((batch, tokens, heads, HEAD), dtype=torch.float64, device=q.device)
    window, sinks = case.get("window", 1 << 30), case.get("sinks", 0)
    step = 256                                             # query tokens looked at together
    first = s["position"].tolist()
    for h in range(kv):
        if case["kind"] == "shared":
            places = torch.arange(case["prefix"], device=q.device)
            pk, pv = (_key_rows(p, s["prefix_pool"][2][0], h, places) for p in s["prefix_pool"][:2])
        for b in range(batch):
            for t0 in range(0, tokens, step):
                n = min(step, tokens - t0)
                at = first[b] + t0
                low = max(0, at - window + 1)
                places = torch.cat([torch.arange(min(sinks, low), device=q.device),
                                    torch.arange(low, at + n, device=q.device)])
                k, v = (_key_rows(p, s["pool"][2][b], h, places) for p in s["pool"][:2])
                mine = torch.arange(at, at + n, device=q.device)[:, None]
                hidden = (places[None] > mine) | ((places[None] <= mine - window) & (places[None] >= sinks))
                hidden = hidden.repeat_interleave(group, 0)
                x = q[b, t0:t0 + n, h * group:(h + 1) * group].reshape(n * group, HEAD).double()
                z = ((x @ k.T) / math.sqrt(HEAD)).masked_fill(hidden, -math.inf)
                if case["kind"] == "shared":
                    z, v = torch.cat([(x @ pk.T) / math.sqrt(HEAD), z], 1), torch.cat([pv, v])
                y = torch.softmax(z, 1) @ v
                out[b, t0:t0 + n, h * group:(h + 1) * group] = y.view(n, group, HEAD)
    return out.reshape(batch * tokens, heads * HEAD)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_sample(state) if case["kind"] == "sample" else _exact_attention(state)
