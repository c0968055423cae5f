"""Several answers to one prompt, as cases that can be timed and checked.

A prompt is run once, its pages are shared by all of its answers, each answer decodes behind them, and what the answers
chose is scored.  Three operators, as a server uses them:

* ``prefix``    decode attention of rows that share their first keys: each group's shared keys are read once for all of its
                rows, every row's own keys follow, one softmax over both;
* ``pages``     the pages that a fork or a move of cached tokens copies, in the tensors of all layers at once;
* ``logprobs``  of each row of logits the log probability of a given token, the entropy and the most likely tokens.

prefix: a row (one token, ``heads`` query heads, query head h reads KV head h / (heads / kv_heads)) sees keys 0 .. kv_len - 1,
out = softmax(scale q . K) V; keys below its group's ``shared`` are read through the block table of the group's first row.
pages: for each move (source, target, n): slots 0 .. n - 1 of page ``target`` become those of page ``source``, in every tensor
[pages, kv_heads, page_size, dim]; all else stays.
logprobs: log softmax(l) at the token; H = - sum p log p; the ``top`` largest, equal ones by the lower id.
"""
import math

import torch

own = False


# ------------------------------------------------------------------------------------------------------------- cases
def _prefix(groups, rows, heads, kv_heads, dim, page, shared, own_keys, dtype="bfloat16"):
    """``groups`` prompts with up to ``rows`` answers each, prompts of up to ``shared`` tokens, answers of up to ``own_keys``."""
    return {"op": "prefix", "groups": groups, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "shared": shared, "own_keys": own_keys, "dtype": dtype}


def _pages(layers, kv_heads, dim, page, parents, children, slots, dtype="bfloat16"):
    """``parents`` pages, each copied to ``children`` others, ``slots`` of its tokens, in the K and V tensors of ``layers``."""
    return {"op": "pages", "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "parents": parents,
            "children": children, "slots": slots, "dtype": dtype}


def _logprobs(rows, vocab, top, masked=False, apart=0):
    """``masked``: most ids are forbidden (-inf), as under a grammar.  ``apart``: columns between a row's end and the next row."""
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "masked": masked, "apart": apart}


def listed():
    return [dict(c, name=n) for n, c in (
        # two answers to a short question, a small model: all latency
        ("prefix-2-short", _prefix(1, 2, 16, 8, 128, 16, 300, 9)),
        # eight samples of a reply behind a system prompt, wide layers
        ("prefix-8", _prefix(1, 8, 32, 8, 128, 16, 4096, 256)),
        # a server under load: six prompts of unlike length, up to twelve answers each, a small model
        ("prefix-six-groups", _prefix(6, 12, 16, 8, 128, 16, 3001, 700)),
        # many heads a KV head: 24 samples of the widest layers
        ("prefix-24-wide", _prefix(1, 24, 64, 8, 128, 16, 8000, 200)),
        # the 32-bit mode, no size is round, pages of no power of two
        ("prefix-float32-odd", _prefix(2, 13, 12, 4, 96, 24, 1501, 77, "float32")),
        # 64 samples behind a long document (the largest)
        ("prefix-64-long", _prefix(1, 64, 32, 8, 128, 16, 32768, 1024)),
        # one request is forked: its last page, nine tokens of it, in 28 layers
        ("fork-1", _pages(28, 8, 128, 16, 1, 1, 9)),
        # a prompt goes to 63 more answers, 36 layers
        ("fork-63", _pages(36, 8, 128, 16, 1, 63, 11)),
        # a cache is made compact: whole pages move, 32-bit, small heads
        ("move-500", _pages(12, 5, 48, 32, 500, 1, 32, "float32")),
        # one user asks for the five likeliest tokens beside the sampled one
        ("logprobs-1", _logprobs(1, 151936, 5)),
        # constrained decoding of 45 requests; odd vocabulary, rows out of a wider buffer
        ("logprobs-45-masked", _logprobs(45, 32003, 20, True, 29)),
        # a portion of a prompt is scored, with the twenty likeliest tokens at each place
        ("logprobs-2048", _logprobs(2048, 151936, 20)),
    )]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: 1 to 64 answers to 1 to 8 prompts of up to 32,768 tokens, heads of 16 to 256; 1 to 1,024 pages in 2 to 64
    layers; 1 to 2,048 rows of 100 to 262,144 logits; at most the largest case's work."""
    op = rng.choice(("prefix", "prefix", "prefix", "pages", "logprobs", "logprobs"))
    if op == "prefix":
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        dim = rng.choice((128, 128, 128, 64, 80, 256, 48, 16, 96))
        kv_heads, per = rng.choice((1, 2, 4, 8, 8, 5)), rng.choice((1, 2, 4, 8, 5, 3))
        groups, rows = rng.choice((1, 1, 1, 2, 3, 8)), _log_int(rng, 1, 64)
        most = 64 * 32 * 32768 * 128 // (2 if dtype == "bfloat16" else 32)
        shared = _log_int(rng, 1, max(2, min(32768, most // (groups * rows * kv_heads * per * dim))))
        return _prefix(groups, rows, kv_heads * per, kv_heads, dim, rng.choice((16, 16, 16, 8, 32, 64, 24)), shared,
                       _log_int(rng, 1, max(2, min(2048, most // (groups * rows * kv_heads * per * dim)))), dtype)
    if op == "pages":
        layers, kv_heads, dim, page = _log_int(rng, 2, 64), rng.choice((1, 2, 4, 8, 5)), rng.choice((128, 128, 64, 48, 80, 256)), rng.choice((16, 16, 8, 32, 24))
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        each = 2 * layers * kv_heads * dim * page * (2 if dtype == "bfloat16" else 4)
        moves = _log_int(rng, 1, max(2, min(1024, 600000000 // each)))
        children = rng.choice((1, 1, _log_int(rng, 1, moves)))
        return _pages(layers, kv_heads, dim, page, max(1, moves // children), children, rng.choice((page, rng.randint(1, page))), dtype)
    rows = _log_int(rng, 1, 2048)
    vocab = _log_int(rng, 100, min(262144, 2048 * 151936 // rows))
    return _logprobs(rows, vocab, rng.choice((0, 1, 5, 20, 32)), rng.random() < 0.2, rng.choice((0, 0, 4, 13)))


def _sizes(case):
    """Of a prefix case: each group's rows and shared keys, each row's keys beyond them (at least the new token's own)."""
    groups, most = case["groups"], case["rows"]
    rows = [max(1, most * (groups - g) // groups) for g in range(groups)]
    shared = [max(1, case["shared"] * (g + 1) // groups) for g in range(groups)]
    own_keys = [1 + (case["own_keys"] - 1) * ((i * 37 + 96) % 97) // 96 for i in range(sum(rows))]
    return rows, shared, own_keys


# ------------------------------------------------------------------------------------------------------ the timed call
def _prepare_prefix(case, gen):
    device, dtype, page, dim, kv_heads = "cuda", getattr(torch, case["dtype"]), case["page"], case["dim"], case["kv_heads"]
    rows, shared, own_keys = _sizes(case)
    tables, at, starts, of = [], 0, [0], []
    total = sum(-(-s // page) + r for s, r in zip(shared, rows)) + sum(-(-k // page) + 1 for k in own_keys)
    order = (torch.randperm(total, generator=gen, device=device) + 1).tolist()
    i = 0
    for g, (count, keys) in enumerate(zip(rows, shared)):
        whole = order[at:at + keys // page]                  # the pages that the group's rows share
        at += len(whole)
        begun = None
        for _ in range(count):
            need = -(-(keys + own_keys[i]) // page) - len(whole)
            mine = order[at:at + need]
            at += need
            if keys % page:
                begun = begun or mine[0]                     # (a fork copies the page that the prompt has begun)
                of.append((begun, mine[0], keys % page))
            tables.append(whole + mine)
            i += 1
        starts.append(i)
    n, width = len(tables), max(len(t) for t in tables)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    # keys and queries behind a per-head norm: scores of a few units, some keys far more alike to the query than others
    k = torch.empty(total + 1, kv_heads, page, dim, device=device, dtype=dtype).normal_(generator=gen)
    v = torch.empty(total + 1, kv_heads, page, dim, device=device, dtype=dtype).normal_(generator=gen)
    for a, b, slots in of:
        k[b, :, :slots] = k[a, :, :slots]
        v[b, :, :slots] = v[a, :, :slots]
    q = (normal(n, case["heads"] * dim) * 1.5).to(dtype)
    table = torch.zeros(n, width, dtype=torch.int32)
    for r, t in enumerate(tables):
        table[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
    lengths = [shared[g] + own_keys[r] for g in range(len(rows)) for r in range(starts[g], starts[g + 1])]
    ints = dict(dtype=torch.int32, device=device)
    return {"q": q, "k": k, "v": v, "table": table.to(device), "cu_q": torch.arange(n + 1, **ints), "kv_len": torch.tensor(lengths, **ints),
            "rows": torch.arange(n, **ints), "groups": torch.tensor([[s, k] for s, k in zip(starts, shared)], **ints),
            "heads": case["heads"], "kv_heads": kv_heads, "dim": dim, "page": page, "scale": dim ** -0.5,
            "most_rows": max(rows), "most_shared": max(shared), "most_own": max(own_keys)}


def _prepare_pages(case, gen):
    device, dtype = "cuda", getattr(torch, case["dtype"])
    moves = case["parents"] * case["children"]
    total = case["parents"] + moves + 2
    pools = torch.empty(2 * case["layers"], total + 1, case["kv_heads"], case["page"], case["dim"], device=device, dtype=dtype)
    pools.normal_(generator=gen)
    order = torch.randperm(total, generator=gen, device=device).cpu() + 1
    source = order[:case["parents"]].repeat_interleave(case["children"])
    target = order[case["parents"]:case["parents"] + moves]
    state = {"pools": pools, "slots": case["slots"], "source": source.to(device), "target": target.to(device),
             "moves": torch.stack([source, target, torch.full_like(source, case["slots"])], 1).to(torch.int32)}
    if own:                                                  # what knows a cache's tensors is made once, with the cache
        from llm_infer_rust_b200.kernels import pages
        state["copier"] = pages.PageCopier(list(pools.unbind(0)))
    return state


def _prepare_logprobs(case, gen):
    device, rows, vocab = "cuda", case["rows"], case["vocab"]
    wide = torch.empty(rows, vocab + case["apart"], device=device)
    logits = wide[:, :vocab].normal_(generator=gen)
    # rows of unlike sharpness, from hardly any choice left to nearly none made
    logits *= torch.exp(1.2 * torch.rand(rows, 1, generator=gen, device=device) + 0.2)
    logits += 3.0
    top = case["top"]
    tokens = torch.randint(vocab, (rows,), generator=gen, device=device)
    if case["masked"]:
        allowed = torch.rand(vocab, generator=gen, device=device) < 0.1
        allowed[torch.randint(vocab, (min(vocab, 2 * top + 1),), generator=gen, device=device)] = True
        allowed[:min(vocab, top + 1)] = True                 # (as many are left as are asked for)
        logits.masked_fill_(~allowed, -math.inf)
        tokens = allowed.nonzero()[:, 0][tokens % int(allowed.sum())]
    return {"logits": logits, "tokens": tokens.to(torch.int32), "top": min(top, vocab)}


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return dict({"prefix": _prepare_prefix, "pages": _prepare_pages, "logprobs": _prepare_logprobs}[case["op"]](case, gen), op=case["op"])


def _plain_prefix(s):
    rows, first, shared, page = s["rows"].long(), s["groups"][:, 0].long(), s["groups"][:, 1].long(), s["page"]
    n, heads, kv_heads, dim = rows.numel(), s["heads"], s["kv_heads"], s["dim"]
    kv_len = s["kv_len"][rows].long()
    q = s["q"].float().view(-1, kv_heads, heads // kv_heads, dim)[s["cu_q"].long()[rows]]
    device = q.device
    place = torch.arange(n, device=device)
    group = torch.searchsorted(first, place, right=True) - 1
    # every group's shared keys, once, against all of its rows
    at = torch.arange(s["most_shared"], device=device)
    pages = s["table"].long()[rows[first]][:, (at // page).clamp(max=s["table"].shape[1] - 1)]
    k, v = s["k"][pages, :, at % page].float(), s["v"][pages, :, at % page].float()
    member = (first[:, None] + torch.arange(s["most_rows"], device=device)).clamp(max=n - 1)
    scores = torch.einsum("grhqd,gphd->grhqp", q[member], k)[group, place - first[group]] * s["scale"]
    seen = at < torch.minimum(shared[group], kv_len)[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    # every row's own keys
    own_at = shared[group][:, None] + torch.arange(s["most_own"], device=device)
    own_pages = s["table"].long()[rows].gather(1, (own_at // page).clamp(max=s["table"].shape[1] - 1))
    own_k, own_v = s["k"][own_pages, :, own_at % page].float(), s["v"][own_pages, :, own_at % page].float()
    own_scores = torch.einsum("rhqd,rphd->rhqp", q, own_k) * s["scale"]
    own_scores = own_scores.masked_fill((own_at >= kv_len[:, None])[:, None, None], -math.inf)
    # one softmax over both
    top = torch.maximum(scores.amax(-1), own_scores.amax(-1)).clamp(min=-3e38)[..., None]
    w, own_w = torch.exp(scores - top), torch.exp(own_scores - top)
    total = (w.sum(-1) + own_w.sum(-1))[..., None]
    shape = (first.numel(), s["most_rows"]) + tuple(w.shape[1:])
    spread = torch.zeros(shape, device=device)
    spread[group, place - first[group]] = w
    out = torch.einsum("grhqp,gphd->grhqd", spread, v)[group, place - first[group]] + torch.einsum("rhqp,rphd->rhqd", own_w, own_v)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.reshape(n, heads * dim).to(s["q"].dtype)


def _plain_pages(s):
    pools, slots = s["pools"], s["slots"]
    pools[:, s["target"], :, :slots] = pools[:, s["source"], :, :slots]
    return pools


def _plain_logprobs(s):
    logits, top = s["logits"], s["top"]
    vocab = logits.shape[1]
    down = logits - logits.amax(1, keepdim=True)
    e = torch.exp(down)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    chosen = down.gather(1, s["tokens"].long()[:, None])[:, 0] - log_total[:, 0]
    entropy = log_total[:, 0] - torch.where(e > 0, e * down, torch.zeros_like(e)).sum(1) / total[:, 0]
    if not top:
        return chosen, entropy
    # equal logits by the lower id: one whole number that falls as the order asks
    bits = (logits + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * 2 ** 20 + (vocab - 1 - torch.arange(vocab, device=logits.device))
    ids = torch.topk(key, top, dim=1).indices
    return chosen, entropy, ids.to(torch.int32), down.gather(1, ids) - log_total


def _own(s):
    if s["op"] == "prefix":
        from llm_infer_rust_b200.kernels import prefix
        out = torch.empty_like(s["q"])
        prefix.prefix_attention(s["q"], s["k"], s["v"], out, s["table"], s["cu_q"], s["kv_len"], s["rows"], s["groups"], s["heads"],
                                s["kv_heads"], s["dim"], s["page"], s["scale"], most_rows=s["most_rows"], most_shared=s["most_shared"],
                                most_own=s["most_own"])
        return out
    if s["op"] == "pages":
        s["copier"].copy(s["moves"])
        return s["pools"]
    from llm_infer_rust_b200.kernels import ops
    found = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    return (found.logprobs, found.entropy) + ((found.top_ids, found.top_logprobs) if s["top"] else ())


def run(state):
    if own:
        return _own(state)
    return {"prefix": _plain_prefix, "pages": _plain_pages, "logprobs": _plain_logprobs}[state["op"]](state)


def work(case):
    if case["op"] == "prefix":
        rows, shared, own_keys = _sizes(case)
        e = 2 if case["dtype"] == "bfloat16" else 4
        keys = sum(shared) + sum(own_keys)
        seen = sum(r * s for r, s in zip(rows, shared)) + sum(own_keys)
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * e + 2 * sum(rows) * case["heads"] * case["dim"] * e,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["op"] == "pages":
        each = 2 * case["layers"] * case["kv_heads"] * case["slots"] * case["dim"] * (2 if case["dtype"] == "bfloat16" else 4)
        return {"bytes": case["parents"] * (1 + case["children"]) * each, "flops": 0}
    rows, vocab, top = case["rows"], case["vocab"], min(case["top"], case["vocab"])
    # a subtraction, an exponential, two sums and a product an element
    return {"bytes": 4 * rows * (vocab + 3 + 2 * top), "flops": 5 * rows * vocab}


# ------------------------------------------------------------------------------------------- the same in 64 bits, apart
def exact(case, seed):
    if case["op"] == "pages":
        return None                                          # (nothing is computed)
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        chosen, entropy, ids, best = [], [], [], []
        for row, token in zip(s["logits"], s["tokens"].tolist()):
            p = torch.log_softmax(row.double(), 0)
            chosen.append(p[token])
            entropy.append(-(p.exp() * p)[p > -math.inf].sum())
            if s["top"]:
                ids.append(torch.sort(row, descending=True, stable=True).indices[:s["top"]])
                best.append(p[ids[-1]])
        found = (torch.stack(chosen), torch.stack(entropy))
        return found + ((torch.stack(ids).to(torch.int32), torch.stack(best)) if s["top"] else ())
    out = []
    per = s["heads"] // s["kv_heads"]
    for r, keys in enumerate(s["kv_len"].tolist()):
        at = torch.arange(keys, device="cuda")
        pages = s["table"][r].long()[at // s["page"]]
        k = s["k"][pages, :, at % s["page"]].double().repeat_interleave(per, 1)
        v = s["v"][pages, :, at % s["page"]].double().repeat_interleave(per, 1)
        q = s["q"][r].double().view(s["heads"], 1, s["dim"])
        p = torch.softmax(torch.matmul(q, k.permute(1, 2, 0)) * s["scale"], -1)
        out.append(torch.matmul(p, v.permute(1, 0, 2)).reshape(-1))
    return torch.stack(out)
