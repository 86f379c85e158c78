"""What a step over trees of drafted tokens adds to a decoder, measured: attention in which a drafted token sees the cached keys and its own
ancestors, sampling with temperature, top-k, top-p and min-p from given uniform numbers, the walk to the drafted tokens that the model agrees
with, and the move of their keys and values to where they belong in the paged cache.

A tree's nodes are an entry's rows in a step, parents in front of their children; node i's keys and values lie at cache position context + i,
and its position in the text is context + its depth.
"""
import itertools
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
MIXED = {"temperature": [0.0, 0.3, 0.8, 1.2], "top_k": [0, 0, 20, 500], "top_p": [1.0, 0.95, 0.9, 0.5], "min_p": [0.0, 0.0, 0.05, 0.2]}
SETTINGS = {"temperature": torch.float32, "top_k": torch.int32, "top_p": torch.float32, "min_p": torch.float32}


# ---- cases ----------------------------------------------------------------------------------------------------------
def _attention(requests, nodes, context, heads, kv_heads, dim, page, window=0, dtype="bfloat16", tree="random"):
    return {"op": "attention", "requests": requests, "nodes": nodes, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "dtype": dtype, "tree": tree}


def _sample(rows, vocab, temperature=0.0, top_k=0, top_p=0.0, min_p=0.0, mixed=False, rounded=False):
    """mixed: rows of requests that ask for different settings (MIXED), greedy ones among them; rounded: logits that a product left in bfloat16."""
    return {"op": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "rounded": rounded}


def _accept(requests, nodes, longest):
    return {"op": "accept", "requests": requests, "nodes": nodes, "longest": longest}


def _keep(requests, nodes, longest, context, layers, kv_heads, dim, page, dtype="bfloat16"):
    return {"op": "keep", "requests": requests, "nodes": nodes, "longest": longest, "context": context, "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype}


def listed():
    return [
        # one user's chat, a draft of eight tokens in a row: latency
        dict(_attention(1, 8, 500, 14, 2, 64, 16, tree="chain"), name="attention_chat"),
        # eight requests deep in their contexts with trees of up to 24 nodes, at the 0.5B sizes of the benchmark
        dict(_attention(8, 24, 4096, 14, 2, 64, 64), name="attention_b8"),
        # small trees of many requests under a sliding window, pages of 16
        dict(_attention(32, 7, 8000, 16, 4, 128, 16, window=1024), name="attention_window"),
        # the 32-bit path
        dict(_attention(4, 13, 1000, 12, 2, 128, 16, dtype="float32"), name="attention_f32"),
        # wide trees over long contexts at the 7B sizes of the benchmark: the largest
        dict(_attention(16, 64, 32768, 28, 4, 128, 64), name="attention_long"),
        # one row: the end of a plain decode step
        dict(_sample(1, 151936, 0.8, 20, 0.95, 0.05), name="sample_chat"),
        # every node of attention_b8's trees, requests with settings of their own
        dict(_sample(192, 151936, mixed=True), name="sample_mixed"),
        # an odd vocabulary, whole rows in the running (temperature and a small min-p only), logits that a product rounded: ties
        dict(_sample(64, 32001, 1.2, 0, 1.0, 0.002, rounded=True), name="sample_flat"),
        dict(_accept(1, 8, 8), name="accept_chat"),
        dict(_accept(256, 64, 16), name="accept_b256"),
        dict(_keep(8, 24, 8, 500, 24, 2, 64, 64), name="keep_b8"),
        dict(_keep(64, 64, 16, 700, 28, 4, 128, 16), name="keep_b64"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "sample", "sample", "accept", "keep"))
    if op == "attention":
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        dim = rng.choice((64, 128, 64, 128, 32, 256, 80))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 3, 4, 6, 7, 8))
        page, window = rng.choice((16, 32, 64, 128)), rng.choice((0, 0, _spread(rng, 100, 4096)))
        requests, nodes = _spread(rng, 1, 48), _spread(rng, 1, 100)
        context = _spread(rng, 1, 32768)
        # at most the largest case's multiply-adds and cached values (in float32 a sixteenth of them)
        share = 1 if dtype == "bfloat16" else 16
        while context > 1 and (requests * heads * nodes * context * dim * share > 16 * 28 * 64 * 32768 * 128 or requests * kv_heads * context * dim * share > 16 * 4 * 32768 * 128):
            context //= 2
        return _attention(requests, nodes, context, heads, kv_heads, dim, page, window, dtype, rng.choice(("random", "random", "chain")))
    if op == "sample":
        settings = rng.uniform(0.3, 2.0), rng.choice((0, 1, 20, 50, 1000)), rng.choice((1.0, 0.95, 0.5)), rng.choice((0.0, 0.01, 0.1))
        return _sample(_spread(rng, 1, 400), _spread(rng, 200, 151936), *settings, mixed=rng.random() < 0.5, rounded=rng.random() < 0.3)
    if op == "accept":
        return _accept(_spread(rng, 1, 256), _spread(rng, 1, 100), rng.randint(1, 20))
    return _keep(_spread(rng, 1, 64), _spread(rng, 2, 64), rng.randint(2, 16), _spread(rng, 1, 700), rng.choice((6, 14, 24, 28)), rng.choice((1, 2, 4)), rng.choice((32, 64, 128)),
                 rng.choice((16, 64)), rng.choice(("bfloat16", "bfloat16", "float32")))


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _part(r, step):
    """The r-th of a sequence that is spread evenly over [0, 1)."""
    return (0.5 + r * step) % 1.0


def _nodes(case):
    """Every request's nodes: from half of the most to all of it."""
    n = case["nodes"]
    return [n if r == 0 else max(1, n - int(_part(r, 0.618034) * n / 2)) for r in range(case["requests"])]


def _contexts(case):
    """Every request's cached keys: from a quarter of the most to all of it."""
    c = case["context"]
    return [c if r == 0 else max(0, c - int(_part(r, 0.754878) * 0.75 * c)) for r in range(case["requests"])]


def _parents(case, nodes, rng):
    """A draft's tree grows at a node that it has already, any of them alike; a chain at the last one."""
    flat = []
    for n in nodes:
        u = torch.rand(n, generator=rng).tolist()
        flat += [-1] + [i - 1 if case.get("tree") == "chain" else min(i - 1, int(u[i] * i)) for i in range(1, n)]
    return flat


def _tables(case, tokens, rng):
    """A block table over shuffled pages, and how many pages there are."""
    page = case["page"]
    pages = [-(-t // page) for t in tokens]
    order = torch.randperm(sum(pages), generator=rng).to(torch.int32)
    table = torch.full((len(tokens), max(pages)), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = order[at:at + n]
        at += n
    return table, at


def prepare(case, seed):
    rng = torch.Generator().manual_seed(seed)
    gpu = torch.Generator("cuda").manual_seed(seed)
    state = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        spread = 1.0 + 3.0 * torch.rand((rows, 1), generator=gpu, device="cuda")             # from unsure rows to sure ones
        logits = torch.randn((rows, vocab), generator=gpu, device="cuda") * spread
        if case["rounded"]:
            logits = logits.bfloat16().float()
        for key, dtype in SETTINGS.items():
            given = torch.tensor(MIXED[key])[torch.randint(0, 4, (rows,), generator=rng)] if case["mixed"] else torch.full((rows,), case[key])
            state[key] = given.to("cuda", dtype)
        state["uniform"] = torch.rand(rows, generator=rng).cuda()
        state["logits"], state["out"] = logits, torch.empty(rows, dtype=torch.int32, device="cuda")
        return state
    nodes = _nodes(case)
    total, requests = sum(nodes), case["requests"]
    starts, parents = [0, *itertools.accumulate(nodes)], _parents(case, nodes, rng)
    state["starts"], state["parents"] = torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(parents, dtype=torch.int32).cuda()
    state["most_nodes"] = max(nodes)
    if case["op"] == "accept":
        # the model agrees with every second drafted token (where several of a node's children would be it, with one of them)
        tokens = torch.randint(0, 32000, (total,), generator=rng, dtype=torch.int32)
        targets = torch.randint(0, 32000, (total,), generator=rng, dtype=torch.int32)
        tokens, targets, agrees = tokens.tolist(), targets.tolist(), torch.rand(total, generator=rng).tolist()
        for first, n in zip(starts, nodes):
            for i in range(first + 1, first + n):
                if agrees[i] < 0.5:
                    targets[first + parents[i]] = tokens[i]
        state["tokens"], state["targets"] = torch.tensor(tokens, dtype=torch.int32).cuda(), torch.tensor(targets, dtype=torch.int32).cuda()
        state["path"] = torch.empty((requests, case["longest"]), dtype=torch.int32, device="cuda")
        state["emitted"] = torch.empty_like(state["path"])
        state["accepted"] = torch.empty(requests, dtype=torch.int32, device="cuda")
        return state
    contexts, dtype = _contexts(case), DTYPES[case["dtype"]]
    table, pages = _tables(case, [c + n for c, n in zip(contexts, nodes)], rng)
    state["context"], state["table"] = torch.tensor(contexts, dtype=torch.int32).cuda(), table.cuda()
    if case["op"] == "keep":
        # a random walk down every tree
        path = torch.full((requests, case["longest"]), -1, dtype=torch.int32)
        accepted = torch.zeros(requests, dtype=torch.int32)
        for r, n in enumerate(nodes):
            own_parents = parents[starts[r]:starts[r + 1]]
            walk = [0]
            while len(walk) < case["longest"]:
                children = [i for i in range(n) if own_parents[i] == walk[-1]]
                if not children:
                    break
                walk.append(children[int(torch.randint(0, len(children), (1,), generator=rng))])
            path[r, :len(walk)], accepted[r] = torch.tensor(walk, dtype=torch.int32), len(walk)
        state["path"], state["accepted"] = path.cuda(), accepted.cuda()
        shape = (case["layers"], pages, 2, case["kv_heads"], case["page"], case["dim"])
        state["kv"] = torch.randn(shape, generator=gpu, device="cuda", dtype=dtype)
        return state
    # the rows of a step come out of the product as q | k | v; three rows behind the last request pad the step
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    qkv = torch.randn((total + 3, (heads + 2 * kv_heads) * dim), generator=gpu, device="cuda", dtype=dtype)
    state["q"] = qkv[:, :heads * dim]
    kv = torch.randn((pages + 1, 2, kv_heads, case["page"], dim), generator=gpu, device="cuda", dtype=dtype)
    state["k"], state["v"] = kv[:, 0], kv[:, 1]
    state["out"] = torch.zeros((total + 3, heads * dim), device="cuda", dtype=dtype)
    state["most_context"] = max(c + n for c, n in zip(contexts, nodes))
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"attention": _run_attention, "sample": _run_sample, "accept": _run_accept, "keep": _run_keep}[case["op"]](state, case)


def _tree_of(state):
    """(rows [R, N] of the nodes, which of them are there, is-ancestor-or-self [R, N, N]) of every request, padded to the most nodes."""
    starts, parents, most = state["starts"].long(), state["parents"].long(), state["most_nodes"]
    nodes = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    there = i < nodes[:, None]
    rows = torch.where(there, starts[:-1, None] + i, 0)
    parent = torch.where(there, parents[rows], -1)
    step = (parent[:, :, None] == i).double()                        # step[i, parent of i] = 1: strictly lower
    reach = torch.linalg.solve_triangular(torch.eye(most, device="cuda", dtype=torch.float64) - step, torch.eye(most, device="cuda", dtype=torch.float64).expand_as(step),
                                          upper=False, unitriangular=True) > 0.5              # 1 + step + step^2 + ...
    return rows, there, reach


def _run_attention(state, case):
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    if own:
        from easy_gpt.cpp_b200 import kernels

        kernels.attention_tree(state["q"], state["k"], state["v"], state["table"], state["starts"], state["context"], state["parents"], state["out"], heads, kv_heads, dim,
                               window or None, dim ** -0.5, state["status"], max_context=state["most_context"])
        return state["out"]
    rows, there, reach = _tree_of(state)
    (requests, most), group, page = rows.shape, heads // kv_heads, case["page"]
    context = state["context"].long()
    keys = torch.arange(state["most_context"], device="cuda")
    pages = state["table"][:, :-(-keys.numel() // page)].long().clamp(min=0)
    k, v = (state[x][pages].transpose(1, 2).reshape(requests, kv_heads, -1, dim)[:, :, :keys.numel()].float() for x in ("k", "v"))
    q = state["q"][rows].view(requests, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, group * most, dim).float()
    depth = reach.sum(-1) - 1
    node = (keys - context[:, None]).clamp(0, most - 1)              # of the keys behind the cached ones
    cached = keys < context[:, None]
    in_tree = torch.gather(reach & there[:, None, :], 2, node[:, None, :].expand(-1, most, -1)) & (keys < context[:, None] + most)[:, None, :]
    seen = torch.where(cached[:, None, :], True, in_tree)
    if window:
        at = torch.where(cached, keys, context[:, None] + torch.gather(depth, 1, node))
        seen &= at[:, None, :] > (context[:, None] + depth)[:, :, None] - window
    scores = (q @ k.transpose(2, 3)).view(requests, kv_heads, group, most, -1) * dim ** -0.5
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    weights /= weights.sum(-1, keepdim=True)
    result = (weights.view(requests, kv_heads, group * most, -1) @ v).view(requests, heads, most, dim).transpose(1, 2).reshape(requests, most, heads * dim)
    state["out"][rows[there]] = result[there].to(state["out"].dtype)
    return state["out"]


def _run_sample(state, case):
    if own:
        from easy_gpt.cpp_b200 import kernels

        kernels.sample_min_p(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["uniform"], state["out"])
        return state["out"]
    # 64 bits: a uniform number next to a token's border decides between two tokens
    x, vocab = state["logits"].double(), case["vocab"]
    temperature, top_p, min_p, uniform = (state[k].double()[:, None] for k in ("temperature", "top_p", "min_p", "uniform"))
    top_k = state["top_k"][:, None]
    index = torch.arange(vocab, device="cuda")
    biggest = x.amax(1, keepdim=True)
    greedy = torch.where(x == biggest, index, vocab).amin(1)
    weight = ((x - biggest) / torch.where(temperature > 0, temperature, 1.0)).exp()
    order = x.sort(dim=1, descending=True, stable=True).indices           # ties: the lower index first
    sorted_weight = weight.gather(1, order)
    sorted_weight = torch.where((top_k > 0) & (index >= top_k), 0.0, sorted_weight)
    before = sorted_weight.cumsum(1) - sorted_weight
    cut = (top_p > 0) & (top_p < 1) & (before >= top_p * sorted_weight.sum(1, keepdim=True)) & (index > 0)
    sorted_weight = torch.where(cut | ((min_p > 0) & (sorted_weight < min_p)), 0.0, sorted_weight)
    kept = torch.zeros_like(weight).scatter_(1, order, sorted_weight)
    cumulated = kept.cumsum(1)
    chosen = (cumulated <= uniform * cumulated[:, -1:]).sum(1)
    last = torch.where(kept > 0, index, 0).amax(1)
    state["out"].copy_(torch.where(temperature[:, 0] > 0, torch.minimum(chosen, last), greedy))
    return state["out"]


def _run_accept(state, case):
    if own:
        from easy_gpt.cpp_b200 import kernels

        kernels.tree_accept(state["tokens"], state["targets"], state["starts"], state["parents"], state["path"], state["accepted"], state["emitted"], state["status"])
        return state["path"], state["accepted"], state["emitted"]
    rows, there, reach = _tree_of(state)
    tokens, targets, parents = (state[k].long()[rows] for k in ("tokens", "targets", "parents"))
    most, longest = rows.shape[1], case["longest"]
    i = torch.arange(most, device="cuda")
    agrees = there & ((i == 0) | ((parents >= 0) & (tokens == targets.gather(1, parents.clamp(min=0)))))
    # of the children of a node that bear its token the first counts
    twin = (parents[:, :, None] == parents[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & (i[:, None] > i) & there[:, None, :]
    agrees &= ~twin.any(2)
    taken = ~(reach & ~agrees[:, None, :]).any(2) & there
    rank = taken.cumsum(1) - 1
    taken &= rank < longest
    path = torch.full((rows.shape[0], max(most, longest) + 1), -1, device="cuda", dtype=torch.long)
    path.scatter_(1, torch.where(taken, rank, max(most, longest)), i.expand_as(rank))
    path = path[:, :longest]
    state["path"].copy_(path)
    state["accepted"].copy_(taken.sum(1))
    state["emitted"].copy_(torch.where(path >= 0, targets.gather(1, path.clamp(min=0)), -1))
    return state["path"], state["accepted"], state["emitted"]


def _run_keep(state, case):
    if own:
        from easy_gpt.cpp_b200 import kernels

        kernels.cache_keep(state["kv"], state["table"], state["context"], state["path"], state["accepted"], state["status"])
        return state["kv"]
    kv, page, context = state["kv"], case["page"], state["context"].long()[:, None]
    j = torch.arange(case["longest"], device="cuda")
    moved = j < state["accepted"][:, None]                           # the others move node 0's row onto itself
    source, target = context + torch.where(moved, state["path"], 0), context + torch.where(moved, j, 0)
    table = state["table"].long()
    source_page, target_page = table.gather(1, source // page), table.gather(1, target // page)
    kv[:, target_page, :, :, target % page] = kv[:, source_page, :, :, source % page]
    return kv


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 24), "flops": 2 * case["rows"] * case["vocab"]}
    nodes = _nodes(case)
    if case["op"] == "accept":
        return {"bytes": 12 * sum(nodes) + case["requests"] * (8 + 8 * case["longest"]), "flops": 0}
    es = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "keep":
        # nodes of a random walk to a leaf that do not lie at their place already, on the average over many trees
        rows = max(1, int(case["requests"] * min(case["longest"] - 1, 0.57 * math.log(case["nodes"]))))
        return {"bytes": 2 * rows * case["layers"] * 2 * case["kv_heads"] * case["dim"] * es, "flops": 0}
    keys = [min(c, case["window"] or c) + n for c, n in zip(_contexts(case), nodes)]
    seen = sum(n * (min(c, case["window"] or c) + 1 + int(math.log(n))) for c, n in zip(_contexts(case), nodes))
    return {"bytes": 2 * sum(keys) * case["kv_heads"] * case["dim"] * es + 2 * sum(nodes) * case["heads"] * case["dim"] * es,
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ---- the same from the definition, in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "sample": _exact_sample, "accept": _exact_accept, "keep": _exact_keep}[case["op"]](state, case)


def _walks(state):
    """Per request: its first row, and every node's line of ancestors, itself last."""
    starts, parents = state["starts"].tolist(), state["parents"].tolist()
    for first, end in zip(starts, starts[1:]):
        lines = []
        for i in range(end - first):
            up = parents[first + i]
            lines.append((lines[up] if up >= 0 else []) + [i])
        yield first, lines


def _exact_attention(state, case):
    heads, kv_heads, dim, page, window = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    out = state["out"].double()
    for r, (first, lines) in enumerate(_walks(state)):
        c, n = int(state["context"][r]), len(lines)
        pages = state["table"][r, :-(-(c + n) // page)].long()
        k, v = (state[x][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :c + n].double() for x in ("k", "v"))
        hidden = torch.ones((n, c + n), dtype=torch.bool)
        for i, line in enumerate(lines):
            reach = window or c + n
            hidden[i, max(0, c + len(line) - reach):c] = False
            hidden[i, [c + a for a in line[-reach:]]] = False
        q = state["q"][first:first + n].double().view(n, kv_heads, heads // kv_heads, dim)
        s = torch.einsum("ngid,gkd->gink", q, k) * dim ** -0.5
        s = s.masked_fill(hidden.cuda(), -math.inf).softmax(-1)
        out[first:first + n] = torch.einsum("gink,gkd->ngid", s, v).reshape(n, heads * dim)
    return out


def _exact_sample(state, case):
    result = []
    for r in range(case["rows"]):
        x = state["logits"][r].double()
        t, k, p, low, u = (float(state[key][r]) for key in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        values, order = torch.sort(-x, stable=True)
        if t <= 0:
            result.append(int(order[0]))
            continue
        w = torch.exp((values[0] - values) / t)
        n = int(k) if 0 < k < len(w) else len(w)
        if 0 < p < 1:
            n = min(n, 1 + int((torch.cumsum(w[:n], 0)[:-1] < p * w[:n].sum()).sum()))
        if low > 0:
            n = min(n, int((w >= low).sum()))
        tokens, by_index = torch.sort(order[:n])
        run = torch.cumsum(w[:n][by_index], 0)
        result.append(int(tokens[min(n - 1, int(torch.searchsorted(run, u * run[-1], right=True)))]))
    return torch.tensor(result, dtype=torch.int32)


def _exact_accept(state, case):
    tokens, targets = state["tokens"].tolist(), state["targets"].tolist()
    path = torch.full((case["requests"], case["longest"]), -1, dtype=torch.int32)
    emitted, accepted = path.clone(), torch.zeros(case["requests"], dtype=torch.int32)
    for r, (first, lines) in enumerate(_walks(state)):
        at, count = 0, 0
        while at is not None and count < case["longest"]:
            path[r, count], emitted[r, count], count = at, targets[first + at], count + 1
            at = next((i for i, line in enumerate(lines) if len(line) > 1 and line[-2] == at and tokens[first + i] == targets[first + at]), None)
        accepted[r] = count
    return path, accepted, emitted


def _exact_keep(state, case):
    kv, page = state["kv"], case["page"]
    for r, (c, count) in enumerate(zip(state["context"].tolist(), state["accepted"].tolist())):
        pages = state["table"][r].tolist()
        for j, node in enumerate(state["path"][r, :count].tolist()):
            kv[:, pages[(c + j) // page], :, :, (c + j) % page] = kv[:, pages[(c + node) // page], :, :, (c + node) % page]
    return kv.double()
