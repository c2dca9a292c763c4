"""Operators of decoding with drafted tokens, as cases that can be timed: attention of a tree of drafted tokens over the cache
(`Attention.forward_draft`), log probabilities of given tokens with entropy and top alternatives (`ops.token_log_probs`) and the walk
that accepts drafted tokens (`ops.accept_draft`).

`own` False: the operators in plain torch operations; True: the framework's.
"""
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
CHUNK = 64


def framework():
    sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "chunk-attention_b200"))
    import chunk_attn
    return chunk_attn


# ---- the cases -------------------------------------------------------------------------------------------------------------
# "attention": rows sequences that share `shared` tokens of prompt and have up to `context` of their own; every one brings a tree of up to
# `nodes` drafted tokens (the first is its last token), each drafted under one of the `reach` before it (reach 1: a chain).
# "log_probs": `rows` rows of logits over `vocab` tokens, `given` tokens named per row, the `top` best reported.
# "accept": trees as above; threshold 0: a drafted token is accepted where it is the model's choice, else also where it is probable enough.

def listed():
    return [
        # one request, a chain of drafted tokens from its own text: the time of a call
        dict(name="chain, one request", kind="attention", dtype="float16", heads=32, kv_heads=32, dim=128, rows=1, shared=0, context=4000, ragged=False, nodes=5, reach=1),
        # a short prompt of a small model, the smallest call
        dict(name="chain, heads of 64", kind="attention", dtype="float16", heads=12, kv_heads=12, dim=64, rows=1, shared=0, context=300, ragged=False, nodes=4, reach=1),
        # requests over one prompt with an answer of their own each
        dict(name="trees 32x(2048+512)", kind="attention", dtype="float16", heads=32, kv_heads=32, dim=128, rows=32, shared=2048, context=512, ragged=False, nodes=13, reach=6),
        # a serving batch of a model with grouped heads
        dict(name="trees, grouped 64x1024", kind="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, rows=64, shared=0, context=1024, ragged=True, nodes=24, reach=10),
        # long documents, wide trees: more queries to a key/value head than a tile has rows
        dict(name="trees, long grouped 8x16000", kind="attention", dtype="bfloat16", heads=64, kv_heads=8, dim=128, rows=8, shared=0, context=16000, ragged=True, nodes=63, reach=24),
        # the fp32 mode
        dict(name="trees fp32 4x288", kind="attention", dtype="float32", heads=32, kv_heads=32, dim=128, rows=4, shared=0, context=288, ragged=True, nodes=9, reach=4),
        # one decoded token with its alternatives: latency
        dict(name="alternatives of one token", kind="log_probs", dtype="float32", rows=1, vocab=32000, given=1, top=5),
        # the nodes of a batch of trees: each node's choice and the probabilities of the tokens drafted under it
        dict(name="nodes of 64 trees", kind="log_probs", dtype="float16", rows=1536, vocab=32000, given=1, top=1),
        # scoring of prompts over a large vocabulary
        dict(name="prompts, large vocabulary", kind="log_probs", dtype="bfloat16", rows=2048, vocab=128000, given=1, top=20),
        # a vocabulary of odd size: rows that start anywhere
        dict(name="prompt, odd vocabulary", kind="log_probs", dtype="float32", rows=517, vocab=50001, given=2, top=8),
        # one request
        dict(name="accept a chain", kind="accept", rows=1, nodes=5, reach=1, threshold=0.0),
        # a large batch of wide trees, tokens accepted by probability
        dict(name="accept in 256 trees", kind="accept", rows=256, nodes=63, reach=24, threshold=0.09),
    ]


LARGEST = dict(kind="attention", dtype="bfloat16", heads=64, kv_heads=8, dim=128, rows=8, shared=0, context=16000, ragged=True, nodes=63, reach=24)
LARGEST_LOGITS = 2048 * 128000


def spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "log_probs", "log_probs", "accept"])
    if kind == "accept":
        return dict(kind=kind, rows=spread(rng, 1, 256), nodes=spread(rng, 1, 64), reach=rng.randint(1, 24), threshold=rng.choice([0.0, 0.09, 0.3]))
    if kind == "log_probs":
        vocab = spread(rng, 1000, 128000)
        return dict(kind=kind, dtype=rng.choice(list(DTYPES)), rows=spread(rng, 1, min(8192, LARGEST_LOGITS // (2 * vocab))), vocab=vocab, given=rng.randint(1, 3), top=rng.randint(1, 20))
    while True:
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        kv_heads = rng.choice([4, 8, 8, 12, 32])
        group = rng.choice([1, 1, 2, 4, 8])
        if dtype == "bfloat16" and group == 1:
            group = 4
        case = dict(kind=kind, dtype=dtype, heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), rows=spread(rng, 1, 64),
                    shared=rng.choice([0, 0, CHUNK * spread(rng, 1, 32)]), context=spread(rng, 1, 16000), ragged=rng.random() < 0.7,
                    nodes=spread(rng, 1, 64), reach=rng.randint(1, 24))
        w, most = work(case), work(LARGEST)
        limit = 16 if dtype == "float32" else 1  # fp32 products run at another rate
        if case["heads"] <= 64 and w["bytes"] <= most["bytes"] and limit * w["flops"] <= most["flops"]:
            return case


# ---- what a case is made of ----------------------------------------------------------------------------------------------------
def item(case):
    return 4 if case["dtype"] == "float32" else 2


def lengths(case):
    """Tokens that each sequence has of its own."""
    n, longest = case["rows"], case["context"]
    return [max(1, longest - (i * 7919) % (longest // 2 + 1)) if case["ragged"] else longest for i in range(n)]


def trees(case):
    """Per sequence the parent of each drafted token, -1 for the first."""
    rng, out = random.Random(case["nodes"] * 1000 + case["rows"]), []
    for i in range(case["rows"]):
        n = case["nodes"] if case["rows"] == 1 or case["reach"] == 1 else max(1, case["nodes"] - (i * 5) % (case["nodes"] // 2 + 1))
        out.append([-1] + [rng.randrange(max(0, j - case["reach"]), j) for j in range(1, n)])
    return out


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def work(case):
    if case["kind"] == "accept":
        n = sum(len(t) for t in trees(case))
        return {"bytes": 4 * n * (5 if case["threshold"] else 3) + 12 * case["rows"], "flops": 4 * n}
    if case["kind"] == "log_probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * item(case) + case["rows"] * (4 + 8 * case["given"] + 8 * case["top"]), "flops": 6 * n}
    own_tokens, t = lengths(case), trees(case)
    nodes, H, G, d = sum(len(x) for x in t), case["heads"], case["kv_heads"], case["dim"]
    cached = case["shared"] + sum(own_tokens)
    pairs = sum(len(x) * (case["shared"] + c) + sum(v + 1 for v in depths(x)) for x, c in zip(t, own_tokens))
    return {"bytes": item(case) * d * (2 * G * (cached + nodes) + 2 * H * nodes), "flops": 4 * d * H * pairs}


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device=DEVICE).mul_(scale).to(dtype)


def table(lists, width):
    """[len(lists), width] of whole numbers, -1 where a list has ended."""
    return torch.tensor([x + [-1] * (width - len(x)) for x in lists], device=DEVICE)


def ancestors(t):
    """[rows, nodes, nodes]: whether node j is node i or one above it."""
    width = max(len(x) for x in t)
    seen = torch.zeros(len(t), width, width, dtype=torch.bool)
    for r, parents in enumerate(t):
        for i, p in enumerate(parents):
            if p >= 0:
                seen[r, i] = seen[r, p]
            seen[r, i, i] = True
    return seen.to(DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "log_probs":
        return prepare_log_probs(case, g)
    t = trees(case)
    offsets = [0]
    for x in t:
        offsets.append(offsets[-1] + len(x))
    if case["kind"] == "accept":
        return prepare_accept(case, g, t, offsets)
    H, G, d, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    shared, tokens = case["shared"], lengths(case)
    starts = [shared]
    for n in tokens:
        starts.append(starts[-1] + n)
    k, v = normal(g, starts[-1], G, d, dtype=dtype), normal(g, starts[-1], G, d, dtype=dtype)
    # scores of a standard deviation of 2, as trained heads have them: some tokens matter, most do not
    q = normal(g, offsets[-1], H, d, dtype=dtype, scale=2.0)
    # keys and values of the drafted tokens as they leave a stacked projection
    kv = normal(g, offsets[-1], 2 * G, d, dtype=dtype)
    state = dict(case=case, q=q, k=kv[:, :G], v=kv[:, G:])
    if own:
        chunk_attn = framework()
        megabytes = 64 + (starts[-1] + case["rows"] * CHUNK * 2) * 2 * G * d * item(case) // 2 ** 20
        if dtype == torch.bfloat16 or H != G:
            cache = chunk_attn.Attention.shaped(n_heads=H, n_kv_heads=G, d_key=d, d_value=d, scale=d ** -0.5, chunk_size=CHUNK, memory_mb=megabytes,
                                                dtype=dtype, device=torch.device(DEVICE))
        else:
            cache = chunk_attn.Attention(n_heads=H, d_head=d, chunk_size=CHUNK, memory_mb=megabytes, dtype=dtype, device=torch.device(DEVICE))
        order = []  # the cache says which row a sequence gets
        for i, n in enumerate(tokens):
            ids = list(range(1, shared + 1)) + [10 ** 6 * (i + 1) + j for j in range(n)]
            row = cache.add_seq(ids, torch.cat([k[:shared], k[starts[i]:starts[i + 1]]]), torch.cat([v[:shared], v[starts[i]:starts[i + 1]]]))
            order.insert(row, i)
        if order != list(range(len(order))):
            raise RuntimeError("sequences of a common prompt are expected in the order they came in")
        return dict(state, cache=cache, draft=chunk_attn.DraftBatch(t, torch.device(DEVICE)))
    pool_rows = [list(range(shared)) + list(range(starts[i], starts[i + 1])) for i in range(case["rows"])]
    nodes = [list(range(offsets[i], offsets[i + 1])) for i in range(case["rows"])]
    return dict(state, cached_k=k, cached_v=v, context=table(pool_rows, max(len(x) for x in pool_rows)), nodes=table(nodes, max(len(x) for x in nodes)), seen=ancestors(t))


def prepare_log_probs(case, g):
    n, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    # logits of a spread of 2.5, and a few tokens in every row that stand out
    logits = normal(g, n, vocab, scale=2.5)
    best = torch.randint(0, vocab, (n, 8), generator=g, device=DEVICE)
    logits.scatter_add_(1, best, normal(g, n, 8, scale=4.0).abs_())
    logits = logits.to(dtype)
    # the tokens that are asked for: one of those, and any others
    tokens = torch.cat([best[:, :1], torch.randint(0, vocab, (n, case["given"] - 1), generator=g, device=DEVICE)], dim=1).reshape(-1).to(torch.int32)
    rows = torch.arange(n, device=DEVICE).repeat_interleave(case["given"]).to(torch.int32)
    state = dict(case=case, logits=logits, tokens=tokens, rows=rows)
    return dict(state, ops=framework().ops) if own else state


def prepare_accept(case, g, t, offsets):
    n = offsets[-1]
    # few token ids, so that a good part of the drafted tokens are the model's choice
    tokens = torch.randint(0, 3, (n,), generator=g, device=DEVICE).to(torch.int32)
    choice = torch.randint(0, 3, (n,), generator=g, device=DEVICE).to(torch.int32)
    log_probs = normal(g, n, scale=2.0).abs_().neg_()
    entropy = normal(g, n, scale=1.5).abs_()
    state = dict(case=case, tokens=tokens, choice=choice, log_probs=log_probs, entropy=entropy)
    if own:
        chunk_attn = framework()
        return dict(state, ops=chunk_attn.ops, draft=chunk_attn.DraftBatch(t, torch.device(DEVICE)))
    width = max(len(x) for x in t)
    return dict(state, nodes=table([list(range(offsets[i], offsets[i + 1])) for i in range(len(t))], width),
                parents=table(t, width), depth=table([depths(x) for x in t], width), seen=ancestors(t))


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"attention": run_attention, "log_probs": run_log_probs, "accept": run_accept}[state["case"]["kind"]](state)


def run_attention(state):
    if own:
        return state["cache"].forward_draft(state["q"], state["k"], state["v"], state["draft"])
    case, context, nodes = state["case"], state["context"], state["nodes"]
    R, N, H, G, d = case["rows"], nodes.shape[1], case["heads"], case["kv_heads"], case["dim"]

    def keys_of(cached, drafted):  # [R, G, context | nodes, d]
        return torch.cat([cached[context.clamp(min=0)], drafted[nodes.clamp(min=0)]], dim=1).float().transpose(1, 2)

    k, v = keys_of(state["cached_k"], state["k"]), keys_of(state["cached_v"], state["v"])
    q = state["q"][nodes.clamp(min=0)].float().view(R, N, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(R, G, H // G * N, d)
    seen = torch.cat([(context >= 0)[:, None, :].expand(R, N, -1), state["seen"]], dim=2)  # [R, N, keys]
    s = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(R, G, H // G, N, -1)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    # a padding node sees the context only; its row is dropped below
    e = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(R, G, H // G * N, -1), v).view(R, G, H // G, N, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(R, N, H, d)
    return out[nodes >= 0].to(state["q"].dtype)


def sortable(x):
    """fp32 values as whole numbers of the same order; what is not a number counts as the lowest value."""
    bits = torch.where(torch.isnan(x), -math.inf, x + 0.0).view(torch.int32).long()
    return torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)


def run_log_probs(state):
    case = state["case"]
    if own:
        return state["ops"].token_log_probs(state["logits"], state["tokens"], state["rows"], case["top"])
    x = state["logits"].float()
    high = x.amax(-1, keepdim=True)
    e = (x - high).exp()
    total = e.sum(-1, dtype=torch.float64)
    log_total = total.log() + high[:, 0].double()
    weighted = torch.where(e > 0, e * x, 0.0).sum(-1, dtype=torch.float64)
    entropy = (log_total - weighted / total).float()
    rows = state["rows"].long()
    log_probs = (x[rows, state["tokens"].long()].double() - log_total[rows]).float()
    # the best by value, of equal ones those with the lowest ids
    order = sortable(x) * 2 ** 31 + torch.arange(case["vocab"] - 1, -1, -1, device=x.device)
    ids = torch.topk(order, case["top"], dim=-1).indices
    return log_probs, entropy, (torch.gather(x, 1, ids).double() - log_total[:, None]).float(), ids.to(torch.int32)


def run_accept(state):
    case, threshold = state["case"], state["case"]["threshold"]
    if own:
        if threshold:
            return state["ops"].accept_draft(state["draft"], state["tokens"], state["choice"], state["log_probs"], state["entropy"], threshold, threshold ** 0.5)
        return state["ops"].accept_draft(state["draft"], state["tokens"], state["choice"])
    nodes, parents, seen = state["nodes"].clamp(min=0), state["parents"].clamp(min=0), state["seen"]
    tokens, choice = state["tokens"][nodes], state["choice"][nodes]
    good = tokens == torch.gather(choice, 1, parents)
    if threshold:
        least = torch.clamp(math.log(threshold ** 0.5) - torch.gather(state["entropy"][nodes], 1, parents), max=math.log(threshold))
        good = good | (state["log_probs"][nodes] >= least)
    good = (good | (state["parents"] < 0)) & (state["nodes"] >= 0)
    whole = ~(seen & ~good[:, None, :]).any(-1) & (state["nodes"] >= 0)
    # the deepest, of equal ones the first
    number = torch.arange(nodes.shape[1], device=nodes.device)
    last = torch.where(whole, state["depth"] * 1024 + 1023 - number, -1).argmax(-1)
    taken = seen[torch.arange(len(last), device=nodes.device), last]
    count = taken.sum(-1)
    path = torch.where(taken, number, 10 ** 6).sort(-1).values[:, :int(case_depth(case))]
    return torch.where(path < 10 ** 6, path, -1).to(torch.int32), count.to(torch.int32), torch.gather(choice, 1, last[:, None])[:, 0]


def case_depth(case):
    """Tokens of the longest path of a case's trees."""
    return 1 + max(max(depths(x)) for x in trees(case))


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "log_probs":
        return exact_log_probs(case, prepare_log_probs(case, g))
    t = trees(case)
    offsets = [0]
    for x in t:
        offsets.append(offsets[-1] + len(x))
    if case["kind"] == "accept":
        return exact_accept(case, prepare_accept(case, g, t, offsets), t)
    H, G, d, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    tokens = lengths(case)
    total = case["shared"] + sum(tokens)
    k, v = normal(g, total, G, d, dtype=dtype), normal(g, total, G, d, dtype=dtype)
    q = normal(g, offsets[-1], H, d, dtype=dtype, scale=2.0)
    kv = normal(g, offsets[-1], 2 * G, d, dtype=dtype)
    out, at = torch.empty(offsets[-1], H, d, dtype=torch.float64, device=DEVICE), case["shared"]
    for r, parents in enumerate(t):
        mine = slice(offsets[r], offsets[r + 1])
        own_rows = slice(at, at + tokens[r])
        at += tokens[r]
        line = []  # what each node sees of the tree
        for p in parents:
            line.append((line[p] if p >= 0 else []) + [len(line)])
        hidden = torch.ones(len(parents), len(parents), dtype=torch.bool, device=DEVICE)
        for i, up in enumerate(line):
            hidden[i, up] = False
        for h in range(H):
            kh = torch.cat([k[:case["shared"], h * G // H], k[own_rows, h * G // H], kv[mine, h * G // H]]).double()
            vh = torch.cat([v[:case["shared"], h * G // H], v[own_rows, h * G // H], kv[mine, G + h * G // H]]).double()
            score = q[mine, h].double() @ kh.T / math.sqrt(d)
            score[:, -len(parents):][hidden] = -math.inf
            out[mine, h] = torch.softmax(score, dim=-1) @ vh
    return out


def exact_log_probs(case, state):
    parts = []
    for block in state["logits"].split(256):
        x = block.double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        parts.append((torch.gather(lp, 1, best), best, -(lp.exp() * lp).sum(-1), lp))
    given = case["given"]
    asked = [torch.gather(p[3], 1, state["tokens"].long().view(-1, given)[i * 256:i * 256 + len(p[3])]) for i, p in enumerate(parts)]
    return torch.cat(asked).reshape(-1), torch.cat([p[2] for p in parts]), torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]).to(torch.int32)


def exact_accept(case, state, t):
    tokens, choice = state["tokens"].tolist(), state["choice"].tolist()
    lp, h = state["log_probs"].double().tolist(), state["entropy"].double().tolist()
    width, at, path, count, following = case_depth(case), 0, [], [], []
    for parents in t:
        best = [0]
        lines = {0: [0]}
        for i, p in enumerate(parents):
            if i == 0 or p not in lines:
                continue
            ok = tokens[at + i] == choice[at + p]
            if case["threshold"] and not ok:
                ok = math.exp(lp[at + i]) >= min(case["threshold"], math.sqrt(case["threshold"]) * math.exp(-h[at + p]))
            if ok:
                lines[i] = lines[p] + [i]
                if len(lines[i]) > len(best):
                    best = lines[i]
        path.append(best + [-1] * (width - len(best)))
        count.append(len(best))
        following.append(choice[at + best[-1]])
        at += len(parents)
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in (path, count, following))
