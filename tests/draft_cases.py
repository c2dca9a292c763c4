"""Decoding with drafted tokens: caches and trees for the tests, and the operators in 64 bits from their definitions."""
import math
import random

import torch

DEV = "cuda:0"


def random_tree(rng, n, reach):
    """Parents of n nodes, each drafted under one of the `reach` before it; the first has none."""
    return [-1] + [rng.randrange(max(0, i - reach), i) for i in range(1, n)] if n else []


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def lines(parents):
    """Every node's ancestors and itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def dirty(nbytes):
    """Memory of the allocator that the next tensor of this size gets, full of NaN patterns: what was never written shows up."""
    t = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV)
    del t


class Case:
    """A cache with sequences in it, their keys and values beside it, and drafted trees."""

    def __init__(self, seed, dtype, kv_heads, group, dk, dv=None, shared=0, own=(10,), nodes=(4,), reach=3, chunk=64, sink=False, scale=None, shaped=None,
                 spread=2.0, trees=None, tpp_threshold=1):
        import chunk_attn
        dv = dk if dv is None else dv
        rng = random.Random(seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.G, self.H, self.dk, self.dv, self.sink = dtype, kv_heads, kv_heads * group, dk, dv, sink
        self.scale = dk ** -0.5 if scale is None else scale
        n_rows = len(own)
        self.trees = trees if trees is not None else [random_tree(rng, n, reach) for n in nodes]
        per_token = kv_heads * (-(-dk // 8) * 8 + -(-dv // 8) * 8) * (4 if dtype == torch.float32 else 2)
        mb = 8 + (shared + sum(own) + n_rows * 2 * chunk + chunk) * per_token // 2 ** 20 * 2
        dirty(mb * 2 ** 20)
        if shaped is None:
            shaped = group > 1 or dv != dk or sink or dtype == torch.bfloat16 or scale is not None
        if shaped:
            self.cache = chunk_attn.Attention.shaped(n_heads=self.H, n_kv_heads=kv_heads, d_key=dk, d_value=dv, scale=self.scale, sink=sink, chunk_size=chunk,
                                                     memory_mb=mb, dtype=dtype, device=torch.device(DEV), tpp_threshold=tpp_threshold)
        else:
            self.cache = chunk_attn.Attention(n_heads=self.H, d_head=dk, chunk_size=chunk, memory_mb=mb, dtype=dtype, device=torch.device(DEV), tpp_threshold=tpp_threshold)

        def normal(*shape, scale=1.0):
            return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(dtype)

        prompt = [rng.randrange(1, 1000) for _ in range(shared)]
        pk, pv = normal(shared, kv_heads, dk), normal(shared, kv_heads, dv)
        self.k, self.v, self.tokens = [], [], []
        for n in own:
            k, v = torch.cat([pk, normal(n, kv_heads, dk)]), torch.cat([pv, normal(n, kv_heads, dv)])
            ids = prompt + [rng.randrange(1000, 10 ** 6) for _ in range(n)]
            row = self.cache.add_seq(ids, k, v)
            self.k.insert(row, k)
            self.v.insert(row, v)
            self.tokens.insert(row, ids)
        self.draft = chunk_attn.DraftBatch(self.trees, torch.device(DEV))
        N = self.draft.n_nodes
        self.qd = normal(N, self.H, dk, scale=spread)
        self.kd, self.vd = normal(N, kv_heads, dk), normal(N, kv_heads, dv)

    def run(self):
        out = self.cache.forward_draft(self.qd, self.kd, self.vd, self.draft)
        assert out.shape == (self.draft.n_nodes, self.H, self.dv) and out.dtype == self.dtype
        return out

    def expected(self):
        return tree_attention(self.qd, self.kd, self.vd, self.trees, self.k, self.v, self.scale, self.sink)

    def tolerance(self, want):
        """Half a rounding step of the result, and what fp32 scores and 16-bit parts of the weights may move it.  A score is a sum of d products:
        off by d 2^-23 sum |q k| scale at most; a weight by that in relation, so the result by twice that of the largest value.  Weights
        enter as hi + lo parts: 2^-16 of the largest value in bf16 and less in fp16; exponentials and their sum 2^-20."""
        q = self.qd.abs().double().flatten(0, 1).amax(0)
        k = torch.cat([self.kd] + self.k).abs().double().flatten(0, 1).amax(0)
        # |q . k| <= |q| |k|, lengths of the longest rows
        q, k = self.qd.double().norm(dim=-1).max().item(), torch.cat([self.kd] + self.k).double().norm(dim=-1).max().item()
        vmax = torch.cat([self.vd] + self.v).abs().max().item()
        score = self.dk * 2.0 ** -23 * q * k * abs(self.scale)
        return torch.finfo(self.dtype).eps / 2 * want.abs() + vmax * (2 * score + 2.0 ** -20 + (2.0 ** -16 if self.dtype == torch.bfloat16 else 0.0))

    def check(self, out=None):
        out = self.run() if out is None else out
        want = self.expected()
        err = (out.double() - want).abs()
        tol = self.tolerance(want)
        assert torch.isfinite(out).all()
        worst = (err - tol).max().item()
        assert worst <= 0, "off by %g, %g allowed" % (err.max().item(), tol[err == err.max()].max().item())
        assert self.cache.device_status() == 0
        return out


def tree_attention(qd, kd, vd, trees, k_rows, v_rows, scale, sink):
    """[n_nodes, H, dv] in fp64: one node at a time over its row's cached tokens and its line."""
    H, G = qd.shape[1], kd.shape[1]
    out = torch.empty(qd.shape[0], H, vd.shape[2], dtype=torch.float64, device=qd.device)
    at = 0
    for parents, kc, vc in zip(trees, k_rows, v_rows):
        kc, vc = kc.double().repeat_interleave(H // G, 1), vc.double().repeat_interleave(H // G, 1)
        for i, line in enumerate(lines(parents)):
            rows = [at + j for j in line]
            k = torch.cat([kc, kd[rows].double().repeat_interleave(H // G, 1)])
            v = torch.cat([vc, vd[rows].double().repeat_interleave(H // G, 1)])
            s = torch.einsum("hd,thd->ht", qd[at + i].double(), k) * scale
            if sink:
                s = torch.cat([s, torch.zeros(H, 1, dtype=torch.float64, device=s.device)], 1)
            p = torch.softmax(s, -1)
            if sink:
                p = p[:, :-1]
            out[at + i] = torch.einsum("ht,thd->hd", p, v)
        at += len(parents)
    return out


def accept(trees, tokens, choice, log_probs=None, entropy=None, epsilon=None, delta=None):
    """(paths, next tokens) by walking down every tree."""
    at, paths, following = 0, [], []
    for parents in trees:
        n = len(parents)
        if n == 0:
            paths.append([])
            following.append(-1)
            continue
        kept = {0: [0]}
        for i in range(1, n):
            p = parents[i]
            if p not in kept:
                continue
            ok = tokens[at + i] == choice[at + p]
            if log_probs is not None and not ok:
                ok = log_probs[at + i] >= min(math.log(epsilon), math.log(delta) - entropy[at + p])
            if ok:
                kept[i] = kept[p] + [i]
        best = max(kept.values(), key=lambda line: (len(line), -line[-1]))
        paths.append(best)
        following.append(choice[at + best[-1]])
        at += n
    return paths, following


def log_probs(logits, tokens, rows, top):
    """fp64: log probabilities, entropy, the best tokens' log probabilities and ids."""
    x = logits.double()
    # a row with a NaN or +infinity in it has no distribution
    x = torch.where((torch.isnan(x) | torch.isposinf(x)).any(-1, keepdim=True), math.nan, x)
    # relative to the largest: next to 3e38 even 64 bits do not hold the log of the number of tokens
    x = x - x.amax(-1, keepdim=True)
    lp = x - x.exp().sum(-1, keepdim=True).log()
    ent = -torch.where(lp > -math.inf, lp.exp() * lp, torch.where(torch.isnan(lp), math.nan, 0.0)).sum(-1)
    order = torch.where(torch.isnan(logits), -math.inf, logits.double())
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp[rows.long(), tokens.long()], ent, torch.gather(lp, 1, ids), ids
