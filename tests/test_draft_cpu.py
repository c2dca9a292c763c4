"""Drafted tokens without a GPU: the batch's tables, its refusals, and the work list, walked in numpy as the kernels walk it."""
import ctypes as C
import math
import random

import numpy as np
import pytest
import torch

import draft_cases as D
from chunk_attn import DraftBatch, PrefixTree, cabi


def test_tables():
    rng = random.Random(0)
    trees = [D.random_tree(rng, n, 6) for n in (5, 0, 1, 64, 65, 256)]
    b = DraftBatch(trees, "cpu")
    assert b.n_rows == 6 and b.n_nodes == 391
    assert list(b.first) == np.cumsum([0] + [len(t) for t in trees]).tolist()
    assert b.depths.tolist() == sum((D.depths(t) for t in trees), [])
    assert b.parents.tolist() == sum(trees, [])
    assert b.row_of.tolist() == [r for r, t in enumerate(trees) for _ in t]
    assert b.max_depth == max(b.depths.tolist())
    assert DraftBatch([], "cpu").n_nodes == 0 and DraftBatch([[]], "cpu").max_depth == -1


@pytest.mark.parametrize("trees", [[[0]], [[-1, 1]], [[-1, 5]], [[-2]], [[-1] * 257]])
def test_batches_refuse(trees):
    with pytest.raises(RuntimeError, match="DraftBatch"):
        DraftBatch(trees, "cpu")


def infos_of(chunk, shared, own, share=True):
    tree = PrefixTree(chunk, 100000, share)
    rows = []
    for i, n in enumerate(own):
        ids = list(range(1, shared + 1)) + [10 ** 5 * (i + 1) + j for j in range(n)]
        rows.insert(tree.add_seq(ids), ids)
    return tree.get_chunks(), rows


def walk(plan, infos, trees, q, kd, vd, pool, G, group):
    """Items to partial results to rows, as the kernels do it, in fp64."""
    H, d, first = G * group, q.shape[2], np.cumsum([0] + [len(t) for t in trees])
    out = np.full((len(q), H, d), np.nan)
    part, written = {}, set()
    line = sum((D.lines(t) for t in trees), [])
    row_of = [r for r, t in enumerate(trees) for _ in t]
    for node0, n_nodes, lst, n_tiles, slot, tree, n_drafted, tokens, *head in plan.items.tolist():
        assert head[:2 * n_tiles] == plan.tiles[2 * lst:2 * (lst + min(4, n_tiles))].tolist()
        assert n_nodes >= 1 and n_nodes * group <= max(plan.info.block_rows, group)
        keys, vals, ids = [], [], []
        for j in range(n_tiles):
            chunk, n = plan.tiles[2 * (lst + j):2 * (lst + j) + 2]
            keys.append(pool[chunk][0][:n])
            vals.append(pool[chunk][1][:n])
        ctx_k = np.concatenate(keys) if keys else np.zeros((0, G, d))
        ctx_v = np.concatenate(vals) if vals else np.zeros((0, G, d))
        assert len(ctx_k) == tokens
        for node in range(node0, node0 + n_nodes):
            extra = []
            if n_drafted:
                assert tree == first[row_of[node]] and node - tree < n_drafted <= len(trees[row_of[node]])
                extra = [tree + j for j in line[node]]
            k, v = np.concatenate([ctx_k, kd[extra]]), np.concatenate([ctx_v, vd[extra]])
            for h in range(H):
                s = k[:, h // group] @ q[node, h]
                m = s.max() if len(s) else -1e30
                e = np.exp(s - m)
                if slot < 0:
                    assert (node, h) not in written
                    written.add((node, h))
                    out[node, h] = e @ v[:, h // group] / e.sum()
                else:
                    assert (slot + node - node0, h) not in part
                    part[slot + node - node0, h] = (m, e.sum(), e @ v[:, h // group])
    for i, node in enumerate(plan.merge_nodes):
        slots = plan.merge_slots[plan.merge_off[i]:plan.merge_off[i + 1]]
        for h in range(H):
            ps = [part.pop((s, h)) for s in slots.tolist()]
            M = max(p[0] for p in ps)
            assert (node, h) not in written
            written.add((node, h))
            out[node, h] = sum(math.exp(p[0] - M) * p[2] for p in ps) / sum(math.exp(p[0] - M) * p[1] for p in ps)
    assert not part and len(written) == len(q) * H
    return out


@pytest.mark.parametrize("shared,own,nodes", [(0, (1,), (1,)), (0, (300,), (5,)), (64, (10, 64, 0), (4, 0, 20)), (192, (5,) * 9, (3,) * 9), (128, (1000, 2), (70, 1)), (16, (15, 17, 33), (0, 0, 3))])
@pytest.mark.parametrize("G,group,block_rows,ctas,threshold", [(1, 1, 128, 296, 1), (2, 4, 64, 8, 1), (3, 2, 16, 592, 2), (1, 3, 2, 40, 1)])
def test_work_lists_cover_every_node_once(shared, own, nodes, G, group, block_rows, ctas, threshold):
    chunk, d = 16, 4
    rng = random.Random(1)
    infos, rows = infos_of(chunk, shared, own)
    trees = [D.random_tree(rng, n, 4) for n in nodes]
    g = np.random.default_rng(0)
    pool = {c[0]: (g.normal(size=(chunk, G, d)), g.normal(size=(chunk, G, d))) for c in infos}
    N = sum(nodes)
    q, kd, vd = g.normal(size=(N, G * group, d)), g.normal(size=(N, G, d)), g.normal(size=(N, G, d))
    first = np.cumsum([0] + list(nodes)).tolist()
    plan = cabi.DraftPlan(infos, first, chunk, threshold, 100000, G, group, block_rows, ctas)
    out = walk(plan, infos, trees, q, kd, vd, pool, G, group)
    # every row's chunks, root first (the list is depth first)
    k_rows, v_rows = [], []
    for r in range(len(own)):
        mine = [c for c in infos if c[2] <= r < c[3] and c[1]]
        k_rows.append(np.concatenate([pool[c[0]][0][:c[1]] for c in mine]) if mine else np.zeros((0, G, d)))
        v_rows.append(np.concatenate([pool[c[0]][1][:c[1]] for c in mine]) if mine else np.zeros((0, G, d)))
        assert len(k_rows[r]) == len(rows[r])
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x))  # noqa: E731
    want = D.tree_attention(t(q), t(kd), t(vd), trees, [t(x) for x in k_rows], [t(x) for x in v_rows], 1.0, False).numpy()
    np.testing.assert_allclose(out, want, rtol=1e-9, atol=1e-12)


def test_long_contexts_are_cut_and_short_ones_are_not():
    infos, _ = infos_of(64, 0, (8000,))
    p = cabi.DraftPlan(infos, [0, 5], kv_heads=8, group=4)
    assert 8 * len(p.items) >= 148 and p.info.n_merge == 5
    infos, _ = infos_of(64, 0, (900,) * 64)
    p = cabi.DraftPlan(infos, [5 * i for i in range(65)], kv_heads=8, group=4)
    assert len(p.items) == 64 and p.info.n_merge == 0


def test_work_lists_refuse():
    ok = [(0, 10, 0, 1)]
    for infos, first in (([(-1, 10, 0, 1)], [0, 2]), ([(5, 10, 0, 1)], [0, 2]), ([(0, 65, 0, 1)], [0, 2]), ([(0, 10, 0, 2)], [0, 2]), ([(0, 10, 1, 1)], [0, 2]), (ok, [0, -1]), (ok, [1, 2])):
        with pytest.raises(cabi.CAError, match="draft plan"):
            cabi.DraftPlan(infos, first, max_chunks=5)
    with pytest.raises(cabi.CAError):
        cabi.DraftPlan(ok, [0, 2], kv_heads=0)
    assert cabi.DraftPlan([], [0]).info.n_items == 0
    assert cabi.DraftPlan([], [0, 0]).info.n_items == 0


class AcceptArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("first", "parent", "depth", "seen")] + [(n, C.c_int32) for n in ("words", "n_rows", "width")] + \
        [(n, C.c_void_p) for n in ("tokens", "choice", "log_probs", "entropy")] + [("epsilon", C.c_double), ("delta", C.c_double)] + \
        [(n, C.c_void_p) for n in ("path", "count", "next")]


class LogProbsArgs(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("row_stride", C.c_int64)] + [(n, C.c_int32) for n in ("n_rows", "vocab", "dtype")] + \
        [("tokens", C.c_void_p), ("rows", C.c_void_p), ("n_tokens", C.c_int32), ("top", C.c_int32)] + \
        [(n, C.c_void_p) for n in ("log_probs", "entropy", "top_log_probs", "top_ids", "scratch")]


def refused(fn, args, what):
    assert fn(C.byref(args), None) != cabi.CA_OK and what in cabi.lib.ca_last_error().decode()


def test_acceptance_refuses_at_the_c_entry():
    """Every call is refused before anything is launched: the addresses are never followed."""
    ok = {n: 4096 for n, t in AcceptArgs._fields_ if t is C.c_void_p}
    ok.update(words=2, n_rows=1, width=1, epsilon=0.1, delta=0.3)
    for name in ("first", "parent", "depth", "seen", "tokens", "choice", "path", "count", "next"):
        refused(cabi.lib.ca_accept_draft, AcceptArgs(**dict(ok, **{name: 0})), "null")
        refused(cabi.lib.ca_accept_draft, AcceptArgs(**dict(ok, **{name: 4098})), "aligned")
    for change, what in (({"n_rows": -1}, "negative"), ({"width": -1}, "negative"), ({"words": 0}, "words"), ({"words": 9}, "words"), ({"entropy": 0}, "together"),
                         ({"log_probs": 0}, "together"), ({"epsilon": 0.0}, "positive"), ({"delta": float("nan")}, "positive"), ({"entropy": 4097}, "aligned")):
        refused(cabi.lib.ca_accept_draft, AcceptArgs(**dict(ok, **change)), what)
    assert cabi.lib.ca_accept_draft(C.byref(AcceptArgs(**dict(ok, n_rows=0))), None) == cabi.CA_OK
    assert cabi.lib.ca_accept_draft(None, None) != cabi.CA_OK


def test_log_probs_refuse_at_the_c_entry():
    ok = {n: 4096 for n, t in LogProbsArgs._fields_ if t is C.c_void_p}
    ok.update(row_stride=100, n_rows=2, vocab=100, dtype=cabi.CA_DTYPE_F32, n_tokens=2, top=3)
    for name in ("logits", "entropy", "scratch", "tokens", "log_probs", "top_ids", "top_log_probs"):
        refused(cabi.lib.ca_token_log_probs, LogProbsArgs(**dict(ok, **{name: 0})), "null")
        refused(cabi.lib.ca_token_log_probs, LogProbsArgs(**dict(ok, **{name: 4098})), "aligned")
    for change, what in (({"n_rows": -1}, "sizes"), ({"n_tokens": -1}, "sizes"), ({"vocab": 0}, "sizes"), ({"vocab": (1 << 28) + 1}, "2^28"), ({"dtype": 9}, "fp16"),
                         ({"top": -1}, "top"), ({"top": 33}, "top"), ({"top": 101}, "top"), ({"vocab": 2}, "top"), ({"row_stride": -1}, "stride"), ({"rows": 4097}, "aligned"),
                         ({"scratch": 4104}, "scratch")):
        refused(cabi.lib.ca_token_log_probs, LogProbsArgs(**dict(ok, **change)), what)
    assert cabi.lib.ca_token_log_probs(None, None) != cabi.CA_OK
    for bad in ((-1, 10, cabi.CA_DTYPE_F32, 1), (1, 0, cabi.CA_DTYPE_F32, 1), (1, 10, 9, 1), (1, 10, cabi.CA_DTYPE_F32, 33)):
        assert cabi.lib.ca_log_probs_scratch(*bad) < 0


def test_log_probs_without_rows_take_a_token_for_every_row():
    """The kernels give every row its token, so another number of them would be read and written behind the arrays' ends, or left unwritten."""
    ok = {n: 4096 for n, t in LogProbsArgs._fields_ if t is C.c_void_p}
    ok.update(row_stride=100, n_rows=4, vocab=100, dtype=cabi.CA_DTYPE_F32, n_tokens=4, top=3, rows=0)
    for change in ({"n_tokens": 3}, {"n_tokens": 5}, {"n_rows": 0}, {"n_tokens": 1, "top": 0}):
        refused(cabi.lib.ca_token_log_probs, LogProbsArgs(**dict(ok, **change)), "one token per row")


def test_log_probs_scratch_goes_by_what_is_asked():
    """A row's part without the best tokens is a few numbers; notes of the best are no more than the row has vectors."""
    size = cabi.lib.ca_log_probs_scratch
    assert size(1 << 20, 100, cabi.CA_DTYPE_F16, 0) < 64 * (1 << 20)
    assert size(1 << 20, 100, cabi.CA_DTYPE_F16, 5) < 128 * (1 << 20)  # 200 bytes of logits a row
    assert size(131072, 32000, cabi.CA_DTYPE_F16, 0) < 64 * 131072 < size(131072, 32000, cabi.CA_DTYPE_F16, 1) < 4096 * 131072
    assert size(1 << 20, 3, cabi.CA_DTYPE_BF16, 3) > 0
