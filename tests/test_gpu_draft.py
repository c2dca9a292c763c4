"""Attention of drafted trees over the cache, the acceptance of drafted tokens and log probabilities, against plain 64-bit forms."""
import ctypes as C
import math
import random

import pytest
import torch

import draft_cases as D

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# ---- attention ---------------------------------------------------------------------------------------------------------------
GEOMETRIES = [  # dtype, kv heads, group, d_key, d_value, chunk, sink
    (F16, 4, 1, 128, 128, 64, False), (F16, 2, 1, 64, 64, 64, False), (F32, 3, 1, 128, 128, 64, False), (F32, 2, 1, 30, 30, 5, False), (F16, 2, 1, 20, 20, 16, False),
    (BF16, 2, 4, 128, 128, 64, False), (BF16, 2, 8, 64, 64, 64, True), (BF16, 1, 3, 128, 64, 64, True), (F16, 2, 2, 64, 128, 64, False), (F32, 2, 4, 96, 40, 32, True),
    (BF16, 1, 5, 80, 80, 64, False), (F32, 1, 2, 256, 256, 64, False), (BF16, 2, 1, 256, 200, 32, True), (F16, 1, 64, 64, 64, 64, False), (BF16, 1, 33, 128, 128, 64, False),
]
BATCHES = [  # shared, own tokens, nodes
    (0, (1,), (1,)), (0, (63, 64, 65), (4, 1, 7)), (128, (5, 200, 64), (3, 0, 20)), (64, (1, 1, 1, 1), (9, 2, 1, 5)), (0, (700,), (64,)), (192, (0, 90), (33, 65)),
]


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_tree_attention(geometry, batch):
    dtype, G, group, dk, dv, chunk, sink = geometry
    shared, own, nodes = batch
    shared = shared // 64 * chunk  # whole chunks, so that they are shared
    D.Case(1, dtype, G, group, dk, dv, shared=shared, own=own, nodes=nodes, reach=5, chunk=chunk, sink=sink).check()


@pytest.mark.parametrize("dtype,group,d", [(F16, 1, 128), (BF16, 8, 128), (BF16, 4, 64), (F32, 1, 64)])
def test_large_trees_and_many_rows(dtype, group, d):
    """More query rows than an item takes, runs that many rows share, pieces of long contexts."""
    D.Case(2, dtype, 2, group, d, shared=320, own=(1500, 3, 64, 0, 130, 700), nodes=(256, 64, 1, 100, 63, 17), reach=40).check()
    D.Case(3, dtype, 1, group, d, own=(9000,), nodes=(5,), reach=1).check()
    D.Case(4, dtype, 4, group, d, shared=128, own=(20,) * 70, nodes=(6,) * 70, reach=3).check()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_trees_of_every_form(dtype):
    """A chain, a star, two trees side by side (nodes without a parent), a lone node."""
    for trees in ([[i - 1 for i in range(40)]], [[-1] + [0] * 39], [[-1, -1, 0, 1, 2, 3, -1]], [[-1]]):
        D.Case(5, dtype, 2, 2, 64, own=(77,), trees=trees).check()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(dtype, scale):
    """Scores turned round, all alike, and so sharp that one key takes all."""
    D.Case(6, dtype, 2, 2, 64, own=(150, 10), nodes=(10, 3), scale=scale, spread=1.0).check()


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64), (F32, 128), (F32, 30)])
def test_values_of_hidden_nodes_do_not_matter(dtype, d):
    """Infinities and NaN in the keys and values of nodes show in the nodes below them only."""
    c = D.Case(7, dtype, 2, 2 if dtype == BF16 else 1, d, own=(70, 65), trees=[[-1, 0, 0, 1, 2, 3], [-1, 0, 1]])
    clean = c.run()
    want = c.expected()
    tol = c.tolerance(want)

    def as_clean(out, rows):
        # rows beside something infinite may be computed in another order: both ways are within the tolerance of the exact result
        assert ((out.double() - want).abs() <= tol)[rows].all()

    for poison in (math.nan, math.inf):
        for t in (c.vd, c.kd):
            keep = t[2].clone()
            t[2] = poison  # node 2 of the first tree; node 4 is below it
            out = c.run()
            as_clean(out, [0, 1, 3, 5, 6, 7, 8])
            assert torch.equal(out[6:], clean[6:])  # another tree
            assert not torch.isfinite(out[2]).any() and not torch.isfinite(out[4]).any()
            t[2] = keep
    c.vd[2, 0, 3] = math.inf  # a single element
    out = c.run()
    group = c.H // c.G
    assert torch.isinf(out[2, :group, 3]).all() and torch.isinf(out[4, :group, 3]).all()
    out[[2, 4], :group, 3] = clean[[2, 4], :group, 3]
    as_clean(out, list(range(9)))
    assert torch.equal(out[:, group:], clean[:, group:])  # other heads


@pytest.mark.parametrize("dtype,group,d", [(F16, 1, 128), (BF16, 4, 128), (F32, 1, 64)])
def test_strided_operands(dtype, group, d):
    """Heads of a stacked projection, heads outermost, and addresses that are no multiple of 16 bytes."""
    c = D.Case(8, dtype, 2, group, d, own=(100, 30), nodes=(12, 5))
    want = c.run()
    n, G, H = c.draft.n_nodes, c.G, c.H
    stacked = torch.cat([c.qd, c.kd, c.vd], 1)
    assert torch.equal(c.cache.forward_draft(stacked[:, :H], stacked[:, H:H + G], stacked[:, H + G:], c.draft), want)
    outer = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (c.qd, c.kd, c.vd)]
    assert torch.equal(c.cache.forward_draft(*outer, c.draft), want)
    odd = []
    for t in (c.qd, c.kd, c.vd):
        buf = torch.full((n * t.shape[1] * (d + 3) + 1,), math.nan, dtype=dtype, device=DEV)
        view = buf[1:].view(n, t.shape[1], d + 3)[:, :, :d]
        view.copy_(t)
        odd.append(view)
    assert torch.equal(c.cache.forward_draft(*odd, c.draft), want)
    one = c.kd[:1].expand(n, G, d)  # the same keys for all nodes
    assert torch.equal(c.cache.forward_draft(c.qd, one, c.vd, c.draft), c.cache.forward_draft(c.qd, one.contiguous(), c.vd, c.draft))


@pytest.mark.parametrize("dtype,group,dk,dv", [(F16, 1, 128, 128), (BF16, 4, 64, 128), (BF16, 8, 128, 64)])
def test_both_kernels(dtype, group, dk, dv):
    """The any-geometry kernel serves what the tensor-core kernel does."""
    from chunk_attn import cabi
    c = D.Case(16, dtype, 2, group, dk, dv, shared=128, own=(300, 64, 5), nodes=(30, 4, 9))
    a = c.check()
    c.cache.set_option(cabi.CA_OPT_DRAFT_TENSOR, 0)
    b = c.check()
    assert not torch.equal(a, b)  # sums in another order: it is another kernel
    c.cache.set_option(cabi.CA_OPT_DRAFT_TENSOR, 1)
    assert torch.equal(a, c.run())


def test_empty_drafts():
    c = D.Case(9, F16, 2, 1, 64, own=(10, 20), nodes=(0, 0))
    assert c.run().shape == (0, 2, 64)
    import chunk_attn
    empty = chunk_attn.Attention(n_heads=2, d_head=64, chunk_size=64, memory_mb=4, dtype=F16, device=torch.device(DEV))
    d = chunk_attn.DraftBatch([], torch.device(DEV))
    t = torch.empty(0, 2, 64, dtype=F16, device=DEV)
    assert empty.forward_draft(t, t, t, d).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype,group", [(F16, 1), (BF16, 4), (F32, 1)])
def test_the_cache_moves_on(dtype, group):
    """The same draft over a cache that appends, accepts (extend_kv), forks and loses rows."""
    c = D.Case(10, dtype, 2, group, 64, shared=64, own=(63, 3, 120), nodes=(4, 6, 3))
    c.check()

    def rows(n):
        return [torch.randn(n, c.G, 64, device=DEV).to(dtype) for _ in range(2)]

    k, v = rows(3)
    c.cache.append_token([1, 2, 3], k, v)
    for i in range(3):
        c.k[i], c.v[i] = torch.cat([c.k[i], k[i:i + 1]]), torch.cat([c.v[i], v[i:i + 1]])
    c.check()
    k, v = rows(7)
    c.cache.extend_kv([2, 0, 1], [[5, 6], [7, 8, 9, 10, 11], []], k, v)
    c.k[2], c.v[2] = torch.cat([c.k[2], k[:2]]), torch.cat([c.v[2], v[:2]])
    c.k[0], c.v[0] = torch.cat([c.k[0], k[2:]]), torch.cat([c.v[0], v[2:]])
    c.check()
    c.cache.remove_seq(1)
    del c.k[1], c.v[1]
    import chunk_attn
    c.trees = [c.trees[0], c.trees[2]]
    keep = [i for i in range(c.draft.n_nodes) if not 4 <= i < 10]
    c.qd, c.kd, c.vd = c.qd[keep], c.kd[keep], c.vd[keep]
    with pytest.raises(RuntimeError, match="one tree per live sequence"):
        c.run()
    c.draft = chunk_attn.DraftBatch(c.trees, torch.device(DEV))
    c.check()
    c.cache.duplicate(0, 1)
    c.k.insert(1, c.k[0])
    c.v.insert(1, c.v[0])
    c.trees = [c.trees[0], [-1], c.trees[1]]
    c.draft = chunk_attn.DraftBatch(c.trees, torch.device(DEV))
    c.qd, c.kd, c.vd = (torch.cat([t[:4], t[:1], t[4:]]) for t in (c.qd, c.kd, c.vd))
    c.check()


def test_extend_kv_is_append_token():
    """Tokens accepted together are the cache that tokens appended one by one make."""
    a, b = (D.Case(11, F16, 2, 1, 64, own=(60, 127), nodes=(3, 3)) for _ in range(2))
    k, v = (torch.randn(2, 70, 2, 64, device=DEV).half() for _ in range(2))
    for i in range(70):
        a.cache.append_token([i, 1000 + i], k[:, i].contiguous(), v[:, i].contiguous())
    b.cache.extend_kv([1, 0], [list(range(1000, 1070)), list(range(70))], torch.cat([k[1], k[0]]), torch.cat([v[1], v[0]]))
    assert torch.equal(a.run(), b.run())
    q = torch.randn(2, 2, 64, device=DEV).half()
    assert torch.equal(a.cache.forward(q), b.cache.forward(q))
    assert [t.n_tokens for t in a.cache.tails] == [t.n_tokens for t in b.cache.tails]


def test_threshold_of_sharing():
    """Chunks of no more sharers than the threshold are walked row by row."""
    for threshold in (1, 2, 3, 8):
        D.Case(12, F16, 2, 1, 128, shared=256, own=(30, 40, 50), nodes=(5, 6, 7), tpp_threshold=threshold).check()


@pytest.mark.parametrize("dtype,group,d", [(F16, 1, 128), (BF16, 4, 64), (F32, 1, 64)])
def test_another_stream_and_a_graph(dtype, group, d):
    c = D.Case(13, dtype, 2, group, d, shared=64, own=(900, 30), nodes=(12, 5))
    want = c.run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = c.run()
        import chunk_attn
        fresh = chunk_attn.DraftBatch(c.trees, torch.device(DEV))
        again = c.cache.forward_draft(c.qd, c.kd, c.vd, fresh)
    # made on the side stream, used here
    third = c.cache.forward_draft(c.qd, c.kd, c.vd, fresh)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want) and torch.equal(third, want)
    tokens = torch.randint(0, 2, (c.draft.n_nodes,), dtype=torch.int32, device=DEV)
    logits = torch.randn(c.draft.n_nodes, 500, device=DEV)
    from chunk_attn import ops
    c.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = c.run()
        lp = ops.token_log_probs(logits, tokens, None, 3)
        acc = ops.accept_draft(c.draft, tokens, lp[3][:, 0].contiguous(), lp[0], lp[1])
    c.qd.mul_(0.5)
    logits.mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, c.run())
    now = ops.token_log_probs(logits, tokens, None, 3)
    assert all(torch.equal(x, y) for x, y in zip(lp, now))
    assert all(torch.equal(x, y) for x, y in zip(acc, ops.accept_draft(c.draft, tokens, now[3][:, 0].contiguous(), now[0], now[1])))
    # the work list of the captured step outlives the tree that it was made from
    before = o.clone()
    k = torch.randn(2, 2, d, device=DEV).to(dtype)
    c.cache.append_token([1, 2], k, k)
    c.run()
    for _ in range(20):
        torch.full((4096,), 7, dtype=torch.int32, device=DEV)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, before)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            chunk_attn.DraftBatch(c.trees, torch.device(DEV))
    torch.cuda.synchronize()


def test_layers_share_their_work_lists():
    import chunk_attn
    c = D.Case(14, F16, 2, 1, 64, own=(100, 40), nodes=(6, 9))
    other = chunk_attn.Attention(c.cache)
    for ids, k, v in zip(c.tokens, c.k, c.v):
        other.add_seq(ids, v, k)  # another layer's numbers
    a = c.run()
    b = other.forward_draft(c.qd, c.kd, c.vd, c.draft)
    torch.testing.assert_close(b.double(), D.tree_attention(c.qd, c.kd, c.vd, c.trees, c.v, c.k, c.scale, False), atol=5e-3, rtol=0)
    assert torch.equal(a, c.run())


def test_refusals():
    import chunk_attn
    c = D.Case(15, F16, 2, 1, 64, own=(10, 20), nodes=(2, 3))
    q, k, v, d = c.qd, c.kd, c.vd, c.draft
    for bad in ((q[:4], k, v), (q.float(), k, v), (q, k[:, :1], v), (q, k, v[:, :, :32]), (q.transpose(0, 2).contiguous().transpose(0, 2), k, v), (q.cpu(), k, v)):
        with pytest.raises(RuntimeError, match="forward_draft"):
            c.cache.forward_draft(*bad, d)
    with pytest.raises(RuntimeError, match="one tree per live sequence"):
        c.cache.forward_draft(q, k, v, chunk_attn.DraftBatch([[-1] * 5], torch.device(DEV)))
    with pytest.raises(RuntimeError, match="another device"):
        c.cache.forward_draft(q, k, v, chunk_attn.DraftBatch(c.trees, torch.device("cpu")))
    latent = chunk_attn.Attention.latent(n_heads=2, latent=64, rotated=32, scale=0.1, memory_mb=4, dtype=BF16, device=torch.device(DEV))
    with pytest.raises(RuntimeError, match="latent"):
        latent.forward_draft(q, k, v, chunk_attn.DraftBatch([], torch.device(DEV)))
    wide = chunk_attn.Attention.shaped(n_heads=130, n_kv_heads=1, d_key=64, d_value=64, scale=0.1, memory_mb=4, dtype=BF16, device=torch.device(DEV))
    one = torch.zeros(3, 1, 64, dtype=BF16, device=DEV)
    wide.add_seq([1, 2, 3], one, one)
    with pytest.raises(RuntimeError, match="query heads"):
        wide.forward_draft(torch.zeros(1, 130, 64, dtype=BF16, device=DEV), one[:1], one[:1], chunk_attn.DraftBatch([[-1]], torch.device(DEV)))
    with pytest.raises(RuntimeError, match="named twice"):
        c.cache.extend_kv([0, 0], [[1], [2]], k[:2], v[:2])
    with pytest.raises(RuntimeError, match="k and v must be"):
        c.cache.extend_kv([0], [[1]], k[:2], v[:2])
    with pytest.raises(RuntimeError, match="out of range"):
        c.cache.extend_kv([2], [[1]], k[:1], v[:1])
    with pytest.raises(RuntimeError, match="capacity"):
        c.cache.extend_kv([0], [[1] * 10 ** 6], k[:1].expand(10 ** 6, 2, 64), v[:1].expand(10 ** 6, 2, 64))
    c.check()


@pytest.mark.parametrize("d,group,nodes", [(64, 1, 4), (64, 1, 12), (64, 1, 30), (64, 4, 64), (128, 1, 8), (128, 1, 12), (128, 1, 30), (128, 4, 64), (80, 4, 30)])
def test_fp32_errors_do_not_grow_with_the_context(d, group, nodes):
    """fp32 operands give fp32 results, whichever kernel multiplies them.  In the 2-norm: a product of two operands is off by 2^-22 of itself at most, so a score
    by 2^-22 |q o k| scale = 2^-22 spread; its sums are rounded some 2^-23 of the score a group, 2^-21 spread together; a weight's
    exponential 2^-22, the second product, its sums and the combination of pieces 2^-20 with it.  No term goes by the number of tokens."""
    for own, spread in (((2,), 2.0), ((300, 90), 2.0), ((16000,), 2.0), ((64000,), 1.0), ((4000, 700), 8.0)):
        c = D.Case(17, F32, 2, group, d, own=own, nodes=(nodes,) * len(own), spread=spread)
        want = c.expected()
        err = ((c.run().double() - want).norm() / want.norm()).item()
        assert err <= 2.0 ** -21 * spread + 2.0 ** -20, (own, spread, err)


# ---- the C entry ---------------------------------------------------------------------------------------------------------------
class DraftArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v")] + [(n, C.c_int64) for n in ("q_node", "q_head", "k_node", "k_head", "v_node", "v_head")] + \
        [("out", C.c_void_p), ("seen", C.c_void_p), ("words", C.c_int32), ("work", C.c_void_p), ("info", C.c_void_p), ("partials", C.c_void_p), ("settled", C.c_int32)]


class CDraft:
    """Trees over a context of the C library, every operand in the caller's hands."""

    def __init__(self, dtype, d, own, nodes, heads=2, chunk=64, reach=4):
        from chunk_attn import PrefixTree, cabi
        self.cabi, lib = cabi, cabi.lib
        g = torch.Generator(device=DEV).manual_seed(0)
        rng = random.Random(0)
        n_chunks = sum(n // chunk + 2 for n in own)
        kind = cabi.CA_DTYPE_F32 if dtype == F32 else cabi.CA_DTYPE_F16
        tree = PrefixTree(chunk, n_chunks, True)
        pool = torch.zeros(n_chunks * heads * 2 * chunk * d * (4 if dtype == F32 else 2), dtype=torch.uint8, device=DEV)
        self.ctx = cabi.Context(heads, d, chunk, kind, pool, n_chunks)

        def normal(*shape, scale=1.0):
            return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(dtype)

        self.k, self.v = [], []
        for i, n in enumerate(own):
            k, v = normal(n, heads, d), normal(n, heads, d)
            row = tree.add_seq([10 ** 5 * (i + 1) + j for j in range(n)])
            mine = [c[0] for c in tree.get_chunks() if c[1] and c[2] <= row < c[3]]
            self.ctx.scatter_prefill(k, v, 0, n, mine)
            self.k.insert(row, k)
            self.v.insert(row, v)
        self.trees = [D.random_tree(rng, n, reach) for n in nodes]
        N = sum(nodes)
        self.qd, self.kd, self.vd = normal(N, heads, d, scale=2.0), normal(N, heads, d), normal(N, heads, d)
        infos, n_infos = cabi.make_infos(tree.get_chunks())
        first = [0]
        for n in nodes:
            first.append(first[-1] + n)
        plan, data = C.c_void_p(), C.POINTER(C.c_int32)()
        self.info = cabi.DraftPlanInfo()
        cabi.check(lib.ca_draft_plan_for_context(self.ctx._h, C.byref(plan), infos, n_infos, (C.c_int32 * len(first))(*first), len(nodes)))
        cabi.check(lib.ca_draft_plan_data(plan, C.byref(data), C.byref(self.info)))
        self.work = torch.tensor(data[:self.info.n_data], dtype=torch.int32)
        lib.ca_draft_plan_destroy(plan)
        self.seen = torch.tensor([[sum(1 << j for j in line), 0] for t in self.trees for line in D.lines(t)], dtype=torch.int32)
        lib.ca_draft_partial_floats.restype = C.c_int64
        floats = lib.ca_draft_partial_floats(self.ctx._h, C.byref(self.info))
        self.partials = torch.full((max(4, floats),), math.nan, device=DEV)
        self.scale, self.dk, self.dtype = d ** -0.5, d, dtype

    def run(self, work, seen, settled=0):
        q, k, v = self.qd, self.kd, self.vd
        out = torch.full(q.shape, math.nan, dtype=q.dtype, device=DEV)
        a = DraftArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_node=q.stride(0), q_head=q.stride(1), k_node=k.stride(0), k_head=k.stride(1),
                      v_node=v.stride(0), v_head=v.stride(1), out=out.data_ptr(), seen=seen.data_ptr(), words=2, work=work.data_ptr(), info=C.addressof(self.info),
                      partials=self.partials.data_ptr(), settled=settled)
        self.cabi.check(self.cabi.lib.ca_draft_attention(self.ctx._h, C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return out

    def want(self):
        return D.tree_attention(self.qd, self.kd, self.vd, self.trees, self.k, self.v, self.scale, False)


C_SHAPES = [  # an even number of nodes: the bits must be 8-byte aligned
    (F16, 64, (700, 30), (12, 6)), (F16, 128, (90, 64, 10), (10, 2, 12)), (F16, 80, (700, 30), (12, 6)), (F16, 80, (300,), (4,)), (F32, 64, (700, 30), (12, 6)), (F32, 128, (65, 5), (3, 1)),
]


@pytest.mark.parametrize("dtype,d,own,nodes", C_SHAPES)
def test_lists_that_a_kernel_writes_right_before(dtype, d, own, nodes):
    """The bits of the trees' lines and the work list are written by kernels ahead of the call, one of which lets its successor start early
    (token_log_probs: the best two ids of a row of logits are a node's bits and 0)."""
    from chunk_attn import ops
    c = CDraft(dtype, d, own, nodes)
    want = c.want()
    tol = D.Case.tolerance(c, want)
    logits = torch.zeros(len(c.seen), 1 << 13, device=DEV, dtype=F16)
    logits[torch.arange(len(c.seen)), c.seen[:, 0].long()] = 2.0
    logits[:, 0] = 1.0
    work, seen = c.work.to(DEV), c.seen.to(DEV)
    settled = c.run(work, seen, 1)
    assert ((settled.double() - want).abs() <= tol).all()
    for _ in range(20):
        # bits by a kernel that its successor may overtake
        assert torch.equal(c.run(work, ops.token_log_probs(logits, top=2)[3]), settled)
        # both by ordinary kernels, on memory that held something else
        late_seen, late = torch.zeros_like(seen), torch.zeros_like(work)
        torch.add(seen, 0, out=late_seen)
        torch.add(work, 0, out=late)
        assert torch.equal(c.run(late, late_seen), settled)
    assert c.ctx.status() == 0


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 80), (F32, 64)])
def test_damaged_work_lists_are_reported(dtype, d):
    """No entry of a work list is followed out of range: the status says that one was wrong, and the next call is right again."""
    c = CDraft(dtype, d, (700, 700), (12, 6))
    work, seen = c.work.to(DEV), c.seen.to(DEV)
    want = c.run(work, seen)
    assert c.ctx.status() == 0 and c.info.n_merge == 18
    damage = [(w + at, x) for w, at, xs in ((0, 0, (-1, 18, 10 ** 9)), (0, 1, (0, -5, 10 ** 9)), (0, 2, (-1, 10 ** 9)), (0, 4, (10 ** 9,)), (0, 5, (-1, 10 ** 9)), (0, 6, (10 ** 9,)),
                                            (c.info.at_nodes, 3, (-1, 18, 10 ** 9)), (c.info.at_off, 2, (-1, 10 ** 9, -2 ** 31)), (c.info.at_slots, 1, (-1, c.info.n_slots, 2 ** 31 - 1)))
              for x in xs]
    for at, x in damage:
        hurt = c.work.clone()
        hurt[at] = x
        c.run(hurt.to(DEV), seen)
        code, status = c.ctx.status_raw()
        assert status == c.cabi.STATUS_BAD_WORK_LIST, (at, x)
        c.ctx.status_clear()
        assert torch.equal(c.run(work, seen), want) and c.ctx.status() == 0


# ---- acceptance --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("thresholds", [None, (0.09, 0.3), (0.5, 0.7)])
def test_acceptance(seed, thresholds):
    import chunk_attn
    from chunk_attn import ops
    rng = random.Random(seed)
    trees = [D.random_tree(rng, n, rng.randint(1, 12)) for n in (1, 0, 5, 64, 33, 256, 32, 65, 2)]
    trees.append(list(range(-1, 255)))
    draft = chunk_attn.DraftBatch(trees, DEV)
    n = draft.n_nodes
    tokens, choice = ([rng.randrange(1 + seed) for _ in range(n)] for _ in range(2))
    lp = torch.tensor([-rng.expovariate(0.7) for _ in range(n)])
    ent = torch.tensor([rng.expovariate(0.7) for _ in range(n)])
    t, ch = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (tokens, choice))
    if thresholds:
        path, count, following = ops.accept_draft(draft, t, ch, lp.to(DEV), ent.to(DEV), *thresholds)
        # a value within rounding of its threshold would say nothing; these are not
        want, after = D.accept(trees, tokens, choice, lp.double().tolist(), ent.double().tolist(), *thresholds)
    else:
        path, count, following = ops.accept_draft(draft, t, ch)
        want, after = D.accept(trees, tokens, choice)
    assert path.shape == (len(trees), 256) and draft.max_depth == 255
    for r, line in enumerate(want):
        assert path[r].tolist() == line + [-1] * (256 - len(line))
    assert count.tolist() == [len(x) for x in want] and following.tolist() == after


def test_acceptance_refuses():
    import chunk_attn
    from chunk_attn import ops
    draft = chunk_attn.DraftBatch([[-1, 0]], DEV)
    t = torch.zeros(2, dtype=torch.int32, device=DEV)
    f = torch.zeros(2, device=DEV)
    for args in ((t[:1], t), (t.long(), t), (t, t.cpu()), (t, t, f), (t, t, f, f.half()), (t, t, f, f, 0.0, 0.5), (t, t, f, f, 0.5, math.nan)):
        with pytest.raises(RuntimeError, match="accept_draft"):
            ops.accept_draft(draft, *args)
    with pytest.raises(RuntimeError, match="one node without a parent"):
        ops.accept_draft(chunk_attn.DraftBatch([[-1, -1]], DEV), t, t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.accept_draft(chunk_attn.DraftBatch([[-1, 0]], "cpu"), t.cpu(), t.cpu())
    nan = ops.accept_draft(draft, t, t + 1, f * math.nan, f)  # not a number: not accepted
    assert nan[0].tolist() == [[0, -1]] and nan[1].tolist() == [1] and nan[2].tolist() == [1]


# ---- log probabilities ---------------------------------------------------------------------------------------------------------
def check_log_probs(logits, top, per_row=2, seed=0):
    """fp32 sums of exponentials: a term is off by 2^-21 of itself (the exponential, and its argument's rounding: |x - max| < 128 or it does not
    count, 2^-24 of that), log and max by 2^-23 of their sizes; the entropy weighs logs with such terms."""
    from chunk_attn import ops
    n, vocab = logits.shape
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, vocab, (n * per_row,), generator=g).to(torch.int32).to(DEV)
    rows = torch.randint(0, n, (n * per_row,), generator=g).to(torch.int32).to(DEV)
    got = ops.token_log_probs(logits, tokens, rows, top)
    want = D.log_probs(logits, tokens, rows, top)
    assert torch.equal(got[3].long(), want[3]), "top tokens differ"
    biggest = torch.nan_to_num(logits.double(), nan=0.0, posinf=0.0, neginf=0.0).abs().max().item()
    for name, a, b in (("log_probs", got[0], want[0]), ("entropy", got[1], want[1]), ("top", got[2], want[2])):
        assert a.dtype == torch.float32 and a.shape == b.shape
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        # the largest difference of two fp32 logits is twice what fp32 holds
        assert torch.equal(torch.isneginf(a), torch.isneginf(b.float())), name
        fine = torch.isfinite(b.float())
        # a difference of numbers of the size of the largest logit, each rounded a few times; relative errors of the terms 2^-17 at most
        # (arguments up to 128 in log2 units), of those that count much less
        tol = 2.0 ** -17 + 2.0 ** -21 * biggest + 2.0 ** -21 * b[fine].abs()
        err = (a.double()[fine] - b[fine]).abs()
        assert (err <= tol).all(), "%s: off by %g" % (name, err.max().item())
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (1, 7, 7), (3, 31, 5), (2, 33, 32), (5, 1000, 1), (1, 32000, 5), (40, 4099, 20), (300, 2050, 3), (2, 100003, 32), (7, 20000, 0), (700, 300, 8)])
def test_log_probs(dtype, n, vocab, top):
    x = torch.randn(n, vocab, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) * 3
    check_log_probs(x.to(dtype), top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,vocab,top", [(2000, 40, 3), (1999, 5001, 9), (100, 150001, 20), (601, 16384, 32), (130, 131077, 0)])
def test_log_probs_of_many_rows(dtype, n, vocab, top):
    """Rows that are cut between CTAs, and CTAs that have several rows."""
    x = torch.randn(n, vocab, device=DEV, generator=torch.Generator(DEV).manual_seed(5)) * 3
    x[n // 2] = -math.inf
    x[n // 2, vocab // 3] = 1.0
    x[n // 3] = 0.25
    x[1, -1] = math.nan
    check_log_probs(x.to(dtype), top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_log_probs_of_odd_rows(dtype):
    """Rows that start at any address, and rows of a wider buffer."""
    buf = (torch.randn(9, 5003, device=DEV) * 4).to(dtype)
    for lo, hi in ((0, 5003), (1, 5000), (3, 4999), (5, 8), (7, 2062)):
        check_log_probs(buf[:, lo:hi], min(6, hi - lo))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_log_probs_with_ties(dtype):
    """Of equal logits the lowest ids come first, wherever they are."""
    g = torch.Generator(DEV).manual_seed(2)
    check_log_probs(torch.randint(-2, 3, (20, 9000), device=DEV, generator=g).to(dtype), 32)
    check_log_probs(torch.zeros(3, 40000, device=DEV, dtype=dtype), 20)
    x = torch.zeros(2, 3000, device=DEV, dtype=dtype)
    x[0, ::2] = -0.0  # equal to 0
    check_log_probs(x, 8)
    for order in (torch.arange(5000, 0, -1), torch.arange(5000)):  # the best come last, and first
        check_log_probs((order.to(DEV).float() * 0.01)[None].expand(3, -1).to(dtype).contiguous(), 16)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_log_probs_of_excluded_tokens(dtype):
    x = (torch.randn(8, 3001, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) * 3).to(dtype)
    inf = math.inf
    x[0, torch.randperm(3001, device=DEV)[:2900]] = -inf
    x[1] = -inf
    x[1, 1234] = 0.5          # one token left
    x[2] = -inf               # none
    x[3, 77] = math.nan
    x[4, 99] = inf
    x[5, ::2] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min  # all alike
    got = check_log_probs(x, 5)
    assert got[3][2].tolist() == [0, 1, 2, 3, 4]
    assert got[1][1].item() == 0 and got[2][1, 0].item() == 0
    y = torch.full((2, 50), torch.finfo(dtype).max, device=DEV, dtype=dtype)
    y[1, ::2] = torch.finfo(dtype).min
    check_log_probs(y, 3)


def check_log_probs_closely(logits, top, more=0.0):
    """What only the differences of a row's logits allow, whatever their size.  The sum of exponentials: a lane adds up to vocab / 256 pairs and some 32
    partial sums, each addition off by 2^-24; a term by 2^-22 (the exponential) and by its argument's rounding, 2^-24 of some 24 log2
    units: 2^-20 together.  That is the log's error, and the result is rounded to fp32.  The entropy weighs logs of up to some 32 with such terms."""
    from chunk_attn import ops
    n, vocab = logits.shape
    tokens = torch.arange(n, dtype=torch.int32, device=DEV) % vocab
    got = ops.token_log_probs(logits, tokens, None, top)
    want = D.log_probs(logits, tokens, torch.arange(n, device=DEV), top)
    assert torch.equal(got[3].long(), want[3]), "top tokens differ"
    close = 2.0 ** -24 * (vocab / 256 + 32) + 2.0 ** -20 + more
    for name, a, b, tol in (("log_probs", got[0], want[0], close), ("entropy", got[1], want[1], 32 * close), ("top", got[2], want[2], close)):
        assert torch.isfinite(a).all(), name
        err = (a.double() - b).abs()
        assert (err <= tol + 2.0 ** -23 * b.abs()).all(), "%s: off by %g" % (name, (err - 2.0 ** -23 * b.abs()).max().item())
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,vocab,kept", [(3, 20000, 300), (700, 8000, 300), (2, 3001, 2), (40, 40000, 5)])
def test_log_probs_of_masked_tokens(dtype, n, vocab, kept):
    """Finite masks of any size, over so many tokens that threads meet nothing else: what is left has the distribution.  Rows of nothing but such logits,
    and of such large ones, too."""
    for mask in (-1e4, -65504.0, -1e9, -2.0 ** 30, -2e9, -1e10, -1e15, -1e20, -1e30, -1e35, -3e38):
        if dtype == F16 and mask < -65504:
            continue
        x = torch.randn(n, vocab, device=DEV, generator=torch.Generator(DEV).manual_seed(6)) * 3
        x[:, kept:] = mask
        got = check_log_probs_closely(x.to(dtype), 5, more=2.0 ** -21 * 16)  # logits of up to 16
        if kept < 5:  # the masked ones follow by their ids
            assert got[3][:, kept:].tolist() == [list(range(kept, 5))] * n
    for high in (-1e30, -1e10, 1e9, 1e10, 1e20, 1e30):
        if dtype == F16:
            continue
        x = torch.full((n, vocab), high, device=DEV)
        x[:, ::3] *= 1.25 if high < 0 else 0.75
        check_log_probs_closely(x.to(dtype), 5)


def test_log_probs_far_from_zero():
    """Large logits: only their differences count."""
    g = torch.Generator(DEV).manual_seed(4)
    check_log_probs(torch.randn(4, 6000, device=DEV, generator=g) + 1000, 4)
    check_log_probs(torch.randn(4, 6000, device=DEV, generator=g) * 300, 4)
    check_log_probs(torch.randn(4, 6000, device=DEV, generator=g) * 1e-6 - 50, 4)


@pytest.mark.parametrize("n,vocab,top", [(64, 6000, 5), (1, 32000, 20), (700, 9001, 3), (3, 100, 0)])
def test_log_probs_do_not_go_by_the_size_of_logits(n, vocab, top):
    """Rows far from zero, and rows with a token that takes nearly all: the error is that of rows around zero."""
    x = torch.randn(n, vocab, device=DEV, generator=torch.Generator(DEV).manual_seed(7)) * 2.5
    for offset in (0.0, 30.0, -30.0, 300.0, -1000.0, 1e4, 1e5, -1e6, 2.0 ** 25, 5e8):
        check_log_probs_closely(x + offset, top)
        y = x + offset
        y[:, 0] = offset + max(40.0, abs(offset) * 2.0 ** -20)
        check_log_probs_closely(y, top)
    check_log_probs_closely(x * 300, top)
    for offset in (30.0, 300.0):  # 16-bit steps of 0.25 (fp16) and 2 (bf16)
        check_log_probs_closely((x + offset).half(), top)
        check_log_probs_closely((x + offset).bfloat16(), top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1, 3, 8, 9, 100, 1024, 4100])
def test_log_probs_of_short_rows_by_the_thousands(dtype, vocab):
    """More notes than a short row has vectors need no room: rising, equal and falling logits, rows that start at any address."""
    n, top = 3000, min(vocab, 7)
    x = torch.randn(n, vocab + 1, device=DEV, generator=torch.Generator(DEV).manual_seed(8)) * 3
    x[::3] = x[::3].sort(-1).values
    x[1::3, :] = 0.5
    check_log_probs_closely(x.to(dtype)[:, 1:], top)
    check_log_probs_closely(x.to(dtype)[:, :vocab].contiguous(), 0)


def test_log_probs_of_named_tokens():
    from chunk_attn import ops
    x = torch.randn(4, 100, device=DEV)
    t = torch.tensor([3, -1, 100, -2], dtype=torch.int32, device=DEV)
    lp, ent, top, ids = ops.token_log_probs(x, t)
    assert top.shape == ids.shape == (4, 0)
    assert lp[1].item() == 0 and torch.isnan(lp[2:]).all()
    assert abs(lp[0].item() - torch.log_softmax(x[0].double(), -1)[3].item()) < 1e-5
    rows = torch.tensor([0, 4, -1, 3], dtype=torch.int32, device=DEV)
    lp = ops.token_log_probs(x, t.clamp(0, 99), rows)[0]
    assert torch.isnan(lp[1]) and torch.isnan(lp[2]) and torch.isfinite(lp[[0, 3]]).all()
    assert ops.token_log_probs(x)[0].shape == (0,)
    none = ops.token_log_probs(x[:0], t[:0], top=2)
    assert [tuple(y.shape) for y in none] == [(0,), (0,), (0, 2), (0, 2)]


def test_log_probs_refuses():
    from chunk_attn import ops
    x = torch.randn(4, 100, device=DEV)
    t = torch.zeros(4, dtype=torch.int32, device=DEV)
    for args in ((x.cpu(),), (x.double(),), (x.t(),), (x[0],), (x, t[:3]), (x, t.long()), (x, None, t), (x, t, t[:2]), (x, t, None, 33), (x, t, None, -1), (x[:, :5], t, None, 6), (x, t.cpu())):
        with pytest.raises(RuntimeError, match="token_log_probs"):
            ops.token_log_probs(*args)
