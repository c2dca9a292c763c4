"""The three operators of drafted tokens together, as the decoder, the host and the command run them: drafted trees through every layer,
log probabilities of the nodes, the accepted line, its keys and values brought to the caches."""
import io
import json
import random
import sys

import pytest
import torch

import test_gpu_llama as L
from chunk_attn import generate
from chunk_attn.models.drafting import PromptLookup
from chunk_attn.models.llama_hf import LlamaConfig, LlamaForCausalLM
from chunk_attn.models.model_host import ModelHost
from chunk_attn.models.registry import load_model
from chunk_attn.models.sequence import Sequence
from llama_dense import dense_logits
from test_gpu_model_folders import gagorax_folder, reference, tokens_for, write_folder  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# fp32 products of a hidden size of 256 over two layers: far below it; the two paths differ by the order of their sums alone
TOL32 = 2e-4


def make_model(dtype, hidden=256, heads=4, vocab=512, seed=0):
    cfg = LlamaConfig(vocab_size=vocab, hidden_size=hidden, intermediate_size=512, num_hidden_layers=2, num_attention_heads=heads,
                      max_position_embeddings=512, chunk_attn_kvcache_gb=0.25, torch_dtype=dtype, torch_device=DEV)
    return LlamaForCausalLM(cfg, seed=seed).to(device=DEV, dtype=dtype).eval()


def prefill(model, caches, prompts):
    seqs = [Sequence(p, max_tokens=400) for p in prompts]
    for s, t in zip(seqs, model(seqs, caches, prefill=True)):
        s.append(t)
    return L.rows_in_cache_order(seqs)


def random_tree(rng, vocab, n):
    return [rng.randrange(vocab) for _ in range(n)], [rng.randrange(-1, i) for i in range(n)]


def tolerance(dtype):
    return TOL32 if dtype == torch.float32 else L.LOGIT_TOL


@pytest.mark.parametrize("dtype,hidden,heads", [(torch.float32, 256, 4), (torch.float16, 512, 4), (torch.float32, 160, 2)], ids=["fp32", "fp16", "heads of 80"])
def test_logits_of_drafted_nodes(dtype, hidden, heads):
    """Each node's scores are those of its line in a dense recomputation; nothing reaches the caches."""
    model = make_model(dtype, hidden, heads)
    caches = model.create_kv_caches()
    rng = random.Random(7)
    running = prefill(model, caches, L.prompts_with_shared_prefix(rng, 512, 130, [5, 60, 1]) + [[9], [rng.randrange(512) for _ in range(63)]])
    before = [c.get_trie().children[0].n_tokens for c in caches]
    trees = []
    for n, seq in zip((12, 0, 40, 3, 7), running):
        tokens, parents = random_tree(rng, 512, n)
        trees.append(([seq[-1]] + tokens, [-1] + [p + 1 for p in parents]))
    with torch.inference_mode():
        hidden_states, batch, _, _ = model.model.draft(running, trees, caches)
        got = model.lm_head(hidden_states).float()
    at = 0
    for seq, (tokens, parents) in zip(running, trees):
        for i in range(len(tokens)):
            line, n = [], i
            while n >= 0:
                line.append(tokens[n])
                n = parents[n]
            ref = dense_logits(model, seq.tokens[:-1] + line[::-1], model.model.cos_sin_cache)[-1]
            assert (got[at] - ref).abs().max().item() < tolerance(dtype), (seq.tokens[:3], i)
            at += 1
    assert at == batch.n_nodes and before == [c.get_trie().children[0].n_tokens for c in caches]


def test_drafts_do_not_change_what_is_decoded():
    """Greedy decoding in fp32 with drafts of the right tokens, of wrong ones and of none, and plain steps between: the same tokens,
    over chunk boundaries and a shared prefix; log probabilities as the dense recomputation has them."""
    model = make_model(torch.float32)
    rng = random.Random(3)
    prompts = L.prompts_with_shared_prefix(rng, 512, 130, [5, 60, 1]) + [[9], [rng.randrange(512) for _ in range(63)]]
    caches = model.create_kv_caches()
    plain = prefill(model, caches, prompts)
    for _ in range(90):
        for s, t in zip(plain, model(plain, caches, prefill=False)):
            s.append(t)
    truth = {tuple(s.prompt_tokens): s.tokens for s in plain}
    for c in caches:
        for _ in plain:
            c.remove_seq(0)
    caches = model.create_kv_caches()
    run = prefill(model, caches, prompts)
    about = {s.id: [] for s in run}
    steps = 0
    while min(len(s) - len(s.prompt_tokens) for s in run) < 80:
        if steps % 7 == 6:
            for s, t in zip(run, model(run, caches, prefill=False)):
                s.append(t)
                about[s.id].append(None)
        else:
            drafts = []
            for i, s in enumerate(run):
                right = truth[tuple(s.prompt_tokens)][len(s):][:(steps + i) % 5]
                tokens, parents = [rng.randrange(512)] + right, [-1] + [-1 if j == 0 else j for j in range(len(right))]
                drafts.append((tokens + [3], parents + [len(tokens) - 1]))
            new, told = model.decode_drafts(run, caches, drafts, top=3)
            for i, (s, ts, ab) in enumerate(zip(run, new, told)):
                assert len(ts) == len(ab) >= min((steps + i) % 5, len(truth[tuple(s.prompt_tokens)]) - len(s)) + 1
                for t, a in zip(ts, ab):
                    s.append(t)
                    about[s.id].append(a)
        steps += 1
    assert steps < 60
    for s in run:
        want = truth[tuple(s.prompt_tokens)]
        assert s.tokens[:len(want)] == want[:len(s)]
        n = min(len(s), len(want))
        ref = torch.log_softmax(dense_logits(model, s.tokens, model.model.cos_sin_cache).double(), -1)
        for j, told in enumerate(about[s.id][:n - len(s.prompt_tokens) - 1]):
            if told is None:
                continue
            row = ref[len(s.prompt_tokens) + j]
            lp, lps, ids = told
            assert abs(lp - row[s.tokens[len(s.prompt_tokens) + 1 + j]].item()) < TOL32
            assert len(ids) == 3 and ids[0] == s.tokens[len(s.prompt_tokens) + 1 + j] and lps[0] == lp
            assert (torch.tensor(lps).double() - row.topk(3).values.cpu()).abs().max() < TOL32
    assert all(c.device_status() == 0 for c in caches)


def test_thresholds_accept_probable_tokens():
    """A drafted token that is not the model's choice is taken where it is probable enough; with a threshold above 1, never."""
    model = make_model(torch.float32)
    for epsilon, taken in ((1e-6, True), (2.0, False)):
        caches = model.create_kv_caches()
        run = prefill(model, caches, [[5, 6, 7], [8, 9]])
        ref = [dense_logits(model, s.tokens, model.model.cos_sin_cache)[-1] for s in run]
        second = [int(r.topk(2).indices[1]) for r in ref]
        new, told = model.decode_drafts(run, caches, [([t], [-1]) for t in second], thresholds=(epsilon, 1e3), top=1)
        for s, t, tok, ab, r in zip(run, second, new, told, ref):
            if taken:
                assert tok[0] == t and len(tok) == 2
                assert abs(ab[0][0] - torch.log_softmax(r.double(), -1)[t].item()) < TOL32 and ab[0][2] == [int(r.argmax())]
            else:
                assert tok == [int(r.argmax())]


def test_decode_drafts_refuses_and_leaves_the_caches():
    model = make_model(torch.float32)
    caches = model.create_kv_caches()
    run = prefill(model, caches, [[5, 6, 7], [8, 9]])
    none = ([], [])
    for bad, what in (([none], "one draft per sequence"), ([none, ([1, 2], [-1])], "one parent"), ([none, ([512], [-1])], "vocabulary"),
                      ([none, ([-1], [-1])], "vocabulary"), ([none, ([1], [0])], "parent"), ([none, ([1] * 256, [-1] * 256)], "256 nodes"),
                      ([none, ([1] * 600, list(range(-1, 599)))], "nodes")):
        with pytest.raises((ValueError, RuntimeError), match=what):
            model.decode_drafts(run, caches, bad)
    assert model.decode_drafts([], caches, []) == ([], [])
    at_end = Sequence([1] * 510)
    assert model.decode_drafts(run, caches, [none, none])[0] == [[t] for t in model_choice(model, run)]
    caches = model.create_kv_caches()
    run = prefill(model, caches, [at_end.tokens])
    with pytest.raises(ValueError, match="max_position_embeddings"):
        model.decode_drafts(run, caches, [([1, 2], [-1, 0])])
    assert len(model.decode_drafts(run, caches, [([1], [-1])])[0][0]) >= 1


def model_choice(model, seqs):
    return [int(dense_logits(model, s.tokens, model.model.cos_sin_cache)[-1].argmax()) for s in seqs]


def test_score():
    """Log probabilities of prompts, ragged, in portions, one token alone among them."""
    model = make_model(torch.float32)
    rng = random.Random(11)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (70, 1, 2, 33)]
    for portion in (1024, 7):
        for prompt, (lp, entropy, top_lp, top_ids) in zip(prompts, model.score(prompts, top=4, portion=portion)):
            n = len(prompt) - 1
            assert lp.shape == entropy.shape == (n,) and top_lp.shape == top_ids.shape == (n, 4)
            ref = torch.log_softmax(dense_logits(model, prompt, model.model.cos_sin_cache).double(), -1)[:n]
            if n:
                want = ref.gather(1, torch.tensor(prompt[1:], device=DEV)[:, None])[:, 0]
                assert (lp - want).abs().max() < TOL32 and (entropy + (ref * ref.exp()).sum(1)).abs().max() < 10 * TOL32
                assert (top_lp - ref.topk(4).values).abs().max() < TOL32
                assert (ref.gather(1, top_ids.long()) - ref.topk(4).values).abs().max() < TOL32
    for bad in ([], [[]], [[512]], [[-1, 2]]):
        with pytest.raises(ValueError):
            model.score(bad)
    assert model.score([[1, 2, 3]])[0][2].shape == (2, 0)


@pytest.mark.parametrize("drafts", [False, True])
def test_host_with_drafts_and_log_probs(drafts):
    model = make_model(torch.float32)
    caches = model.create_kv_caches()
    rng = random.Random(3)
    prompts = L.prompts_with_shared_prefix(rng, 512, 100, [4, 30, 64, 9, 1, 17]) + [[1, 2, 3] * 7]
    lens, asked = [12, 40, 7, 70, 25, 1, 33], [None, 0, 2, 5, None, 1, 32]
    host = ModelHost(model, caches, max_batch_size=4, draft=PromptLookup(6, 2, 2) if drafts else None)
    host.cycle_time = 0.05
    with host:
        seqs = [host.predict_async(p, n, k) for p, n, k in zip(prompts, lens, asked)]
        results = [s.get_result(timeout=120) for s in seqs]
    for p, n, k, seq, toks in zip(prompts, lens, asked, seqs, results):
        assert toks[:len(p)] == p and len(toks) == len(p) + n
        ref = torch.log_softmax(dense_logits(model, toks, model.model.cos_sin_cache).double(), -1)
        assert len(seq.token_log_probs) == (0 if k is None else n)
        for t in range(n):
            row, tok = ref[len(p) - 1 + t], toks[len(p) + t]
            assert row[tok] >= row.max() - 2 * TOL32
            if k is not None:
                lp, lps, ids = seq.token_log_probs[t]
                assert abs(lp - row[tok].item()) < TOL32 and len(lps) == len(ids) == k
                if k:
                    assert (torch.tensor(lps).double() - row.topk(k).values.cpu()).abs().max() < TOL32
    assert all(len(c.get_trie().children) == 0 for c in caches) and all(c.device_status() == 0 for c in caches)
    if drafts:
        assert host.n_drafted > 0


def test_command(tmp_path, monkeypatch, capsys):
    fields = {"vocab_size": 64, "hidden_size": 128, "intermediate_size": 96, "num_hidden_layers": 2, "num_attention_heads": 2,
              "max_position_embeddings": 128}
    direct = LlamaForCausalLM(LlamaConfig(torch_device=DEV, chunk_attn_kvcache_gb=0.1, torch_dtype=torch.float32, **fields), seed=3).to(DEV, torch.float32)
    write_folder(tmp_path, dict(fields, architectures=["LlamaForCausalLM"]), direct.state_dict())
    monkeypatch.setattr(generate, "load_model", lambda *a, **k: load_model(*a, chunk_attn_kvcache_gb=0.1, **k))
    outs = []
    for extra in ([], ["--draft-tokens", "5"], ["--draft-tokens", "5", "--log-probs", "2"], ["--log-probs", "0"]):
        monkeypatch.setattr(sys, "stdin", io.StringIO("5 9 33 2\n7 7 7 7 7\n"))
        assert generate.main(["--model", str(tmp_path), "--dtype", "float32", "--max-new-tokens", "20"] + extra) == 0
        outs.append(capsys.readouterr().out.splitlines())
    assert len(outs[0]) == 2 and outs[1] == outs[0] and outs[2][::2] == outs[0] and outs[3][::2] == outs[0]
    about = json.loads(outs[2][1])
    tokens = [int(t) for t in outs[0][0].split()]
    assert len(about) == 20 and [a[2][0] for a in about] == tokens[4:] and all(a[0] == a[1][0] and len(a[1]) == 2 for a in about)
    for bad in (["--draft-tokens", "-1"], ["--draft-tokens", "256"], ["--log-probs", "33"]):
        with pytest.raises(SystemExit):
            generate.main(["--model", str(tmp_path)] + bad)


def test_log_probs_of_a_model_without_drafts(gagorax_folder, monkeypatch, capsys):  # noqa: F811
    """The host takes log probabilities from any model's scores; drafts are refused where the model has no step for them."""
    cfg, w, path = gagorax_folder
    prompts = [tokens_for(cfg, n, n) for n in (3, 70)]
    text = "\n".join(" ".join(map(str, p)) for p in prompts) + "\n"
    args = ["--model", str(path / "m"), "--dtype", "float32", "--max-new-tokens", "5"]
    monkeypatch.setattr(sys, "stdin", io.StringIO(text))
    assert generate.main(args + ["--log-probs", "2"]) == 0
    lines = capsys.readouterr().out.splitlines()
    for p, line, about in zip(prompts, lines[::2], lines[1::2]):
        toks = [int(t) for t in line.split()]
        ref = torch.log_softmax(torch.tensor(reference(cfg, w, toks)).double(), -1)
        for t, (lp, lps, ids) in enumerate(json.loads(about)):
            row = ref[len(p) - 1 + t]
            # the scores themselves are compared to 1e-3 where this model is tested
            assert ids[0] == toks[len(p) + t] and abs(lp - row[ids[0]].item()) < 1e-3 and max(abs(l - row[i].item()) for l, i in zip(lps, ids)) < 1e-3
    monkeypatch.setattr(sys, "stdin", io.StringIO(text))
    with pytest.raises(ValueError, match="does not decode drafted"):
        generate.main(args + ["--draft-tokens", "2"])
