"""Drafts from a sequence's own text, and the host's decode steps over drafts, without a GPU."""
import random

import pytest

import test_model_host_cpu as H
from chunk_attn.models.drafting import PromptLookup, cut
from chunk_attn.models.model_host import ModelHost


def test_prompt_lookup():
    look = PromptLookup(n_tokens=4, ngram=2, lines=1)
    assert look([1, 2, 3, 4, 9, 1, 2], 8) == ([3, 4, 9, 1], [-1, 0, 1, 2])
    assert look([1, 2, 3, 4, 9, 1, 2], 2) == ([3, 4], [-1, 0])
    assert look([1, 2, 3], 8) == ([], []) and look([5], 8) == ([], []) and look([1, 1], 0) == ([], [])
    assert look([7, 7], 8) == ([7], [-1])
    two = PromptLookup(n_tokens=6, ngram=2, lines=2)
    # "1 2" stood twice before: 3 4 .. last, 3 5 .. first; they share 3
    tokens, parents = two([1, 2, 3, 5, 6, 1, 2, 3, 4, 8, 1, 2], 3)
    assert tokens == [3, 4, 8, 5, 6] and parents == [-1, 0, 1, 0, 3]
    for bad in ((0, 1, 1), (256, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            PromptLookup(*bad)


def test_drafts_are_trees_of_the_text():
    rng = random.Random(0)
    for _ in range(200):
        tokens = [rng.randrange(4) for _ in range(rng.randint(1, 40))]
        look = PromptLookup(rng.randint(1, 9), rng.randint(1, 4), rng.randint(1, 3))
        depth = rng.randint(0, 9)
        drafted, parents = look(tokens, depth)
        assert len(drafted) == len(parents) <= look.n_tokens
        assert len(set(zip(parents, drafted))) == len(drafted)
        deep = []
        for i, p in enumerate(parents):
            assert -1 <= p < i
            deep.append(1 if p < 0 else deep[p] + 1)
        assert max(deep, default=0) <= depth


def scan(look, tokens, depth):
    """The definition: the latest places after the longest ending that stood before."""
    for n in range(min(look.ngram, len(tokens) - 1), 0, -1):
        places = [i + n for i in range(len(tokens) - n - 1, -1, -1) if tokens[i:i + n] == tokens[-n:]][:look.lines]
        if places and depth > 0:
            return look._tree([tokens[i:i + depth] for i in places])
    return [], []


def test_followers_draft_what_the_text_says():
    rng = random.Random(2)
    for _ in range(100):
        look = PromptLookup(rng.randint(1, 9), rng.randint(1, 4), rng.randint(1, 3))
        follower, tokens, words = look.follow(), [], rng.randint(1, 6)
        for _ in range(rng.randint(1, 30)):
            tokens += [rng.randrange(words) for _ in range(rng.randint(0, 4))]
            depth = rng.randint(0, 6)
            want = scan(look, tokens, depth)
            assert look(tokens, depth) == want
            assert follower(tokens, depth) == want
    follower = look.follow()
    follower([1, 2, 3], 4)
    with pytest.raises(ValueError, match="shorter"):
        follower([1, 2], 4)


class Counted(list):
    """Counts the elements that are read."""
    read = 0

    def __getitem__(self, i):
        x = super().__getitem__(i)
        Counted.read += len(x) if isinstance(i, slice) else 1
        return x


def test_a_draft_does_not_go_through_the_text_again():
    look = PromptLookup(8)
    tokens = Counted(range(16000))
    Counted.read = 0
    assert look(tokens, 8) == ([], [])
    assert Counted.read < 2 * 16000  # a call by itself: once
    follower = look.follow()
    follower(tokens, 8)
    Counted.read = 0
    for i in range(10):
        tokens.append(20000 + i)
        assert follower(tokens, 8) == ([], [])
    assert Counted.read < 10 * 32


def test_the_host_gives_every_sequence_a_drafter():
    look, made = PromptLookup(4), []

    class Source:
        def __call__(self, tokens, depth):
            raise AssertionError("the followers draft")

        def follow(self):
            made.append(look.follow())
            return made[-1]

    host = ModelHost(DraftingModel(), [H.TreeCache()], max_batch_size=2, draft=Source())
    host.cycle_time = 0.02
    prompts = [[1, 2, 3, 1, 2], [4, 4, 4], [5, 6]]
    with host:
        seqs = [host.predict_async(p, 20) for p in prompts]
        for seq, p in zip(seqs, prompts):
            assert seq.get_result(timeout=60) == H.rollout(p, 20)
    assert len(made) == 3


class DraftingModel(H.TreeModel):
    """Takes drafted tokens as the decoder does: the longest line that its own next tokens agree with."""

    def decode_drafts(self, seqs, kv_caches, drafts, thresholds, top):
        for cache in kv_caches:
            assert H.tree_rows(cache.tree) == [s.tokens[:-1] for s in seqs]
        new = []
        for r, (seq, (tokens, parents)) in enumerate(zip(seqs, drafts)):
            line, kept = -1, []
            while True:
                want = H.next_token(seq.tokens + kept)
                step = [i for i in range(len(tokens)) if parents[i] == line and tokens[i] == want]
                if not step:
                    break
                line = step[0]
                kept.append(want)
            new.append(kept + [want])
            for cache in kv_caches:
                cache.tree.extend_seq(r, [seq[-1]] + kept)
        return new, [[(0.0, [], [])] * len(t) for t in new]


@pytest.mark.parametrize("batch", [1, 3])
def test_host_over_drafts(batch):
    """Every request's tokens are those of plain decoding, in fewer steps when the drafts are right, whatever the drafts are."""
    rng = random.Random(1)
    prompts = [[rng.randrange(1000) for _ in range(n)] for n in (3, 9, 4, 17, 8)]
    lens = [12, 1, 30, 7, 19]
    truth = {tuple(p): H.rollout(p, 40) for p in prompts}

    def oracle(tokens, depth):  # a right line of three, and a wrong one beside it
        rest = next(t for p, t in truth.items() if tuple(t[:len(tokens)]) == tuple(tokens))[len(tokens):][:min(3, depth)]
        return rest + [5], list(range(-1, len(rest) - 1)) + [-1]

    steps = []
    for draft in (lambda t, d: ([], []), lambda t, d: ([1, 2], [-1, 0]) if d > 1 else ([], []), oracle):
        caches = [H.TreeCache(), H.TreeCache()]
        host = ModelHost(DraftingModel(), caches, max_batch_size=batch, draft=draft)
        host.cycle_time = 0.02
        with host:
            seqs = [host.predict_async(p, n) for p, n in zip(prompts, lens)]
            for seq, p, n in zip(seqs, prompts, lens):
                assert seq.get_result(timeout=60) == H.rollout(p, n)
        steps.append(host.n_decode_steps)
    assert steps[0] == steps[1] and steps[2] < steps[0] / 2
    assert host.n_accepted > 0 and host.n_drafted > host.n_accepted


def test_a_draft_beyond_the_end_is_cut():
    caches = [H.TreeCache()]
    host = ModelHost(DraftingModel(), caches, max_batch_size=2, draft=lambda t, depth: (H.rollout(t, 9)[len(t):], list(range(-1, 8))))
    host.cycle_time = 0.02
    with host:
        for n in (1, 2, 4, 13):
            assert host.predict([4, 5, 6], n) == H.rollout([4, 5, 6], n)


def test_host_refuses():
    with pytest.raises(ValueError, match="does not decode drafted"):
        ModelHost(H.TreeModel(), [], draft=PromptLookup())
    host = ModelHost(H.TreeModel(), [H.TreeCache()])
    host.stopped = False
    with pytest.raises(ValueError, match="log_probs"):
        host.predict_async([1], 1, log_probs=33)


class LimitedModel(DraftingModel):
    """Has positions for no more than `limit` tokens, as decoders do, and refuses steps that need more."""
    limit = 12

    def decode_drafts(self, seqs, kv_caches, drafts, thresholds, top):
        for seq, (tokens, parents) in zip(seqs, drafts):
            deep = []
            for p in parents:
                deep.append(1 if p < 0 else deep[p] + 1)
            if len(seq) - 1 + max(deep, default=0) >= self.limit:
                raise ValueError("sequence exceeds the last position")
        return super().decode_drafts(seqs, kv_caches, drafts, thresholds, top)


def test_a_draft_beyond_the_last_position_does_not_fail_the_host():
    """Requests that end at the model's last position are served whatever the draft brings beyond it."""
    def draft(tokens, depth):
        return H.rollout(tokens, 9)[len(tokens):] + [1, 2, 3], list(range(-1, 8)) + [-1, 9, 10]

    host = ModelHost(LimitedModel(), [H.TreeCache()], max_batch_size=2, draft=draft)
    host.cycle_time = 0.02
    with host:
        for n in (2, 4, 9, 10):
            assert host.predict([4, 5, 6], n) == H.rollout([4, 5, 6], n)
        assert host.failure is None


def test_cut():
    assert cut(([7, 8, 9, 5, 6], [-1, 0, 1, -1, 3]), 2) == ([7, 8, 5, 6], [-1, 0, -1, 2])
    assert cut(([7, 8, 9], [-1, 0, 1]), 3) == ([7, 8, 9], [-1, 0, 1]) and cut(([7, 8], [-1, -1]), 0) == ([], [])
    for bad in (([1], []), ([1], [0]), ([1, 2], [-1, -2])):
        with pytest.raises(ValueError):
            cut(bad, 4)
