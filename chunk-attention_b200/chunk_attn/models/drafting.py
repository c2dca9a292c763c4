"""Drafted tokens: guesses at the tokens that come next, which one decode step of a model checks together.

A draft is (tokens, parents): a tree below the sequence's last token.  parents[i] is the number of the token that tokens[i] would
follow, a lower one, or -1 for the sequence's last token.  The model attends to the cached tokens and to each drafted token's own line
(`Attention.forward_draft`), and keeps the longest line that it agrees with (`ops.accept_draft`).
"""


def cut(draft, depth):
    """The draft without what stands deeper than `depth` tokens."""
    tokens, parents = draft
    if len(tokens) != len(parents):
        raise ValueError("one parent per drafted token is required")
    deep, at, kept = [], {-1: -1}, ([], [])  # at: the new numbers of those that stay
    for i, (token, p) in enumerate(zip(tokens, parents)):
        if not -1 <= p < i:
            raise ValueError("a drafted token's parent must be a token before it, or -1")
        deep.append(1 if p < 0 else deep[p] + 1)
        if deep[i] <= depth:
            at[i] = len(kept[0])
            kept[0].append(token)
            kept[1].append(at[p])
    return kept


class PromptLookup:
    """Drafts from the sequence's own text: where its last tokens have stood before, what followed them is drafted.

    n_tokens: drafted tokens at most; ngram: the longest ending that is looked for (then shorter ones); lines: how many earlier
    places, the latest first, share the draft; equal beginnings are drafted once."""

    def __init__(self, n_tokens=8, ngram=3, lines=2):
        if not 1 <= n_tokens <= 255 or ngram < 1 or lines < 1:
            raise ValueError("n_tokens must be 1 to 255, ngram and lines positive")
        self.n_tokens, self.ngram, self.lines = n_tokens, ngram, lines

    def __call__(self, tokens, depth):
        """A draft of at most `depth` tokens in a line; ([], []) when nothing is found."""
        if depth < 1:
            return [], []
        return self._drafted(tokens, depth, (i for i in range(len(tokens) - 1, 0, -1) if tokens[i - 1] == tokens[-1]))

    def follow(self):
        """A drafter of one sequence, to which tokens are only ever appended: it keeps where every token has stood, so that a draft goes through the
        places of the last one alone.  (16000 tokens without the last one among them: a call of its own 0.8 ms, a follower's 2 us.)"""
        return _Follower(self)

    def _drafted(self, tokens, depth, candidates):
        """candidates: the places that the last token stands before, latest first."""
        # found[n - 1]: the latest places that follow the last n tokens
        found = [[] for _ in range(min(self.ngram, len(tokens) - 1))]
        for i in candidates if found else ():
            for n, places in enumerate(found, 1):
                if n > i or tokens[i - n] != tokens[-n]:
                    break
                if len(places) < self.lines:
                    places.append(i)
            if len(found[-1]) == self.lines:
                break
        longest = next((places for places in reversed(found) if places), [])
        return self._tree([tokens[i:i + depth] for i in longest])

    def _tree(self, lines):
        drafted, parents, known = [], [], {}
        # the latest place has the first half of the tokens, or all of them if it is the only one
        for i, line in enumerate(lines):
            at, room = -1, self.n_tokens if i else (self.n_tokens + len(lines) - 1) // len(lines)
            for token in line:
                if (at, token) not in known:
                    if len(drafted) >= room:
                        break
                    known[at, token] = len(drafted)
                    drafted.append(token)
                    parents.append(at)
                at = known[at, token]
        return drafted, parents


class _Follower:
    def __init__(self, lookup):
        self.lookup = lookup
        self.latest = {}   # token: the latest place behind it
        self.before = [0]  # of every place, the one before behind the same token; 0: none

    def __call__(self, tokens, depth):
        if max(1, len(tokens)) < len(self.before):
            raise ValueError("a drafter follows one sequence, which does not get shorter")
        for i in range(len(self.before), len(tokens)):
            self.before.append(self.latest.get(tokens[i - 1], 0))
            self.latest[tokens[i - 1]] = i
        return self.lookup._drafted(tokens, depth, self._places(tokens[-1])) if depth > 0 and tokens else ([], [])

    def _places(self, token):
        i = self.latest.get(token, 0)
        while i:
            yield i
            i = self.before[i]
