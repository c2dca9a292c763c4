"""Drafted tokens: guesses at the tokens that come next, which one decode step of a model checks together.

A draft is (tokens, parents): a tree below the sequence's last token.  parents[i] is the number of the token that tokens[i] would
follow, a lower one, or -1 for the sequence's last token.  The model attends to the cached tokens and to each drafted token's own line
(`Attention.forward_draft`), and keeps the longest line that it agrees with (`ops.accept_draft`).
"""


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
        for n in range(min(self.ngram, len(tokens) - 1), 0, -1):
            ending = tokens[-n:]
            places = []
            for i in range(len(tokens) - n - 1, -1, -1):
                if tokens[i:i + n] == ending:
                    places.append(i + n)
                    if len(places) == self.lines:
                        break
            if places:
                return self._tree([tokens[i:i + depth] for i in places])
        return [], []

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
