"""Continuous-batching loop around a model and its per-layer KV caches.

Surface and iteration order of the reference's ModelHost (src/chunk_attn/models/model_host.py:13-134):
every iteration (1) retires finished sequences from every cache, (2) prefills the requests that
arrived, inserting each at the row its prefill returned, (3) runs one decode step over everything
that is running.  `running_seqs` is therefore always in the caches' DFS row order, which is the
order `Attention.forward` expects its query rows in.

Unlike the reference, an exception on the worker thread does not leave callers blocked: it is
handed to every sequence in flight and to every later `predict`.
"""
import queue
import threading

import torch

from chunk_attn import ops

from ..logger import logger
from .drafting import cut
from .sequence import Sequence


class ModelHost:
    def __init__(self, model_obj, kv_caches, max_batch_size=32, draft=None, thresholds=None):
        """draft(tokens, depth) -> (drafted tokens, parents): decode steps check drafted tokens, for models with
        `decode_drafts`; thresholds as there.  A draft with `follow()` gives every sequence a drafter of its own."""
        if draft is not None and not hasattr(model_obj, "decode_drafts"):
            raise ValueError("%s does not decode drafted tokens" % type(model_obj).__name__)
        self.model_obj = model_obj
        self.kv_caches = kv_caches
        self.running_seqs = []
        self.max_batch_size = max_batch_size
        self.peak_batch_size = 0
        self.stopped = True
        self.cycle_time = 1.0
        self.failure = None
        self.n_decode_steps = 0
        self.draft, self.thresholds = draft, thresholds
        self.n_drafted = self.n_accepted = 0
        self.batch_queue = queue.Queue(maxsize=2 * max_batch_size)
        self.thread = None

    # ---- client side ---------------------------------------------------------------------------
    def predict_async(self, prompt_tokens, max_tokens, log_probs=None):
        """log_probs: k >= 0, also keep every generated token's log probability and the k best tokens (`Sequence`)."""
        if self.failure is not None:
            raise RuntimeError("model host failed: %r" % (self.failure,))
        if self.stopped:
            raise RuntimeError("model host is stopped, can't predict anymore")
        if len(prompt_tokens) == 0:
            raise ValueError("empty prompt")
        if log_probs is not None and not 0 <= log_probs <= 32:
            raise ValueError("log_probs must be 0 to 32")
        seq = Sequence(prompt_tokens=prompt_tokens, max_tokens=max_tokens, log_probs=log_probs)
        self.batch_queue.put(seq)
        return seq

    def predict(self, prompt_tokens, max_tokens):
        return self.predict_async(prompt_tokens, max_tokens).get_result()

    def start(self):
        if not self.stopped:
            raise RuntimeError("model host is already started")
        self.stopped = False
        self.thread = threading.Thread(target=self.run_iterations, name="chunk-attn-model-host", daemon=True)
        self.thread.start()

    def stop(self):
        self.stopped = True
        if self.thread is not None:
            self.thread.join()
            self.thread = None

    def __enter__(self):
        self.start()
        return self

    def __exit__(self, exc_type, exc_val, exc_tb):
        self.stop()

    # ---- worker side ---------------------------------------------------------------------------
    def get_new_requests(self):
        new_seqs = []
        if len(self.running_seqs) == 0:  # idle: block until something arrives (or a cycle passes)
            try:
                new_seqs.append(self.batch_queue.get(block=True, timeout=self.cycle_time))
            except queue.Empty:
                pass
        while len(new_seqs) + len(self.running_seqs) < self.max_batch_size:
            try:
                new_seqs.append(self.batch_queue.get(block=False))
            except queue.Empty:
                break
        return new_seqs

    def retire_finished(self):
        """Drop finished sequences from the batch and from every layer's cache (rows shift down as the
        reference's index arithmetic assumes, model_host.py:88-102)."""
        kept = []
        n_removed = 0
        for idx, seq in enumerate(self.running_seqs):
            if seq.finished():
                for kv_cache in self.kv_caches:
                    kv_cache.remove_seq(idx - n_removed)
                n_removed += 1
                logger.debug("finished the seq %s", seq.id)
                seq.set_result_ready()
            else:
                kept.append(seq)
        self.running_seqs = kept
        return n_removed

    def next_tokens(self, seqs, prefill):
        """The model's next token of each sequence; where log probabilities are asked for, those too."""
        top = max((s.log_probs for s in seqs if s.log_probs is not None), default=None)
        if top is None:
            return self.model_obj(seqs, self.kv_caches, prefill=prefill)
        logits = self.model_obj.logits(seqs, self.kv_caches, prefill)
        _, _, best_lp, best = ops.token_log_probs(logits, top=max(1, min(top, logits.shape[1])))
        best_lp, best = best_lp.tolist(), best.tolist()
        for seq, lps, ids in zip(seqs, best_lp, best):
            if seq.log_probs is not None:
                seq.token_log_probs.append((lps[0], lps[:seq.log_probs], ids[:seq.log_probs]))
        return [ids[0] for ids in best]

    def decode_drafts(self):
        """One decode step over drafted tokens.  The draft is asked for lines that end with the sequence; what a longer one brings
        beyond its end is dropped before the model sees it (it may be beyond the model's last position, too)."""
        seqs = self.running_seqs
        for s in seqs:
            if s.drafter is None:
                s.drafter = self.draft.follow() if hasattr(self.draft, "follow") else self.draft
        left = [s.max_tokens + len(s.prompt_tokens) - len(s) - 1 for s in seqs]
        drafts = [cut(s.drafter(s.tokens, n), n) for s, n in zip(seqs, left)]
        top = max((s.log_probs for s in seqs if s.log_probs is not None), default=0)
        new, told = self.model_obj.decode_drafts(seqs, self.kv_caches, drafts, self.thresholds, top)
        for seq, (drafted, _), tokens, about in zip(seqs, drafts, new, told):
            self.n_drafted += len(drafted)
            self.n_accepted += len(tokens) - 1
            for token, (lp, lps, ids) in zip(tokens, about):
                if seq.finished():
                    break
                seq.append(token)
                if seq.log_probs is not None:
                    seq.token_log_probs.append((lp, lps[:seq.log_probs], ids[:seq.log_probs]))

    def step(self):
        """One iteration of the serving loop; returns the number of sequences that were decoded."""
        self.retire_finished()
        arrived = self.get_new_requests()
        if arrived:
            logger.debug("prefill of %d new seqs, %d running", len(arrived), len(self.running_seqs))
            new_tokens = self.next_tokens(arrived, prefill=True)
            for seq, tok in zip(arrived, new_tokens):
                seq.append(tok)
            for seq in arrived:  # same order as the caches inserted them: rows stay aligned
                self.running_seqs.insert(seq.index, seq)
        self.peak_batch_size = max(self.peak_batch_size, len(self.running_seqs))
        # a one-token request is complete after its prefill; it must not be decoded
        live = [s for s in self.running_seqs if not s.finished()]
        if len(live) != len(self.running_seqs):
            self.retire_finished()
        if self.running_seqs:
            if self.draft is not None:
                self.decode_drafts()
            else:
                for seq, tok in zip(self.running_seqs, self.next_tokens(self.running_seqs, prefill=False)):
                    seq.append(tok)
            self.n_decode_steps += 1
        return len(self.running_seqs)

    @torch.inference_mode()
    def run_iterations(self):
        try:
            while not self.stopped:
                self.step()
            # a stop request lets nothing hang: whatever is still running leaves the caches (last row
            # first, so the remaining rows keep their indices) and is reported as cancelled
            for idx in reversed(range(len(self.running_seqs))):
                for kv_cache in self.kv_caches:
                    kv_cache.remove_seq(idx)
            self._fail_all(RuntimeError("model host stopped before the sequence finished"), record=False)
        except BaseException as e:  # noqa: BLE001 - handed to the callers, not swallowed
            self._fail_all(e, record=True)

    def _fail_all(self, error, record):
        if record:
            logger.error("model host failed: %r", error)
            self.failure = error
            self.stopped = True
        for seq in self.running_seqs:
            seq.set_error(error)
        self.running_seqs = []
        while True:
            try:
                self.batch_queue.get(block=False).set_error(error)
            except queue.Empty:
                break
