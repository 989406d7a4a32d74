"""Greedy speculative decoding over two resident models: the verify loop of
examples/spec_decode_70b.rs:213-336 on librq.  A draft model proposes K
tokens one at a time; the target scores [last, d_1 .. d_K] in one forward
(rq_llama_forward_all, M = K+1 rows through the small-M kernels); the
longest prefix the target agrees with is accepted plus the target's own
next token (the bonus); both KV caches are truncated to the accepted
length.  With greedy sampling the output equals the target's greedy
decode, whatever the draft proposes.

With a temperature the draft's tokens are drawn from its probabilities, and
the target accepts or replaces them by rq_spec_verify, so that the output is
distributed as the target's own samples, whatever the draft proposes."""
from __future__ import annotations

from collections import deque

from .linear import Context

try:  # greedy decoding needs neither torch nor its binding
    import torch
except Exception:  # pragma: no cover
    torch = None
_rqtorch = None  # the binding, from the first verification on


def spec_verify(p, drafts, u, r, q=None, n_drafts=None):
    """(tokens [batch, n + 1], accepted [batch]) int32: the drafted tokens
    drafts [batch, n] checked against the target's probabilities p [batch, n +
    1, vocab] and those they were drawn from, q [batch, n, vocab] (None: each
    was certain), with the uniform numbers u [batch, n] and r [batch]
    (float32); rq_spec_verify of include/rq.h.  n_drafts [batch] (int32)
    limits a row's drafts.  A row of tokens is the accepted drafts, one drawn
    token and -1s; with n = 0 the call samples from p."""
    global _rqtorch
    if _rqtorch is None:
        from . import _rqtorch
    return _rqtorch.spec_verify(Context.of(p), p, drafts, u, r, q, n_drafts)


class SpecDecoder:
    def __init__(self, target, draft, k: int = 4, adaptive: bool = False, window: int = 4, temperature: float = 0.0,
                 seed: int = 0):
        """temperature 0: greedy.  Above: sampling on one GPU, its random
        numbers drawn from ``seed``."""
        self.target, self.draft = target, draft
        self.temperature = float(temperature)
        if self.temperature > 0:
            self.device = torch.device("cuda", target.ctx.device)
            self.gen = torch.Generator(device=self.device).manual_seed(seed)
        self.k_max = k
        self.adaptive, self.window = adaptive, window
        self.stats = {"target_forwards": 0, "draft_forwards": 0, "accepted": 0, "proposed": 0}

    # ---- sampling: probabilities on the device, tokens by rq_spec_verify
    def _probs(self, model, ids, pos, every):
        """softmax(logits / temperature) of the last (or every) position,
        [1, rows, vocab]."""
        rows = len(ids) if every else 1
        out = torch.empty((rows, model.cfg["vocab"]), dtype=torch.float32, device=self.device)
        if every:
            model.forward_all(ids, pos, logits_out=out)
        else:
            model.forward(ids, pos, logits_out=out[0])
        return torch.softmax(out.div_(self.temperature), -1)[None]

    def _uniform(self, *shape):
        return torch.rand(*shape, device=self.device, generator=self.gen)

    def _draw(self, p):
        """A token from p [1, 1, vocab]: the verification of no draft."""
        none = torch.empty((1, 0), dtype=torch.int32, device=self.device)
        return spec_verify(p, none, self._uniform(1, 0), self._uniform(1))[0]

    def _propose(self, last, index_pos, k):
        """k drafted tokens on top of ``last`` and their probabilities."""
        drafts, probs, cur = [], [], last
        for j in range(k):
            if self.temperature > 0:
                probs.append(self._probs(self.draft, [cur], index_pos + j, False))
                cur = int(self._draw(probs[-1]))
            else:
                _, cur = self.draft.forward([cur], index_pos + j, want_logits=False)
            drafts.append(cur)
            self.stats["draft_forwards"] += 1
        return drafts, probs

    def _verify(self, last, drafts, probs, index_pos):
        """(accepted, next token) of the drafts, by one target forward."""
        k = len(drafts)
        self.stats["target_forwards"] += 1
        if self.temperature > 0:
            p = self._probs(self.target, [last] + drafts, index_pos, True)
            tokens, accepted = spec_verify(p, torch.tensor([drafts], dtype=torch.int32, device=self.device).reshape(1, k),
                                           self._uniform(1, k), self._uniform(1), q=torch.cat(probs, 1) if k else None)
            n = int(accepted)
            return n, int(tokens[0, n])
        _, pred = self.target.forward_all([last] + drafts, index_pos)
        for j in range(k):
            if pred[j] != drafts[j]:
                return j, pred[j]
        return k, pred[k]

    def generate(self, prompt_ids, max_new_tokens: int) -> list:
        t, d = self.target, self.draft
        prompt = [int(v) for v in prompt_ids]
        if self.temperature > 0:
            last = int(self._draw(self._probs(t, prompt, 0, False)))
        else:
            _, last = t.forward(prompt, 0, want_logits=False)
        d.forward(prompt, 0, want_logits=False)
        self.stats["target_forwards"] += 1
        self.stats["draft_forwards"] += 1
        out = [last]
        index_pos = len(prompt)
        k_now = self.k_max
        recent: deque = deque()
        while len(out) < max_new_tokens:
            # 1. draft K tokens: inputs last, d_1 .. d_{K-1}
            drafts, probs = self._propose(last, index_pos, k_now)
            # 2. verify [last, d_1 .. d_K] in one target forward
            # 3. longest accepted prefix, then the bonus token
            accepted, bonus = self._verify(last, drafts, probs, index_pos)
            self.stats["accepted"] += accepted
            self.stats["proposed"] += k_now
            out.extend(drafts[:accepted] + [bonus])
            # 4. caches: every position before the bonus
            if k_now > 0 and accepted == k_now:
                d.forward([drafts[-1]], index_pos + k_now, want_logits=False)
                self.stats["draft_forwards"] += 1
            new_len = index_pos + accepted + 1
            t.truncate_caches(new_len)
            d.truncate_caches(new_len)
            # 5. adaptive K (spec_decode_70b.rs:305-326)
            if self.adaptive:
                recent.append((accepted, k_now))
                if len(recent) > self.window:
                    recent.popleft()
                acc = sum(a for a, _ in recent)
                att = sum(b for _, b in recent)
                rate = acc / att if att else 1.0
                if len(recent) >= 2 and rate < 0.40 and k_now > 0:
                    k_now -= 1
                    recent.clear()
                elif len(recent) >= self.window and rate > 0.70 and k_now < self.k_max:
                    k_now += 1
                    recent.clear()
            index_pos = new_len
            last = bonus
        return out[:max_new_tokens]
