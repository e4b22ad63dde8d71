"""The plugin form of a model that answers with logits: a subclass says what the model answers, everything that the
reference's plugin surface asks of a model (``sample``, ``sample1``, ``calc_ml2p``, ``parse_file``; lib4mc/MonteCarloParent.py:11-69)
runs on ``montecarlo_amd.logits``.  The keys it samples stay on the GPU and go to ``MonteCarloLib`` as any other model's."""
from __future__ import annotations

import abc
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import dist as mcd
from .lib4mc.MonteCarloParent import MonteCarlo, SampleKeys
from .logits import OUTSIDE, SKIP, logits_draw, logits_keys, logits_score


def default_batch(tokens: int, max_len: int) -> int:
    """Passwords at a time: 65536, or as many as their answers' [batch, max_len, tokens] logits stay below 2^31 with."""
    return max(1, min(1 << 16, (1 << 31) // (tokens * max_len)))


class LogitsMonteCarlo(MonteCarlo):
    """``vocabulary``: the text of every token, the end symbol's at position ``end``.  A password is its tokens and the end
    symbol; one of ``max_len`` tokens needs no end symbol (so the probabilities of all strings up to that length add up to
    1) and longer ones are impossible.  ``batch``: passwords the model is asked about at a time (``default_batch``).

    Samples carry the probability of the tokens that were drawn, ``calc_ml2p`` that of the tokens that ``encode`` gives: of a
    sub-word vocabulary, in which a password has several encodings, each speaks of one of them.  Scores are sums of 32 bits per
    token: a sample's key and its password's score, or those of batches of other sizes, may differ in their last bits."""

    def __init__(self, vocabulary: Sequence[str], end: int, max_len: int = 32, temperature: float = 1.0,
                 batch: Optional[int] = None, device=None):
        self.vocabulary, self.end, self.max_len = list(vocabulary), int(end), int(max_len)
        if not 0 <= self.end < len(self.vocabulary) or self.max_len < 1 or (batch is not None and batch < 1):
            raise ValueError("end: a position of the vocabulary; max_len and batch: at least 1")
        self.temperature = float(temperature)
        self.batch = default_batch(len(self.vocabulary), self.max_len) if batch is None else int(batch)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._ids = {text: i for i, text in enumerate(self.vocabulary) if i != self.end}
        if type(self).encode is LogitsMonteCarlo.encode:
            chars = [text for i, text in enumerate(self.vocabulary) if len(text) == 1 and i != self.end]
            twice = next((c for c in chars if chars.count(c) > 1), None) if len(set(chars)) < len(chars) else None
            if twice is not None:                           # (samples would hold either, scores only know the last)
                raise ValueError(f"vocabulary: two tokens are {twice!r}")

    @abc.abstractmethod
    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        """[B, t] tokens (int64; any value behind a password's end) -> [B, t + 1, V] logits on the GPU: place i speaks of token
        i given the i before it.  More logits than tokens (rows padded to a multiple) are cut to the vocabulary's."""

    def next_logits(self, tokens: torch.Tensor) -> torch.Tensor:
        """[B, t] tokens -> [B, V] logits of the next one (a model with a state of its own keeps it here)."""
        return self.logits(tokens)[:, -1]

    def _of_vocabulary(self, x: torch.Tensor) -> torch.Tensor:
        n = len(self.vocabulary)
        if x.shape[-1] < n:
            raise ValueError(f"the model answers with {x.shape[-1]} logits for a vocabulary of {n}")
        return x[..., :n]

    def encode(self, pwd: str) -> List[int]:
        """A password's tokens; ``OUTSIDE`` (or any other id that is none) for what the vocabulary does not hold.  One character a
        token, unless overridden."""
        return [self._ids.get(c, OUTSIDE) for c in pwd]

    # ---- sampling (lib4mc/MonteCarloParent.py:33-46) ---------------------------------------------------------------
    @torch.no_grad()
    def _sample_batch(self, n: int, seed: int, first: int) -> Tuple[torch.Tensor, torch.Tensor]:
        tokens = torch.full((n, self.max_len), SKIP, dtype=torch.int64, device=self.device)
        ml2p = torch.zeros((n, self.max_len), dtype=torch.float32, device=self.device)
        live = torch.ones(n, dtype=torch.bool, device=self.device)
        for step in range(self.max_len):
            x = self._of_vocabulary(self.next_logits(tokens[:, :step].clamp(min=0)))
            r = logits_draw(x, seed=seed, first_id=first, draw=step, temperature=self.temperature, live=live)
            tokens[:, step], ml2p[:, step] = r.tokens, r.ml2p
            live = live & (r.tokens != self.end) & (r.tokens != OUTSIDE)
            if not bool(live.any()):
                break
        keys = logits_keys(ml2p)
        if bool((tokens == OUTSIDE).any()):
            raise RuntimeError("the model left a sample without a next token (logits all -inf, or NaN or +inf among them)")
        return tokens, keys

    def _sampled_strings(self, tokens: torch.Tensor) -> List[str]:
        return ["".join(self.vocabulary[t] for t in row if t >= 0 and t != self.end) for row in tokens.tolist()]

    def sample(self, size: int, sampled_pwds: Dict[str, List] = None, clearIfNotNone: bool = True):
        seed, first = self._claim_ids(size)
        group, n_global = mcd.active_group(), size
        if group is not None:
            lo, size = mcd.shard_range(n_global, torch.distributed.get_rank(group), torch.distributed.get_world_size(group))
            first += lo
        want, parts, distinct = isinstance(sampled_pwds, dict), [], {}
        for at in range(0, size, self.batch):
            tokens, keys = self._sample_batch(min(self.batch, size - at), seed, first + at)
            parts.append(keys)
            if want:
                for pwd, x in zip(self._sampled_strings(tokens), keys.tolist()):
                    distinct.setdefault(pwd, [x, 0])[1] += 1
        if want:
            if group is not None:
                merged, distinct = mcd.merge_distinct([(p, x, c) for p, (x, c) in distinct.items()], group), {}
                for pwd, x, c in merged:
                    distinct.setdefault(pwd, [x, 0])[1] += c
            if clearIfNotNone:
                sampled_pwds.clear()
            sampled_pwds.update(distinct)
        keys = torch.cat(parts) if parts else torch.empty(0, dtype=torch.float64, device=self.device)
        return SampleKeys(keys, group=group, n_global=n_global if group is not None else None)

    def sample1(self) -> Tuple[float, str]:
        seed, first = self._claim_ids(1)
        tokens, keys = self._sample_batch(1, seed, first)
        return float(keys[0]), self._sampled_strings(tokens)[0]

    # ---- scoring (lib4mc/MonteCarloParent.py:17-24, 48-69) ---------------------------------------------------------
    def calc_ml2p(self, pwd: str) -> Tuple[float, List[str]]:
        ml2p, parts = self.score_batch([pwd])
        return ml2p[0], parts[0]

    @torch.no_grad()
    def score_batch(self, pwds: List[str]):
        pwds = list(pwds)
        ml2p: List[float] = []
        parts: List[List[str]] = []
        for at in range(0, len(pwds), self.batch):
            ids = [self.encode(p) for p in pwds[at:at + self.batch]]
            # (a password that is too long, or holds the end or what is no token -- SKIP too, which would count as certain --, is
            # impossible whatever its other tokens are: it stands as one unknown token, and the model is asked nothing else)
            whole = [not r or len(r) <= self.max_len and min(r) >= 0 and max(r) < len(self.vocabulary) and self.end not in r for r in ids]
            rows = [[OUTSIDE] if not w else r + [self.end] if len(r) < self.max_len else r for r, w in zip(ids, whole)]
            width = max(len(r) for r in rows)
            tokens = torch.tensor([r + [SKIP] * (width - len(r)) for r in rows], dtype=torch.int64, device=self.device)
            x = self._of_vocabulary(self.logits(tokens[:, :-1].clamp(min=0)))
            scores = logits_score(x, tokens, temperature=self.temperature)
            keys = logits_keys(scores.ml2p).tolist()
            if any(k != k for k in keys):
                raise RuntimeError("the model's logits hold NaN or +inf")
            ml2p += keys
            parts += [[self.vocabulary[t] for t in r] if k < 1022.0 else [p]
                      for p, r, k in zip(pwds[at:at + self.batch], ids, keys)]
        return ml2p, parts
