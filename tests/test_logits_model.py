"""The plugin of models that answer with logits (montecarlo_amd.logits_simulator) without a GPU: what it hands to the model and
to the operators, which are stood in for by the definitions."""
import math

import numpy as np
import pytest
import torch

from montecarlo_amd import logits_simulator as ls
from montecarlo_amd.logits import LogitScores
from tests.logits_ref import OUTSIDE, SKIP, Row


class Model(ls.LogitsMonteCarlo):
    """Logits by place; keeps what it was asked and what was scored."""

    def __init__(self, texts="ab", seed=1, wide=0, **kw):
        kw.setdefault("max_len", 4)
        super().__init__(list(texts) + ["<end>"], len(texts), device="cpu", **kw)
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randn(self.max_len + 1, len(self.vocabulary) + wide, generator=g)
        self.asked, self.scored = [], []

    def logits(self, tokens):
        self.asked.append(tokens)
        return self.table[:tokens.shape[1] + 1].expand(tokens.shape[0], -1, -1)


@pytest.fixture(autouse=True)
def definitions(monkeypatch):
    def score(x, tokens, temperature=1.0):
        assert x.shape[:-1] == tokens.shape
        rows = [Row(r, temperature).score(t)[0] for r, t in zip(x.reshape(-1, x.shape[-1]).numpy(), tokens.reshape(-1).tolist())]
        return LogitScores(torch.tensor(rows).view(tokens.shape))

    def keys(ml2p):
        s = ml2p.double().sum(-1)
        return torch.where(s == math.inf, 1022.0, s)

    monkeypatch.setattr(ls, "logits_score", score)
    monkeypatch.setattr(ls, "logits_keys", keys)


@pytest.mark.parametrize("bad", [SKIP, -7, 3, 1 << 40])
def test_an_encoding_that_leaves_the_vocabulary_is_impossible(bad):
    class Odd(Model):
        def encode(self, pwd):
            return [bad if c == "?" else i for c, i in zip(pwd, super().encode(pwd))]

    m = Odd()
    ml2p, parts = m.score_batch(["a?b", "?", "ab", "b?", "abab"])
    assert [x == 1022.0 for x in ml2p] == [True, True, False, True, False]
    assert parts[0] == ["a?b"] and parts[2] == ["a", "b"]
    for t in m.asked:                                       # the model sees no id that it does not know
        assert int(t.min()) >= 0 and int(t.max()) < len(m.vocabulary)
    want = sum(Row(m.table[i].numpy(), 1.0).score(t)[0] for i, t in enumerate([0, 1, 2]))
    assert abs(ml2p[2] - want) < 1e-5


def draws(monkeypatch, m):
    """logits_draw stood in for by the first most probable token, and what it was given."""
    seen = []

    def draw(x, seed, first_id, draw, temperature, live):
        seen.append(x.shape)
        from montecarlo_amd.logits import LogitDraws
        return LogitDraws(torch.where(live, x.argmax(-1), SKIP).int(), torch.zeros(x.shape[0]))

    monkeypatch.setattr(ls, "logits_draw", draw)
    return seen


def test_a_model_of_fewer_logits_than_tokens_is_refused_and_padding_is_not_looked_at(monkeypatch):
    m = Model()
    want = m.score_batch(["ab", "a"])
    m.table = m.table[:, :2]
    with pytest.raises(ValueError, match="2 logits for a vocabulary of 3"):
        m.score_batch(["ab"])
    seen = draws(monkeypatch, m)
    with pytest.raises(ValueError, match="2 logits for a vocabulary of 3"):
        m.sample(5)
    wide = Model(wide=5)                                    # (rows padded to a multiple of eight)
    wide.table = torch.cat([Model().table, torch.full((5, 5), 30.0)], 1)
    assert wide.score_batch(["ab", "a"]) == want
    strings = {}
    assert len(wide.sample(5, strings)) == 5 and all(s == (5, 3) for s in seen)
    assert set("".join(strings)) <= set("ab")


def test_a_model_that_answers_nan_is_an_error_when_scoring_too():
    m = Model()
    m.table[1, 0] = math.nan
    with pytest.raises(RuntimeError, match="NaN"):
        m.score_batch(["bb", "ab"])
    with pytest.raises(RuntimeError, match="NaN"):
        m.calc_ml2p("ab")
    m.table[1, 0] = math.inf
    with pytest.raises(RuntimeError, match="NaN"):
        m.score_batch(["bb"])


def test_characters_that_two_tokens_share_are_refused():
    with pytest.raises(ValueError, match="'a'"):
        Model("aba")
    Model(["ab", "ab", "<pad>", "<pad>", "", "", "a"])      # (texts that no character is encoded as)

    class Own(Model):
        def encode(self, pwd):
            return [0 for _ in pwd]

    assert Own("aba").encode("a") == [0]                    # an encoding of one's own may know them apart


@pytest.mark.parametrize("tokens,max_len,batch", [(3, 4, 1 << 16), (97, 32, 1 << 16), (257, 64, 1 << 16), (32768, 32, 2048), (131072, 64, 256), (1 << 20, 1 << 12, 1)])
def test_the_default_batch_knows_the_width_of_the_answer(tokens, max_len, batch):
    """At most 2^31 logits at a time ([batch, places, tokens]), and what was there for models of few tokens."""
    m = Model([chr(0x4E00 + i) if i < 20000 else f"t{i}" for i in range(tokens - 1)], max_len=1)
    assert m.batch == 1 << 16 if tokens * 2 * (1 << 16) <= 1 << 31 else m.batch * tokens <= 1 << 31
    assert ls.default_batch(tokens, max_len) == batch
    assert Model("ab", batch=70000).batch == 70000
