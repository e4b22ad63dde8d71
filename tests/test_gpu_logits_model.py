"""A model that answers with logits behind the plugin surface (montecarlo_amd.logits_simulator)."""
import io
import itertools
import math

import numpy as np
import pytest
import torch

from montecarlo_amd import logits as lg
from montecarlo_amd.lib4mc.MonteCarloLib import MonteCarloLib
from montecarlo_amd.logits_simulator import LogitsMonteCarlo
from oracle.philox import uniform53
from tests.logits_ref import Row, steps_of

pytestmark = pytest.mark.gpu


class Bigram(LogitsMonteCarlo):
    """Logits by the token before; row V is the start's."""

    def __init__(self, letters, seed, **kw):
        super().__init__(list(letters) + ["<end>"], len(letters), **kw)
        g = torch.Generator().manual_seed(seed)
        v = len(self.vocabulary)
        self.table = (torch.randn(v + 1, v, generator=g) * 1.5).to(torch.bfloat16)
        self.table[:, 1] = -math.inf                      # a letter the model never says
        self.table = self.table.to(self.device)

    def logits(self, tokens):
        start = torch.full((tokens.shape[0], 1), len(self.vocabulary), device=tokens.device)
        return self.table[torch.cat([start, tokens], 1)]


def key_of(m, pwd):
    """-log2 p of a password in 64 bits, and how far off the sum of float32 scores may be."""
    rows = [Row(r, m.temperature) for r in m.table.double().cpu().numpy()]
    prev, s, tol = len(m.vocabulary), 0.0, 0.0
    ids = [m.vocabulary.index(c) for c in pwd]
    for t in ids + ([m.end] if len(ids) < m.max_len else []):
        v, d = rows[prev].score(t)
        s, tol, prev = s + v, tol + d, t
    return s, tol + 1e-12


def test_probabilities_of_all_strings_add_up_to_one():
    m = Bigram("abc", 1, max_len=4)
    every = ["".join(p) for n in range(5) for p in itertools.product("abc", repeat=n)]
    ml2p, parts = m.score_batch(every)
    for pwd, x, part in zip(every, ml2p, parts):
        if "b" in pwd:
            assert x == 1022.0 and part == [pwd]
        else:
            want, tol = key_of(m, pwd)
            assert abs(x - want) <= tol and "".join(part) == pwd
    assert abs(sum(2.0 ** -x for x in ml2p) - 1) < 1e-5
    assert m.calc_ml2p("abcab")[0] == 1022.0 and m.calc_ml2p("axe")[0] == 1022.0


def test_a_password_that_holds_the_end_is_impossible():
    class Careless(Bigram):
        def encode(self, pwd):
            return [len(self.vocabulary) - 1 if c == "$" else self.vocabulary.index(c) for c in pwd]

    m = Careless("abc", 1, max_len=4)
    ml2p, parts = m.score_batch(["a$c", "$", "ac", ""])
    assert ml2p[:2] == [1022.0, 1022.0] and parts[:2] == [["a$c"], ["$"]]
    assert ml2p[2] < 1022.0 and ml2p[3] < 1022.0


def test_samples_are_the_streams_and_come_with_their_scores():
    m = Bigram("abcdefg", 2, max_len=9, batch=700, temperature=0.8)
    m.seed(11, first_id=5)
    seen = {}
    keys = m.sample(2000, seen)
    assert len(keys) == 2000 and sum(c for _, c in seen.values()) == 2000
    rows = [Row(r, 0.8) for r in m.table.double().cpu().numpy()]
    got = np.array(keys.tolist())
    for i in range(0, 2000, 37):
        prev, pwd = len(m.vocabulary), ""
        for step in range(9):
            t, margin = rows[prev].draw(uniform53(11, 5 + i, step))
            assert margin > 1e-12
            if t == m.end:
                break
            pwd, prev = pwd + m.vocabulary[t], t
        want, tol = key_of(m, pwd)
        assert abs(got[i] - want) <= tol
        assert pwd in seen
    ml2p, _ = m.score_batch(list(seen))
    for (pwd, (x, _)), y in zip(seen.items(), ml2p):
        assert abs(x - y) <= 2 * key_of(m, pwd)[1]
    m.seed(11, first_id=5)
    again = m.sample(2000)
    assert again.tolist() == got.tolist()
    m.seed(11, first_id=5 + 41)
    x, pwd = m.sample1()
    assert x == got[41] and pwd in seen


def test_the_whole_flow_to_guess_numbers():
    m = Bigram("abcdefgh", 3, max_len=6)
    m.seed(4)
    keys = m.sample(50000)
    raw = np.sort(np.array(keys.tolist()))
    mc = MonteCarloLib(keys)
    lines = ["ab", "acdc", "ah", "ah", "", "zz", "ccccccc", "dead"]
    scored = m.parse_file(io.StringIO("\n".join(lines) + "\n"))
    assert sorted((p, c) for p, c, _ in scored) == sorted((p, lines.count(p)) for p in set(lines))
    pos = np.cumsum(2.0 ** (raw - math.log2(len(raw))))
    prev = 0
    for (pwd, rank_x, _, rank, _, _), (p, _, x) in zip(mc.ml2p_iter2gc(scored), scored):
        i = int(np.searchsorted(raw, x, side="right"))
        want = math.ceil(max(pos[i - 1] if i else 1, prev + 1))
        assert pwd == p and abs(rank - want) <= 1e-9 * want + 1
        prev = rank


def test_the_model_is_asked_without_gradients():
    asked = []

    class Trained(Bigram):
        def logits(self, tokens):
            asked.append(torch.is_grad_enabled())
            return super().logits(tokens)

    m = Trained("abc", 2, max_len=3)
    m.table.requires_grad_()
    want = Bigram("abc", 2, max_len=3).score_batch(["ac", "a"])
    assert m.score_batch(["ac", "a"]) == want and len(m.sample(5)) == 5
    assert asked and not any(asked) and torch.is_grad_enabled()


def test_a_model_that_leaves_nothing_is_an_error():
    m = Bigram("ab", 1)
    m.table[:] = -math.inf
    with pytest.raises(RuntimeError, match="next token"):
        m.sample(10)
    with pytest.raises(ValueError):
        Bigram("ab", 1, max_len=0)
    assert len(Bigram("ab", 1).sample(0)) == 0


def test_a_model_learns_its_corpus():
    """The gradient in a training loop of a table of logits: the analytic optimum (relative frequencies) is a fixed point."""
    m = Bigram("abcd", 5, max_len=5)
    pwds = ["ac", "acd", "ad", "da", "c", "acdc"] * 3
    v = len(m.vocabulary)
    rows = [[m.vocabulary.index(c) for c in p] + [m.end] for p in pwds]
    tokens = torch.tensor([r + [lg.SKIP] * (5 - len(r)) for r in rows]).cuda()
    prev = torch.cat([torch.full((len(rows), 1), v).cuda(), tokens[:, :-1].clamp(min=0)], 1)
    count = torch.zeros(v + 1, v, dtype=torch.float64)
    for a, b in zip(prev.cpu().view(-1).tolist(), tokens.cpu().view(-1).tolist()):
        if b >= 0:
            count[a, b] += 1
    table = torch.log(count).float().cuda().requires_grad_()          # p = relative frequency; never seen: -inf
    x = table[prev]
    w = torch.full(tokens.shape, math.log(2) / int((tokens >= 0).sum()), device="cuda")
    x.backward(lg.logits_gradient(x, tokens, w).grad)
    # sums of at most 18 gradients, each off by its bound (p and the roundings of p - 1)
    assert table.grad.abs().max().item() <= 18 * 2.0 ** -24 * (steps_of(v) + 8) / int((tokens >= 0).sum())


def test_passwords_that_are_certain_keep_their_place():
    """A sharpened model whose commonest password is certain up to a rounding at every place: keys are 0 or above, and guess numbers of
    all passwords are those of 64 bits on the same keys."""
    m = Bigram("abcdef", 7, max_len=8, temperature=0.02)
    m.table[:] = -9.0
    v = len(m.vocabulary)
    g = torch.Generator().manual_seed(1)
    m.table[:, :] += torch.rand(v + 1, v, generator=g).to(m.table)
    for a, b in ((v, 0), (0, 2), (2, 3), (3, 4), (4, m.end)):         # "acde", each step far above the others
        m.table[a, b] = 5.0 + 0.37 * a
    m.seed(2)
    keys = m.sample(5000)
    raw = np.array(keys.tolist())
    assert raw.min() >= 0 and not np.signbit(raw).any() and (raw < 1e-5).all()
    assert m.sample1()[1] == "acde" and 0 <= m.calc_ml2p("acde")[0] < 1e-5
    # certain ones among others (continuations that were forced): the index of all of them in order
    other = Bigram("abcdef", 8, max_len=8)
    other.seed(3)
    mixed = torch.cat([keys.tensor, other.sample(3000).tensor])[torch.randperm(8000, generator=g).to(m.device)]
    srt = np.sort(mixed.cpu().numpy())
    pos = np.cumsum(2.0 ** (srt - math.log2(8000)))
    mc = MonteCarloLib(mixed.clone())
    for x in [0.0, 1e-7, float(srt[2500]), float(srt[4999]), 0.5, float(srt[6000]), float(srt[7999])]:
        i = int(np.searchsorted(srt, x, side="right"))
        assert abs(mc.ml2p2rank(x) - (pos[i - 1] if i else 1)) <= 1e-9 * pos[-1], x
