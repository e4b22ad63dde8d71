"""The operators on logits (montecarlo_amd.logits) against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from montecarlo_amd import logits as lg
from montecarlo_amd.lib4mc.MonteCarloLib import MonteCarloLib
from oracle.philox import uniform53
from tests.logits_ref import OUTSIDE, SKIP, Row, steps_of

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
VOCABS = [1, 2, 3, 7, 8, 9, 15, 31, 64, 97, 128, 200, 255, 257, 509, 512, 1000, 1025, 2048, 3001, 4099, 8192, 16385, 50001]


def make(rows, vocab, dtype, seed, scale=2.5):
    """Logits with a few tokens switched off and, as far as there are rows, one of every awkward kind."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    x[:, torch.rand(vocab, generator=g) < 0.03] = -math.inf
    low = torch.finfo(dtype).min
    kinds = [lambda r: r.fill_(-math.inf), lambda r: r.fill_(low), lambda r: r.fill_(0.25),
             lambda r: r.copy_(torch.where(torch.arange(vocab) % 3 == 0, low, -math.inf)),
             lambda r: r.copy_(torch.arange(vocab) / 64.0), lambda r: r.copy_(-torch.arange(vocab) / 64.0),
             lambda r: r.fill_(-math.inf)[vocab // 2:vocab // 2 + 1].fill_(3.0),
             lambda r: r[vocab - 1:].fill_(math.nan), lambda r: r[vocab // 3:vocab // 3 + 1].fill_(math.inf),
             lambda r: r.copy_(torch.round(r)), lambda r: r.copy_(torch.where(r > 0, 0.0, -0.0)),
             lambda r: r[::2].fill_(low)]
    for i, kind in enumerate(kinds):
        if 2 * i + 1 < rows:
            kind(x[2 * i + 1])
    return x.to(dtype)


def tokens_for(x, seed):
    g = torch.Generator().manual_seed(seed)
    rows, vocab = x.shape
    t = torch.randint(0, vocab, (rows,), generator=g)
    pick = torch.arange(rows) % 5
    best = x.float().nan_to_num(nan=-1e9, posinf=-1e9, neginf=-1e9).argmax(-1)
    t = torch.where(pick == 1, best, t)
    t[pick == 4] = torch.tensor([OUTSIDE, SKIP, vocab, -77])[torch.randint(0, 4, (int((pick == 4).sum()),), generator=g)]
    return t


def near(got, want, tol, what):
    if math.isfinite(want):
        assert abs(got - want) <= tol, (what, got, want, tol)
    else:
        assert got == want or (math.isnan(got) and math.isnan(want)), (what, got, want)


def check_score(x, toks, r, temperature, top):
    xs = x.double().cpu().numpy().reshape(-1, x.shape[-1])
    ts = toks.cpu().numpy().reshape(-1)
    ml2p, ent = r.ml2p.cpu().numpy().reshape(-1), r.entropy.cpu().numpy().reshape(-1)
    ids = r.top_tokens.cpu().numpy().reshape(-1, top) if top else None
    vals = r.top_ml2p.cpu().numpy().reshape(-1, top) if top else None
    for i in range(len(xs)):
        ref = Row(xs[i], temperature)
        near(ml2p[i], *ref.score(ts[i]), ("ml2p", i))
        near(ent[i], *ref.h(ts[i]), ("entropy", i))
        if top:
            want_ids, want = ([SKIP] * top, [0.0] * top) if ts[i] == SKIP else ref.top(top)
            assert ids[i].tolist() == want_ids, i
            for k in range(top):
                tol = ref.score(want_ids[k])[1] if want_ids[k] >= 0 else 0.0
                near(vals[i][k], want[k], tol, ("top", i, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_score(vocab, dtype):
    rows = 29 if vocab < 5000 else 25
    x = make(rows, vocab, DTYPES[dtype], vocab)
    toks = tokens_for(x, vocab + 1)
    t = [1.0, 0.6, 1.9][vocab % 3]
    top = min(vocab, [5, 1, 64, 20][vocab % 4])
    check_score(x, toks, lg.logits_score(x.cuda(), toks.cuda(), temperature=t, entropy=True, top=top), t, top)
    plain = lg.logits_score(x.cuda(), toks.int().cuda(), temperature=t)
    assert plain.entropy is None and plain.top_tokens is None
    for i in range(rows):
        near(plain.ml2p[i].item(), *Row(x[i].double().numpy(), t).score(toks[i].item()), i)


@pytest.mark.parametrize("vocab,dtype", [(200003, "bf16"), (170001, "fp32"), (300000, "fp16")])
def test_score_of_few_very_wide_rows(vocab, dtype):
    x = make(25, vocab, DTYPES[dtype], vocab)
    toks = tokens_for(x, 5)
    check_score(x, toks, lg.logits_score(x.cuda(), toks.cuda(), temperature=0.9, entropy=True, top=33), 0.9, 33)
    base = torch.empty(25, vocab + 1, dtype=x.dtype).cuda()
    base[:, 1:] = x.cuda()
    check_score(x, toks, lg.logits_score(base[:, 1:], toks.cuda(), entropy=True, top=2), 1.0, 2)


@pytest.mark.parametrize("vocab,rows", [(97, 5000), (64, 1023), (700, 777), (5000, 300), (40000, 3)])
def test_score_many_rows_agree_with_the_same_rows_alone(vocab, rows):
    """Whatever way a launch takes with many rows and with few, each row's alternatives are the same and its score is within
    the bound of the definition."""
    x = make(rows, vocab, torch.bfloat16, 5)
    toks = tokens_for(x, 6)
    xd, td = x.cuda(), toks.cuda()
    many = lg.logits_score(xd, td, entropy=True, top=7)
    for i in list(range(0, rows, max(1, rows // 40))) + [rows - 1]:
        one = lg.logits_score(xd[i], td[i], entropy=True, top=7)
        assert torch.equal(one.top_tokens, many.top_tokens[i])
        ref = Row(x[i].double().numpy(), 1.0)
        for r, j in ((many.ml2p[i], one.ml2p),):
            near(r.item(), *ref.score(toks[i].item()), i)
            near(j.item(), *ref.score(toks[i].item()), i)
        near(many.entropy[i].item(), *ref.h(toks[i].item()), i)
        near(one.entropy.item(), *ref.h(toks[i].item()), i)


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "sawtooth", "two_values", "few_left", "one_left", "spikes"])
@pytest.mark.parametrize("vocab,dtype", [(1000, "fp32"), (20000, "bf16"), (131073, "fp32"), (70000, "fp16"), (170001, "bf16")])
def test_top_in_orders_that_are_hard(kind, vocab, dtype):
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"ascending": i * (30.0 / vocab), "descending": -i * (30.0 / vocab), "equal": torch.zeros(vocab), "sawtooth": (i % 1024) / 64,
         "two_values": (i % 7 == 3).float(), "few_left": torch.where(i % (vocab // 10) == 5, i / vocab, torch.tensor(-math.inf)),
         "one_left": torch.where(i == vocab - 1, 1.0, torch.tensor(-math.inf)), "spikes": torch.where(i % 2048 == 0, 5.0, 0.0)}[kind]
    x = x.to(DTYPES[dtype])
    toks = torch.tensor([vocab // 2, 0, SKIP])
    for rows in (1, 3):
        xs = x.expand(rows, vocab)
        r = lg.logits_score(x.cuda().expand(rows, vocab), toks[:rows].cuda(), entropy=True, top=40)
        check_score(xs, toks[:rows], r, 1.0, 40)


@pytest.mark.parametrize("bits", [0x7FFFFFFF, 0x7F800001, -1])
@pytest.mark.parametrize("vocab,rows", [(200000, 3), (200000, 1030), (40000, 4), (4000, 9)])
def test_alternatives_beside_nan_of_any_bits(vocab, rows, bits):
    """Equal logits and, where one thread has them, more NaNs than alternatives: no row's selection may count these."""
    x = torch.ones(rows, vocab, device="cuda")
    for u in range(16):                                     # vectors that lie 256 lanes apart
        x[0, u * 1024:u * 1024 + 4].view(torch.int32).fill_(bits) if u * 1024 + 4 <= vocab else None
    x[1].view(torch.int32).fill_(bits)
    x[2, vocab - 1:].view(torch.int32).fill_(bits)
    toks = torch.arange(rows)
    r = lg.logits_score(x, toks.cuda(), entropy=True, top=min(64, vocab))
    check_score(x[:4].cpu(), toks[:4], lg.LogitScores(*(t[:4] for t in r)), 1.0, 64)


def test_score_takes_any_strides():
    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 5, 40, generator=g).to(torch.float16).cuda()
    toks = torch.randint(0, 33, (6, 5), generator=g).cuda()
    for x, t in ((base[:, :-1, :33], toks[:, 1:]), (base[::2, 1:, 3:36], toks[::2, :-1]), (base[:, :, 7:40].transpose(0, 1), toks.t()),
                 (base[:, :1, 1:34].expand(6, 4, 33), toks[:, :4]), (base[2:3, :, :33], toks[2:3]), (base[:, 2, 5:38], toks[:, 2])):
        r = lg.logits_score(x, t, entropy=True, top=4)
        assert r.ml2p.shape == x.shape[:-1] and r.top_tokens.shape == (*x.shape[:-1], 4)
        check_score(x.contiguous(), t.contiguous(), r, 1.0, 4)


@pytest.mark.parametrize("temperature", [1e-30, 1e-5, 0.01, 300.0, 1e30])
@pytest.mark.parametrize("vocab", [33, 700, 9001])
def test_temperatures_far_from_one(vocab, temperature):
    x = make(25, vocab, torch.float32, vocab + 9)
    toks = tokens_for(x, 2)
    g = torch.Generator().manual_seed(vocab)
    u, w, v = torch.rand(25, generator=g, dtype=torch.float64), torch.rand(25, generator=g), torch.rand(25, generator=g)
    check_score(x, toks, lg.logits_score(x.cuda(), toks.cuda(), temperature=temperature, entropy=True, top=3), temperature, 3)
    check_draw(x, u, None, lg.logits_draw(x.cuda(), u.cuda(), temperature=temperature), temperature)
    check_gradient(x, toks, w, v, lg.logits_gradient(x.cuda(), toks.cuda(), w.cuda(), entropy_weights=v.cuda(), temperature=temperature),
                   temperature, "fp32")


@pytest.mark.parametrize("vocab,rows,dtype,top", [(97, 20000, "bf16", 64), (200, 40000, "fp32", 33), (4096, 900, "fp16", 64), (3001, 3000, "bf16", 64),
                                                  (262144, 1100, "fp32", 64)])
def test_many_alternatives_of_many_rows(vocab, rows, dtype, top):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5).to(DTYPES[dtype])
    some = list(range(26)) + [rows // 2, rows - 1]
    x[:26] = make(26, vocab, DTYPES[dtype], vocab).cuda()
    toks = torch.zeros(rows, dtype=torch.int64)
    r = lg.logits_score(x, toks.cuda(), entropy=True, top=top)
    check_score(x[some].cpu(), toks[some], lg.LogitScores(*(t[some] for t in r)), 1.0, top)


def test_more_rows_than_a_grid_is_wide():
    rows = (1 << 26) + 77                                   # 64 of them a workgroup, 2^20 workgroups a line of the grid
    x = torch.zeros(rows, 3, dtype=torch.bfloat16, device="cuda")
    x[-40:] = make(40, 3, torch.bfloat16, 1).cuda()
    toks = torch.zeros(rows, dtype=torch.int32, device="cuda")
    r = lg.logits_score(x, toks)
    check_score(x[-40:].cpu(), toks[-40:].cpu(), lg.logits_score(x[-40:], toks[-40:], entropy=True), 1.0, 0)
    assert torch.equal(r.ml2p[-40:].view(torch.int32), lg.logits_score(x[-40:], toks[-40:]).ml2p.view(torch.int32))
    assert bool((r.ml2p[:-40] == r.ml2p[0]).all()) and abs(r.ml2p[0].item() - math.log2(3)) < 1e-6
    del x, r
    rows = (1 << 20) + 5                                    # one a workgroup
    x = torch.zeros(rows, 2052, dtype=torch.float32, device="cuda")
    x[-1, 7] = 20.0
    d = lg.logits_draw(x, torch.full((rows,), 0.5, dtype=torch.float64, device="cuda"))
    assert d.tokens[-1].item() == 7 and bool((d.tokens[:-1] == 1026).all())
    s = lg.logits_score(x, torch.full((rows,), 7, device="cuda"), top=1)
    assert s.top_tokens[-1].item() == 7 and bool((s.top_tokens[:-1] == 0).all())


def test_rows_beyond_32_bits_of_offset():
    base = torch.empty(2_200_000_400, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, 2, 100), (2_200_000_100, 150, 1))
    x.copy_(make(4, 100, torch.bfloat16, 8).view(2, 2, 100))
    toks = torch.tensor([[3, 4], [5, 6]]).cuda()
    check_score(x.contiguous(), toks, lg.logits_score(x, toks, entropy=True, top=3), 1.0, 3)
    w = torch.ones(2, 2).cuda()
    assert torch.equal(lg.logits_gradient(x, toks, w).grad.isnan().any(-1), lg.logits_gradient(x.contiguous(), toks, w).grad.isnan().any(-1))
    assert torch.equal(lg.logits_gradient(x, toks, w).grad.nan_to_num(), lg.logits_gradient(x.contiguous(), toks, w).grad.nan_to_num())
    rows = base.as_strided((2, 100), (2_200_000_100, 1))
    u = torch.tensor([0.3, 0.9], dtype=torch.float64).cuda()
    assert torch.equal(lg.logits_draw(rows, u).tokens, lg.logits_draw(rows.contiguous(), u).tokens)


# ---- gradient ------------------------------------------------------------------------------------------------------
HALF = {"fp32": (2.0 ** -24, 0.0), "fp16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}


def check_gradient(x, toks, w, v, r, temperature, dtype):
    eps, least = HALF[dtype]
    vocab = x.shape[-1]
    xs, ts, ws = x.double().cpu().numpy().reshape(-1, vocab), toks.cpu().numpy().reshape(-1), w.double().cpu().numpy().reshape(-1)
    vs = v.double().cpu().numpy().reshape(-1) if v is not None else np.zeros(len(ts))
    got, ml2p = r.grad.double().cpu().numpy().reshape(-1, vocab), r.ml2p.cpu().numpy().reshape(-1)
    for i in range(len(ts)):
        ref = Row(xs[i], temperature)
        near(ml2p[i], *ref.score(ts[i]), ("ml2p", i))
        if v is not None:
            near(r.entropy.reshape(-1)[i].item(), *ref.h(ts[i]), ("entropy", i))
        want, tol = ref.grad(ts[i], ws[i], vs[i], eps, least)
        if ref.bad and ts[i] != SKIP:
            assert np.isnan(got[i]).all(), i
        else:
            off = np.abs(got[i] - want) - tol
            assert off.max() <= 0, (i, int(off.argmax()), got[i][off.argmax()], want[off.argmax()], tol[off.argmax()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_gradient(vocab, dtype):
    rows = 27
    x = make(rows, vocab, DTYPES[dtype], vocab + 7)
    toks = tokens_for(x, vocab + 2)
    g = torch.Generator().manual_seed(vocab)
    w, v = torch.rand(rows, generator=g) + 0.1, torch.rand(rows, generator=g) - 0.5
    t = [1.0, 1.7, 0.5][vocab % 3]
    xd, td = x.cuda(), toks.cuda()
    r = lg.logits_gradient(xd, td, w.cuda(), temperature=t)
    assert r.entropy is None and r.grad.shape == x.shape and r.grad.dtype == x.dtype
    check_gradient(x, toks, w, None, r, t, dtype)
    r = lg.logits_gradient(xd, td.int(), w.cuda(), entropy_weights=v.cuda(), temperature=t)
    check_gradient(x, toks, w, v, r, t, dtype)
    mine = xd.clone()
    same = lg.logits_gradient(mine, td, w.cuda(), entropy_weights=v.cuda(), temperature=t, out=mine)
    assert same.grad is mine
    assert torch.equal(mine.nan_to_num(nan=7.0), r.grad.nan_to_num(nan=7.0))


@pytest.mark.parametrize("vocab,rows", [(97, 2050), (600, 500), (9000, 260), (70001, 2), (131072, 3), (200003, 5)])
def test_gradient_of_a_sequence(vocab, rows):
    length = 5
    x = make(rows * length, vocab, torch.bfloat16, 4).view(rows, length, vocab)
    toks = tokens_for(x.view(-1, vocab), 9).view(rows, length)
    w = torch.rand(rows, 1).expand(rows, length)            # one weight a password, broadcast over its tokens
    v = torch.rand(rows, length)
    r = lg.logits_gradient(x.cuda()[:, :-1], toks.cuda()[:, 1:], w.cuda()[:, 1:], entropy_weights=v.cuda()[:, 1:])
    pick = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:6]
    sub = lg.LogitGradient(r.ml2p[pick], r.entropy[pick], r.grad[pick])
    check_gradient(x[pick][:, :-1], toks[pick][:, 1:], w[pick][:, 1:], v[pick][:, 1:], sub, 1.0, "bf16")


def test_gradient_is_the_difference_of_the_scores():
    """The scores themselves, a step up and a step down: with h = 1/16 the central difference is off by at most h^2 / 6 of the third
    derivative (below 1/ln 2 / 4 in bits) and by two scores' errors over 2 h."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(1, 33, generator=g).cuda()
    toks = torch.tensor([4]).cuda()
    grad = lg.logits_gradient(x, toks, torch.ones(1).cuda()).grad[0]
    h = 1 / 16
    step = torch.eye(33).cuda() * h
    up = lg.logits_score(x + step, toks.expand(33)).ml2p
    down = lg.logits_score(x - step, toks.expand(33)).ml2p
    tol = h * h / 6 / math.log(2) / 4 + 2 * Row(x[0].double().cpu().numpy(), 1.0).score(4)[1] * 2 / (2 * h)
    assert ((up - down) / (2 * h) - grad).abs().max().item() <= tol


def test_gradient_in_a_training_step():
    """logits.backward(grad) is the gradient of the loss for what the logits were made of (float64 differences of the loss)."""
    g = torch.Generator().manual_seed(2)
    hid, emb = torch.randn(12, 8, generator=g).cuda(), torch.randn(8, 40, generator=g).cuda().requires_grad_()
    toks = torch.randint(0, 40, (12,), generator=g).cuda()
    x = hid @ emb
    w = torch.full((12,), math.log(2) / 12, device="cuda")
    x.backward(lg.logits_gradient(x, toks, w).grad)
    ref = emb.detach().double().requires_grad_()
    torch.nn.functional.cross_entropy(hid.double() @ ref, toks).backward()
    # (a product of 12 terms with logits and gradients of 32 bits)
    assert (emb.grad.double() - ref.grad).abs().max().item() < 64 * 2.0 ** -24 * hid.abs().max().item()


# ---- draw ----------------------------------------------------------------------------------------------------------
def check_draw(x, u, live, r, temperature):
    xs = x.double().cpu().numpy()
    toks, ml2p = r.tokens.cpu().numpy().reshape(-1), r.ml2p.cpu().numpy().reshape(-1)
    close = 0
    for i in range(len(xs)):
        if live is not None and not live[i]:
            assert toks[i] == SKIP and ml2p[i] == 0.0
            continue
        ref = Row(xs[i], temperature)
        want, margin = ref.draw(float(u[i]))
        if margin < 1e-11:                           # (64 bits themselves cannot tell here)
            close += 1
            want = int(toks[i])
        assert toks[i] == want, (i, toks[i], want, margin)
        if want == OUTSIDE:
            assert math.isnan(ml2p[i]) if ref.bad else ml2p[i] == math.inf
        else:
            near(ml2p[i], *ref.score(want), ("ml2p", i))
    return close


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_draw(vocab, dtype):
    rows = 61
    x = make(rows, vocab, DTYPES[dtype], vocab + 3)
    g = torch.Generator().manual_seed(vocab)
    u = torch.rand(rows, generator=g, dtype=torch.float64)
    live = torch.rand(rows, generator=g) < 0.8
    t = [1.0, 0.7, 2.2][vocab % 3]
    check_draw(x, u, None, lg.logits_draw(x.cuda(), u.cuda(), temperature=t), t)
    check_draw(x, u, live, lg.logits_draw(x.cuda(), u.cuda(), temperature=t, live=live.cuda()), t)


@pytest.mark.parametrize("vocab", [3, 97, 513, 5000, 70000])
def test_draw_at_and_beside_the_borders(vocab):
    """Uniforms a few parts in 10^7 and 10^10 beside the running sums, where 32 bits cannot tell and 64 do, and those at 0 and near 1."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(vocab, generator=g) * 2).to(torch.float16)
    c = np.cumsum(np.exp(x.double().numpy() - x.double().max().item()))
    c /= c[-1]
    at = c[np.unique(np.linspace(0, vocab - 1, 24).astype(int))]
    us = np.concatenate([at + s * d for s in (-1, 1) for d in (1e-10, 3e-8, 1e-6)] + [[0.0, 1e-300, 1 - 2.0 ** -53, 0.5]])
    us = np.clip(us, 0, 1 - 2.0 ** -53)
    u = torch.from_numpy(us)
    xs = x.cuda().expand(len(us), vocab)
    close = check_draw(x.expand(len(us), vocab), u, None, lg.logits_draw(xs, u.cuda()), 1.0)
    assert close <= 8, close


@pytest.mark.parametrize("rows", [600, 40])
@pytest.mark.parametrize("vocab,dtype", [(2305, "fp32"), (4099, "fp16"), (20001, "bf16"), (50001, "fp16"), (66001, "bf16"), (33001, "fp32"),
                                         (140001, "fp16")])
def test_draw_beside_the_borders_of_many_rows(vocab, dtype, rows):
    """As above for every way that rows of many tokens are drawn, down to where 64 bits leave it to the definition: numpy's running
    sums are right to 1e-12 here (vocab roundings of 2^-53), a tenth of the least distance."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(vocab, generator=g) * 2).to(DTYPES[dtype])
    x[torch.rand(vocab, generator=g) < 0.05] = -math.inf
    x[0] = 1.0
    w = np.exp(x.double().numpy() - x.double().max().item())
    c = np.cumsum(w)
    c /= c[-1]
    at = np.unique(np.concatenate([[0], np.linspace(0, vocab - 1, rows // 8 + 1).astype(int)]))
    at = at[w[at] > 1e-6][:rows // 8]
    us = np.concatenate([c[at] + s * d for s in (-1, 1) for d in (1.5e-11, 8e-11, 2e-8, 1e-6)])
    us = np.clip(np.concatenate([us, np.linspace(0, 1, rows, endpoint=False)])[:rows], 0, 1 - 2.0 ** -53)
    r = lg.logits_draw(x.cuda().expand(rows, vocab), torch.from_numpy(us).cuda())
    want = np.searchsorted(c, us, side="right")
    assert r.tokens.tolist() == want.tolist()
    ml2p = -np.log2(w[want] / w.sum())
    assert np.all(np.abs(r.ml2p.cpu().numpy() - ml2p) <= 2.0 ** -24 * (steps_of(vocab) + np.abs(ml2p)))


@pytest.mark.parametrize("vocab,dtype", [(4099, "fp16"), (20001, "bf16"), (66001, "bf16"), (140001, "fp32")])
def test_draw_of_many_rows_outside_zero_to_one(vocab, dtype):
    x = torch.full((600, vocab), 2.0, dtype=DTYPES[dtype], device="cuda")
    x[:, 0] = -math.inf
    x[:, vocab - 700:] = -math.inf
    u = torch.tensor([-1.0, math.nan, 1.0, 5.0, math.inf, 1 - 2.0 ** -53] * 100, dtype=torch.float64)
    last = vocab - 701
    assert lg.logits_draw(x, u.cuda()).tokens.tolist() == [1, 1, last, last, last, last] * 100


@pytest.mark.parametrize("vocab", [5, 97, 3000, 60000])
def test_draw_outside_zero_to_one(vocab):
    x = torch.zeros(5, vocab)
    x[:, 0] = x[:, vocab - 1] = -math.inf
    u = torch.tensor([-1.0, math.nan, 1.0, 5.0, math.inf], dtype=torch.float64)
    assert lg.logits_draw(x.cuda(), u.cuda()).tokens.tolist() == [1, 1, vocab - 2, vocab - 2, vocab - 2]


@pytest.mark.parametrize("vocab", [41, 2000, 33000])
def test_draw_takes_the_stream_of_the_samplers(vocab):
    x = make(40, vocab, torch.float32, 2)
    for draw in (0, 1, 6, 7):
        u = [uniform53(77, (1 << 32) - 5 + i, draw) for i in range(40)]
        r = lg.logits_draw(x.cuda(), seed=77, first_id=(1 << 32) - 5, draw=draw)
        assert torch.equal(r.tokens, lg.logits_draw(x.cuda(), torch.tensor(u, dtype=torch.float64).cuda()).tokens)
        check_draw(x, u, None, r, 1.0)


def test_draw_frequencies():
    x = torch.tensor([0.0, math.log(2), -math.inf, math.log(5)]).cuda().expand(80000, 4)
    n = torch.bincount(lg.logits_draw(x, seed=5).tokens.long(), minlength=4).double() / 80000
    assert (n.cpu() - torch.tensor([1 / 8, 2 / 8, 0, 5 / 8])).abs().max() < 5 * math.sqrt(0.25 / 80000)


@pytest.mark.parametrize("rows", [700, 40])
@pytest.mark.parametrize("vocab,dtype,temperature", [(5, "fp32", 1.0), (97, "bf16", 1.0), (97, "fp32", 1e-4), (600, "fp16", 0.7), (4099, "fp16", 1.0), (20001, "bf16", 1.0),
                                                     (20001, "fp32", 1e-4), (66001, "bf16", 1.0), (33001, "fp32", 1.0), (140001, "fp16", 1.0), (140001, "fp32", 1e-3)])
def test_a_drawn_token_comes_with_one_value_whatever_its_uniform(vocab, dtype, rows, temperature):
    """The -log2 p of a token is that of the row, not that of the way its uniform was decided on (32 bits, 64, the definition): equal
    samples have equal keys."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(vocab, generator=g) * 2).to(DTYPES[dtype])
    x[::max(2, vocab // 9)] = x.max() + 3                   # ten tokens that hold half of the row or more
    c = np.cumsum(np.exp((x.double().numpy() - x.double().max().item()) / temperature))
    c /= c[-1]
    top = np.nonzero(np.diff(c, prepend=0.0) > 0.02)[0][:6]
    assert len(top) >= 2
    us = np.concatenate([[c[at] - d for d in (1.5e-11, 8e-11, 2e-8, 3e-7, 1e-4, 1e-3)] for at in top])
    us = np.clip(np.concatenate([us, np.linspace(0, 1, rows, endpoint=False)])[:rows], 0, 1 - 2.0 ** -53)
    d = lg.logits_draw(x.cuda().expand(rows, vocab), torch.from_numpy(us).cuda(), temperature=temperature)
    toks, bits = d.tokens.cpu().numpy(), d.ml2p.cpu().numpy().view(np.int32)
    for t in top:
        mine = bits[toks == t]
        assert len(mine) >= 6 and len(set(mine.tolist())) == 1, (t, len(mine), sorted(set(d.ml2p.cpu().numpy()[toks == t].tolist())))


# ---- keys ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("batch,length", [(1, 0), (1, 1), (3, 5), (257, 24), (1000, 1), (65, 300), (70001, 9), (2, 40000)])
def test_keys(batch, length):
    g = torch.Generator().manual_seed(batch)
    m = torch.empty(batch, length).exponential_(0.3, generator=g)
    if length > 2:
        m[::7, 1] = math.inf
    lengths = torch.randint(-1, length + 2, (batch,), generator=g)
    n = lengths.clamp(0, length)
    rows = m.double().numpy()
    want = [math.fsum(r[:k]) if np.isfinite(r[:k]).all() else 1022.0 for r, k in zip(rows, n.tolist())]

    def same(got, want):
        got = got.cpu().numpy()
        assert got.dtype == np.float64 and len(got) == len(want)
        # at most `length` additions of positive numbers, each off by half a step of 64 bits
        assert np.all(np.abs(got - want) <= np.maximum(length, 1) * 2.0 ** -53 * np.array(want))

    md = m.cuda()
    same(lg.logits_keys(md, lengths.cuda()), want)
    same(lg.logits_keys(md, lengths.int().cuda()), want)
    wide = torch.empty(batch, length + 3).cuda()
    wide[:, 1:length + 1] = md
    same(lg.logits_keys(wide[:, 1:length + 1], lengths.cuda()), want)
    if length:
        same(lg.logits_keys(md.t().contiguous().t(), lengths.cuda()), want)
    same(lg.logits_keys(md), [math.fsum(r) if np.isfinite(r).all() else 1022.0 for r in rows])
    packed = torch.cat([m[i, :k] for i, k in enumerate(n.tolist())]) if batch < 2000 else m[torch.arange(length)[None] < n[:, None]]
    off = torch.zeros(batch + 1, dtype=torch.int64)
    off[1:] = n.cumsum(0)
    same(lg.logits_keys(packed.cuda(), offsets=off.cuda()), want)


def test_keys_of_bad_offsets_and_nan():
    m = torch.tensor([1.0, 2.0, 4.0, math.nan]).cuda()
    off = torch.tensor([0, 2, 1, 3, 99, -5, 0, 0, 4]).cuda()
    got = lg.logits_keys(m, offsets=off).tolist()
    assert got[:2] == [3.0, 0.0] and got[2] == 6.0 and got[3:7] == [0.0, 0.0, 0.0, 0.0] and math.isnan(got[7])
    assert lg.logits_keys(torch.empty(0).cuda(), offsets=torch.zeros(4, dtype=torch.int64).cuda()).tolist() == [0.0] * 3


# ---- many rows of many tokens: a launch that gives each row a workgroup (or several, one batch of rows after another) ---
@pytest.mark.parametrize("vocab,rows,dtype", [(2305, 1500, "fp32"), (5003, 1100, "bf16"), (20001, 1100, "fp16"), (33001, 1030, "fp32"),
                                              (40001, 1030, "bf16"), (66001, 1030, "fp32"), (100003, 600, "bf16"), (131071, 300, "fp16"),
                                              (140001, 500, "bf16")])
def test_many_wide_rows(vocab, rows, dtype):
    dt = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5).to(dt)
    some = list(range(26)) + [rows // 2, rows - 2, rows - 1]
    x[:26] = make(26, vocab, dt, vocab).cuda()
    cg = torch.Generator().manual_seed(vocab)
    toks = torch.randint(0, vocab, (rows,), generator=cg)
    toks[:26] = tokens_for(x[:26].cpu(), 3)
    w, v = torch.rand(rows, generator=cg), torch.rand(rows, generator=cg) - 0.5
    u = torch.rand(rows, generator=cg, dtype=torch.float64)
    r = lg.logits_score(x, toks.cuda(), entropy=True, top=6)
    sub = lg.LogitScores(*(t[some] for t in r))
    check_score(x[some].cpu(), toks[some], sub, 1.0, 6)
    d = lg.logits_draw(x, u.cuda(), temperature=0.9)
    check_draw(x[some].cpu(), u[some], None, lg.LogitDraws(d.tokens[some], d.ml2p[some]), 0.9)
    # every row, against each other: the drawn token's score, and gradients that sum to 0 (their roundings apart)
    again = lg.logits_score(x, d.tokens, temperature=0.9).ml2p
    fine = torch.isfinite(again)
    assert (again - d.ml2p)[fine].abs().max().item() <= 2.0 ** -24 * (4 * steps_of(vocab) + 400)
    for kw in ({}, {"entropy_weights": v.cuda()}):
        gr = lg.logits_gradient(x, toks.cuda(), w.cuda(), **kw)
        sub = lg.LogitGradient(gr.ml2p[some], gr.entropy[some] if kw else None, gr.grad[some])
        check_gradient(x[some].cpu(), toks[some], w[some], v[some] if kw else None, sub, 1.0, dtype)
        mine = x.clone()
        lg.logits_gradient(mine, toks.cuda(), w.cuda(), out=mine, **kw)
        assert torch.equal(mine.nan_to_num(nan=7.0), gr.grad.nan_to_num(nan=7.0))
        # rows that begin at an odd element, in and out of step with their gradient
        base = torch.empty(rows, vocab + 1, dtype=dt, device="cuda")
        base[:, 1:] = x
        odd = lg.logits_gradient(base[:, 1:], toks.cuda(), w.cuda(), **kw)
        for a, b in ((odd.grad, gr.grad),):
            near_enough = (a.float() - b.float()).nan_to_num().abs() <= 2 * torch.finfo(dt).eps * b.float().nan_to_num().abs() + 1e-5 * b.float().nan_to_num().abs().amax(-1, keepdim=True) + 2.0 ** -24
            assert bool(near_enough.all())
    base = torch.empty(rows, vocab + 1, dtype=dt, device="cuda")
    base[:, 1:] = x
    odd = lg.logits_score(base[:, 1:], toks.cuda(), entropy=True, top=6)
    assert torch.equal(odd.top_tokens, r.top_tokens)
    assert torch.equal(lg.logits_draw(base[:, 1:], u.cuda(), temperature=0.9).tokens, d.tokens)


# ---- as they are used ----------------------------------------------------------------------------------------------
def test_from_logits_to_guess_numbers():
    """Samples of a small model drawn step by step, their keys, the rank index, and the guess numbers of scored passwords: all against
    64 bits on the same uniforms."""
    vocab, end, longest, n = 30, 29, 12, 4000
    g = torch.Generator().manual_seed(9)
    table = torch.randn(vocab, vocab, generator=g) * 1.5
    table[:, end] += 1.0
    dev = table.cuda().to(torch.bfloat16)
    last = torch.full((n,), 0, device="cuda")
    live = torch.ones(n, dtype=torch.bool, device="cuda")
    toks, ml2p = [], []
    for step in range(longest):
        r = lg.logits_draw(dev[last], seed=3, draw=step, live=live)
        toks.append(r.tokens)
        ml2p.append(r.ml2p)
        live = live & (r.tokens != end)
        last = r.tokens.clamp(min=0).long()
    toks, ml2p = torch.stack(toks, 1), torch.stack(ml2p, 1)
    keys = lg.logits_keys(ml2p)
    rows = [Row(r, 1.0) for r in dev.double().cpu().numpy()]
    want = []
    for i in range(0, n, 40):
        prev, s, tol = 0, 0.0, 0.0
        for step in range(longest):
            t, margin = rows[prev].draw(uniform53(3, i, step))
            assert margin > 1e-12 and t == int(toks[i, step])
            v, d = rows[prev].score(t)
            s, tol, prev = s + v, tol + d, t
            if t == end:
                break
        assert abs(float(keys[i]) - s) <= tol + 1e-12
        want.append(s)
    # the same strings scored as a batch of sequences: the same keys to within twice the bound
    before = torch.cat([torch.zeros(n, 1, dtype=torch.long, device="cuda"), toks[:, :-1].clamp(min=0).long()], 1)
    scored = lg.logits_keys(lg.logits_score(dev[before], toks).ml2p)
    assert (scored - keys).abs().max().item() <= 2 * longest * max(r.score(k)[1] for r in rows for k in range(vocab) if r.p[k] > 0)
    mc = MonteCarloLib(keys.clone())
    ks = np.sort(keys.cpu().numpy())
    pos = np.cumsum(2.0 ** (ks - math.log2(n)))
    x = float(ks[n // 2]) + 1e-9
    assert abs(mc.ml2p2rank(x) - pos[np.searchsorted(ks, x, side="right") - 1]) <= 1e-9 * pos[-1]
    gc = mc.ml2p_iter2gc([("a", 1, float(ks[10])), ("b", 2, float(ks[n - 10]))])
    assert gc[0][3] >= 1 and gc[1][3] > gc[0][3]


def test_other_stream_and_repeated_runs_are_the_same():
    x = make(700, 5003, torch.bfloat16, 1).cuda()
    t = tokens_for(x.cpu(), 1).cuda()
    w = torch.rand(700).cuda()
    u = torch.rand(700, dtype=torch.float64).cuda()

    def all_of():
        a, b, c = lg.logits_score(x, t, entropy=True, top=9), lg.logits_gradient(x, t, w, entropy_weights=w), lg.logits_draw(x, u)
        return [v.view(torch.int32) if v.dtype == torch.float32 else v.view(torch.int16) if v.dtype == torch.bfloat16 else v
                for v in (*a, *b, *c, lg.logits_keys(a.ml2p.nan_to_num().view(70, 10)))]

    first = all_of()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = all_of()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    assert all(torch.equal(p, q) for p, q in zip(first, all_of()))


@pytest.mark.parametrize("rows,vocab", [(5, 33), (3, 40000), (300, 9000), (2000, 97)])
def test_captured_and_replayed(rows, vocab):
    x = make(rows, vocab, torch.float32, 1).cuda()
    t = tokens_for(x.cpu(), 1).cuda()
    w = torch.rand(rows).cuda()
    u = torch.rand(rows, dtype=torch.float64).cuda()
    k = min(vocab, 6)

    def all_of():
        a = lg.logits_score(x, t, entropy=True, top=k)
        return [*a, *lg.logits_gradient(x, t, w, entropy_weights=w), *lg.logits_draw(x, u), lg.logits_keys(a.ml2p.view(rows, 1))]

    all_of()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of()
    for seed in range(4):
        x.copy_(make(rows, vocab, torch.float32, 20 + seed))
        u.uniform_(generator=None)
        graph.replay()
        torch.cuda.synchronize()
        want = all_of()
        torch.cuda.synchronize()
        for p, q in zip(held, want):
            assert torch.equal(p.nan_to_num(nan=3.0), q.nan_to_num(nan=3.0))


def test_captured_wide_rows_with_workspaces():
    """Two graphs of calls that are cut into parts, replayed in turn with eager work between them."""
    x = make(9, 200003, torch.float32, 3).cuda()
    t = tokens_for(x.cpu(), 1).cuda()
    w = torch.rand(9).cuda()
    u = torch.rand(9, dtype=torch.float64).cuda()

    def all_of():
        return [*lg.logits_score(x, t, entropy=True, top=20), *lg.logits_gradient(x, t, w, entropy_weights=w), *lg.logits_draw(x, u)]

    all_of()
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(all_of())
    for seed in range(3):
        x.copy_(make(9, 200003, torch.float32, 30 + seed))
        u.uniform_(generator=None)
        graphs[0].replay()
        want = all_of()
        graphs[1].replay()
        torch.cuda.synchronize()
        for mine in held:
            for p, q in zip(mine, want):
                assert torch.equal(p.nan_to_num(nan=3.0), q.nan_to_num(nan=3.0))


def test_two_streams_and_two_threads_at_once():
    import threading
    xs = [make(9, 200003, torch.bfloat16, 5 + i).cuda() for i in range(2)] + [make(3000, 97, torch.float16, 9).cuda()]
    ts = [tokens_for(x.cpu(), 1).cuda() for x in xs]
    us = [torch.rand(x.shape[0], dtype=torch.float64).cuda() for x in xs]
    ws = [torch.rand(x.shape[0]).cuda() for x in xs]

    def all_of(i):
        return [*lg.logits_score(xs[i], ts[i], entropy=True, top=8), *lg.logits_gradient(xs[i], ts[i], ws[i], entropy_weights=ws[i]),
                *lg.logits_draw(xs[i], us[i])]

    want = [all_of(i) for i in range(3)]
    torch.cuda.synchronize()
    got, errors = [[] for _ in xs], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i].append(all_of(i))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for i in range(3):
        for run in got[i]:
            for p, q in zip(run, want[i]):
                assert torch.equal(p.nan_to_num(nan=3.0), q.nan_to_num(nan=3.0))


def test_a_gradient_in_the_logits_place_is_noticed():
    """What autograd saved of the logits is overwritten: its backward refuses, and works where the logits were not needed."""
    a = torch.randn(4, 50, device="cuda", requires_grad=True)
    t, w = torch.arange(4).cuda(), torch.ones(4).cuda()
    x = a.tanh()
    g = lg.logits_gradient(x, t, w, out=x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        x.backward(g.grad)
    x = a * 2.0
    want = lg.logits_gradient(x, t, w).grad
    x.backward(lg.logits_gradient(x, t, w, out=x.detach()).grad)
    assert torch.equal(a.grad, want * 2.0)


def test_refusals():
    x = torch.zeros(4, 6, 10).cuda()
    t = torch.zeros(4, 6, dtype=torch.int64).cuda()
    w = torch.ones(4, 6).cuda()
    u = torch.zeros(6, dtype=torch.float64).cuda()
    for exc, call in [
        (TypeError, lambda: lg.logits_score(x.double(), t)), (ValueError, lambda: lg.logits_score(x, t[:, 1:])),
        (TypeError, lambda: lg.logits_score(x, t.float())), (ValueError, lambda: lg.logits_score(x, t.cpu())),
        (ValueError, lambda: lg.logits_score(x.transpose(1, 2), t)), (ValueError, lambda: lg.logits_score(x[..., :0], t)),
        (ValueError, lambda: lg.logits_score(x[None], t[None])), (ValueError, lambda: lg.logits_score(x, t, top=11)),
        (ValueError, lambda: lg.logits_score(x, t, top=-1)), (ValueError, lambda: lg.logits_score(x, t, temperature=0)),
        (ValueError, lambda: lg.logits_score(x, t, temperature=math.nan)), (TypeError, lambda: lg.logits_gradient(x, t, w.double())),
        (ValueError, lambda: lg.logits_gradient(x, t, w[0])), (ValueError, lambda: lg.logits_gradient(x, t, w, entropy_weights=w[:2])),
        (ValueError, lambda: lg.logits_gradient(x, t, w, out=x.half())), (ValueError, lambda: lg.logits_gradient(x, t, w, out=x[:, :, :9])),
        (ValueError, lambda: lg.logits_gradient(x[:, :5], t[:, :5], w[:, :5], out=x.view(-1)[:200].view(4, 5, 10))),
        (ValueError, lambda: lg.logits_draw(x, seed=1)), (ValueError, lambda: lg.logits_draw(x[0])),
        (ValueError, lambda: lg.logits_draw(x[0], u, seed=1)), (TypeError, lambda: lg.logits_draw(x[0], u.float())),
        (ValueError, lambda: lg.logits_draw(x[0], u[1:])), (TypeError, lambda: lg.logits_draw(x[0], u, live=t[0, :])),
        (TypeError, lambda: lg.logits_keys(w.double())), (ValueError, lambda: lg.logits_keys(w, t[0])),
        (TypeError, lambda: lg.logits_keys(w, t[:, 0].float())), (ValueError, lambda: lg.logits_keys(w, offsets=t[0])),
        (ValueError, lambda: lg.logits_keys(w[0], t[0], offsets=t[0])), (ValueError, lambda: lg.logits_keys(w, t[:, 0].cpu())),
    ]:
        with pytest.raises(exc):
            call()


def test_no_rows():
    x = torch.zeros(0, 5, 7).cuda()
    t = torch.zeros(0, 5, dtype=torch.int64).cuda()
    w = torch.zeros(0, 5).cuda()
    assert lg.logits_score(x, t, entropy=True, top=2).top_tokens.shape == (0, 5, 2)
    assert lg.logits_gradient(x, t, w).grad.shape == (0, 5, 7)
    assert lg.logits_draw(x[:, 0], seed=1).tokens.shape == (0,)
    assert lg.logits_keys(w).shape == (0,)


# ---- alternatives of rows whose parts, or vectors, are fewer than the launch's largest --------------------------------
@pytest.mark.parametrize("vocab,rows,dtype,top", [(262208, 600, "bf16", 10), (262145, 512, "bf16", 5), (262208, 300, "fp32", 33), (262208, 600, "fp32", 8),
                                                  (524289, 1024, "bf16", 5), (300001, 700, "fp16", 64)])
def test_alternatives_of_shorter_last_parts(vocab, rows, dtype, top):
    """The largest logits in a row's last part (17 chunks a part and 16 in the last one), in its first element and anywhere, every row
    against a sort by logit and id."""
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.0).to(DTYPES[dtype])
    at = torch.randint(vocab - vocab // 5, vocab, (rows, top // 2 + 1), generator=g, device="cuda")
    x.scatter_(1, at, torch.rand(rows, top // 2 + 1, generator=g, device="cuda").mul_(4).add_(12).to(x.dtype))
    x[::3, 0] = 14.0
    x[::4] = torch.randn((rows + 3) // 4, vocab, generator=g, device="cuda").sub_(60.0).to(x.dtype)      # (no logit near 0)
    r = lg.logits_score(x, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=top)
    order = torch.arange(vocab, 0, -1, device="cuda")
    for i in range(0, rows, 64):
        bits = (x[i:i + 64].float() + 0.0).view(torch.int32)
        keys = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + order
        want = torch.topk(keys, top, dim=-1).indices
        assert torch.equal(r.top_tokens[i:i + 64].long(), want), i


# ---- nothing is below 0 ------------------------------------------------------------------------------------------------
def not_negative(t, most=None):
    """No sign bit anywhere (rank indexes sort the bits), and at most `most` where that is given."""
    bits = t.contiguous().view(torch.int64 if t.dtype == torch.float64 else torch.int32)
    assert bool((bits >= 0).all()), t[t.view(-1) < 0][:5] if t.dim() == 1 else t.min()
    assert most is None or t.max().item() <= most


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("vocab,rows", [(1, 900), (5, 900), (97, 900), (97, 20000), (700, 900), (3001, 900), (9001, 900), (20001, 600), (20001, 9), (66001, 600),
                                        (140001, 520), (200003, 9)])
def test_certain_tokens_score_0_and_never_less(vocab, rows, dtype):
    """Rows with one token left and rows whose others are 30 below it, at many logits and temperatures: -log2 p and entropy are 0 or
    a rounding above it.  (A power and a logarithm of a number in (1/2, 1], off by a step of 2^-23 of their value each: below 2^-21;
    `vocab` others of 2^-43 add no more than 2^-24.)"""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    at = torch.arange(rows, device="cuda") * 7 % vocab
    value = torch.linspace(-100, 100, rows, device="cuda")
    x = torch.full((rows, vocab), -math.inf, device="cuda")
    x.scatter_(1, at[:, None], value[:, None])
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64) * 0.999
    w = torch.rand(rows, generator=g, device="cuda")
    for others in (False, True):
        if others:
            x = torch.where(x == -math.inf, value[:, None] - 30.5, x)
        xs = x.to(DTYPES[dtype])
        for t in (1.0, 0.7, 0.05) if others else (1.0, 0.02, 0.7, 3.1, 40.0):
            r = lg.logits_score(xs, at, temperature=t, entropy=True, top=1)
            # (30 below it in bits of 1.44 / T: the others together are below vocab * 2^-43 of the row, their entropy 45 times that)
            most = 2.0 ** -21 + vocab * 2.0 ** -43 * 45 * others
            for v in (r.ml2p, r.entropy, r.top_ml2p.view(-1), lg.logits_score(xs, at, temperature=t).ml2p):
                not_negative(v, most)
            assert torch.equal(r.top_tokens[:, 0].long(), at)
            gr = lg.logits_gradient(xs, at, w, entropy_weights=w, temperature=t)
            not_negative(gr.ml2p, most)
            not_negative(gr.entropy, most)
            d = lg.logits_draw(xs, u, temperature=t)
            assert torch.equal(d.tokens.long(), at) or others
            not_negative(d.ml2p)
            not_negative(d.ml2p[d.tokens == at], most)


def test_keys_are_never_below_0():
    m = torch.tensor([[-6e-8, 3e-8, 0.0], [-0.0, -0.0, -0.0], [-6e-8, 1.0, 0.0], [-1e-7, math.inf, 0.0], [-1e-7, math.nan, 0.0]]).cuda()
    off = torch.arange(0, 16, 3).cuda()
    many = m[:3].repeat(2000, 1)
    for got in (lg.logits_keys(m), lg.logits_keys(m.view(-1), offsets=off)):
        not_negative(got[:4])
        assert got[:2].tolist() == [0.0, 0.0] and got[2].item() == 1.0 + float(m[2, 0]) and got[3].item() == 1022.0 and math.isnan(got[4].item())
    not_negative(lg.logits_keys(many.view(-1), offsets=torch.arange(0, 18001, 3).cuda()))


@pytest.mark.parametrize("temperature", [1e30, 1e29, 1e10])
@pytest.mark.parametrize("vocab,rows", [(5, 7), (97, 3000), (700, 7), (9001, 7), (9001, 600), (200003, 3)])
def test_logits_further_apart_than_the_type_reaches(vocab, rows, temperature):
    """The difference of two float32 logits may pass the largest float32 number where the exponent that it stands for does not."""
    x = make(rows, vocab, torch.float32, vocab)
    for i, (hi, lo) in enumerate([(3e38, -3e38), (3.4e38, -3.4e38), (2e38, -2.5e38)]):
        x[2 * i % rows] = torch.where(torch.arange(vocab) % 3 == i % 3, hi, lo)
    some = list(range(min(rows, 7)))
    toks = torch.arange(rows) % vocab
    g = torch.Generator().manual_seed(vocab)
    w, u = torch.rand(rows, generator=g), torch.rand(rows, generator=g, dtype=torch.float64)
    r = lg.logits_score(x.cuda(), toks.cuda(), temperature=temperature, entropy=True, top=min(4, vocab))
    check_score(x[some], toks[some], lg.LogitScores(*(t[some] for t in r)), temperature, min(4, vocab))
    gr = lg.logits_gradient(x.cuda(), toks.cuda(), w.cuda(), entropy_weights=w.cuda(), temperature=temperature)
    check_gradient(x[some], toks[some], w[some], w[some], lg.LogitGradient(*(t[some] for t in gr)), temperature, "fp32")
    d = lg.logits_draw(x.cuda(), u.cuda(), temperature=temperature)
    check_draw(x[some], u[some], None, lg.LogitDraws(d.tokens[some], d.ml2p[some]), temperature)


@pytest.mark.parametrize("vocab,rows", [(5, 9), (97, 300), (700, 9), (3001, 40), (9001, 40), (20001, 600), (200003, 9)])
def test_nan_and_infinities_beside_each_other(vocab, rows):
    """+inf, -inf and NaN in one row, in either order and beside logits whose scaled values overflow: NaN, and no token."""
    x = torch.zeros(rows, vocab)
    for i in range(min(rows, 9)):
        first, second = [(math.inf, math.nan), (math.nan, math.inf), (3e38, math.nan), (math.nan, 3e38), (-math.inf, math.nan), (math.inf, math.inf),
                         (math.inf, -math.inf), (3e38, math.inf), (math.inf, 3e38)][i]
        x[i, 0], x[i, vocab - 1] = first, second
    toks = torch.arange(rows) % vocab
    w, u = torch.ones(rows), torch.full((rows,), 0.25, dtype=torch.float64)
    for t in (1.0, 1e-5):
        r = lg.logits_score(x.cuda(), toks.cuda(), temperature=t, entropy=True, top=2)
        g = lg.logits_gradient(x.cuda(), toks.cuda(), w.cuda(), entropy_weights=w.cuda(), temperature=t)
        d = lg.logits_draw(x.cuda(), u.cuda(), temperature=t)
        n = min(rows, 9)
        for v in (r.ml2p, r.entropy, r.top_ml2p[:, 0], g.ml2p, g.entropy, d.ml2p):
            assert bool(v[:n].isnan().all()) and not bool(v[n:].isnan().any())
        assert bool((r.top_tokens[:n] == OUTSIDE).all()) and bool((d.tokens[:n] == OUTSIDE).all())
        assert bool(g.grad[:n].isnan().all()) and bool(torch.isfinite(g.grad[n:]).all())
