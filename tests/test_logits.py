"""The operators on logits without a GPU: the definitions against differences, and what the C ABI refuses."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from montecarlo_amd import _native as nv
from montecarlo_amd import logits as lg
from tests.logits_ref import OUTSIDE, SKIP, Row


@pytest.mark.parametrize("vocab,temperature,tok", [(1, 1.0, 0), (5, 0.7, 3), (17, 1.6, 0), (17, 1.0, OUTSIDE), (6, 1.0, SKIP)])
def test_gradient_formula_is_the_differences(vocab, temperature, tok):
    rng = np.random.default_rng(vocab)
    x = rng.normal(size=vocab) * 2
    a, b, h = 0.7, -0.4, 1e-5

    def loss(v):
        r = Row(v, temperature)
        m = r.score(tok)[0]
        return (a * m if math.isfinite(m) else 0.0) + b * r.h(tok)[0]

    got = Row(x, temperature).grad(tok, a, b, 0.0, 0.0)[0]
    for i in range(vocab):
        d = np.zeros(vocab)
        d[i] = h
        # (the central difference is off by h^2 / 6 times the third derivative, and by the losses' rounding over h)
        assert abs((loss(x + d) - loss(x - d)) / (2 * h) - got[i]) < 1e-8


def _score(**over):
    a = dict(logits=None, dtype=0, outer=1, inner=1, vocab=8, os=0, is_=8, tokens=None, tb=8, tos=0, tis=1, t=1.0, ml2p=None,
             ent=None, top=0, ids=None, vals=None, ws=None, wsb=0, stream=None)
    a.update(over)
    return nv.lib.mc_logits_score(*a.values())


BUF = (C.c_char * 4096)()
ADDR = C.addressof(BUF) & ~63 | 0


@pytest.mark.parametrize("over", [
    dict(),                                                     # no logits
    dict(logits=ADDR),                                          # no tokens
    dict(logits=ADDR, tokens=ADDR),                             # no output
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, dtype=3),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, vocab=0),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, vocab=1 << 31),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, outer=1 << 20, inner=1 << 20),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, outer=1 << 63, inner=2),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, tb=2),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, t=0.0),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, t=-1.0),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, t=math.nan),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, t=math.inf),
    dict(logits=ADDR + 2, tokens=ADDR, ml2p=ADDR),              # float32 at an odd half word
    dict(logits=ADDR + 1, tokens=ADDR, ml2p=ADDR, dtype=2),
    dict(logits=ADDR, tokens=ADDR + 4, ml2p=ADDR),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, top=65, ids=ADDR, vals=ADDR, vocab=100),
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, top=9, ids=ADDR, vals=ADDR),      # more than tokens
    dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, top=2, ids=ADDR),
])
def test_score_refuses(over):
    assert _score(**over) == -1
    assert nv.lib.mc_last_error().startswith(b"mc_logits_score: ")


@pytest.mark.parametrize("name,args", [
    ("mc_logits_gradient", [ADDR, 0, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, None, 0, 1, None, 0, 0, ADDR, None, ADDR, None, 0, None]),
    ("mc_logits_gradient", [ADDR, 0, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, ADDR, 0, 1, None, 0, 0, ADDR, None, None, None, 0, None]),
    ("mc_logits_gradient", [ADDR, 0, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, ADDR, 0, 1, None, 0, 0, ADDR, None, ADDR + 2, None, 0, None]),
    ("mc_logits_gradient", [ADDR, 7, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, ADDR, 0, 1, None, 0, 0, ADDR, None, ADDR, None, 0, None]),
    ("mc_logits_draw", [ADDR, 0, 1, 8, 8, 1.0, None, 0, 0, 0, None, None, ADDR, None, 0, None]),
    ("mc_logits_draw", [ADDR, 0, 1, 8, 8, 0.0, None, 0, 0, 0, None, ADDR, ADDR, None, 0, None]),
    ("mc_logits_draw", [ADDR, 0, 1 << 31, 8, 8, 1.0, None, 0, 0, 0, None, ADDR, ADDR, None, 0, None]),
    ("mc_logits_draw", [None, 0, 1, 8, 8, 1.0, None, 0, 0, 0, None, ADDR, ADDR, None, 0, None]),
    ("mc_logits_keys", [ADDR, ADDR, ADDR, 8, 1, 0, 1, ADDR, None]),
    ("mc_logits_keys", [ADDR, None, ADDR, 2, 1, 0, 1, ADDR, None]),
    ("mc_logits_keys", [None, None, None, 0, 1, 4, 4, ADDR, None]),
    ("mc_logits_keys", [ADDR, None, None, 0, 1, 4, 4, None, None]),
    ("mc_logits_keys", [ADDR, None, None, 0, 1 << 50, 4, 4, ADDR, None]),
])
def test_the_others_refuse(name, args):
    assert getattr(nv.lib, name)(*args) == -1
    assert nv.lib.mc_last_error().startswith(name.encode() + b": ")


def test_a_workspace_that_is_too_small_is_refused():
    need = nv.lib.mc_logits_score_workspace_bytes(0, 2, 300000, 5)
    assert need > 0 and nv.lib.mc_logits_score_workspace_bytes(0, 2, 100, 5) == 0
    big = dict(logits=ADDR, tokens=ADDR, ml2p=ADDR, inner=2, vocab=300000, top=5, ids=ADDR, vals=ADDR)
    for ws, size in ((None, need), (ADDR, need - 1), (ADDR + 8, need)):
        assert _score(**big, ws=ws, wsb=size) == -6
    need = nv.lib.mc_logits_gradient_workspace_bytes(2, 2, 300000)
    assert need > 0
    assert nv.lib.mc_logits_gradient(ADDR, 2, 1, 2, 300000, 0, 300000, ADDR, 8, 0, 1, 1.0, ADDR, 0, 1, None, 0, 0, ADDR, None, ADDR, ADDR,
                                     need - 1, None) == -6
    need = nv.lib.mc_logits_draw_workspace_bytes(1, 2, 100000)
    assert need > 0
    assert nv.lib.mc_logits_draw(ADDR, 1, 2, 100000, 100000, 1.0, None, 0, 0, 0, None, ADDR, ADDR, ADDR, need - 1, None) == -6


def test_nothing_to_do_is_fine_without_a_gpu():
    assert _score(inner=0) == 0
    assert _score(outer=0, inner=5) == 0
    assert nv.lib.mc_logits_draw(None, 0, 0, 8, 8, 1.0, None, 0, 0, 0, None, None, None, None, 0, None) == 0
    assert nv.lib.mc_logits_keys(None, None, None, 0, 0, 0, 0, None, None) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(3, 5)
    t = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: lg.logits_score(x, t), lambda: lg.logits_gradient(x, t, torch.ones(3)),
                 lambda: lg.logits_draw(x, seed=1), lambda: lg.logits_keys(x)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_the_plugin_form_is_abstract_and_checks_its_arguments():
    from montecarlo_amd.logits_simulator import LogitsMonteCarlo

    class Model(LogitsMonteCarlo):
        def logits(self, tokens):
            raise NotImplementedError

    with pytest.raises(TypeError):
        LogitsMonteCarlo(["a", "<end>"], 1, device="cpu")
    for end, max_len, batch in ((2, 4, 1), (-1, 4, 1), (1, 0, 1), (1, 4, 0)):
        with pytest.raises(ValueError):
            Model(["a", "<end>"], end, max_len=max_len, batch=batch, device="cpu")
    m = Model(["a", "b", "<end>"], 2, device="cpu")
    assert m.encode("abz") == [0, 1, OUTSIDE]
    assert m._sampled_strings(torch.tensor([[0, 1, 2, SKIP], [2, SKIP, SKIP, SKIP]])) == ["ab", ""]


def test_the_multiplication_that_stands_for_a_division():
    """make_div / at of csrc/mc_logits.h in whole numbers: exact for every row number below 2^31."""
    rng = np.random.default_rng(1)
    for d in [1, 2, 3, 5, 7, 16, 31, 97, 1000, 65535, 65536, 65537, (1 << 30) - 1, 1 << 30, (1 << 31) - 1] + rng.integers(1, 1 << 31, 300).tolist():
        shift = 0
        while (1 << shift) < d:
            shift += 1
        mul = ((1 << (31 + shift)) + d - 1) // d
        assert mul < 1 << 32
        rows = {0, 1, d - 1, d, d + 1, 2 * d - 1, (1 << 31) - 1, ((1 << 31) - 1) // d * d, ((1 << 31) - 1) // d * d - 1}
        for r in list(rows) + rng.integers(0, 1 << 31, 20).tolist():
            if 0 <= r < 1 << 31:
                assert (((r << 1) * mul) >> 32) >> shift == r // d, (r, d)


def test_the_polynomial_of_the_draw():
    """2^f on [-1/2, 1/2] as csrc/mc_logits_draw.hip has it: off by less than 4.1e-11 of its value, with room to the margin."""
    import os
    import re
    from decimal import Decimal, getcontext
    getcontext().prec = 40
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "montecarlo_amd", "csrc", "mc_logits_draw.hip")).read()
    body = src[src.index("double power_of("):src.index("return __hiloint2double")]
    c = [Decimal(float.fromhex(h)) for h in re.findall(r"(0x1\.[0-9a-f]+p[+-]\d+)", body)]
    assert len(c) == 8                                      # from the highest power down
    worst = Decimal(0)
    for i in range(-500, 501):
        f = Decimal(i) / 1000
        p = Decimal(0)
        for k in c:
            p = p * f + k
        worst = max(worst, abs(p / (f * Decimal(2).ln()).exp() - 1))
    margin = float(re.search(r"MARGIN = ([0-9e.-]+);", src).group(1))
    assert worst < Decimal("4.1e-11") and margin >= 2 * float(worst)


def test_the_cells_of_alternatives_fit_what_is_allocated():
    """Rows of cells that k_logits_score writes (csrc/mc_logits_score.hip) against those its LDS is counted for, in whole numbers: of
    every part of a row cut into parts, of whole rows, and of rows whose first element stays before their vectors."""
    import os
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "montecarlo_amd", "csrc", "mc_logits_score.hip")).read()
    kernel = src[src.index("void k_logits_score(Rows a"):src.index("// the parts of a row joined")]
    # the kernel fills cells of as many chunks as the host counted: it does not spread its own chunks anew
    assert re.search(r"per_cell = sp\.per_cell;", kernel) and "CELL_ROWS" not in kernel

    def up(a, b):
        return -(-a // b)

    def cells(vecs, lanes):                                # cell_chunks, cell_bytes
        per_cell = up(up(vecs, 4 * lanes), 16)
        return per_cell, up(up(vecs, 4 * lanes), per_cell)

    rng = np.random.default_rng(5)
    vocabs = [16384 * 8 * k + d for k in range(1, 9) for d in (-9, -1, 0, 1, 2, 64, 4097)] + [262208, 262145, 524289, 1 << 20, (1 << 31) - 65]
    vocabs += np.exp(rng.uniform(math.log(4097), math.log(3e6), 400)).astype(int).tolist()
    for vocab in vocabs:
        for rows in (1, 3, 25, 256, 257, 300, 512, 600, 1023, 1024, 4096):
            for size in (2, 4):
                per = 16 // size
                nvec, shift = up(vocab, per), 0
                while vocab > 160000 and shift < 6 and (rows << shift) < 1024 and (nvec >> (shift + 1)) >= 1024:
                    shift += 1
                for mine in {nvec, up(vocab - 1, per) if size == 2 else nvec}:
                    if shift:
                        vecs = up(up(nvec, 1 << shift), 1024) * 1024
                        per_cell, room = cells(vecs, 256)
                        used = [up(up(max(0, min(mine, (p + 1) * vecs) - p * vecs), 1024), per_cell) for p in range(1 << shift)]
                    else:
                        lanes = 1024 if nvec >= 16384 or (rows <= 256 and nvec >= 2048) else 256
                        per_cell, room = cells(nvec, lanes)
                        used = [up(up(mine, 4 * lanes), per_cell)]
                    assert max(used) <= room <= 16, (vocab, rows, size, used, room)


def test_kernels_load_nothing_of_skipped_rows():
    """Every place where a kernel looks at where a row begins (which loads the first element of rows of two bytes at an odd one) lies
    behind the question whether the row is skipped, or is told."""
    import os
    import re
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "montecarlo_amd", "csrc")
    head = open(os.path.join(here, "mc_logits.h")).read()
    body = head[head.index("Span span_of("):head.index("// vector v of a row;")]
    assert "bool read" in body and re.search(r"read \? element<DT>\(row, 0\) : -INFINITY", body)
    seen = 0
    for name in ("score", "gradient", "draw"):
        src = open(os.path.join(here, f"mc_logits_{name}.hip")).read()
        for kernel in re.split(r"\n__global__ ", src)[1:]:
            for m in re.finditer(r"span_of<DT>\(([^;]*)\)[,;]", kernel):
                seen += 1
                before = kernel[:m.start()]
                told = "tok != MC_TOKEN_SKIP" in m.group(1)
                asked = re.search(r"if \((tok == MC_TOKEN_SKIP|d\.live && !d\.live\[row\])\) \{.*?return;|(== MC_TOKEN_SKIP|!d\.live\[row\]\))\) return;"
                                  r"|if \(tok != MC_TOKEN_SKIP\) \{", before, re.S)
                assert told or asked, (name, kernel[:60])
    assert seen >= 9


@pytest.mark.parametrize("name,args,which", [
    ("mc_logits_score", [ADDR, 0, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, ADDR, ADDR, 2, ADDR, ADDR, None, 0, None], {12: 2, 13: 2, 15: 2, 16: 2}),
    ("mc_logits_gradient", [ADDR, 0, 1, 1, 8, 0, 8, ADDR, 8, 0, 1, 1.0, ADDR, 0, 1, ADDR, 0, 1, ADDR, ADDR, ADDR, None, 0, None], {12: 2, 15: 1, 18: 2, 19: 2}),
    ("mc_logits_draw", [ADDR, 0, 1, 8, 8, 1.0, ADDR, 0, 0, 0, None, ADDR, ADDR, None, 0, None], {6: 4, 11: 2, 12: 2}),
    ("mc_logits_keys", [ADDR, ADDR, None, 0, 1, 0, 1, ADDR, None], {0: 2, 1: 4, 7: 4}),
    ("mc_logits_keys", [ADDR, None, ADDR, 8, 1, 4, 4, ADDR, None], {0: 1, 2: 4, 7: 4}),
    ("mc_logits_keys", [ADDR, None, ADDR, 4, 1, 4, 4, ADDR, None], {2: 2}),
])
def test_what_is_not_aligned_to_its_type_is_refused(name, args, which):
    for i, off in which.items():
        mine = list(args)
        mine[i] += off
        assert getattr(nv.lib, name)(*mine) == -1, (name, i)
        assert b"aligned" in nv.lib.mc_last_error(), (name, i)
