"""The operators on logits in 64 bits, straight from their definitions, with the error bounds of sums held in 32 bits."""
import math

import numpy as np

from montecarlo_amd.logits import OUTSIDE, SKIP

U = 2.0 ** -24          # half a step of float32, relative


def steps_of(vocab):
    """Additions in a row behind each other that a kernel may make: a thread's share of a row and the joining of threads."""
    return 64 + vocab / 128


class Row:
    """One row of logits (float64 values) at a temperature."""

    def __init__(self, x, temperature):
        self.x, self.t = np.asarray(x, dtype=np.float64), float(temperature)
        self.vocab = len(self.x)
        self.bad = bool(np.isnan(self.x).any() or (self.x == math.inf).any())
        self.empty = not self.bad and not (self.x > -math.inf).any()
        if self.bad or self.empty:
            return
        with np.errstate(under="ignore"):
            self.y = (self.x - self.x.max()) / self.t * math.log2(math.e)
            self.w = np.exp2(self.y)
        self.z = math.fsum(self.w)
        self.lz = math.log2(self.z)
        self.p = self.w / self.z
        there = self.p > 0
        self.yp = np.where(there, self.y, 0.0)
        self.entropy = self.lz - math.fsum(self.p * self.yp)
        # relative error of Z: that of the weights (three roundings of the exponent, the power's own step), and the sums'
        self.dz = U * (2.1 * math.fsum(self.p * -self.yp) + 2 + steps_of(self.vocab))

    def score(self, tok):
        """(-log2 p of the token, how far off a kernel may be)."""
        if tok == SKIP:
            return 0.0, 0.0
        if self.bad:
            return math.nan, 0.0
        if self.empty or not 0 <= tok < self.vocab or self.x[tok] == -math.inf:
            return math.inf, 0.0
        v = self.lz - self.y[tok]
        if v > 3.4028234663852886e38:               # (the result is a float32: beyond its largest number it rounds to +inf)
            return math.inf, 0.0
        return v, 1.45 * self.dz + U * (3 * abs(self.y[tok]) + 2 * self.lz + abs(v) + 1e-30)

    def h(self, tok=0):
        if tok == SKIP:
            return 0.0, 0.0
        if self.bad:
            return math.nan, 0.0
        if self.empty:
            return 0.0, 0.0
        mean, square = math.fsum(self.p * -self.yp), math.fsum(self.p * self.yp ** 2)
        tol = 1.45 * self.dz + mean * (self.dz + U * (steps_of(self.vocab) + 6)) + 2.1 * U * square
        return self.entropy, tol + U * (2 * self.lz + abs(self.entropy))

    def top(self, k):
        """ids and -log2 p of the k largest."""
        if self.bad or self.empty:
            return [OUTSIDE] * k, [math.nan if self.bad else math.inf] * k
        order = sorted(range(self.vocab), key=lambda i: (-self.x[i], i))[:k]
        ids, vals = [], []
        for i in order:
            # (an exponent beyond what 32 bits hold is a probability of 0)
            gone = self.x[i] == -math.inf or self.y[i] < -3.4e38
            ids.append(OUTSIDE if gone else i)
            vals.append(math.inf if gone else self.lz - self.y[i])
        return ids, vals

    def grad(self, tok, a, b, eps, least):
        """d (a ml2p + b entropy) / dx and how far off it may be: `eps`, `least` half a step of the output type and of its
        smallest numbers."""
        if tok == SKIP or self.empty:
            return np.zeros(self.vocab), np.zeros(self.vocab)
        if self.bad:
            return np.full(self.vocab, math.nan), np.zeros(self.vocab)
        hit = np.zeros(self.vocab)
        A = a / math.log(2) / self.t if 0 <= tok < self.vocab else 0.0
        if A:
            hit[tok] = 1.0
        B = b / self.t
        lp = self.yp - self.lz + self.entropy
        g = A * (self.p - hit) - B * self.p * np.where(self.p > 0, lp, 0.0)
        dp = self.dz + U * (2.1 * np.abs(self.yp) + 8)
        dl = U * 3 * np.abs(self.yp) + self.h()[1] + 1.45 * self.dz + U * (np.abs(lp) + self.lz + self.entropy)
        tol = self.p * (abs(A) + abs(B) * np.abs(lp)) * dp + abs(B) * self.p * dl + U * 4 * (abs(A) * hit + np.abs(g))
        return g, tol * (1 + eps) + eps * np.abs(g) + least + 1e-37 * (abs(A) + abs(B) * 200)

    def draw(self, u):
        """(token, how far u Z is from the ends of its interval as a share of Z)."""
        if self.bad or self.empty:
            return OUTSIDE, 1.0
        w = np.exp((self.x - self.x.max()) / self.t)
        c = np.cumsum(w)
        target = max(u, 0.0) * c[-1]
        last = int(np.nonzero(w > 0)[0][-1])
        i = min(int(np.searchsorted(c, target, side="right")), last)
        lo = c[i - 1] if i else 0.0
        return i, min(abs(target - lo) if i else 1.0, abs(c[i] - target) if i < last else 1.0) / c[-1]
