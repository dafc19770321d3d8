"""Plain implementations of a beam search's step in 64 bits, on the CPU, and what a result is held to."""
import numpy as np

from oracle import oracle as O
from tests.edit_util import edit_row

# An output's distance from the exact score. A lane adds at most 8 fp32 terms in an accumulator and joins those in two
# more additions: 10 u of the sum (u = 2^-24). A term exp(-d) is off by u d for the subtraction, the factor log2 e / T and the
# product each, and by 2 u for the exponential: with its weight exp(-d), 3 / e u + 2 u of the sum at most. 14 u < 2^-20 of the
# sum is as much of its logarithm. The output then rounds to fp32: u of its value.
TOL = 2.0 ** -20
U = 2.0 ** -24


def log_softmax64(x, T):
    """fp64 log-probabilities of fp32 logits (-inf or NaN: no token), T <= 0 as 1; None where there is no token."""
    x = np.asarray(x, np.float32)
    T = float(np.float32(T)) if T > 0 else 1.0
    on = x > -np.inf
    if not on.any():
        return None
    M = float(x[on].max())
    lp = np.full(x.shape, -np.inf)
    if M == np.inf:
        lp[x == np.inf] = -np.log(float((x == np.inf).sum()))
        return lp
    d = (x[on].astype(np.float64) - M) / T
    lp[on] = d - np.log(np.exp(d).sum())
    return lp


class Step:
    """A step's exact candidates: c[r] a row's scores [V] in fp64 (-inf: none), x[r] its edited logits."""

    def __init__(self, x, score, row_off, n, eos=-1, p=None, bias=None, allowed=None):
        R = len(x)
        self.off, self.n, self.eos = np.asarray(row_off, np.int64), n, eos
        self.S = len(self.off) - 1
        of = np.repeat(np.arange(self.S), np.diff(self.off))
        self.x, self.c = [], []
        for r in range(R):
            s = of[r]
            e = edit_row(x[r], None, [], bias[s] if bias else (), None)
            if p is not None and p["softcap"][s] > 0:
                e = O.softcap(np.asarray(x[r], np.float32).copy(), float(p["softcap"][s]))
                for t, b in (bias[s] if bias else ()):
                    if 0 <= t < e.size:
                        e[t] = np.float32(e[t]) + np.float32(b)
            if allowed is not None and allowed[r] is not None:
                e = np.where(allowed[r], e, -np.inf).astype(np.float32)
            lp = log_softmax64(e, float(p["temperature"][s]) if p is not None else 1.0)
            a = float(np.float32(score[r])) if score is not None else 0.0
            c = np.full(e.shape, -np.inf) if lp is None or not a > -np.inf else a + lp
            with np.errstate(over="ignore"):
                c[~(c.astype(np.float32) > -np.inf)] = -np.inf
            self.x.append(e)
            self.c.append(c)

    def check(self, out):
        """Holds a result without keep_slots to the definition: scores within the tolerance, nothing better left out, exact
        order within a row, and equal candidates by row."""
        got = {k: v.cpu().numpy() for k, v in out.items()}
        n = self.n
        for s in range(self.S):
            rows = range(int(self.off[s]), int(self.off[s + 1]))
            C = [self.c[r].copy() for r in rows]
            ends = [c[self.eos] if 0 <= self.eos < c.size else -np.inf for c in C]
            for c in C:
                if 0 <= self.eos < c.size:
                    c[self.eos] = -np.inf
            flat = np.sort(np.concatenate([c[c > -np.inf] for c in C]) if C else np.zeros(0))[::-1]
            k = min(n, flat.size)
            p, t, v = got["parent"][s], got["tok"][s], got["score"][s].astype(np.float64)
            assert np.all(p[k:] == -1) and np.all(t[k:] == -1) and np.all(v[k:] == -np.inf), (s, k, p, t, v)
            assert np.all((p[:k] >= 0) & (p[:k] < len(C))), (s, p)
            want = np.array([C[p[j]][t[j]] for j in range(k)])
            tol = TOL + U * np.abs(want)
            assert np.all(want > -np.inf), (s, p, t, want)
            with np.errstate(invalid="ignore"):
                assert np.all((np.abs(v[:k] - want) <= tol) | (v[:k] == want)), (s, v[:k], want)
                # the j-th of them is as good as the exact j-th
                assert np.all((np.abs(want - flat[:k]) <= 2 * TOL) | (want == flat[:k])), (s, want, flat[:k])
            assert len(set(zip(p[:k].tolist(), t[:k].tolist()))) == k, (s, p, t)
            for w in range(len(C)):                            # a row's tokens: its largest, in order, none left out
                mine = t[:k][p[:k] == w]
                x = np.where(C[w] > -np.inf, self.x[rows[w]], -np.inf) + 0.0
                order = np.lexsort((np.arange(x.size), -x))[:mine.size]
                assert np.array_equal(mine, order), (s, w, mine, order)
            for j in range(k - 1):                             # equal ones: the lower row first
                assert want[j] >= want[j + 1] or want[j + 1] - want[j] <= 2 * TOL
                if want[j] == want[j + 1] and np.array_equal(C[p[j]], C[p[j + 1]]):
                    assert p[j] <= p[j + 1], (s, p)
            self._check_done(s, got, C, ends, flat)

    def _check_done(self, s, got, C, ends, flat):
        n, d = self.n, int(got["done"][s])
        dp, dv = got["done_parent"][s], got["done_score"][s].astype(np.float64)
        assert 0 <= d <= min(n, len(C)), (s, d)
        assert np.all(dp[d:] == -1) and np.all(dv[d:] == -np.inf), (s, d, dp, dv)
        assert len(set(dp[:d].tolist())) == d, (s, dp)
        for j in range(d):
            e = ends[dp[j]]
            assert e > -np.inf and (dv[j] == e or abs(dv[j] - e) <= TOL + U * abs(e)), (s, j, dv[j], e)
            assert j == 0 or ends[dp[j - 1]] >= e - 2 * TOL, (s, dp)
        for w, e in enumerate(ends):
            if not e > -np.inf:
                continue
            others = np.concatenate([flat, [o for i, o in enumerate(ends) if i != w and o > -np.inf]])
            sure = int((others > e + 2 * TOL).sum())
            same = int((C[w] == e).sum())                      # (of the same row and logit: behind it)
            maybe = int((others > e - 2 * TOL).sum()) - same
            if maybe < n:
                assert w in dp[:d], (s, w, e, dp)
            if sure >= n:
                assert w not in dp[:d], (s, w, e, dp)


def slots(parent, n):
    """Places of new beams (best first) where they keep their parents': place j of the result holds beam order[j]."""
    order, late = [-1] * n, []
    for j, p in enumerate(parent):
        if 0 <= p < n and order[p] < 0:
            order[p] = j
        else:
            late.append(j)
    for i in range(n):
        if order[i] < 0:
            order[i] = late.pop(0)
    return order


def fork(hists, row_off, parent, tok):
    """New histories, a list of lists."""
    out = []
    for s, ps in enumerate(parent):
        for j, p in enumerate(ps):
            ok = 0 <= p < row_off[s + 1] - row_off[s]
            out.append(list(hists[row_off[s] + p]) + ([int(tok[s][j])] if tok is not None else []) if ok else [])
    return out
