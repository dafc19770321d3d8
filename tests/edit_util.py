"""Plain implementations of the edited logits, sampling under them and log-probabilities, on the CPU."""
import numpy as np

from oracle import oracle as O


def unpack(words, V):
    """Truth values [n, V] from mask words."""
    w = np.ascontiguousarray(words).view(np.uint8)
    return np.unpackbits(w.reshape(w.shape[0], -1), axis=1, bitorder="little")[:, :V].astype(bool)


def edit_row(x, p, hist, bias=(), allowed=None):
    """One row's edited logits in fp32, each step rounded as the oracle rounds it; not allowed: -inf. bias: (id, value)s."""
    row = np.asarray(x, np.float32).copy()
    if p is not None and p["softcap"] > 0:
        row = O.softcap(row, float(p["softcap"]))
    for t, b in bias:
        if 0 <= t < row.size:
            row[t] = np.float32(row[t]) + np.float32(b)
    if p is not None:
        row = O.penalize(row, hist, p)
    if allowed is not None:
        row[~allowed] = -np.inf
    return row


def edit_row64(x, p, hist, bias=(), allowed=None):
    """The same in fp64, and a bound of what rounding every step to fp32 (by at most u = 2^-24 relative) adds up to."""
    u = 2.0 ** -24
    row = np.asarray(x, np.float64).copy()
    err = np.zeros_like(row)
    if p is not None and p["softcap"] > 0:
        cap = float(p["softcap"])
        row = cap * np.tanh(row / cap)
        err += 4 * u * np.abs(row)             # a divide, a tanh within an ulp (2u), a multiply; tanh' <= tanh(y) / y
    for t, b in bias:
        if 0 <= t < row.size:
            row[t] += float(np.float32(b))
            err[t] += u * abs(row[t])
    if p is not None and p["repeat_last_n"] != 0 and len(hist):
        L = len(hist)
        b = L - int(p["repeat_last_n"]) if 0 < p["repeat_last_n"] < L else 0
        b = max(b, int(p["penalty_from"]))
        ids, cnt = np.unique(np.asarray(hist[b:], np.int64), return_counts=True)
        rep, fq, pres = float(p["repetition_penalty"]), float(p["frequency_penalty"]), float(p["presence_penalty"])
        for t, c in zip(ids, cnt):
            if not 0 <= t < row.size:
                continue
            if rep != 1.0:
                row[t] = row[t] / rep if row[t] > 0 else row[t] * rep
                err[t] = err[t] * max(rep, 1 / rep) + u * abs(row[t])
            if fq != 0.0 or pres != 0.0:
                s = c * fq + pres
                row[t] -= s
                err[t] += u * (abs(c * fq) + abs(s) + abs(row[t]))
    if allowed is not None:
        row[~allowed] = -np.inf
    return row, err


def neutral(p):
    q = p.copy()
    q["repetition_penalty"], q["frequency_penalty"], q["presence_penalty"] = 1.0, 0.0, 0.0
    q["repeat_last_n"], q["penalty_from"], q["softcap"] = 0, 0, 0.0
    return q


def sample_row(x, p, hist, u, bias=(), allowed=None, kcap=0):
    """dict(tok, keep, ids, probs, ncand) of one row: the oracle's sampler on the edited row, its candidates the logits above
    -inf. A row without one: token -1, nothing kept."""
    row = edit_row(x, p, hist, bias, allowed)
    is_cand = row > -np.inf
    if not is_cand.any():
        return dict(tok=-1, keep=0, ids=np.zeros(0, np.int32), probs=np.zeros(0), ncand=0)
    if p["temperature"] <= 0 or p["top_k"] == 1:
        tok = int(np.argmax(np.where(is_cand, row, -np.inf)))
        return dict(tok=tok, keep=1, ids=np.array([tok], np.int32), probs=np.ones(1), ncand=1)
    row[~is_cand] = np.nan
    tok, ids, probs, keep, ncand = O.sample(row, np.zeros(0, np.int32), neutral(p), u, max(kcap, min(x.size, 4096)))
    return dict(tok=tok, keep=keep, ids=ids, probs=probs, ncand=ncand)


def logprob_row(x, t=None, n=0, cap=0.0, T=1.0, bias=(), allowed=None):
    """(lp, rank, ids, top) of one row in fp64, on logits edited as the kernel edits them (fp32 bias sums)."""
    p = O.make_params(1, softcap=cap, repetition_penalty=1.0)[0]
    row = edit_row(x, p, [], bias, allowed)
    row[np.isnan(row)] = -np.inf
    live = np.flatnonzero(row > -np.inf)
    v = row.astype(np.float64)
    lp = np.full(row.size, -np.inf)
    if live.size:
        m = v.max()
        if np.isinf(m):
            lp[v == m] = -np.log((v == m).sum())
        else:
            d = (v[live] - m) / T
            lp[live] = d - np.log(np.exp(d).sum())
    out_lp, rank = -np.inf, 0
    if t is not None and 0 <= t < row.size and row[t] > -np.inf:
        out_lp, rank = lp[t], 1 + int((row > row[t]).sum())
    order = live[np.lexsort((live, -v[live]))][:n]
    ids = np.full(n, -1)
    top = np.full(n, -np.inf)
    ids[:order.size], top[:order.size] = order, lp[order]
    return out_lp, rank, ids, top


def masks(rng, kind, n, V):
    """Truth values [n, V]: "few" (a handful, low ids mostly), "most" (all but 3 %), "block" (one run of ids), "none" (nothing
    allowed), "last" (the last token alone)."""
    a = np.zeros((n, V), bool)
    for r in range(n):
        if kind == "few":
            a[r, rng.integers(0, max(V // 8, 1), min(V, 20))] = True
        elif kind == "most":
            a[r] = rng.random(V) >= 0.03
        elif kind == "block":
            lo = int(rng.integers(0, V))
            a[r, lo:lo + max(1, V // 5)] = True
        elif kind == "last":
            a[r, V - 1] = True
    return a


def bias_lists(rng, S, V, n):
    """S lists of about n (id, value), ids ascending and some of them twice."""
    out = []
    for _ in range(S):
        ids = np.sort(rng.integers(0, V, int(rng.integers(0, 2 * n + 1))))
        out.append([(int(t), float(np.float32(rng.choice([rng.uniform(-4, 4), -100.0, -np.inf], p=[0.8, 0.15, 0.05])))) for t in ids])
    return out


def csr(lists):
    off = np.zeros(len(lists) + 1, np.int64)
    off[1:] = np.cumsum([len(r) for r in lists])
    flat = [e for r in lists for e in r]
    return np.array([t for t, _ in flat], np.int32), np.array([b for _, b in flat], np.float32), off
