"""Beam search: selection over a stream's beams and tokens, histories and model states following their beams, with plain forms.

A program that searches instead of sampling keeps n beams per stream (a stream is one request). A step selects the best
continuations of a stream's beams over the whole vocabulary, gives each new beam its parent's history with the token behind
it, and gives its cache rows what the parent's held. The cases below call the C ABI of include/ferro_sampler.h through the
package's ctypes binding, with device pointers the program already holds; with `own` false the same results come from
elementary torch operations.

Selection: row r of a stream has the score a_r, and its token t the candidate
    c(r, t) = a_r + (x_t - max x) / T - log sum_j exp((x_j - max x) / T),    x = logit + bias over the allowed tokens.
The n best that do not end the text are the new beams; those that do (eos) are ended hypotheses where fewer than n
candidates of any kind come before them. Equal candidates: those that end the text first, then the lower row, in a row the
larger logit, then the lower token. Beams come by score, or with `slots` in their parents' places: a parent's best child in the parent's slot, the
others in the free ones, ascending, so that a state is copied only for a parent's further children.
"""
import ctypes
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1}


def _select(name, S, W, n, V, **kw):
    """S streams of W rows, n new beams each, V logits per row. mask: as a grammar makes them, "keys" (a handful to a few
    hundred tokens), "text" (all but a few per cent) or "mixed" (both kinds and unmasked rows); NB biases per stream (on the
    average, ragged); dead: rows of each stream whose beam has ended (score -inf)."""
    c = dict(name=name, call="select", S=S, W=W, n=n, V=V, type="f32", T=1.0, mask="none", NB=0, eos=True, slots=True, dead=0)
    c.update(kw)
    return c


def _hist(name, S, W, n, H, **kw):
    """Histories of H ids on the average (ragged over the streams; a stream's beams are of one length)."""
    c = dict(name=name, call="hist", S=S, W=W, n=n, H=H)
    c.update(kw)
    return c


def _states(name, S, W, n, N, **kw):
    """N state buffers of S * W rows (in place: n = W; else S * n rows in another buffer). layout "fixed": `heads` blocks of
    `dim` values a row; "heads": a cache [rows, heads, cap, dim], "tokens": [rows, cap, heads, dim], of which positions
    from the prompt's end (`prompt`, ragged) to the present length (L, ragged) differ between the beams of a stream.
    pad: values between one row and the next."""
    c = dict(name=name, call="states", S=S, W=W, n=n, N=N, layout="heads", heads=8, dim=64, cap=1024, prompt=0, L=0, pad=0,
             type="bf16", place=True)
    c.update(kw)
    return c


def listed():
    return [
        # one interactive request, four beams on a small vocabulary: latency
        _select("beam_single", 1, 4, 4, 65536),
        # the step behind the prompts: one row per stream opens its beams
        _select("beam_first", 16, 1, 8, 262144, slots=False),
        # the serving batch: 16 requests of four beams on the large vocabulary
        _select("beam_serving", 16, 4, 4, 262144, T=0.9),
        # structured output: half of the beams inside a grammar, biases per request, two beams of each request ended
        _select("beam_grammar", 8, 8, 8, 151936, mask="mixed", NB=30, dead=2),
        # n-best lists: the widest beams, fp16 logits, an odd vocabulary, best first
        _select("beam_wide", 2, 64, 64, 100003, type="f16", slots=False),
        # batch translation of many documents from bf16 logits
        _select("beam_batch", 128, 8, 8, 151936, type="bf16"),
        # the histories of one request
        _hist("hist_single", 1, 4, 4, 300),
        # of a serving batch
        _hist("hist_serving", 64, 8, 8, 2048),
        # of long documents, 33 MB in and out
        _hist("hist_long", 32, 8, 8, 32768),
        # convolution states of one request: small fixed buffers of many layers
        _states("states_conv", 1, 4, 4, 20, layout="fixed", heads=1, dim=4096, type="f32"),
        # keys and values of a serving batch, in place
        _states("states_serving", 16, 4, 4, 16, prompt=256, L=768),
        # prompt caches opened into beams, another buffer
        _states("states_expand", 16, 1, 4, 16, layout="tokens", cap=1024, L=1000, place=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same kinds: every size over its range, odd ones among them."""
    call = rng.choice(["select", "select", "hist", "states"])
    n = rng.choice([rng.randint(2, 8), rng.randint(2, 16), _log_int(rng, 1, 64)])
    W = rng.choice([n, n, n, 1])
    if call == "select":
        V = rng.choice([65536, 262144, 151936, rng.randint(32000, 262144), rng.randint(1000, 262144)])
        S = _log_int(rng, 1, max(1, min(256, (1 << 26) // V // W)))
        c = _select("", S, W, n, V, type=rng.choice(["f32", "bf16", "f16"]), T=rng.choice([1.0, round(rng.uniform(0.5, 1.5), 2)]),
                    mask=rng.choice(["none", "none", "keys", "text", "mixed"]), NB=rng.choice([0, 0, _log_int(rng, 1, 300)]),
                    eos=rng.random() < 0.8, slots=rng.random() < 0.6, dead=rng.randint(0, W // 3))
    elif call == "hist":
        H = _log_int(rng, 16, 32768)
        c = _hist("", _log_int(rng, 1, max(1, min(256, (1 << 23) // H // max(n, W)))), W, n, H)
    else:
        layout = rng.choice(["fixed", "heads", "tokens"])
        heads, dim, N = rng.choice([1, 2, 4, 8, rng.randint(1, 16)]), rng.choice([64, 128, rng.randint(20, 200)]), rng.randint(1, 32)
        cap = 1 if layout == "fixed" else _log_int(rng, 64, 4096)
        dim = rng.choice([1024, 4096, rng.randint(100, 9000)]) if layout == "fixed" else dim
        kind = rng.choice(["bf16", "f16", "f32", "u8"])
        place = W == n and rng.random() < 0.6
        row = heads * dim * cap * SIZES[kind] * N * (n if place else n + W)
        S = _log_int(rng, 1, max(1, min(128, (1 << 30) // row)))
        while row * S > (1 << 30) and N > 1:
            row, N = row // N * (N - 1), N - 1
        L = rng.randint(1, cap)
        c = _states("", S, W, n, N, layout=layout, heads=heads, dim=dim, cap=cap, L=L, prompt=rng.choice([0, rng.randint(0, L)]),
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), type=kind, place=place)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _ragged(rs, S, n):
    """S lengths with mean n: from a quarter of n to 7/4 of it."""
    if S == 1 or n == 0:
        return np.full(S, n, np.int64)
    return rs.permutation(np.linspace(n // 4, 2 * n - n // 4, S).astype(np.int64))


def _offsets(n):
    off = np.zeros(len(n) + 1, np.int64)
    off[1:] = np.cumsum(n)
    return off


def _masks(case, R, rs, g):
    """(words [n, words of V bits] int32, mask of each row, -1: none). Bit t % 32 of word t / 32: token t is allowed."""
    V = case["V"]
    words = (V + 31) // 32
    kinds = {"keys": [1], "text": [2], "mixed": [0, 1, 2, 1, 0, 2]}[case["mask"]]
    kind = rs.permutation(np.resize(kinds, R))
    of = np.full(R, -1, np.int32)
    of[kind > 0] = np.arange(int((kind > 0).sum()), dtype=np.int32)
    n, kind = int((kind > 0).sum()), kind[kind > 0]
    ok = torch.zeros((n, words * 32), dtype=torch.bool, device="cuda")
    for m in range(n):
        if kind[m] == 2:
            ok[m] = torch.rand(words * 32, device="cuda", generator=g) >= 0.03
        else:                                      # most structural tokens sit low in the vocabulary
            c = int(np.exp(rs.uniform(math.log(4.0), math.log(300.0))))
            t = np.where(rs.random_sample(c) < 0.7, rs.randint(0, max(1, V // 64), c), rs.randint(0, V, c))
            ok[m, torch.from_numpy(t).cuda()] = True
    bit = 1 << torch.arange(32, dtype=torch.int64, device="cuda")
    out = torch.zeros((max(n, 1), words), dtype=torch.int32, device="cuda")
    for a in range(0, n, 32):
        out[a:a + 32][:min(32, n - a)] = (ok[a:a + 32].view(-1, words, 32) * bit).sum(2).to(torch.int32)
    return out, of


def _moved(W):
    """(beams of a stream that are copies, parents they are copies of) where beams keep their slots."""
    m = W // 2
    return m, min(m, max(1, (W - m) // 2)) if m else 0


def _parents(case, rs):
    """[S, n] parents as a selection leaves them. In place the beams keep their slots: a parent stays where it is and the
    slots of half of the beams are given to further children of others. Else by score: any order."""
    S, W, n = case["S"], case["W"], case["n"]
    p = np.zeros((S, n), np.int32)
    for s in range(S):
        if W == n and case.get("place", False):
            m, d = _moved(W)
            at = rs.permutation(W)
            p[s] = np.arange(W)
            if m:
                p[s, at[:m]] = at[m:][np.arange(m) % d]
        else:
            p[s] = np.minimum(rs.geometric(min(1.0, 2.0 / max(W, 1)), n) - 1, W - 1)
            p[s] = rs.permutation(p[s])
    return p


def _inputs(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator("cuda").manual_seed(seed)
    S, W, n = case["S"], case["W"], case["n"]
    d = {"case": case}
    if case["call"] == "select":
        V, R = case["V"], S * W
        ld = -(-V // 128) * 128                    # an lm_head writes its rows padded to a multiple of 128
        x = torch.randn(R, ld, device="cuda", generator=g) * 2.0
        at = torch.randint(0, V, (R, 12), device="cuda", generator=g)       # a dozen tokens of each row stand out
        x.scatter_add_(1, at, 5.0 + 3.0 * torch.randn(R, 12, device="cuda", generator=g))
        eos = int(rs.randint(0, min(V, 1000)))
        if case["eos"]:                            # the text may well end at some beams
            x[:, eos] += torch.from_numpy(np.where(rs.random_sample(R) < 0.4, 12.0, 0.0).astype(np.float32)).cuda()
        d["x"], d["ld"], d["eos"] = x.to(DTYPES[case["type"]]), ld, eos if case["eos"] else -1
        a = -rs.uniform(2.0, 60.0, (S, 1)) - rs.exponential(1.5, (S, W))
        for s in range(S):
            a[s, rs.permutation(W)[:case["dead"]]] = -np.inf
        d["score"] = torch.from_numpy(a.reshape(-1).astype(np.float32)).cuda()
        if case["mask"] != "none":
            d["mask"], of = _masks(case, R, rs, g)
            d["mask_of"] = torch.from_numpy(of).cuda()
        if case["NB"]:
            ids = [np.unique(rs.randint(0, V, int(k))).astype(np.int32) for k in _ragged(rs, S, case["NB"])]
            off = _offsets([len(i) for i in ids])
            ids = np.concatenate(ids)
            val = rs.uniform(-3.0, 3.0, ids.size).astype(np.float32)
            val[rs.random_sample(ids.size) < 0.2] = -100.0
            d["b_ids"], d["b_val"], d["b_off"] = (torch.from_numpy(t).cuda() for t in (ids, val, off))
            d["n_bias"] = int(off[-1])
        d["row_off"] = torch.arange(0, R + 1, W, dtype=torch.int64, device="cuda")
        return d
    p = _parents(case, rs)
    d["parent"] = torch.from_numpy(p.reshape(-1)).cuda()
    if case["call"] == "hist":
        H = np.repeat(_ragged(rs, S, case["H"]), W)
        off = _offsets(H)
        d["hist"] = torch.from_numpy(rs.randint(0, 65536, int(off[-1])).astype(np.int32)).cuda()
        d["off"] = torch.from_numpy(off).cuda()
        d["row_off"] = torch.arange(0, S * W + 1, W, dtype=torch.int64, device="cuda")
        d["tok"] = torch.from_numpy(rs.randint(0, 65536, S * n).astype(np.int32)).cuda()
        d["n_out"] = int(sum(H.reshape(S, W)[np.arange(S)[:, None], p].reshape(-1) + 1))
        return d
    heads, dim, cap, pad = case["heads"], case["dim"], case["cap"], case["pad"]

    def buffers(rows, fill):
        out = []
        for _ in range(case["N"]):
            shape = (heads, cap, dim) if case["layout"] != "tokens" else (cap, heads, dim)
            flat = torch.zeros((rows, heads * cap * dim + pad), dtype=DTYPES[case["type"]], device="cuda")
            if fill and case["type"] == "u8":
                flat.copy_(torch.randint(0, 256, flat.shape, device="cuda", generator=g, dtype=torch.uint8))
            elif fill:
                flat.copy_(torch.randn(flat.shape, device="cuda", generator=g))
            out.append(flat[:, :heads * cap * dim].view(rows, *shape))
        return out

    d["src"] = buffers(S * W, True)
    d["dst"] = d["src"] if case["place"] else buffers(S * n, False)
    L = np.minimum(_ragged(rs, S, case["L"]), cap) if case["layout"] != "fixed" else np.ones(S, np.int64)
    d["len"] = torch.from_numpy(L.astype(np.int32)).cuda()
    d["from"] = torch.from_numpy(np.minimum(_ragged(rs, S, case["prompt"]), L).astype(np.int32)).cuda()
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        _bind(d)
    return d


# ------------------------------------------------------------------------------------------------ the framework's calls
def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _bind(d):
    """The call's argument list, as a program holds it from step to step."""
    import ferro_amd as F
    from ferro_amd._lib import check, lib
    c = d["case"]
    S, W, n = c["S"], c["W"], c["n"]
    ctx = F.Context.default()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    i32 = functools.partial(torch.zeros, dtype=torch.int32, device="cuda")
    f32 = functools.partial(torch.zeros, dtype=torch.float32, device="cuda")
    keep = [ctx]
    if c["call"] == "select":
        hp = np.zeros(S, F.PARAMS_DTYPE)
        hp["temperature"] = c["T"]
        rec = torch.from_numpy(hp.view(np.uint8).copy()).cuda()
        e = None
        if c["mask"] != "none" or c["NB"]:
            ed = F.Edits(mask=d.get("mask"), mask_of=d.get("mask_of"),
                         bias=(d["b_ids"], d["b_val"], d["b_off"]) if c["NB"] else None)
            e = ctypes.byref(ed.c)
            keep.append(ed)
        out = {"parent": i32((S, n)), "tok": i32((S, n)), "score": f32((S, n)), "done": i32(S), "done_parent": i32((S, n)),
               "done_score": f32((S, n))}
        kind = {"f32": F.F32, "bf16": F.BF16, "f16": F.F16}[c["type"]]
        fn, args = lib().fs_beam_select, (
            ctx.h, _ptr(d["x"]), kind, d["ld"], S, S * W, c["V"], _ptr(d["row_off"]), _ptr(d["score"]), _ptr(rec), e, d["eos"],
            n, F.BEAM_KEEP_SLOTS if c["slots"] else 0, _ptr(out["parent"]), _ptr(out["tok"]), _ptr(out["score"]),
            _ptr(out["done"]), _ptr(out["done_parent"]), _ptr(out["done_score"]), stream)
        keep.append(rec)
    elif c["call"] == "hist":
        out = {"hist": i32(d["n_out"]), "off": torch.zeros(S * n + 1, dtype=torch.int64, device="cuda")}
        fn, args = lib().fs_hist_fork, (
            ctx.h, S, _ptr(d["hist"]), _ptr(d["off"]), _ptr(d["row_off"]), n, _ptr(d["parent"]), _ptr(d["tok"]),
            _ptr(out["hist"]), d["n_out"], _ptr(out["off"]), stream)
    else:
        states = F.States(d["src"], dst=d["dst"], pos_dim={"fixed": None, "heads": 2, "tokens": 1}[c["layout"]])
        out = d["dst"]
        fn, args = lib().fs_reorder_states, (
            ctx.h, len(states), states.c, S, W, n, _ptr(d["parent"]), _ptr(d["from"]), _ptr(d["len"]), stream)
        keep.append(states)
    d["own"] = (functools.partial(fn, *args), out, check, keep)


# ------------------------------------------------------------------------------------------------ the plain forms
def _allowed(d):
    """[R, V] truth values."""
    t = torch.arange(d["case"]["V"], device="cuda")
    rows = [((words[:, t >> 5] >> (t & 31).to(torch.int32)) & 1).bool() for words in d["mask"].split(16)]
    rows.append(torch.ones((1, d["case"]["V"]), dtype=torch.bool, device="cuda"))       # mask -1: the last row
    return torch.cat(rows)[d["mask_of"].long()]


def _plain_select(d):
    c = d["case"]
    S, W, n, V = c["S"], c["W"], c["n"], c["V"]
    x = d["x"][:, :V].float()
    if c["NB"]:
        k = d["b_off"][1:] - d["b_off"][:-1]
        b = torch.zeros((S, V), device="cuda")
        b[torch.repeat_interleave(torch.arange(S, device="cuda"), k, output_size=d["n_bias"]), d["b_ids"].long()] = d["b_val"]
        x = x + b.repeat_interleave(W, 0)
    if c["mask"] != "none":
        x = x.masked_fill(~_allowed(d), -math.inf)
    T = torch.full((), c["T"], dtype=torch.float32, device="cuda").double()
    m = x.max(1, keepdim=True).values.clamp(min=-3e38).double()
    z = torch.log(torch.cat([torch.exp((r.double() - mr) / T).sum(1, keepdim=True)
                             for r, mr in zip(x.split(64), m.split(64))]))
    a = d["score"][:, None].double()
    score = lambda v: a + ((v.double() - m) / T - z)
    # a row's best tokens but eos, and eos by itself (before others of its score)
    if c["eos"]:
        e = score(x[:, d["eos"]:d["eos"] + 1])
        x = x.clone() if x.data_ptr() == d["x"].data_ptr() else x      # (the logits are read only)
        x[:, d["eos"]] = -math.inf
    v, idx = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(n, V)
    v, idx = v[:, :k], idx[:, :k]
    cand = torch.where(v > -math.inf, score(v), -math.inf)
    cand, at = torch.sort(cand.view(S, W * k), dim=1, descending=True, stable=True)     # by row, then by logit
    if W * k < n:
        cand = torch.nn.functional.pad(cand, (0, n - W * k), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, n - W * k))
    cand, at = cand[:, :n], at[:, :n]
    live = cand.float() > -math.inf
    parent = torch.where(live, at // k, -1).to(torch.int32)
    tok = torch.where(live, torch.gather(idx.reshape(S, W * k), 1, at), -1).to(torch.int32)
    best = torch.where(live, cand.float(), -math.inf)
    done = torch.zeros(S, dtype=torch.int32, device="cuda")
    done_parent = torch.full((S, n), -1, dtype=torch.int32, device="cuda")
    done_score = torch.full((S, n), -math.inf, device="cuda")
    if c["eos"]:
        e = e.view(S, W)
        e, row = torch.sort(torch.where(e.float() > -math.inf, e, -math.inf), dim=1, descending=True, stable=True)
        before = torch.arange(W, device="cuda")[None] + (cand[:, None, :] > e[:, :, None]).sum(2)
        ended = (e > -math.inf) & (before < n)
        done = ended.sum(1).to(torch.int32)
        k = min(W, n)
        done_parent[:, :k] = torch.where(ended, row, -1)[:, :k].to(torch.int32)
        done_score[:, :k] = torch.where(ended, e, -math.inf)[:, :k].float()
    if c["slots"]:
        i = torch.arange(n, device="cuda")
        earlier = ((parent[:, :, None] == parent[:, None, :]) & (i[None, :] < i[:, None])).any(2)
        first = live & ~earlier & (parent < n)
        used = torch.zeros((S, n + 1), dtype=torch.bool, device="cuda")
        used.scatter_(1, torch.where(first, parent, n).long(), True)
        free = torch.sort(used[:, :n].int(), dim=1, stable=True).indices
        turn = torch.cumsum((~first).int(), 1) - 1
        slot = torch.where(first, parent.long(), torch.gather(free, 1, turn.clamp(min=0).long()))
        parent, tok, best = (torch.empty_like(t).scatter_(1, slot, t) for t in (parent, tok, best))
    return {"parent": parent, "tok": tok, "score": best, "done": done, "done_parent": done_parent, "done_score": done_score}


def _plain_hist(d):
    c = d["case"]
    S, W, n = c["S"], c["W"], c["n"]
    row = torch.arange(S, device="cuda").repeat_interleave(n) * W + d["parent"].long()
    length = (d["off"][1:] - d["off"][:-1])[row]
    off = torch.zeros(S * n + 1, dtype=torch.int64, device="cuda")
    off[1:] = torch.cumsum(length + 1, 0)
    of = torch.repeat_interleave(torch.arange(S * n, device="cuda"), length + 1, output_size=d["n_out"])
    i = torch.arange(d["n_out"], device="cuda") - off[of]
    at = d["off"][row[of]] + torch.minimum(i, (length[of] - 1).clamp(min=0))
    ids = torch.where(i < length[of], d["hist"][at.clamp(max=d["hist"].numel() - 1)], d["tok"][of])
    return {"hist": ids, "off": off}


def _plain_states(d):
    c = d["case"]
    S, W, n = c["S"], c["W"], c["n"]
    row = torch.arange(S, device="cuda").repeat_interleave(n) * W + d["parent"].long()
    fixed = c["layout"] == "fixed"
    i = torch.arange(c["cap"], device="cuda")
    of = torch.arange(S, device="cuda").repeat_interleave(n)
    mine = (i[None] >= d["from"][of][:, None]) & (i[None] < d["len"][of][:, None])
    mine = mine.view(S * n, 1, -1, 1) if c["layout"] == "heads" else mine.view(S * n, -1, 1, 1)
    for src, dst in zip(d["src"], d["dst"]):
        new = src[row]
        dst.copy_(new if fixed else torch.where(mine, new, dst))
    return d["dst"]


def run(state):
    if own:
        fn, out, check, _ = state["own"]
        check(fn(), state["case"]["call"])
        return out
    return {"select": _plain_select, "hist": _plain_hist, "states": _plain_states}[state["case"]["call"]](state)


# ------------------------------------------------------------------------------------------------ what is compared
def work(case):
    S, W, n = case["S"], case["W"], case["n"]
    if case["call"] == "select":
        R, V, size = S * (W - case["dead"]), case["V"], SIZES[case["type"]]
        masked, few = {"none": (0.0, 0.0), "keys": (1.0, 1.0), "text": (1.0, 0.0), "mixed": (4 / 6, 2 / 6)}[case["mask"]]
        read = R * (V * (1.0 - masked + 0.97 * (masked - few)) + 80 * few)
        return {"bytes": int(read * size + R * masked * V / 8 + 8 * S * case["NB"] + 4 * S * W + 20 * S * n),
                "flops": int(4 * read)}
    if case["call"] == "hist":
        # (parents by a geometric law: about half of a stream's beams have children)
        read = S * (W if W == 1 else (W + 1) // 2) * case["H"]
        return {"bytes": int(4 * read + 4 * S * n * (case["H"] + 1) + 12 * S * n), "flops": 0}
    used = case["dim"] * case["heads"] * SIZES[case["type"]]
    if case["layout"] != "fixed":
        used *= max(0, min(case["L"], case["cap"]) - case["prompt"])
    m, d = _moved(W) if case["place"] else (n, 1 if W == 1 else (W + 1) // 2)
    return {"bytes": int(case["N"] * S * used * (m + d) + 4 * S * n), "flops": 0}


def exact(case, seed):
    """The new beams' and the ended hypotheses' scores in 64 bits, stream by stream; ids, counts and copies have no such
    value."""
    if case["call"] != "select":
        return None
    d = _inputs(case, seed)
    S, W, n, V = case["S"], case["W"], case["n"], case["V"]
    T = float(np.float32(case["T"]))
    off = d["b_off"].cpu().numpy() if case["NB"] else None
    of = d["mask_of"].cpu().numpy() if case["mask"] != "none" else None
    shift = torch.arange(32, dtype=torch.int32, device="cuda")
    best = np.full((S, n), -np.inf)
    ended = np.full((S, n), -np.inf)
    a = d["score"].cpu().numpy().astype(np.float64)
    for s in range(S):
        rows, eos = [], []
        for w in range(W):
            r = s * W + w
            if a[r] == -np.inf:
                continue
            x = d["x"][r, :V].double()
            if off is not None:
                at = slice(int(off[s]), int(off[s + 1]))
                x[d["b_ids"][at].long()] = (x[d["b_ids"][at].long()] + d["b_val"][at].double()).float().double()
            if of is not None and of[r] >= 0:
                x[((d["mask"][int(of[r])][:, None] >> shift) & 1).reshape(-1)[:V] == 0] = -math.inf
            lp = torch.log_softmax(x / T, 0) + a[r]
            if case["eos"]:
                eos.append((float(lp[d["eos"]]), w))
                lp[d["eos"]] = -math.inf
            top = torch.topk(lp, min(n, V))
            rows += [(v, w, i) for i, v in enumerate(top.values.cpu().tolist())]
        rows = [e for e in sorted(rows, key=lambda e: (-e[0], e[1], e[2])) if e[0] > -np.inf][:n]
        eos = sorted((e for e in eos if e[0] > -np.inf), key=lambda e: (-e[0], e[1]))
        k = 0
        for i, (v, _) in enumerate(eos):
            if i + sum(e[0] > v for e in rows) < n:
                ended[s, k] = v
                k += 1
        at = list(range(len(rows)))
        if case["slots"]:
            taken, late = {}, []
            for j, (_, w, _) in enumerate(rows):
                if w < n and w not in taken:
                    taken[w] = j
                else:
                    late.append(j)
            free = [i for i in range(n) if i not in taken]
            at = [0] * len(rows)
            for slot, j in list(taken.items()) + list(zip(free, late)):
                at[j] = slot
        for j, (v, _, _) in enumerate(rows):
            best[s, at[j]] = v
    score, done = (torch.from_numpy(t).cuda() for t in (best, ended))
    return {"parent": None, "tok": None, "score": score, "done": None, "done_parent": None, "done_score": done}
