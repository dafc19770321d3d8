"""Logit edits, sampling under them and log-probabilities: the calls a serving program makes, with their plain forms.

A program that serves structured output, tool calls and OpenAI-style `logit_bias` / `logprobs` holds, beside the logits,
a bitmask of the tokens that a row's grammar allows and a short list of (token, bias) pairs per request. The cases below
call the C ABI of include/ferro_sampler.h through the package's ctypes binding, with device pointers the program already
holds; with `own` false the same results come from elementary torch operations.

An edited logit is pen(cap(l) + bias): the model's final softcap, the request's bias, then the repetition and the
frequency / presence penalties over the row's history, each step rounded to fp32 as ferro's sampler rounds its steps; a
token whose mask bit is 0, or whose edited logit is NaN or -inf, is no candidate.
"""
import ctypes
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PARAMS = dict(T=1.0, k=0, p=1.0, min_p=0.0, rep=1.0, freq=0.0, pres=0.0, last_n=-1, softcap=0.0)


def _case(name, call, B, V, **kw):
    """call: the entry point. B rows (verify: streams of M rows) of V logits, H history ids per row, NB biases per row (both
    on the average, ragged). mask: "none", "keys" (a grammar's structural position: a handful to a few hundred tokens),
    "text" (inside a string: all but a few per cent) or "mixed" (rows of both kinds and unmasked ones). mixed: every
    row has parameters of its own. kcap: candidates returned; n: the largest log-probabilities returned."""
    c = dict(name=name, call=call, B=B, V=V, M=1, H=0, NB=0, mask="none", type="f32", logits="mixture", mixed=False,
             kcap=0, n=0)
    c.update(PARAMS)
    c.update(kw)
    return c


def listed():
    return [
        # one interactive tool call: a single row at a position where the grammar allows few tokens
        _case("tool_call_row", "sample", 1, 65536, H=256, mask="keys", logits="spikes", T=0.7, k=40, p=0.95, rep=1.1, kcap=5),
        # deterministic structured output: a small greedy batch with frequency / presence penalties
        _case("json_greedy", "sample", 8, 65536, H=256, NB=4, mask="mixed", logits="normal", T=0.0, freq=0.5, pres=0.3),
        # the serving batch: 64 sessions on the large vocabulary, some in a grammar, some with biases, the candidates'
        # probabilities returned
        _case("json_serving", "sample", 64, 262144, H=512, NB=8, mask="mixed", T=0.8, k=64, p=0.95, rep=1.05, kcap=64),
        # speculative decoding of structured output: every row of a window has the mask its drafts lead to
        _case("verify_grammar", "verify", 16, 65536, M=17, H=64, mask="text", logits="normal", T=0.0),
        # top-p alone (top_k = 0), the usual setting of OpenAI-style clients, half of them in a grammar
        _case("nucleus_grammar", "sample", 32, 151936, H=300, mask="mixed", T=0.8, p=0.95, pres=0.2),
        # clients that each set their own parameters and long bias lists, on a large batch
        _case("mixed_clients", "sample", 256, 262144, H=1024, NB=100, mask="mixed", mixed=True),
        # the edited row itself, for a program that samples on the host or reads the row back
        _case("edit_row", "edit", 1, 65536, H=512, NB=16, mask="text", rep=1.1),
        # a bf16 head's logits made fp32 on the way, the whole batch edited for a sampler of the program's own
        _case("edit_bf16", "edit", 64, 262144, H=512, NB=30, mask="mixed", type="bf16", rep=1.05, freq=0.2, pres=0.1),
        # fp16 logits with the final softcap, odd vocabulary, long histories
        _case("edit_f16_capped", "edit", 24, 100003, H=4096, NB=300, mask="text", type="f16", rep=1.2, softcap=30.0),
        # the probability of one sampled token and the top five, for a single streamed answer
        _case("logprobs_row", "logprobs", 1, 65536, n=5),
        # the same for a serving batch, under the masks and biases the tokens were sampled with, top 20
        _case("logprobs_serving", "logprobs", 64, 262144, NB=8, mask="mixed", n=20, T=0.8),
        # scoring a prompt (or a rollout): every position's next token, from bf16 logits
        _case("score_prompt", "logprobs", 1024, 151936, type="bf16", n=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same kinds: every size over its range, odd ones among them."""
    c = dict(rng.choice(listed()))
    del c["name"]
    c["V"] = V = rng.choice([65536, 262144, rng.randint(32000, 262144), rng.randint(1000, 262144)])
    c["mask"] = rng.choice(["none", "keys", "text", "mixed", "mixed"])
    if c["call"] == "logprobs":
        c["type"] = rng.choice(["f32", "bf16", "f16"])
        c["n"] = rng.choice([0, 1, rng.randint(2, 20)])
        c["B"] = _log_int(rng, 1, max(1, min(1024, (1 << 27) // V)))
        c["T"] = rng.choice([1.0, round(rng.uniform(0.3, 1.5), 2)])
        c["NB"] = rng.choice([0, _log_int(rng, 1, 300)])
        return c
    c["H"] = _log_int(rng, 16, 2048)
    c["NB"] = rng.choice([0, _log_int(rng, 1, 300)])
    if c["call"] == "verify":
        c["M"] = rng.randint(2, 17)
    c["B"] = max(1, _log_int(rng, 1, max(1, min(256, (1 << 24) // V))) // c["M"])
    if c["call"] == "edit":
        c["type"] = rng.choice(["f32", "bf16", "f16"])
        c["softcap"] = rng.choice([0.0, 0.0, 30.0])
        c["rep"] = rng.choice([1.0, round(rng.uniform(0.9, 1.3), 2)])
        c["freq"] = rng.choice([0.0, round(rng.uniform(-0.5, 1.0), 2)])
    elif not c["mixed"] and c["T"] > 0:
        c["T"] = round(rng.uniform(0.3, 1.3), 2)
        c["k"] = rng.choice([0, rng.randint(10, 64), rng.randint(10, 64), _log_int(rng, 65, 1024)])
        c["p"] = rng.choice([1.0, round(rng.uniform(0.8, 1.0), 3)])
        c["rep"] = rng.choice([1.0, round(rng.uniform(0.95, 1.3), 2)])
        c["last_n"] = rng.choice([-1, -1, 64])
    if c["call"] == "sample":
        c["kcap"] = rng.choice([0, rng.randint(1, 64)]) if c["k"] else 0
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _logits(case, R, ld, g):
    randn = functools.partial(torch.randn, dtype=torch.float32, device="cuda", generator=g)
    if case["logits"] == "mixture":    # 90% N(0, 1.5), 10% Student-t(3) * 4
        x = randn(R, ld)
        chi = randn(R, ld).square_().add_(randn(R, ld).square_()).add_(randn(R, ld).square_())
        pick = torch.rand((R, ld), device="cuda", generator=g) < 0.1
        x = torch.where(pick, 4.0 * x * torch.rsqrt(chi / 3.0), 1.5 * x)
    else:
        x = 2.0 * randn(R, ld)
        if case["logits"] == "spikes":  # 8 tokens of each row stand out by 12
            at = torch.randint(0, case["V"], (R, 8), device="cuda", generator=g)
            x.scatter_add_(1, at, torch.full((R, 8), 12.0, device="cuda"))
    return x.clamp_(-60000.0, 60000.0).to(DTYPES[case["type"]])


def _ragged(rs, S, n):
    """S lengths with mean n: from a quarter of n to 7/4 of it."""
    if S == 1 or n == 0:
        return np.full(S, n, np.int64)
    return rs.permutation(np.linspace(n // 4, 2 * n - n // 4, S).astype(np.int64))


def _offsets(n):
    off = np.zeros(len(n) + 1, np.int64)
    off[1:] = np.cumsum(n)
    return off


def _histories(case, rs):
    """CSR histories of Zipf(1.1) ids."""
    S, V = case["B"], case["V"]
    off = _offsets(_ragged(rs, S, case["H"]))
    cdf = np.cumsum(np.arange(1, V + 1, dtype=np.float64) ** -1.1)
    ids = np.searchsorted(cdf, rs.random_sample(int(off[-1])) * cdf[-1]).clip(0, V - 1).astype(np.int32)
    return ids, off


def _biases(case, rs):
    """CSR biases, ids ascending within a row: a fifth of them bans (-100), the others push a token up or down."""
    S, V = case["B"], case["V"]
    rows = [np.unique(rs.randint(0, V, int(n))).astype(np.int32) for n in _ragged(rs, S, case["NB"])]
    ids = np.concatenate(rows) if rows else np.zeros(0, np.int32)
    val = rs.uniform(-3.0, 3.0, ids.size).astype(np.float32)
    val[rs.random_sample(ids.size) < 0.2] = -100.0
    return ids, val, _offsets([r.size for r in rows])


def _masks(case, R, rs, g):
    """(words [n, W] int32, mask of each row, -1: none). Bit t % 32 of word t / 32: token t is allowed."""
    V = case["V"]
    W = (V + 31) // 32
    kinds = {"keys": [1], "text": [2], "mixed": [0, 1, 2, 1, 2, 2]}[case["mask"]]
    kind = rs.permutation(np.resize(kinds, R))
    of = np.full(R, -1, np.int32)
    of[kind > 0] = np.arange(int((kind > 0).sum()), dtype=np.int32)
    n = int((kind > 0).sum())
    kind = kind[kind > 0]
    at, tok = [], []
    for m in np.flatnonzero(kind == 1):            # most structural tokens sit low in the vocabulary
        c = int(np.exp(rs.uniform(math.log(4.0), math.log(300.0))))
        low = rs.random_sample(c) < 0.7
        tok.append(np.where(low, rs.randint(0, max(1, V // 64), c), rs.randint(0, V, c)))
        at.append(np.full(c, m))
    ok = torch.zeros((n, W * 32), dtype=torch.bool, device="cuda")
    if at:
        ok[torch.from_numpy(np.concatenate(at)).cuda(), torch.from_numpy(np.concatenate(tok)).cuda()] = True
    for m in np.flatnonzero(kind == 2):
        ok[int(m)] = torch.rand(W * 32, device="cuda", generator=g) >= 0.03
    bit = 1 << torch.arange(32, dtype=torch.int64, device="cuda")
    words = torch.empty((n, W), dtype=torch.int32, device="cuda")
    for a in range(0, n, 32):
        words[a:a + 32] = (ok[a:a + 32].view(-1, W, 32) * bit).sum(2).to(torch.int32)
    return words, of


def _params(case, rs):
    B = case["B"]
    p = {k: np.full(B, case[k], np.int32 if k in ("k", "last_n") else np.float32) for k in PARAMS}
    if case["mixed"]:
        T = rs.uniform(0.3, 1.5, B)
        T[rs.random_sample(B) < 0.05] = 0.0
        p["T"] = T.astype(np.float32)
        p["k"] = np.floor(np.exp(rs.uniform(0.0, math.log(2048.0), B))).astype(np.int32).clip(1, 2048)
        p["p"] = rs.uniform(0.8, 1.0, B).astype(np.float32)
        p["rep"] = rs.uniform(1.0, 1.3, B).astype(np.float32)
        p["freq"] = rs.uniform(0.0, 1.0, B).astype(np.float32)
        p["pres"] = rs.uniform(0.0, 1.0, B).astype(np.float32)
    return p


def _inputs(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator("cuda").manual_seed(seed)
    B, V, M = case["B"], case["V"], case["M"]
    R = B * M
    d = {"case": case, "ld": -(-V // 128) * 128}   # an lm_head writes its rows padded to a multiple of 128
    d["x"] = _logits(case, R, d["ld"], g)
    d["p"] = _params(case, rs)
    if case["H"]:
        ids, off = _histories(case, rs)
        d["hist"], d["off"], d["n_hist"] = torch.from_numpy(ids).cuda(), torch.from_numpy(off).cuda(), int(off[-1])
    if case["NB"]:
        ids, val, off = _biases(case, rs)
        d["b_ids"], d["b_val"], d["b_off"] = (torch.from_numpy(a).cuda() for a in (ids, val, off))
        d["n_bias"] = int(off[-1])
    if case["mask"] != "none":
        d["mask"], of = _masks(case, R, rs, g)
        d["mask_of"] = torch.from_numpy(of).cuda()
    if case["call"] in ("sample", "verify"):
        d["u"] = torch.from_numpy(rs.random_sample(R)).cuda()
    if case["call"] == "verify":       # a draft is a token the row may well emit four times out of five
        x = d["x"][:, :V].float()
        if "mask" in d:
            x = x.masked_fill(~_allowed(d), -math.inf)
        best = x.argmax(1).cpu().numpy().reshape(B, M)
        rows = rs.randint(0, V, (B, M))
        rows[:, 1:] = np.where(rs.random_sample((B, M - 1)) < 0.8, best[:, :-1], rows[:, 1:])
        d["rows"] = torch.from_numpy(rows.reshape(-1).astype(np.int32)).cuda()
        d["row_off"] = torch.arange(0, R + 1, M, dtype=torch.int64, device="cuda")
    if case["call"] == "logprobs":     # the token that was sampled or follows in the text: mostly a likely one
        top = d["x"][:, :V].float().argmax(1).cpu().numpy()
        d["tok"] = torch.from_numpy(np.where(rs.random_sample(R) < 0.5, top, rs.randint(0, V, R)).astype(np.int32)).cuda()
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["dp"] = {k: torch.from_numpy(v).cuda() for k, v in d["p"].items()}
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
    B, V, M, ld = c["B"], c["V"], c["M"], d["ld"]
    R = B * M
    hp = np.zeros(B, F.PARAMS_DTYPE)
    for field, key in (("temperature", "T"), ("top_k", "k"), ("top_p", "p"), ("min_p", "min_p"),
                       ("repetition_penalty", "rep"), ("frequency_penalty", "freq"), ("presence_penalty", "pres"),
                       ("repeat_last_n", "last_n"), ("softcap", "softcap")):
        hp[field] = d["p"][key]
    rec = torch.from_numpy(hp.view(np.uint8).copy()).cuda()
    ed = F.Edits(mask=d.get("mask"), mask_of=d.get("mask_of"),
                 bias=(d["b_ids"], d["b_val"], d["b_off"]) if c["NB"] else None)
    ctx = F.Context.default()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    i32 = functools.partial(torch.zeros, dtype=torch.int32, device="cuda")
    f32 = functools.partial(torch.zeros, dtype=torch.float32, device="cuda")
    hist, off, e = _ptr(d.get("hist")), _ptr(d.get("off")), ctypes.byref(ed.c)
    host = hp.ctypes.data_as(ctypes.c_void_p)
    kind = {"f32": F.F32, "bf16": F.BF16, "f16": F.F16}[c["type"]]
    if c["call"] == "sample":
        out = {"tok": i32(B), "keep": i32(B)}
        if c["kcap"]:
            out["ids"] = i32((B, c["kcap"]))
            out["probs"] = torch.zeros((B, c["kcap"]), dtype=torch.float64, device="cuda")
        fn, args = lib().fs_sample_edited, (
            ctx.h, _ptr(d["x"]), ld, B, V, hist, off, _ptr(rec), host, e, _ptr(d["u"]), _ptr(out["tok"]), c["kcap"],
            _ptr(out.get("ids")), _ptr(out.get("probs")), _ptr(out["keep"]), stream)
    elif c["call"] == "verify":
        out = {"tok": i32(R), "accepted": i32(B)}
        fn, args = lib().fs_verify_edited, (
            ctx.h, _ptr(d["x"]), ld, B, R, V, _ptr(d["rows"]), _ptr(d["row_off"]), hist, off, _ptr(rec), host, e,
            _ptr(d["u"]), -1, _ptr(out["tok"]), _ptr(out["accepted"]), stream)
    elif c["call"] == "edit":
        buf = f32((B, ld))
        out = {"logits": buf[:, :V]}
        fn, args = lib().fs_edit_batch, (ctx.h, _ptr(d["x"]), kind, ld, B, V, hist, off, _ptr(rec), e, _ptr(buf), ld, stream)
    else:
        out = {"lp": f32(B), "rank": i32(B)}
        if c["n"]:
            out.update(ids=i32((B, c["n"])), top=f32((B, c["n"])))
        fn, args = lib().fs_logprobs, (
            ctx.h, _ptr(d["x"]), kind, ld, B, V, _ptr(rec), e, _ptr(d["tok"]), c["n"], _ptr(out["lp"]), _ptr(out["rank"]),
            _ptr(out.get("ids")), _ptr(out.get("top")), stream)
    d["own"] = (functools.partial(fn, *args), out, check, (rec, hp, ed, ctx))


# ------------------------------------------------------------------------------------------------ the plain forms
def _allowed(d):
    """[R, V] truth values."""
    V = d["case"]["V"]
    t = torch.arange(V, device="cuda")
    rows = []
    for words in d["mask"].split(16):
        rows.append(((words[:, t >> 5] >> (t & 31).to(torch.int32)) & 1).bool())
    rows.append(torch.ones((1, V), dtype=torch.bool, device="cuda"))       # mask -1: the last row
    return torch.cat(rows)[d["mask_of"].long()]


def _row_of(off, total):
    """The row of each entry of a CSR list."""
    n = off[1:] - off[:-1]
    return torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=total)


def _counts(d):
    """[R, V] occurrences in each row's penalty window: the history's last ids and, in a window, the drafts fed before."""
    c = d["case"]
    B, V, M = c["B"], c["V"], c["M"]
    off, ids = d["off"], d["hist"].long()
    row = _row_of(off, d["n_hist"])
    if M == 1:
        if c["last_n"] > 0:
            fresh = torch.arange(d["n_hist"], device="cuda") >= off[1:][row] - c["last_n"]
            row, ids = row[fresh], ids[fresh]
        n = torch.zeros((B, V), device="cuda")
        n.index_put_((row, ids), torch.ones((), device="cuda"), accumulate=True)
        return n
    n = torch.zeros((B, M, V), device="cuda")
    for r in range(M):                             # row r's history: the stream's, then the drafts of rows 1 .. r
        i, s = ids, row
        if c["last_n"] > 0:
            fresh = torch.arange(d["n_hist"], device="cuda") >= off[1:][row] - (c["last_n"] - r)
            i, s = ids[fresh], row[fresh]
        n[:, r].index_put_((s, i), torch.ones((), device="cuda"), accumulate=True)
        fed = d["rows"].view(B, M)[:, 1:r + 1].long()
        if c["last_n"] > 0:
            fed = fed[:, max(0, r - c["last_n"]):]
        n[:, r].scatter_add_(1, fed, torch.ones(fed.shape, device="cuda"))
    return n.view(B * M, V)


def _edited(d, penalties=True):
    """The edited logits in fp32, and which tokens are candidates."""
    c = d["case"]
    V, M, p = c["V"], c["M"], d["dp"]
    x = d["x"][:, :V].float()
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    if c["NB"]:
        b = torch.zeros((c["B"], V), device="cuda")
        b[_row_of(d["b_off"], d["n_bias"]), d["b_ids"].long()] = d["b_val"]
        x = x + (b.repeat_interleave(M, 0) if M > 1 else b)
    if penalties and c["H"] and (c["mixed"] or c["rep"] != 1.0 or c["freq"] or c["pres"]):
        n = _counts(d)
        rep, freq, pres = (p[k].repeat_interleave(M)[:, None] for k in ("rep", "freq", "pres"))
        y = torch.where(rep != 1.0, torch.where(x > 0, x / rep, x * rep), x)
        y = y - (n * freq + pres)
        x = torch.where(n > 0, y, x)
    ok = x > -math.inf
    if c["mask"] != "none":
        ok = ok & _allowed(d)
    return x, ok


def _sample(d):
    """Token and kept count: candidates in the order (logit, lower id first), softmax in 64 bits, min-p, top-p, the draw."""
    c, p = d["case"], d["dp"]
    V, M = c["V"], c["M"]
    x, ok = _edited(d)
    x = x.masked_fill(~ok, -math.inf)
    v, idx = torch.sort(x, dim=1, descending=True, stable=True)
    T, k, top_p, min_p = (p[key].repeat_interleave(M)[:, None] for key in ("T", "k", "p", "min_p"))
    greedy = (T <= 0) | (k == 1)
    k = torch.where(greedy, 1, torch.where((k > 0) & (k < V), k, V))
    k = torch.minimum(k, ok.sum(1, keepdim=True))
    at = torch.arange(V, device="cuda")[None]
    e = torch.exp((v - v[:, :1]).double() / torch.where(greedy, 1.0, T).double())
    e = torch.where(at < k, e, 0.0)
    pr = e / e.sum(1, keepdim=True)
    keep = torch.where(min_p > 0, (pr >= pr[:, :1] * min_p.double()).sum(1, keepdim=True).clamp(min=1), k)
    keep = torch.minimum(keep, k)
    cs = torch.cumsum(pr, 1)
    past = torch.where(top_p < 1, (cs < top_p.double()).sum(1, keepdim=True) + 1, V)
    keep = torch.minimum(keep, past)
    r = d["u"][:, None] * torch.gather(cs, 1, (keep - 1).clamp(min=0).long())
    pick = torch.minimum((cs < r).sum(1, keepdim=True), keep - 1).clamp(min=0)
    tok = torch.gather(idx, 1, pick.long())
    tok = torch.where(k > 0, tok, -1)
    out = {"tok": tok[:, 0].to(torch.int32), "keep": torch.where(k > 0, keep, 0)[:, 0].to(torch.int32)}
    if c["kcap"]:
        n = c["kcap"]
        live = at[:, :n] < k
        out["ids"] = torch.where(live, idx[:, :n], 0).to(torch.int32)
        out["probs"] = torch.where(live, pr[:, :n], 0.0)
    return out


def _logprobs(d):
    c = d["case"]
    x, ok = _edited(d, penalties=False)
    x = x.masked_fill(~ok, -math.inf)
    T = d["dp"]["T"][:, None].double()
    m = x.max(1, keepdim=True).values
    z = torch.log(torch.exp((x - m) / T.float()).double().sum(1, keepdim=True))
    t = d["tok"].long()[:, None]
    xt = torch.gather(x, 1, t)
    lp = (xt - m).double() / T - z
    rank = torch.where(xt > -math.inf, (x > xt).sum(1, keepdim=True) + 1, 0)
    out = {"lp": lp[:, 0].float(), "rank": rank[:, 0].to(torch.int32)}
    if c["n"]:
        v, idx = torch.sort(x, dim=1, descending=True, stable=True)
        v, idx = v[:, :c["n"]], idx[:, :c["n"]]
        live = v > -math.inf
        out["ids"] = torch.where(live, idx, -1).to(torch.int32)
        out["top"] = ((v - m).double() / T - z).float()
    return out


def run(state):
    if own:
        fn, out, check, _ = state["own"]
        check(fn(), state["case"]["call"])
        return out
    c = state["case"]
    if c["call"] == "edit":
        x, ok = _edited(state)
        if c["mask"] != "none":
            x = x.masked_fill(~_allowed(state), -math.inf)
        return {"logits": x}
    if c["call"] == "logprobs":
        return _logprobs(state)
    out = _sample(state)
    if c["call"] == "sample":
        return out
    tok, B, M = out["tok"], c["B"], c["M"]
    same = tok.view(B, M)[:, :-1] == state["rows"].view(B, M)[:, 1:]
    return {"tok": tok, "accepted": (1 + torch.cumprod(same.int(), 1).sum(1)).to(torch.int32)}


# ------------------------------------------------------------------------------------------------ what is compared
def work(case):
    B, V, M = case["B"], case["V"], case["M"]
    R, size = B * M, {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    # shares of the rows that are masked, and of a row's logits that have to be read
    masked, few = {"none": (0.0, 0.0), "keys": (1.0, 1.0), "text": (1.0, 0.0), "mixed": (5 / 6, 2 / 6)}[case["mask"]]
    text = masked - few
    read = R * (V * (1.0 - masked + 0.97 * text) + 80 * few)
    bytes_ = read * size + R * masked * V / 8 + 4 * B * case["H"] + 8 * B * case["NB"]
    flops = read * 2
    if case["call"] == "edit":
        bytes_ += 4 * R * V
        flops = R * V * (20 if case["softcap"] else 2)
    elif case["call"] == "logprobs":
        bytes_ += R * (12 + 8 * case["n"])
        flops = read * 4
    else:
        bytes_ += R * (8 + 12 * case["kcap"])
    return {"bytes": int(bytes_), "flops": int(flops)}


def exact(case, seed):
    """Edited logits, candidates' probabilities and log-probabilities in 64 bits, row by row; tokens, counts, ranks and ids
    have no such value. Sampling's definition rounds each edit, and a candidate's distance from the largest, to fp32."""
    call, n = case["call"], case["n"] or case["kcap"]
    if call == "verify" or (call == "sample" and n == 0):
        return None
    d = _inputs(case, seed)
    B, V = case["B"], case["V"]
    host = {k: d[k].cpu().numpy() for k in ("off", "hist", "b_off", "b_ids", "b_val", "mask_of") if k in d}
    lp = torch.empty(B, dtype=torch.float64, device="cuda")
    top = torch.zeros((B, max(n, 1)), dtype=torch.float64, device="cuda")
    rows = torch.empty((B, V) if call == "edit" else (0,), dtype=torch.float64, device="cuda")
    shift = torch.arange(32, dtype=torch.int32, device="cuda")
    step = (lambda t: t.float().double()) if call == "sample" else (lambda t: t)
    for r in range(B):
        x = d["x"][r, :V].double()
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        if case["NB"]:
            a, b = host["b_off"][r], host["b_off"][r + 1]
            x[torch.from_numpy(host["b_ids"][a:b]).cuda().long()] += torch.from_numpy(host["b_val"][a:b]).cuda().double()
            x = step(x)
        if call != "logprobs" and case["H"]:
            h = host["hist"][host["off"][r]:host["off"][r + 1]]
            h = h[-case["last_n"]:] if case["last_n"] > 0 else h
            ids, cnt = np.unique(h, return_counts=True)
            ids, cnt = torch.from_numpy(ids).cuda().long(), torch.from_numpy(cnt).cuda().double()
            rep, freq, pres = (float(d["p"][k][r]) for k in ("rep", "freq", "pres"))
            y = x[ids]
            x[ids] = step(step(torch.where(y > 0, y / rep, y * rep)) - step(step(cnt * freq) + pres))
        if case["mask"] != "none" and host["mask_of"][r] >= 0:
            bits = (d["mask"][int(host["mask_of"][r])][:, None] >> shift) & 1
            x[bits.reshape(-1)[:V] == 0] = -math.inf
        if call == "edit":
            rows[r] = x
            continue
        T = float(d["p"]["T"][r])
        if call == "sample":
            k = int(d["p"]["k"][r])
            greedy = T <= 0 or k == 1
            k = min(1 if greedy else k if 0 < k < V else V, int((x > -math.inf).sum()))
            v = torch.topk(x, k).values
            pr = torch.softmax(step(v - v[0]) / (1.0 if greedy else T), 0)
            top[r, :min(k, n)] = pr[:n]
            continue
        x = x / T
        z = torch.logsumexp(x, 0)
        lp[r] = x[int(d["tok"][r])] - z
        if n:
            m = min(n, V)
            top[r, :m] = torch.topk(x, m).values - z
    if call == "edit":
        return {"logits": rows}
    if call == "sample":
        return {"tok": None, "keep": None, "ids": None, "probs": top}
    return {"lp": lp, "rank": None, **({"ids": None, "top": top} if n else {})}
