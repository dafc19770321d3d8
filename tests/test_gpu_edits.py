"""GPU: edited logits, sampling under edits and log-probabilities against plain implementations (tests/edit_util.py)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from oracle import oracle as O  # noqa: E402
from tests import edit_util as U  # noqa: E402
from tests.parity_util import boundary_row  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def histories(rng, S, V, H):
    hs = [rng.integers(-1, max(V // 4, 1), int(n)).astype(np.int32) for n in rng.integers(0, 2 * H + 1, S)]
    off = np.zeros(S + 1, np.int64)
    off[1:] = np.cumsum([len(h) for h in hs])
    return hs, (np.concatenate(hs) if len(hs) else np.zeros(0, np.int32)).astype(np.int32), off


class Batch:
    """B rows of V logits with histories, parameters, masks and biases."""

    def __init__(self, seed, B, V, kind="most", nb=5, H=40, records=None, **params):
        rng = self.rng = np.random.default_rng(seed)
        S = records or B
        self.B, self.V = B, V
        self.x = W.mixture_logits(rng, B, V)
        self.hs, self.hist, self.off = histories(rng, S, V, H)
        self.p = W.make_params(S, **params)
        self.u = rng.random(B)
        self.bias = U.bias_lists(rng, S, V, nb) if nb else [[]] * S
        self.allowed, self.of = None, np.full(B, -1, np.int32)
        if kind:
            kinds = [kind] if isinstance(kind, str) else list(kind)
            # fewer masks than rows, some rows unmasked, masks shared between rows
            n = max(1, B - B // 4)
            self.allowed = np.concatenate([U.masks(rng, kinds[i % len(kinds)], 1, V) for i in range(n)])
            self.of = rng.integers(-1, n, B).astype(np.int32)
            self.of[0] = 0
        self.ed = F.Edits(mask=None if self.allowed is None else U_pack(self.allowed),
                          mask_of=None if self.allowed is None else self.of, bias=U.csr(self.bias))

    def ok(self, r):
        return None if self.of[r] < 0 else self.allowed[self.of[r]]


def U_pack(a):
    """Mask words with every bit past the vocabulary set (they must not matter), rows one word longer than needed."""
    n, V = a.shape
    pad = np.ones((n, (-V) % 32 + 32), bool)
    return F.Edits.pack(np.concatenate([a, pad], 1))


# ------------------------------------------------------------------------------------------------ edit_batch
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,V,kind,cap", [(1, 1, "most", 0.0), (3, 5, "last", 0.0), (2, 33, "few", 30.0), (5, 1023, "block", 0.0),
                                          (3, 4101, "most", 30.0), (2, 70001, ("few", "none", "most"), 0.0),
                                          (40, 20000, ("most", "block"), 0.0), (1, 65536, None, 0.0)])
def test_edit_batch(dtype, B, V, kind, cap):
    b = Batch(hash((B, V)) % 1000, B, V, kind, nb=min(V, 30), H=60, repetition_penalty=1.2, frequency_penalty=0.3,
              presence_penalty=0.1, softcap=cap)
    b.p["repeat_last_n"][::2] = 16
    b.p["repetition_penalty"][::3] = 0.9
    b.p["penalty_from"][1::3] = 4
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    x = cuda(b.x).clamp(-60000, 60000).to(t)
    x[0, V // 2] = float("nan") if cap == 0 else 1.0
    got = F.edit_batch(x, b.p, b.hist, b.off, edits=b.ed).cpu().numpy()
    xs = x.float().cpu().numpy()
    for r in range(B):
        want = U.edit_row(xs[r], b.p[r], b.hs[r], b.bias[r], b.ok(r))
        np.testing.assert_array_equal(got[r], want, err_msg=f"row {r}")        # the same fp32 steps
        w64, err = U.edit_row64(xs[r], b.p[r], b.hs[r], b.bias[r], b.ok(r))
        fin = np.isfinite(w64) & np.isfinite(err)
        assert np.array_equal(np.isfinite(got[r]), np.isfinite(w64))
        assert np.all(np.abs(got[r].astype(np.float64) - w64)[fin] <= err[fin] * 1.001)


def test_edit_batch_in_place_strided_and_rows_behind():
    """A strided view edited in place leaves the padding and the rows behind as they were; out into a wider buffer."""
    b = Batch(3, 4, 1003, "most", repetition_penalty=1.3)
    buf = torch.full((6, 1024), 7.25, device="cuda")
    buf[:4, :1003] = cuda(b.x)
    got = F.edit_batch(buf[:4], b.p, b.hist, b.off, edits=b.ed, V=1003, out=buf[:4])
    assert got.data_ptr() == buf.data_ptr()
    want = np.stack([U.edit_row(b.x[r], b.p[r], b.hs[r], b.bias[r], b.ok(r)) for r in range(4)])
    h = buf.cpu().numpy()
    np.testing.assert_array_equal(h[:4, :1003], want)
    assert np.all(h[:4, 1003:] == 7.25) and np.all(h[4:] == 7.25)
    wide = torch.full((4, 1200), 7.25, device="cuda")
    F.edit_batch(cuda(b.x), b.p, b.hist, b.off, edits=b.ed, out=wide)
    h = wide.cpu().numpy()
    np.testing.assert_array_equal(h[:, :1003], want)
    assert np.all(h[:, 1003:] == 7.25)
    # an unaligned bf16 view, no parameters, no edits: a conversion
    y = torch.randn((3, 71), device="cuda").to(torch.bfloat16)[:, 1:]
    assert torch.equal(F.edit_batch(y), y.float())


# ------------------------------------------------------------------------------------------------ sampling
SETS = {
    "greedy": dict(temperature=0.0, repetition_penalty=1.2),
    "greedy_counts": dict(temperature=0.0, repetition_penalty=1.0, frequency_penalty=0.5, presence_penalty=0.2),
    "small_k": dict(temperature=0.8, top_k=40, top_p=0.95, repetition_penalty=1.1),
    "small_k_up": dict(temperature=0.9, top_k=20, top_p=0.9, repetition_penalty=0.8),
    "small_k_cap": dict(temperature=0.8, top_k=50, repetition_penalty=1.05, softcap=20.0),
    "mid_k": dict(temperature=1.0, top_k=300, top_p=0.97, min_p=0.001, repetition_penalty=1.1, frequency_penalty=0.2),
    "every": dict(temperature=0.9, top_k=0, top_p=0.95, repetition_penalty=1.05, presence_penalty=0.2),
    "every_flat": dict(temperature=1.5, top_k=0, repetition_penalty=1.0),
    "every_min_p": dict(temperature=1.0, top_k=0, min_p=0.02, repetition_penalty=1.1),
    "large_k": dict(temperature=1.0, top_k=3000, top_p=0.99, repetition_penalty=1.1),
}


def check_rows(b, tok, keep, kcap=0, ids=None, probs=None, rows_of=None):
    """Every row against the plain implementation; returns the rows whose draw lies at a boundary."""
    near = 0
    for r in range(b.B):
        s, hist = rows_of(r) if rows_of else (r, b.hs[r])
        p = b.p[s]
        want = U.sample_row(b.x[r], p, hist, b.u[r], b.bias[s], b.ok(r), kcap=kcap)
        m = min(want["ncand"], kcap)
        if m:
            np.testing.assert_array_equal(ids[r, :m], want["ids"][:m], err_msg=f"row {r}")
            np.testing.assert_allclose(probs[r, :m], want["probs"][:m], rtol=1e-12, atol=1e-300, err_msg=f"row {r}")
        if tok[r] != want["tok"] or (keep is not None and keep[r] != want["keep"]):
            assert p["temperature"] > 0 and want["ncand"] > 0, f"row {r}: {tok[r]} for {want['tok']}"
            assert boundary_row(want["probs"], want["keep"], b.u[r], float(p["top_p"]), float(p["min_p"])), \
                f"row {r}: {tok[r]} for {want['tok']}, kept {keep[r] if keep is not None else None} for {want['keep']}"
            near += 1
    return near


@pytest.mark.parametrize("route", ["host", "device"])
@pytest.mark.parametrize("kind", ["most", "few", "block", ("most", "few", "none", "last"), None])
@pytest.mark.parametrize("name", list(SETS))
def test_sample_edited(name, kind, route):
    for B, V in ((1, 1), (3, 70), (9, 5003), (5, 33000)):
        b = Batch(B * 7 + V, B, V, kind, nb=min(V, 20), **SETS[name])
        kcap = 8 if name in ("greedy", "small_k", "mid_k") else 0
        out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, kcap=kcap, route=route, edits=b.ed)
        h = {k: None if out[k] is None else out[k].cpu().numpy() for k in ("tok", "keep", "cand_ids", "cand_probs")}
        near = check_rows(b, h["tok"], h["keep"], kcap, h["cand_ids"], h["cand_probs"])
        assert near <= 1, (B, V, near)


def test_sample_edited_mixed_batch():
    """Rows of every kind in one batch, on the large vocabulary: masks of all kinds, long bias lists."""
    B, V = 24, 151939
    b = Batch(11, B, V, ("most", "few", "block", "none", "last", "most"), nb=400, H=300)
    for r, s in enumerate(np.resize(np.array(list(SETS)), B)):
        if s in ("large_k", "every_min_p", "small_k_cap"):
            s = "mid_k"
        for k, v in dict(dict(top_p=1.0, min_p=0.0, frequency_penalty=0.0, presence_penalty=0.0), **SETS[s]).items():
            b.p[k][r] = v
    for route in ("host", "device"):
        out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, route=route, edits=b.ed)
        near = check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy())
        assert near <= 1


def test_no_edits_equal_the_plain_call():
    """Edits without masks and biases: the plain call's tokens, on rows of finite logits."""
    for name in SETS:
        b = Batch(5, 6, 9001, None, nb=0, **SETS[name])
        a = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off)
        e = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=F.Edits())
        assert torch.equal(a["tok"], e["tok"]) and torch.equal(a["keep"], e["keep"]), name


@pytest.mark.parametrize("name", ["greedy", "small_k", "mid_k", "every"])
def test_infinities_nan_and_lowest_values(name):
    """NaN, infinities and the type's lowest value, in allowed and in masked places; rows with nothing left."""
    B, V = 8, 6007
    b = Batch(21, B, V, "most", nb=0, H=0, **dict(SETS[name], frequency_penalty=0.0, presence_penalty=0.0, repetition_penalty=1.0))
    b.of[:] = np.minimum(np.arange(B), b.allowed.shape[0] - 1)
    b.ed = F.Edits(mask=U_pack(b.allowed), mask_of=b.of)
    lowest = np.finfo(np.float32).min
    bad = ~b.allowed
    for r in range(B):
        m = bad[b.of[r]]
        b.x[r, m] = [np.inf, np.nan, -np.inf, lowest, 100.0, np.nan, np.inf, 3e38][r]
    b.x[1, ::3] = np.nan
    b.x[2, 5:] = -np.inf                                       # five candidates at most
    b.x[3, 2:] = lowest                                        # a model's own mask: the lowest value is a number
    b.x[4] = -np.inf                                           # nothing left
    b.x[5] = np.nan
    b.x[6, 0] = np.nan                                         # (ferro's greedy scan would keep index 0)
    out = F.sample_batch(cuda(b.x), b.p, b.u, edits=b.ed)
    tok, keep = out["tok"].cpu().numpy(), out["keep"].cpu().numpy()
    b.hs = [np.zeros(0, np.int32)] * B
    assert check_rows(b, tok, keep) == 0
    assert tok[4] == -1 and tok[5] == -1 and keep[4] == 0 and keep[5] == 0


def test_argmax_edited():
    b = Batch(8, 7, 4099, ("few", "most", "none"), temperature=0.7, repetition_penalty=1.3)
    tok = F.argmax_batch(cuda(b.x), b.hist, b.off, b.p, edits=b.ed).cpu().numpy()
    dev = F.argmax_batch(cuda(b.x), b.hist, b.off, cuda(b.p.view(np.uint8)), edits=b.ed).cpu().numpy()
    none = F.argmax_batch(cuda(b.x), edits=b.ed).cpu().numpy()
    g = b.p.copy()
    g["temperature"] = 0.0
    free = W.make_params(1, temperature=0.0, repetition_penalty=1.0)[0]
    for r in range(7):
        want = U.sample_row(b.x[r], g[r], b.hs[r], 0.0, b.bias[r], b.ok(r))["tok"]
        assert tok[r] == dev[r] == want
        assert none[r] == U.sample_row(b.x[r], free, [], 0.0, b.bias[r], b.ok(r))["tok"]


# ------------------------------------------------------------------------------------------------ windows
def window_batch(seed, S, V, kind, ms, **params):
    off = np.zeros(S + 1, np.int64)
    off[1:] = np.cumsum(ms)
    R = int(off[-1])
    b = Batch(seed, R, V, kind, nb=10, records=S, **params)
    b.row_off = off
    stream = np.repeat(np.arange(S), ms)
    fed = b.rng.integers(0, V, R).astype(np.int32)

    def rows_of(r):
        s = stream[r]
        return s, np.concatenate([b.hs[s], fed[off[s] + 1:r + 1]])

    for r in range(R):                             # a draft is the row's own token four times out of five
        s, hist = rows_of(r)
        if r + 1 < off[s + 1] and b.rng.random() < 0.8:
            t = U.sample_row(b.x[r], b.p[s], hist, b.u[r], b.bias[s], b.ok(r))["tok"]
            fed[r + 1] = max(t, 0)
    b.fed, b.rows_of = fed, rows_of
    return b


def accepted(b, tok, eos):
    acc = []
    for s in range(b.row_off.size - 1):
        r0, m = int(b.row_off[s]), int(b.row_off[s + 1] - b.row_off[s])
        n = 0
        for r in range(m):
            n = r + 1
            if tok[r0 + r] < 0 or (eos >= 0 and tok[r0 + r] == eos) or r + 1 >= m or tok[r0 + r] != b.fed[r0 + r + 1]:
                break
        acc.append(n)
    return np.array(acc, np.int32)


@pytest.mark.parametrize("route", ["host", "device"])
@pytest.mark.parametrize("name", ["greedy", "greedy_counts", "small_k", "mid_k", "every", "free"])
@pytest.mark.parametrize("kind", ["most", ("few", "most", "none"), None])
def test_verify_edited(name, kind, route):
    params = SETS.get(name, dict(temperature=0.0, repetition_penalty=1.0))
    for S, V, ms in ((1, 50, [1]), (3, 4111, [1, 5, 2]), (2, 33000, [17, 40])):
        b = window_batch(S + V, S, V, kind, ms, **params)
        eos = int(b.fed[1]) if b.fed.size > 1 else -1
        tok, acc = F.verify(cuda(b.x), b.fed, b.row_off, b.p, b.u, b.hist, b.off, eos_id=eos, route=route, edits=b.ed)
        tok, acc = tok.cpu().numpy(), acc.cpu().numpy()
        assert check_rows(b, tok, None, rows_of=b.rows_of) == 0
        np.testing.assert_array_equal(acc, accepted(b, tok, eos))


def test_a_masked_draft_is_never_accepted():
    """A window whose row has no candidate ends there, also where the next draft is token 0."""
    V, m = 4096, 4
    x = np.zeros((m, V), np.float32)
    x[:, 0] = 5.0
    p = W.make_params(1, temperature=0.0, repetition_penalty=1.0)
    allowed = np.ones((m, V), bool)
    allowed[1] = False
    for route in ("host", "device"):
        tok, acc = F.verify(cuda(x), np.zeros(m, np.int32), [0, m], p, edits=F.Edits(mask=F.Edits.pack(allowed)), route=route)
        assert tok.tolist() == [0, -1, 0, 0] and acc.tolist() == [2]


# ------------------------------------------------------------------------------------------------ decode steps
@pytest.mark.parametrize("route", ["host", "device"])
@pytest.mark.parametrize("name", ["greedy", "small_k", "mid_k", "every"])
def test_decode_loop_edited(name, route):
    """Steps with a new mask each: draws, tokens and histories follow the plain loop; a row without a candidate appends -1
    (and, sampled, consumes its draw)."""
    B, V, steps = 5, 8009, 4
    rng = np.random.default_rng(31)
    p = W.make_params(B, **SETS[name])
    seeds = np.arange(1, B + 1, dtype=np.uint64) * 77
    drng = F.DeviceRng(seeds)
    engines = [O.MT64(int(s)) for s in seeds]
    hs = [rng.integers(0, V, 3 * i).astype(np.int32) for i in range(B)]
    hist = cuda(np.concatenate(hs).astype(np.int32))
    off = np.concatenate([[0], np.cumsum([len(h) for h in hs])]).astype(np.int64)
    doff = cuda(off)
    for step in range(steps):
        x = W.mixture_logits(rng, B, V)
        allowed = np.concatenate([U.masks(rng, k, 1, V) for k in ("few", "most", "block", "none" if step == 1 else "last", "most")])
        bias = U.bias_lists(rng, B, V, 6)
        ed = F.Edits(mask=U_pack(allowed), bias=U.csr(bias))
        tok, keep, hist, doff = F.decode_step(cuda(x), p, drng, hist, doff, route=route, edits=ed)
        greedy = SETS[name]["temperature"] <= 0
        for r in range(B):
            u = 0.0 if greedy else O.canonical(engines[r].next())
            want = U.sample_row(x[r], p[r], hs[r], u, bias[r], allowed[r])
            assert int(tok[r]) == want["tok"] and int(keep[r]) == want["keep"], (step, r)
            hs[r] = np.append(hs[r], np.int32(want["tok"]))
        h, o = hist.cpu().numpy(), doff.cpu().numpy()
        np.testing.assert_array_equal(h[:o[-1]], np.concatenate(hs))
    assert drng.error() == 0
    # without histories
    tok, keep, h1, o1 = F.decode_step(cuda(x), p, drng, route=route, edits=ed)
    assert o1.tolist() == list(range(B + 1)) and torch.equal(h1[:B], tok)


# ------------------------------------------------------------------------------------------------ log-probabilities
def lp_tolerance(lp):
    """fp32 terms: the difference to the maximum (u = 2^-24) and its product with log2 e / T, itself rounded (2u), relative to
    an argument of at most 30 where a term matters (below e^-30 they sum to less than u), the exponential (an ulp, 2u) and
    at most 10 additions (u each; the chunks' sums are added in fp64): the sum is off by at most (3 * 30 + 2 + 10) u relative,
    its logarithm by as much absolutely, and 200u is above it. The result is rounded to fp32."""
    return 200 * 2.0 ** -24 + np.abs(lp) * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,V,n,kind,T,cap", [(1, 1, 1, "most", 1.0, 0.0), (4, 7, 20, "few", 0.7, 0.0), (3, 33, 5, ("none", "last"), 1.0, 0.0),
                                              (6, 4100, 64, "block", 1.3, 30.0), (5, 65536, 20, ("most", "few"), 0.8, 0.0),
                                              (70, 20011, 3, ("most", None, "few"), 1.0, 0.0), (2, 151936, 0, None, 0.6, 0.0)])
def test_logprobs(dtype, B, V, n, kind, T, cap):
    kinds = None if kind is None else tuple(k or "most" for k in ([kind] if isinstance(kind, str) else kind))
    b = Batch(B + V, B, V, kinds, nb=min(V, 40), temperature=T, softcap=cap)
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    x = cuda(b.x).clamp(-60000, 60000).to(t)
    if B > 2:
        x[1, ::5] = float("nan")
        x[2, ::2] = float("-inf")
    tok = b.rng.integers(-1, V + 1, B).astype(np.int32)
    xs = x.float().cpu().numpy()
    tok[0] = np.nanargmax(xs[0])
    out = F.logprobs(x, tok, n, params=b.p, edits=b.ed)
    h = {k: None if v is None else v.cpu().numpy() for k, v in out.items()}
    only = F.logprobs(x, None, n, params=b.p, edits=b.ed) if n else None
    for r in range(B):
        lp, rank, ids, top = U.logprob_row(xs[r], int(tok[r]), n, cap, float(np.float32(T)), b.bias[r], b.ok(r))
        assert h["rank"][r] == rank, r
        if np.isinf(lp):
            assert h["lp"][r] == lp
        else:
            assert abs(h["lp"][r] - lp) <= lp_tolerance(lp), (r, h["lp"][r], lp)
        if n:
            np.testing.assert_array_equal(h["ids"][r], ids)
            fin = np.isfinite(top)
            assert np.array_equal(np.isfinite(h["top"][r]), fin)
            assert np.all(np.abs(h["top"][r][fin] - top[fin]) <= lp_tolerance(top[fin]))
    if n:
        assert torch.equal(only["ids"], out["ids"]) and torch.equal(only["top"], out["top"]) and only["lp"] is None


@pytest.mark.parametrize("V", [5, 4096, 50000])
def test_logprobs_ties_and_infinities(V):
    """Thousands of equal logits (the lowest ids first), +inf sharing the mass, one value alone."""
    x = torch.zeros((5, V), device="cuda")
    x[1] = torch.arange(V, device="cuda") % 3
    x[2, ::2] = float("inf")
    x[3] = float("-inf")
    x[3, V // 2] = -3.4e38
    x[4] = -0.0
    x[4, 1] = 0.0
    n = min(V, 64)
    tok = [V - 1, 2, 2, V // 2, 0]
    out = F.logprobs(x, tok, n)
    for r in range(5):
        lp, rank, ids, top = U.logprob_row(x[r].cpu().numpy(), tok[r], n)
        assert out["ids"][r].tolist() == ids.tolist() and int(out["rank"][r]) == rank, r
        got = out["top"][r].cpu().numpy()
        fin = np.isfinite(top)
        assert np.array_equal(np.isfinite(got), fin) and np.all(np.abs(got[fin] - top[fin]) <= lp_tolerance(top[fin]))
        assert abs(float(out["lp"][r]) - lp) <= lp_tolerance(lp)


def test_logprobs_sum_to_one():
    x = torch.randn((3, 64), device="cuda") * 5
    top = F.logprobs(x, n=64)["top"].double()
    assert torch.all((top.exp().sum(1) - 1).abs() < 64 * lp_tolerance(10.0))


# ------------------------------------------------------------------------------------------------ errors, streams, graphs
def test_a_mask_index_past_the_masks_allows_nothing():
    ctx = F.Context()
    x = torch.randn((3, 5000), device="cuda")
    ed = F.Edits(mask=F.Edits.pack(np.ones((1, 5000), bool)), mask_of=[0, 1, -7])
    for params in (dict(temperature=0.0), dict(top_k=20, temperature=1.0), dict(top_k=200, temperature=1.0)):
        p = W.make_params(3, repetition_penalty=1.0, **params)
        for route in ("host", "device"):
            tok = F.sample_batch(x, p, np.full(3, 0.5), ctx=ctx, edits=ed, route=route)["tok"].tolist()
            assert tok[1] == -1 and tok[0] >= 0 and tok[2] >= 0
            assert F.device_error(ctx) == 8
    assert torch.isneginf(F.edit_batch(x, edits=ed, ctx=ctx)[1]).all() and F.device_error(ctx) == 8
    out = F.logprobs(x, [0, 0, 0], 2, edits=ed, ctx=ctx)
    assert out["ids"][1].tolist() == [-1, -1] and out["lp"][1] == float("-inf") and F.device_error(ctx) == 8


def test_refusals_on_device_tensors():
    x = torch.randn((2, 64), device="cuda")
    ed = F.Edits(mask=np.full((2, 1), -1, np.int32))
    with pytest.raises(F.SamplerError):
        F.edit_batch(x, edits=ed)                              # masks of 32 tokens for 64
    with pytest.raises(F.SamplerError):
        F.edit_batch(x.double())
    with pytest.raises(F.SamplerError):
        F.logprobs(x, [0, 1, 2])
    with pytest.raises(F.SamplerError):
        F.logprobs(x, n=65)
    with pytest.raises(F.SamplerError):
        F.edit_batch(x, out=torch.empty((2, 64), device="cuda", dtype=torch.float16))
    with pytest.raises(F.SamplerError):
        F.sample_batch(x, W.make_params(2), [0.5, 0.5], edits=F.Edits(bias=[{}]))


def test_on_another_stream():
    """Calls given a stream wait for what the current one made."""
    b = Batch(17, 6, 40000, ("most", "few"), **SETS["small_k"])
    x = cuda(b.x)
    want = F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=b.ed)["tok"]
    lp = F.logprobs(x, want, 5, edits=b.ed)
    st = torch.cuda.Stream()
    for _ in range(5):
        y = torch.empty_like(x)
        for _ in range(20):
            y.copy_(x)                                         # work on the current stream ahead of the call
        got = F.sample_batch(y, b.p, b.u, b.hist, b.off, edits=b.ed, stream=st)["tok"]
        st.synchronize()
        assert torch.equal(got, want)
        g = F.logprobs(y, want, 5, edits=b.ed, stream=st)
        e = F.edit_batch(y, b.p, b.hist, b.off, edits=b.ed, stream=st)
        st.synchronize()
        assert torch.equal(g["lp"], lp["lp"]) and torch.equal(g["ids"], lp["ids"])
        assert torch.equal(e, F.edit_batch(x, b.p, b.hist, b.off, edits=b.ed))


@pytest.mark.parametrize("name", ["greedy", "small_k", "mid_k", "every", "large_k"])
def test_captured_calls_replay(name):
    """Sampling, log-probabilities and edited rows in one graph, as a decode loop runs them: every replay, with other masks,
    biases and logits written into the same buffers and eager calls in between, equals the eager calls."""
    B, V = 5, 30011
    b = Batch(41, B, V, ("most", "few"), **SETS[name])
    ctx = F.Context()
    ld = V + (-V) % 4
    x = torch.zeros((B, ld), device="cuda")
    x[:, :V] = cuda(b.x)
    p, u, hist, off = cuda(b.p.view(np.uint8)), cuda(b.u), cuda(b.hist), cuda(b.off)

    def step():
        out = F.sample_batch(x, p, u, hist, off, V=V, edits=b.ed, ctx=ctx)
        lp = F.logprobs(x, out["tok"], 5, edits=b.ed, V=V, ctx=ctx)
        return out["tok"], out["keep"], lp["lp"], lp["rank"], lp["ids"], F.edit_batch(x, p, hist, off, edits=b.ed, V=V, ctx=ctx)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for i in range(4):
        x[:, :V] = torch.randn((B, V), device="cuda") * 2
        b.ed.mask[0] = torch.randint(-2 ** 31, 2 ** 31 - 1, b.ed.mask[0].shape, dtype=torch.int64, device="cuda").to(torch.int32)
        b.ed.bias.copy_(torch.randn_like(b.ed.bias))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(torch.nan_to_num(a.double(), nan=1e300), torch.nan_to_num(c.double(), nan=1e300)), i


def test_capture_refuses_to_grow():
    """A captured call whose workspace would have to grow is refused; the capture goes on."""
    b = Batch(43, 3, 9000, "most", **SETS["large_k"])
    ctx = F.Context()
    x, p, u = cuda(b.x), cuda(b.p.view(np.uint8)), cuda(b.u)
    hist, off = cuda(b.hist), cuda(b.off)
    g = torch.cuda.CUDAGraph()
    y = torch.zeros(3, device="cuda")
    with torch.cuda.graph(g):
        with pytest.raises(F.SamplerError, match="allocation"):
            F.sample_batch(x, p, u, hist, off, edits=b.ed, ctx=ctx)
        with pytest.raises(F.SamplerError, match="allocation"):
            F.logprobs(x, n=3, ctx=ctx)
        y.add_(1.0)
    g.replay()
    torch.cuda.synchronize()
    assert y.tolist() == [1.0, 1.0, 1.0]


def test_a_rollout_as_a_program_runs_it():
    """bf16 logits made fp32 by edit_batch, sampled, scored and appended for three steps: edit_batch and the plain sampler
    agree with the sampler under the same edits."""
    B, V = 6, 20003
    b = Batch(51, B, V, ("most", "few"), temperature=0.9, top_k=50, top_p=0.95, repetition_penalty=1.1)
    hist, off = cuda(b.hist), cuda(b.off)
    q = U.neutral(b.p)
    for step in range(3):
        x16 = (torch.randn((B, V), device="cuda") * 2).to(torch.bfloat16)
        x = F.edit_batch(x16)                                  # converted
        tok = F.sample_batch(x, b.p, b.u, hist, off, edits=b.ed)["tok"]
        rows = F.edit_batch(x16, b.p, hist, off, edits=b.ed)
        live = rows > float("-inf")
        k = min(50, int(live.sum(1).min()))
        assert k > 0
        same = F.sample_batch(torch.where(live, rows, float("nan")), q, b.u)["tok"]
        assert torch.equal(tok, same)
        lp = F.logprobs(x16, tok, edits=b.ed)["lp"]
        assert torch.isfinite(lp).all()
        hist, off = F.hist_append(hist, off, tok)
    assert off[-1].item() == b.off[-1] + 3 * B
