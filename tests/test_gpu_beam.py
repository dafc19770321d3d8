"""GPU: a beam search's selection, histories and states against plain implementations (tests/beam_util.py)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from ferro_amd import _lib  # noqa: E402
from tests import beam_util as BU  # noqa: E402
from tests import edit_util as U  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Rows:
    """Streams of rows of V logits of a type (x: as the kernels read them, y: their fp32 values) with scores."""

    def __init__(self, seed, counts, V, kind="f32", logits=None, dead=0.0):
        rng = self.rng = np.random.default_rng(seed)
        self.off = np.zeros(len(counts) + 1, np.int64)
        self.off[1:] = np.cumsum(counts)
        R = int(self.off[-1])
        x = W.mixture_logits(rng, R, V) if logits is None else logits(rng, R, V)
        self.x = torch.from_numpy(np.clip(x, -60000, 60000) if kind == "f16" else x).to(TYPES[kind]).cuda()
        self.y = self.x.float().cpu().numpy()
        self.score = (-rng.uniform(0, 40) - rng.exponential(2.0, R)).astype(np.float32)
        self.score[rng.random(R) < dead] = -np.inf

    def run(self, n, eos=-1, p=None, ed=None, bias=None, allowed=None, **kw):
        step = BU.Step(self.y, self.score, self.off, n, eos, p, bias, allowed)
        args = dict(eos_id=eos, params=p, row_off=self.off, edits=ed, **kw)
        out = F.beam_select(self.x, cuda(self.score), n, **args)
        step.check(out)
        kept = F.beam_select(self.x, cuda(self.score), n, keep_slots=True, **args)
        for s in range(len(self.off) - 1):
            order = BU.slots(out["parent"][s].tolist(), n)
            for k in ("parent", "tok", "score"):
                assert torch.equal(kept[k][s], out[k][s][order]), (s, k, kept[k][s], out[k][s], order)
        for k in ("done", "done_parent", "done_score"):
            assert torch.equal(kept[k], out[k]), k
        return out


# ------------------------------------------------------------------------------------------------ selection
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 3, 4, 7, 64, 257, 1000, 4096, 4097, 16389, 50001])
def test_select_sizes_and_types(V, kind):
    r = Rows(V, [4, 4, 1, 0, 7], V, kind)
    r.run(4, eos=min(V - 1, 2))
    r.run(1)
    r.run(9, eos=0)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 16, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_select_widths(n, kind):
    r = Rows(n, [n, n, 1], 5003, kind)
    r.run(n, eos=int(r.y[0].argmax()))
    r = Rows(100 + n, [n], 70, kind)                           # more beams than a row has tokens
    r.run(n, eos=5)


@pytest.mark.parametrize("V,counts", [(65536, [4]), (151936, [8, 8]), (262144, [1, 1, 1]), (100003, [16, 3])])
def test_select_large_vocabularies(V, counts):
    r = Rows(V, counts, V)
    out = r.run(8, eos=int(r.y[0].argmax()))
    assert int(out["done"][0]) >= 0
    Rows(V + 1, counts, V, "bf16").run(20, eos=7)


def test_select_many_streams():
    Rows(5, [5] * 300, 777).run(5, eos=3)
    Rows(6, list(np.random.default_rng(6).integers(0, 9, 500)), 301, "f16", dead=0.3).run(6, eos=3)


def test_select_many_rows_of_a_stream():
    """More rows than a wave has lanes, more of them than new beams."""
    Rows(8, [200, 65, 64, 63], 333).run(10, eos=2)
    Rows(9, [130], 100, "bf16").run(64, eos=2)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_select_ties(kind):
    """Logits of few values, alike rows: lower rows and lower tokens first, eos before its equals."""
    def few(rng, R, V):
        return rng.integers(0, 3, (1, V)).astype(np.float32).repeat(R, 0)
    r = Rows(3, [4, 5], 999, kind, few)
    r.score[:] = -1.5
    for eos in (-1, int(r.y[0].argmax())):
        out = r.run(6, eos=eos)
        t = np.flatnonzero(r.y[0] == 2)
        t = t[t != eos]
        assert out["parent"][0].tolist() == [0] * 6 and out["tok"][0].tolist() == t[:6].tolist()
        assert int(out["done"][0]) == (4 if eos >= 0 else 0)
    Rows(4, [3], 2000, kind, lambda rng, R, V: np.zeros((R, V), np.float32)).run(64, eos=1999)


@pytest.mark.parametrize("n", [5, 20, 64])
def test_select_ties_of_many_rows(n):
    """More equal candidates than there is room for: alike rows, of one value and of few, dead ones among them."""
    for seed, counts, V, values in ((40, [70, 130], 200, 1), (41, [64], 90, 1), (42, [17, 65], 300, 3), (43, [20], 64, 2)):
        r = Rows(seed, counts, V, "bf16", lambda rng, R, V: rng.integers(0, values, (1, V)).astype(np.float32).repeat(R, 0))
        r.score[:] = -2.0
        r.score[[0, 9]] = -np.inf
        out = r.run(n, eos=int(r.y[0].argmax()))
        t = [i for i in np.flatnonzero(r.y[0] == r.y[0].max()) if i != int(r.y[0].argmax())][:n]
        assert out["parent"][0].tolist()[:len(t)] == [1] * len(t) and out["tok"][0].tolist()[:len(t)] == t
        # scores apart by less than the rows' candidates
        r.score = (-2.0 - 0.01 * r.rng.random(r.score.size)).astype(np.float32)
        r.run(n, eos=0)


def test_select_dead_rows():
    """Rows of score -inf or NaN do not matter, whatever they hold; streams of dead rows alone have no beam."""
    r = Rows(11, [4, 4, 4], 3001)
    r.score[[1, 4, 5, 6, 7, 9]] = -np.inf
    r.score[10] = np.nan
    r.y[1] = r.y[9] = np.nan
    r.x[1] = r.x[9] = float("nan")
    out = r.run(4, eos=17)
    assert out["parent"][1].tolist() == [-1] * 4 and int(out["done"][1]) == 0
    assert set(out["parent"][0].tolist()) <= {0, 2, 3}


def test_select_scores_far_apart():
    r = Rows(12, [6], 2000)
    r.score[:] = [0.0, -1e30, 3e38, -3e38, 1e-30, np.inf]
    r.run(8)
    r.score[:] = [-3.4028e38, -3.4e38, -np.inf, -3.4e38, -3.4e38, -3.4e38]
    r.run(8)


def test_select_infinities_and_nan():
    V = 1201
    r = Rows(13, [5, 2, 3], V)
    y = r.y
    y[0, 5] = np.inf                                           # one
    y[1, [7, 900]] = np.inf                                    # two share the probability
    y[2, :] = -np.inf                                          # no token
    y[3, ::2] = np.nan
    y[4, 1:] = -np.inf                                         # one token
    y[5, :] = np.nan
    y[7, 3] = 3.0e38
    y[8, :] = -3.0e38
    y[9, :600] = -np.inf
    r.x = torch.from_numpy(y).cuda()
    r.run(4, eos=5)
    r.run(40)


@pytest.mark.parametrize("T", [0.0, 0.05, 0.7, 3.0, 100.0, 1e-30, 1e30])
def test_select_temperatures(T):
    r = Rows(14, [4, 3], 3000)
    p = W.make_params(2, temperature=T)
    r.run(5, eos=9, p=p)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_select_softcap_and_temperatures_by_stream(kind):
    r = Rows(15, [4, 3, 2, 5], 5000, kind)
    p = W.make_params(4, temperature=1.0)
    p["softcap"] = [30.0, 0.0, 5.0, 30.0]
    p["temperature"] = [1.0, 0.5, 0.0, 2.0]
    r.run(6, eos=11, p=p)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("V", [5, 1000, 40001])
def test_select_masks_and_biases(kind, V):
    counts = [4, 6, 1, 5]
    R = sum(counts)
    r = Rows(16 + V, counts, V, kind)
    rng = r.rng
    allowed = [None if i % 4 == 0 else rng.random(V) < (0.95 if i % 4 == 1 else min(1.0, 20 / V)) for i in range(R)]
    allowed[2] = np.zeros(V, bool)                             # a row whose mask leaves nothing
    masks = np.stack([np.ones(V, bool) if m is None else m for m in allowed])
    of = np.where([m is None for m in allowed], -1, np.arange(R)).astype(np.int32)
    bias = U.bias_lists(rng, 4, V, 9)
    bias[1] = [(0, -np.inf)] + [b for b in bias[1] if b[0] > 0]
    ed = F.Edits(mask=F.Edits.pack(masks), mask_of=of, bias=U.csr(bias))
    r.run(5, eos=V // 2, ed=ed, bias=bias, allowed=allowed)
    p = W.make_params(4, temperature=0.8)
    p["softcap"] = 20.0
    r.run(3, eos=0, p=p, ed=ed, bias=bias, allowed=allowed)


def test_select_mask_index_past_the_masks():
    V = 500
    r = Rows(17, [2, 2], V)
    ed = F.Edits(mask=F.Edits.pack(np.ones((1, V), bool)), mask_of=np.array([0, 1, -1, 7], np.int32))
    out = F.beam_select(r.x, cuda(r.score), 3, row_off=r.off, edits=ed)
    assert F.device_error() == _lib.FS_DEVERR_MASK
    assert set(out["parent"].reshape(-1).tolist()) == {0}


def test_select_rows_alike_and_no_scores():
    """Without row_off: streams of equal parts; without scores: zeros; strided rows; other outputs left out."""
    r = Rows(18, [3, 3, 3, 3], 1500)
    a = F.beam_select(r.x, cuda(r.score), 4, row_off=r.off, eos_id=2)
    b = F.beam_select(r.x, cuda(r.score.reshape(4, 3)), 4, eos_id=2)
    c = F.beam_select(r.x, cuda(r.score), 4, streams=4, eos_id=2)
    wide = torch.full((12, 1600), 50.0, device="cuda")
    wide[:, :1500] = r.x
    d = F.beam_select(wide, cuda(r.score), 4, streams=4, eos_id=2, V=1500)
    e = F.beam_select(r.x.t().contiguous().t(), cuda(r.score), 4, streams=4, eos_id=2)   # repacked
    for o in (b, c, d, e):
        for k in a:
            assert torch.equal(a[k], o[k]), k
    z = F.beam_select(r.x, None, 4, streams=4)
    o = F.beam_select(r.x, torch.zeros(12, device="cuda"), 4, streams=4)
    for k in z:
        assert torch.equal(z[k], o[k]), k


def test_select_is_one_result():
    """Two calls, and calls on other contexts and streams, give the same bits."""
    r = Rows(19, [8] * 6, 30011, "bf16")
    a = F.beam_select(r.x, cuda(r.score), 8, row_off=r.off, eos_id=2, keep_slots=True)
    s = torch.cuda.Stream()
    b = F.beam_select(r.x, cuda(r.score), 8, row_off=r.off, eos_id=2, keep_slots=True, ctx=F.Context(), stream=s)
    s.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_select_refusals():
    x, a = torch.zeros((4, 64), device="cuda"), torch.zeros(4, device="cuda")
    for bad in (dict(n=0), dict(n=65), dict(streams=3), dict(streams=None), dict(row_off=[0, 2, 5]), dict(row_off=[0, 3, 2, 4]),
                dict(score=torch.zeros(3, device="cuda")), dict(params=W.make_params(3)),
                dict(edits=F.Edits(mask=np.zeros((2, 2), np.int32))), dict(logits=x.double()), dict(V=65)):
        kw = dict(logits=x, score=a, n=4, streams=2)
        kw.update(bad)
        if "row_off" in kw:
            del kw["streams"]
        with pytest.raises(F.SamplerError):
            F.beam_select(**kw)


# ------------------------------------------------------------------------------------------------ histories
def hists(rng, rows, H):
    hs = [rng.integers(0, 1 << 20, int(k)).astype(np.int32) for k in rng.integers(0, 2 * H + 1, rows)]
    off = np.zeros(rows + 1, np.int64)
    off[1:] = np.cumsum([len(h) for h in hs])
    return hs, np.concatenate(hs + [np.zeros(0, np.int32)]).astype(np.int32), off


def same_hists(out, off, want):
    off = off.cpu().numpy()
    assert off.tolist() == np.concatenate([[0], np.cumsum([len(h) for h in want])]).astype(int).tolist()
    assert out.cpu().numpy()[:off[-1]].tolist() == [t for h in want for t in h]


@pytest.mark.parametrize("S,n,H", [(1, 1, 0), (1, 4, 1), (3, 4, 50), (1, 64, 9), (70, 8, 33), (2, 3, 5000), (700, 2, 3), (5, 7, 2049),
                                   (2500, 1, 4), (40, 64, 60)])
def test_fork(S, n, H):
    rng = np.random.default_rng(S * n + H)
    hs, flat, off = hists(rng, S * n, H)
    parent = rng.integers(-1, n, (S, n)).astype(np.int32)
    tok = rng.integers(0, 1 << 20, (S, n)).astype(np.int32)
    ro = np.arange(0, S * n + 1, n)
    for t in (tok, None):
        out, o = F.hist_fork(flat, off, cuda(parent), None if t is None else cuda(t))
        same_hists(out, o, BU.fork(hs, ro, parent, t))
    # the capacity to the id; a history array that does not begin at 0
    want = BU.fork(hs, ro, parent, tok)
    total = sum(len(h) for h in want)
    out, o = F.hist_fork(np.concatenate([np.full(5, -9, np.int32), flat]), off + 5, cuda(parent), cuda(tok), out_cap=total)
    same_hists(out, o, want)


def test_fork_of_ragged_rows():
    """The first step: a row per stream opens n beams; and streams of other numbers of rows."""
    rng = np.random.default_rng(1)
    for counts in ([1, 1, 1], [3, 1, 5, 2], [64, 1]):
        ro = np.concatenate([[0], np.cumsum(counts)])
        hs, flat, off = hists(rng, int(ro[-1]), 40)
        parent = np.stack([rng.integers(0, c, 4) for c in counts]).astype(np.int32)
        tok = rng.integers(0, 99, parent.shape).astype(np.int32)
        out, o = F.hist_fork(flat, off, parent, tok, row_off=ro)
        same_hists(out, o, BU.fork(hs, ro, parent, tok))


def test_fork_errors():
    rng = np.random.default_rng(2)
    hs, flat, off = hists(rng, 8, 30)
    parent = np.array([[0, 1, 2, 3], [3, 2, 9, 0]], np.int32)
    tok = np.arange(8, dtype=np.int32).reshape(2, 4)
    out, o = F.hist_fork(flat, off, parent, tok)
    same_hists(out, o, BU.fork(hs, [0, 4, 8], parent, tok))   # (the parent past the rows: an empty history)
    assert F.device_error() == _lib.FS_DEVERR_PARENT
    parent[1, 2] = 1
    want = [t for h in BU.fork(hs, [0, 4, 8], parent, tok) for t in h]
    for cap in (0, 1, len(want) - 1):
        buf = torch.full((len(want) + 64,), -7, dtype=torch.int32, device="cuda")
        o = torch.empty(9, dtype=torch.int64, device="cuda")
        P = F.sampler._ptr
        ctx = F.Context.default()
        keep = [cuda(a) for a in (flat, off, parent, tok)]
        _lib.check(_lib.lib().fs_hist_fork(ctx.h, 2, P(keep[0]), P(keep[1]), None, 4, P(keep[2]), P(keep[3]), P(buf), cap, P(o),
                                           F.sampler._stream()), "fs_hist_fork")
        assert F.device_error() == _lib.FS_DEVERR_HIST_APPEND
        got = buf.cpu().tolist()
        assert got[:cap] == want[:cap] and got[cap:] == [-7] * (len(got) - cap)
    out, o = F.hist_fork(np.zeros(0, np.int32), np.zeros(9, np.int64), parent, tok)
    same_hists(out, o, [[int(t)] for t in tok.reshape(-1)])
    for bad in (dict(tok=tok[:1]), dict(hist_off=off[:-1]), dict(row_off=[0, 8]), dict(row_off=[0, 3, 4]), dict(parent=parent[0])):
        kw = dict(hist=flat, hist_off=off, parent=parent, tok=tok)
        kw.update(bad)
        with pytest.raises(F.SamplerError):
            F.hist_fork(**kw)


# ------------------------------------------------------------------------------------------------ states
def filled(shape, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    if dtype == torch.uint8:
        return torch.randint(0, 256, shape, device="cuda", generator=g, dtype=dtype)
    if dtype == torch.int64:
        return torch.randint(0, 1 << 60, shape, device="cuda", generator=g, dtype=dtype)
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def moved(src, dst, parent, pos=None, start=None, length=None):
    """What dst becomes."""
    S, n = parent.shape
    n_src = src.shape[0] // S
    old, out = src.cpu(), dst.cpu().clone()
    for s in range(S):
        for j in range(n):
            p = int(parent[s, j])
            if p < 0 or p >= n_src:
                continue
            a, b = old[s * n_src + p], out[s * n + j]
            if pos is None:
                b.copy_(a)
            else:
                m = min(a.shape[pos - 1], b.shape[pos - 1])
                lo = max(int(start[s]) if start is not None else 0, 0)
                hi = min(int(length[s]) if length is not None else m, m)
                if lo < hi:
                    b.narrow(pos - 1, lo, hi - lo).copy_(a.narrow(pos - 1, lo, hi - lo))
    return out


def parents(rng, S, n, n_src, kind):
    if kind == "perm" and n == n_src:
        return np.stack([rng.permutation(n) for _ in range(S)]).astype(np.int32)
    if kind == "same" and n == n_src:
        return np.tile(np.arange(n, dtype=np.int32), (S, 1))
    return rng.integers(-1 if kind == "some" else 0, n_src, (S, n)).astype(np.int32)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("kind", ["perm", "some", "any", "same"])
def test_states_in_place(n, kind):
    rng = np.random.default_rng(n)
    S = 3
    p = parents(rng, S, n, n, kind)
    start, length = np.array([0, 3, 5], np.int32), np.array([40, 17, 99], np.int32)
    for dtype, shape, pos in ((torch.bfloat16, (2, 40, 16), 2), (torch.float32, (40, 3, 5), 1), (torch.uint8, (3, 40, 7), 2),
                              (torch.float16, (1, 40, 129), 2), (torch.float32, (600,), None), (torch.bfloat16, (3, 7), None),
                              (torch.int64, (33,), None)):
        x = filled((S * n, *shape), dtype, n)
        want = moved(x, x, p, pos, start, length)
        F.reorder_states(F.States([x], pos_dim=pos), cuda(p), cuda(start), cuda(length))
        assert torch.equal(x.cpu(), want), (dtype, shape)


@pytest.mark.parametrize("n_src,n", [(1, 4), (1, 64), (4, 1), (3, 5), (5, 3), (64, 64), (1, 1), (20, 9)])
def test_states_into_other_buffers(n_src, n):
    rng = np.random.default_rng(n_src * 100 + n)
    S = 4
    p = parents(rng, S, n, n_src, "some")
    start, length = np.array([0, 0, 7, 30], np.int32), np.array([0, 64, 50, 30], np.int32)
    src = [filled((S * n_src, 2, 64, 24), torch.bfloat16, 1), filled((S * n_src, 2, 64, 24), torch.bfloat16, 2)]
    dst = [filled((S * n, 2, 100, 24), torch.bfloat16, 3), filled((S * n, 2, 50, 24), torch.bfloat16, 4)]
    want = [moved(a, b, p, 2, start, length) for a, b in zip(src, dst)]
    was = [a.clone() for a in src]
    F.reorder_states(F.States(src, dst, pos_dim=2), cuda(p), cuda(start), cuda(length))
    for a, b, c, d in zip(src, dst, want, was):
        assert torch.equal(b.cpu(), c) and torch.equal(a, d)


def test_states_strides():
    """Rows, blocks and positions any stride apart: keys and values in one buffer, positions before heads, padded rows, rows in
    the middle, unaligned bytes."""
    rng = np.random.default_rng(5)
    S, n = 2, 6
    p = parents(rng, S, n, n, "perm")
    length = np.array([9, 13], np.int32)
    kv = filled((S * n, 13, 2, 4, 10), torch.bfloat16, 1)      # [rows, positions, k / v, heads, dim]
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = [moved(k, k, p, 1, None, length), moved(v, v, p, 1, None, length)]
    F.reorder_states(F.States([k, v], pos_dim=1), cuda(p), length=cuda(length))
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    m = filled((13, S * n, 3, 8), torch.float32, 2).transpose(0, 1)       # rows in the middle
    want = moved(m, m, p, 1, None, length)
    F.reorder_states(F.States([m], pos_dim=1), cuda(p), length=cuda(length))
    assert torch.equal(m.cpu(), want)
    for cut in (1, 2, 3, 8):                                   # unaligned rows and pointers
        u = filled((S * n, 3 * 13 * 5 + cut + 4), torch.uint8, 3)
        t = u[:, cut:cut + 195].unflatten(1, (3, 13, 5))
        want, edge = moved(t, t, p, 2, None, length), u[:, :cut].clone()
        F.reorder_states(F.States([t], pos_dim=2), cuda(p), length=cuda(length))
        assert torch.equal(t.cpu(), want) and torch.equal(u[:, :cut], edge)
    g = filled((S * n, 2, 3, 13, 16), torch.float16, 4)        # groups and heads fold into blocks
    want = moved(g, g, p, 3, None, length)
    F.reorder_states(F.States([g], pos_dim=3), cuda(p), length=cuda(length))
    assert torch.equal(g.cpu(), want)


def test_states_many_and_mixed():
    """More states than a launch takes, of several widths and kinds in one call; empty ones; lengths out of range."""
    rng = np.random.default_rng(6)
    S, n = 5, 4
    p = parents(rng, S, n, n, "any")
    start = np.array([-3, 0, 4, 90, 2], np.int32)
    length = np.array([5, 1000, 3, 99, -1], np.int32)
    xs, dims = [], []
    for i in range(75):
        kind = i % 4
        xs.append(filled((S * n, 2, 20 + i, 8) if kind == 0 else (S * n, 11 + i) if kind == 1 else (S * n, 20, 3, i + 1)
                         if kind == 2 else (S * n, 2, 0, 8), [torch.float32, torch.bfloat16, torch.uint8, torch.float32][kind], i))
        dims.append([2, None, 1, 2][kind])
    want = [moved(x, x, p, d, start, length) for x, d in zip(xs, dims)]
    F.reorder_states(F.States(xs, pos_dim=dims), cuda(p), cuda(start), cuda(length))
    for i, (x, w) in enumerate(zip(xs, want)):
        assert torch.equal(x.cpu(), w), i


def test_states_large():
    """A state that takes many workgroups of a stream, and many streams."""
    rng = np.random.default_rng(7)
    x = filled((8, 8, 4096, 64), torch.bfloat16, 1)
    p = parents(rng, 2, 4, 4, "perm")
    start, length = np.array([100, 0], np.int32), np.array([4001, 4096], np.int32)
    want = moved(x, x, p, 2, start, length)
    F.reorder_states(F.States([x], pos_dim=2), cuda(p), cuda(start), cuda(length))
    assert torch.equal(x.cpu(), want)
    y = filled((1400, 500), torch.float32, 2)
    p = parents(rng, 700, 2, 2, "any")
    want = moved(y, y, p)
    F.reorder_states([y], cuda(p))
    assert torch.equal(y.cpu(), want)


def test_states_errors():
    x = filled((8, 100), torch.float32, 1)
    p = np.array([[0, 1, 2, 3], [1, 4, 0, -1]], np.int32)
    want = moved(x, x, p)
    F.reorder_states([x], cuda(p))
    assert F.device_error() == _lib.FS_DEVERR_PARENT
    assert torch.equal(x.cpu(), want)
    y = torch.zeros((8, 4, 6), device="cuda")
    with pytest.raises(F.SamplerError):
        F.reorder_states([x[:7]], p)                           # rows that are not streams' rows
    with pytest.raises(F.SamplerError):
        F.reorder_states([x.cpu()], p)
    with pytest.raises(F.SamplerError):
        F.reorder_states([x], p, start=np.zeros(3, np.int32))
    with pytest.raises(F.SamplerError):
        F.reorder_states([x], p[0])
    with pytest.raises(F.SamplerError):                        # overlapping buffers that are not in place
        F.reorder_states(F.States([x[:4]], [x]), np.array([[0, 1, 2, 3], [1, 1, 0, 1]], np.int32))
    with pytest.raises(F.SamplerError):
        F.States([y], [torch.zeros((8, 5, 6), device="cuda")])
    with pytest.raises(F.SamplerError):
        F.States([y], pos_dim=0)
    with pytest.raises(F.SamplerError):
        F.States([y.transpose(1, 2)], pos_dim=1)               # what lies behind a position is not packed
