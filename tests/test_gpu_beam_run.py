"""GPU: whole beam searches by beam_select, hist_fork and reorder_states, as a program runs them, against a search on the CPU;
captured steps; other streams; offsets past 32 bits."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import _lib  # noqa: E402
from tests import beam_util as BU  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


class Model:
    """Logits from the last token and the sum of a cache of embeddings, in values whose sums are exact in fp32: multiples of
    2^-9 below 2^12 however they are added."""

    def __init__(self, seed, V, dim=8):
        g = np.random.default_rng(seed)
        self.V, self.dim = V, dim
        self.last = (g.integers(-1500, 1500, (V, V)) / 512).astype(np.float32)
        self.emb = g.integers(-2, 3, (V, dim)).astype(np.float32)
        self.out = (g.integers(-120, 120, (dim, V)) / 512).astype(np.float32)
        self.dev = [torch.from_numpy(a).cuda() for a in (self.last, self.emb, self.out)]

    def host(self, toks):
        return self.last[toks[-1]] + self.emb[np.array(toks)].sum(0) @ self.out

    def device(self, last, cache, length):
        """cache [rows, heads, positions, dim / heads], length [rows]"""
        m = torch.arange(cache.shape[2], device="cuda")[None, None, :, None] < length[:, None, None, None]
        s = torch.where(m, cache, 0.0).sum(2).reshape(cache.shape[0], -1)
        return self.dev[0][last.long()] + (s.double() @ self.dev[2].double()).float()


def search(model, prompts, n, steps, eos):
    """A stream's beams and ended hypotheses by the definition: [(tokens, score)] sorted, [(tokens, score)] as they ended."""
    out = []
    for prompt in prompts:
        beams, ended = [(list(prompt), np.float32(0))], []
        for _ in range(steps):
            cand = []
            for i, (toks, score) in enumerate(beams):
                lp = BU.log_softmax64(model.host(toks), 1.0)
                cand += [(-(float(score) + lp[t]), t != eos, i, t) for t in range(model.V)]
            cand.sort()
            new = []
            for rank, (c, _, i, t) in enumerate(cand):
                if t == eos and rank < n:
                    ended.append((beams[i][0] + [t], np.float32(-c)))
                elif t != eos and len(new) < n:
                    new.append((beams[i][0] + [t], np.float32(-c)))
            beams = new
        out.append((beams, ended))
    return out


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("seed,S,n,V,steps", [(1, 3, 4, 211, 12), (2, 1, 1, 50, 9), (3, 5, 7, 97, 10), (4, 2, 17, 131, 6), (5, 2, 64, 300, 4)])
def test_search(seed, S, n, V, steps, slots):
    model = Model(seed, V)
    rng = np.random.default_rng(seed)
    prompts = [rng.integers(1, V, int(rng.integers(1, 6))).tolist() for _ in range(S)]
    eos = 0
    want = search(model, prompts, n, steps, eos)
    # the prompts' caches: a row per stream, then a row per beam; beams of a stream share the prompt's positions
    cap, heads = 32, 2
    start = np.array([len(p) for p in prompts], np.int32)
    pc = torch.zeros((S, heads, cap, model.dim // heads), device="cuda")
    for s, p in enumerate(prompts):
        e = model.dev[1][torch.tensor(p, device="cuda")]                   # [len, dim]
        pc[s, :, :len(p)] = e.view(len(p), heads, -1).transpose(0, 1)
    cache = torch.full((S * n, heads, cap, model.dim // heads), float("nan"), device="cuda")
    hist = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device="cuda")
    off = torch.tensor(np.concatenate([[0], np.cumsum(start)]), dtype=torch.int64, device="cuda")
    start = torch.from_numpy(start).cuda()
    length, ended = start.clone(), [[] for _ in range(S)]
    logits = model.device(torch.tensor([p[-1] for p in prompts], device="cuda"), pc, length)
    score, ro = None, np.arange(S + 1)
    live = F.States([cache], pos_dim=2)
    for step in range(steps):
        out = F.beam_select(logits, score, n, eos_id=eos, row_off=ro, keep_slots=slots)
        h, o = hist.cpu().numpy(), off.cpu().numpy()
        for s in range(S):
            for j in range(int(out["done"][s])):
                r = int(ro[s]) + int(out["done_parent"][s, j])
                ended[s].append((h[o[r]:o[r + 1]].tolist() + [eos], float(out["done_score"][s, j])))
        hist, off = F.hist_fork(hist, off, out["parent"], out["tok"], row_off=ro)
        if step == 0:                                          # the prompts' rows open the beams
            F.reorder_states(F.States([pc], [cache], pos_dim=2), out["parent"], length=length)
        else:
            F.reorder_states(live, out["parent"], start=start, length=length)
        ro, score = np.arange(0, S * n + 1, n), out["score"].view(-1)
        tok = out["tok"].view(-1).clamp(min=0)
        rows = length.repeat_interleave(n).long()
        cache[torch.arange(S * n, device="cuda"), :, rows] = model.dev[1][tok.long()].view(S * n, heads, -1)
        length = length + 1
        logits = model.device(tok, cache, length.repeat_interleave(n))
    h, o = hist.cpu().numpy(), off.cpu().numpy()
    got = out["score"].cpu().numpy()
    for s in range(S):
        rows = sorted(range(n), key=lambda j: (-got[s, j], j)) if slots else range(n)
        beams, done = want[s]
        assert [h[o[s * n + j]:o[s * n + j + 1]].tolist() for j in rows] == [b[0] for b in beams], s
        # a step adds TOL and two roundings of the score
        err = [steps * (BU.TOL + 2 * BU.U * abs(b[1])) for b in beams]
        assert np.all(np.abs(got[s][list(rows)] - [b[1] for b in beams]) <= err), s
        assert [e[0] for e in ended[s]] == [e[0] for e in done], s
        assert all(abs(a[1] - b[1]) <= steps * (BU.TOL + 2 * BU.U * abs(b[1])) for a, b in zip(ended[s], done)), s


def test_search_under_a_grammar():
    """Masks by row and biases by stream, of which one stream runs out of tokens: its beams die, the other goes on."""
    V, n = 300, 3
    rng = np.random.default_rng(7)
    x = [rng.normal(0, 2, (2 * n, V)).astype(np.float32) for _ in range(3)]
    allowed = rng.random((2 * n, V)) < 0.3
    none = allowed.copy()
    none[:n] = False
    bias = [[(5, 2.0), (7, -np.inf)], [(9, 1.5)]]
    score = np.zeros(2 * n, np.float32)
    for x_, ok in zip(x, (allowed, none, allowed)):
        from tests import edit_util as U
        ed = F.Edits(mask=F.Edits.pack(ok), bias=U.csr(bias))
        off = np.arange(0, 2 * n + 1, n)
        out = F.beam_select(torch.from_numpy(x_).cuda(), torch.from_numpy(score).cuda(), n, eos_id=11, row_off=off, edits=ed)
        BU.Step(x_, score, off, n, 11, None, bias, list(ok)).check(out)
        score = out["score"].cpu().numpy().reshape(-1)
    assert out["parent"][0].tolist() == [-1] * n and out["parent"][1].min() >= 0


# ------------------------------------------------------------------------------------------------ graphs and streams
def step_calls(ctx, S, n, V, x, score, hist, off, states, stream):
    """The three launches of a step on fixed buffers."""
    P, L = F.sampler._ptr, _lib.lib()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    b = dict(parent=i32(S, n), tok=i32(S, n), out=torch.zeros((S, n), device="cuda"), done=i32(S), dp=i32(S, n),
             ds=torch.zeros((S, n), device="cuda"), hist=i32(hist.numel() * n + S * n), off=torch.zeros(S * n + 1, dtype=torch.int64, device="cuda"))

    def run():
        st = ctypes.c_void_p(stream())
        _lib.check(L.fs_beam_select(ctx.h, P(x), F.F32, V, S, S * n, V, None, P(score), None, None, 3, n, 1, P(b["parent"]), P(b["tok"]),
                                    P(b["out"]), P(b["done"]), P(b["dp"]), P(b["ds"]), st), "select")
        _lib.check(L.fs_hist_fork(ctx.h, S, P(hist), P(off), None, n, P(b["parent"]), P(b["tok"]), P(b["hist"]), b["hist"].numel(),
                                  P(b["off"]), st), "fork")
        _lib.check(L.fs_reorder_states(ctx.h, len(states), states.c, S, n, n, P(b["parent"]), None, None, st), "states")
    return b, run


@pytest.mark.parametrize("S,n,V", [(3, 4, 4096), (2, 33, 30000), (1, 1, 5000)])
def test_captured_steps(S, n, V):
    """A step recorded into a graph and replayed on new inputs, eager calls of another context between the replays."""
    g = torch.Generator("cuda").manual_seed(S)
    x = torch.zeros((S * n, V), device="cuda")
    score = torch.zeros(S * n, device="cuda")
    hist = torch.arange(S * n * 7, dtype=torch.int32, device="cuda")
    off = torch.arange(0, S * n * 7 + 1, 7, dtype=torch.int64, device="cuda")
    cache = torch.zeros((S * n, 2, 9, 8), device="cuda")
    other = torch.zeros_like(cache)
    cur = lambda: torch.cuda.current_stream().cuda_stream
    ctx = F.Context()
    kept, captured = step_calls(ctx, S, n, V, x, score, hist, off, F.States([cache]), cur)
    want, eager = step_calls(F.Context(), S, n, V, x, score, hist, off, F.States([other]), cur)
    captured()                                                 # warm: the workspaces are there
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    for i in range(4):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g) * 2)
        score.copy_(-torch.rand(score.shape, device="cuda", generator=g) * 9)
        cache.copy_(torch.randn(cache.shape, device="cuda", generator=g))
        other.copy_(cache)
        graph.replay()
        eager()
        torch.cuda.synchronize()
        for k in ("parent", "tok", "out", "done", "dp", "ds", "off"):
            assert torch.equal(kept[k], want[k]), (i, k)
        m = int(kept["off"][-1])
        assert torch.equal(kept["hist"][:m], want["hist"][:m]) and torch.equal(cache, other), i


def test_capture_refuses_to_grow():
    """A recorded call whose workspace would have to grow is refused, and the capture goes on."""
    x = torch.randn((8, 8192), device="cuda")
    ctx = F.Context()
    F.beam_select(x[:1], None, 2, streams=1, ctx=ctx)
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        with pytest.raises(F.SamplerError, match="allocation"):
            F.beam_select(x, None, 2, streams=2, ctx=ctx)
        y += 1
    graph.replay()
    torch.cuda.synchronize()
    assert y.tolist() == [1.0] * 4
    a = F.beam_select(x, None, 2, streams=2, ctx=ctx)
    b = F.beam_select(x, None, 2, streams=2)
    assert torch.equal(a["tok"], b["tok"]) and torch.equal(a["score"], b["score"])


def test_two_streams_and_contexts_at_once():
    """Steps on two streams, a context each, in flight together."""
    S, n, V = 4, 6, 20000
    runs = []
    for i in range(2):
        g = torch.Generator("cuda").manual_seed(i)
        x, score = torch.randn((S * n, V), device="cuda", generator=g) * 2, -torch.rand(S * n, device="cuda", generator=g)
        hist = torch.randint(0, V, (S * n * 50,), device="cuda", generator=g, dtype=torch.int32)
        off = torch.arange(0, S * n * 50 + 1, 50, dtype=torch.int64, device="cuda")
        cache = torch.randn((S * n, 4, 64, 32), device="cuda", generator=g)
        runs.append((x, score, hist, off, cache))
    want = []
    for x, score, hist, off, cache in runs:
        c = cache.clone()
        out = F.beam_select(x, score, n, streams=S, eos_id=5, keep_slots=True)
        h, o = F.hist_fork(hist, off, out["parent"], out["tok"])
        F.reorder_states([c], out["parent"])
        want.append((out, h, o, c))
    torch.cuda.synchronize()
    streams, ctxs, got = [torch.cuda.Stream() for _ in runs], [F.Context() for _ in runs], []
    for _ in range(5):
        got = []
        for (x, score, hist, off, cache), st, ctx in zip(runs, streams, ctxs):
            c = cache.clone()
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                out = F.beam_select(x, score, n, streams=S, eos_id=5, keep_slots=True, ctx=ctx)
                h, o = F.hist_fork(hist, off, out["parent"], out["tok"], ctx=ctx)
                F.reorder_states([c], out["parent"], ctx=ctx)
            got.append((out, h, o, c))
        torch.cuda.synchronize()
        for (a, h, o, c), (b, h2, o2, c2) in zip(got, want):
            assert all(torch.equal(a[k], b[k]) for k in a)
            assert torch.equal(o, o2) and torch.equal(h[:int(o[-1])], h2[:int(o[-1])]) and torch.equal(c, c2)


# ------------------------------------------------------------------------------------------------ large
def room(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GiB of free memory")


def test_states_past_32_bits():
    """Rows 4.5 GB apart, of which the last positions move."""
    room(16)
    x = torch.empty((2, 4_500_000, 1000), dtype=torch.uint8, device="cuda")
    tail = x[:, -10_000:]
    tail.copy_(torch.randint(0, 256, tail.shape, dtype=torch.uint8, device="cuda"))
    want = tail.flip(0).clone()
    F.reorder_states(F.States([x], pos_dim=1), np.array([[1, 0]], np.int32), start=[4_490_000], length=[4_500_000])
    assert torch.equal(x[:, -10_000:], want)


def test_histories_past_32_bits():
    """Seventeen beams of one history of 2^28 ids: 4.6 billion new ids."""
    room(32)
    L = 1 << 28
    hist = torch.arange(L, dtype=torch.int32, device="cuda")
    tok = torch.arange(17, dtype=torch.int32, device="cuda").view(1, 17)
    out, off = F.hist_fork(hist, [0, L], np.zeros((1, 17), np.int32), tok, row_off=[0, 1], out_cap=17 * (L + 1))
    assert off.tolist() == [j * (L + 1) for j in range(18)]
    rows = out.view(17, L + 1)
    assert torch.equal(rows[:, L], tok[0])
    for j in (0, 7, 8, 16):
        assert torch.equal(rows[j, :L], hist), j


def test_logits_past_32_bits():
    """9000 rows of 262144 bf16 logits: the last streams' result is that of their rows alone."""
    room(16)
    S, n, V = 2250, 4, 262144
    x = torch.empty((S * n, V), dtype=torch.bfloat16, device="cuda").normal_()
    score = -torch.rand(S * n, device="cuda")
    a = F.beam_select(x, score, n, streams=S, eos_id=9)
    # (rows split otherwise: sums, and with them scores, may differ in the last bit)
    b = F.beam_select(x[-40:], score[-40:], n, streams=10, eos_id=9)
    for k in ("parent", "tok", "done", "done_parent"):
        assert torch.equal(a[k][-10:], b[k]), k
    assert torch.allclose(a["score"][-10:], b["score"], rtol=2 * BU.U, atol=2 * BU.TOL)


def test_many_histories():
    """More rows than a workgroup keeps the offsets of, some thousands of streams."""
    rng = np.random.default_rng(3)
    for S, n in ((1000, 9), (20000, 1), (5000, 4)):
        lens = rng.integers(0, 6, S * n)
        off = np.concatenate([[0], np.cumsum(lens)])
        flat = rng.integers(0, 1000, int(off[-1])).astype(np.int32)
        parent = rng.integers(-1, n, (S, n)).astype(np.int32)
        tok = rng.integers(0, 1000, (S, n)).astype(np.int32)
        hs = [flat[off[r]:off[r + 1]] for r in range(S * n)]
        out, o = F.hist_fork(flat, off, parent, tok)
        want = BU.fork(hs, np.arange(0, S * n + 1, n), parent, tok)
        o = o.cpu().numpy()
        assert o.tolist() == np.concatenate([[0], np.cumsum([len(h) for h in want])]).astype(int).tolist()
        assert out.cpu().numpy()[:o[-1]].tolist() == [t for h in want for t in h]
