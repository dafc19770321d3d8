"""GPU: calls of the beam search that a long run, a captured one or an unusual program makes (tests/beam_util.py)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import _lib  # noqa: E402
from tests import beam_util as BU  # noqa: E402
from tests.test_gpu_beam import Rows  # noqa: E402
from tests.test_gpu_beam_run import Model, search  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------------------------------------------ selection
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("counts,n,V", [([4, 4], 4, 5000), ([1, 0, 3, 0, 0], 3, 70001), ([5, 0, 9], 8, 4099), ([0, 0, 40], 64, 300),
                                        ([70, 2], 20, 900)])
def test_select_rows_behind_the_last_stream(counts, n, V, kind):
    """A padded batch: offsets on the device, rows behind the last stream's (whose mask indices and scores mean nothing), in a
    context that goes on to other calls; a stream that ends past the rows ends with them; no stream has a row."""
    r = Rows(n, counts, V, kind)
    R, pad = int(r.off[-1]), 7
    x = torch.cat([r.x, torch.full((pad, V), 9.0, device="cuda", dtype=r.x.dtype)])
    ctx, all_on = F.Context(), np.full(R + pad, -1, np.int32)
    all_on[R:] = 99
    ed = F.Edits(mask=F.Edits.pack(np.ones((1, V), bool)), mask_of=all_on)
    alone = F.beam_select(r.x, cuda(r.score), n, eos_id=3, row_off=r.off, ctx=ctx)
    BU.Step(r.y, r.score, r.off, n, 3).check(alone)
    past, none = r.off.copy(), np.zeros_like(r.off)
    past[-1] += 1000
    live = torch.zeros(pad, device="cuda")
    for i in range(3):
        padded = F.beam_select(x, torch.cat([cuda(r.score), live + i]), n, eos_id=3, row_off=cuda(r.off), edits=ed, ctx=ctx)
        cut = F.beam_select(r.x, cuda(r.score), n, eos_id=3, row_off=cuda(past), ctx=ctx)
        empty = F.beam_select(x, None, n, eos_id=3, row_off=cuda(none), ctx=ctx)
        again = F.beam_select(r.x, cuda(r.score), n, eos_id=3, row_off=r.off, ctx=ctx)
        for k in ("parent", "tok", "done", "done_parent"):
            assert torch.equal(padded[k], alone[k]) and torch.equal(cut[k], alone[k]) and torch.equal(again[k], alone[k]), (i, k)
            assert torch.all(empty[k] == (0 if k == "done" else -1)), k
        for k in ("score", "done_score"):                      # (rows split otherwise: the last bit of a sum)
            assert torch.allclose(padded[k], alone[k], rtol=2 * BU.U, atol=2 * BU.TOL), (i, k)
            assert torch.equal(cut[k], alone[k]) and torch.equal(again[k], alone[k]) and torch.all(empty[k] == -np.inf), (i, k)
    assert F.device_error(ctx) == 0


@pytest.mark.parametrize("n", [16, 17, 40, 63, 64])
@pytest.mark.parametrize("V", [300, 20000, 262144])
def test_select_dead_streams_of_few_rows(n, V):
    """Streams of one to five rows, dead ones between live ones: a wave or a workgroup a row, and rows that end by themselves."""
    r = Rows(n, [1, 1, 2, 1, 4, 3, 5, 5, 1], V, "bf16")
    for dead in ([0], [1, 2, 3], [4, 5, 7], [8, 10, 11], [12, 13, 14, 15, 16, 17, 21], range(22), [0, 4, 22]):
        r.score = (-r.rng.exponential(2.0, 23)).astype(np.float32)
        r.score[list(dead)] = -np.inf
        out = r.run(n, eos=int(r.y[3].argmax()))
        for s in range(9):
            if np.all(r.score[r.off[s]:r.off[s + 1]] == -np.inf):
                assert out["parent"][s].tolist() == [-1] * n and int(out["done"][s]) == 0


def test_select_dead_rows_after_better_ones():
    """What an earlier call's rows left in the workspace does not come back for dead ones."""
    for n, counts in ((4, [4]), (64, [1, 4, 5]), (8, [9, 70])):
        r = Rows(3, counts, 5000)
        ctx, best = F.Context(), Rows(4, counts, 5000)
        best.score[:] = 1000.0
        best.x[:, 7] = float("inf")
        r.score[::2] = -np.inf
        for _ in range(3):
            F.beam_select(best.x, cuda(best.score), n, row_off=best.off, eos_id=5, ctx=ctx)
            out = F.beam_select(r.x, cuda(r.score), n, row_off=r.off, eos_id=5, ctx=ctx)
            BU.Step(r.y, r.score, r.off, n, 5).check(out)


def test_select_outputs_beside_inputs():
    """Outputs in one buffer with the scores and offsets, next to them on both sides, are taken."""
    S, n, V = 2, 4, 3000
    r = Rows(5, [n] * S, V)
    want = F.beam_select(r.x, cuda(r.score), n, eos_id=3, row_off=r.off)
    buf = torch.full((64,), -7, dtype=torch.int32, device="cuda")
    at = dict(parent=(0, 8), score_in=(8, 16), tok=(16, 24), score=(24, 32), off=(32, 38), done=(38, 40), dp=(40, 48), ds=(48, 56))
    v = {k: buf[a:b] for k, (a, b) in at.items()}
    v["score_in"].view(torch.float32).copy_(cuda(r.score))
    v["off"].view(torch.int64).copy_(cuda(r.off))
    ctx, p = F.Context.default(), F.sampler._ptr
    _lib.check(_lib.lib().fs_beam_select(ctx.h, p(r.x), F.F32, r.x.stride(0), S, S * n, V, p(v["off"]), p(v["score_in"]), None, None,
                                         3, n, 0, p(v["parent"]), p(v["tok"]), p(v["score"]), p(v["done"]), p(v["dp"]), p(v["ds"]),
                                         F.sampler._stream()), "select")
    assert torch.equal(v["parent"].view(S, n), want["parent"]) and torch.equal(v["tok"].view(S, n), want["tok"])
    assert torch.equal(v["score"].view(torch.float32).view(S, n), want["score"]) and torch.equal(v["done"], want["done"])
    assert v["off"].view(torch.int64).tolist() == r.off.tolist() and torch.all(buf[56:] == -7)


def test_captured_select_of_smaller_batches():
    """A recorded call of nine rows, replayed for batches of fewer rows and streams: what changes is in the offsets' tensor."""
    n, V = 3, 6000
    ctx, r = F.Context(), Rows(8, [9], V)
    score, off = cuda(r.score), cuda(np.array([0, 3, 6, 9]))
    F.beam_select(r.x, score, n, eos_id=4, row_off=off, ctx=ctx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.beam_select(r.x, score, n, eos_id=4, row_off=off, ctx=ctx)
    for cut in ([0, 3, 6, 9], [0, 3, 3, 3], [0, 0, 0, 0], [0, 1, 2, 3], [0, 0, 4, 8], [0, 0, 0, 1], [0, 9, 9, 9], [0, 0, 0, 0],
                [0, 3, 6, 9]):
        off.copy_(torch.tensor(cut))
        graph.replay()
        m = cut[-1]
        BU.Step(r.y[:m], r.score[:m], np.array(cut), n, 4).check(out)
    assert F.device_error(ctx) == 0


def test_select_scores_in_host_memory():
    """Scores as an array or a list, [streams, rows each] or [rows], as the other arguments may be."""
    r = Rows(6, [3, 3, 3, 3], 700)
    want = F.beam_select(r.x, cuda(r.score), 4, streams=4)
    two = r.score.reshape(4, 3)
    for score, kw in ((two, {}), (two.tolist(), {}), (torch.from_numpy(two), {}), (r.score, dict(streams=4)),
                      (two.astype(np.float64), {})):
        out = F.beam_select(r.x, score, 4, **kw)
        assert all(torch.equal(out[k], want[k]) for k in want)
    for score in (r.score, r.score.tolist(), None, two[:3], 1.0):
        with pytest.raises(F.SamplerError):
            F.beam_select(r.x, score, 4)


# ------------------------------------------------------------------------------------------------ histories
@pytest.mark.parametrize("how", ["default", "max_len", "stream"])
@pytest.mark.parametrize("S,n,steps", [(3, 8, 200), (1, 64, 60), (40, 1, 60)])
def test_fork_room_over_a_long_search(how, S, n, steps):
    """A search's histories in buffers that grow by a token per beam and step, as its ids do."""
    rng = np.random.default_rng(S)
    stream = torch.cuda.Stream() if how == "stream" else None
    lens = rng.integers(1, 20, S)
    longest = int(lens.max())
    off = np.concatenate([[0], np.cumsum(lens)])
    ids = rng.integers(0, 1 << 20, int(off[-1])).astype(np.int32)
    host = [ids[off[s]:off[s + 1]].tolist() for s in range(S)]
    hist, off, ro = cuda(ids), cuda(off), np.arange(S + 1)
    for step in range(steps):
        parent = rng.integers(0, 1 if step == 0 else n, (S, n)).astype(np.int32)
        tok = rng.integers(0, 1 << 20, (S, n)).astype(np.int32)
        host = BU.fork(host, ro if step == 0 else np.arange(0, S * n + 1, n), parent, tok)
        hist, off = F.hist_fork(hist, off, cuda(parent), cuda(tok), row_off=ro if step == 0 else None, stream=stream,
                                max_len=longest + step if how == "max_len" else None)
        assert hist.numel() <= S * n * (longest + step + 1), step
        assert hist.numel() >= sum(len(h) for h in host), step
    torch.cuda.synchronize()
    end = off.tolist()
    assert end == np.concatenate([[0], np.cumsum([len(h) for h in host])]).tolist()
    assert hist[:end[-1]].tolist() == [t for h in host for t in h]


def test_fork_room_of_offsets_on_the_host():
    """Offsets in host memory, streams of unlike rows: room for n of a stream's longest, for any parents."""
    off, ro = np.array([2, 5, 5, 14, 15]), [0, 0, 3, 4]
    hist = cuda(np.arange(100, dtype=np.int32))
    parent, tok = np.array([[-1, -1], [2, 2], [0, 0]], np.int32), np.arange(6, dtype=np.int32).reshape(3, 2)
    for t in (tok, None):
        out, o = F.hist_fork(hist, off, parent, t, row_off=ro)
        again, _ = F.hist_fork(hist, cuda(off.astype(np.int32))[None], parent, t, row_off=cuda(np.array(ro, np.int32))[None])
        assert again.numel() == out.numel() and torch.equal(again[:int(o[-1])], out[:int(o[-1])])
        assert out.numel() == 2 * (0 + 9 + 1) + (6 if t is not None else 0)
        want = BU.fork([np.arange(a, b) for a, b in zip(off, off[1:])], ro, parent, t)
        assert out[:int(o[-1])].tolist() == [x for h in want for x in h]


def test_fork_room_in_a_captured_call():
    """A recorded call does not wait: it has room for any parents of whatever hist holds at a replay."""
    hist, off = cuda(np.arange(24, dtype=np.int32)), cuda(np.arange(0, 25, 6))
    parent, tok = cuda(np.zeros((2, 2), np.int32)), cuda(np.full((2, 2), 99, np.int32))
    ctx = F.Context()
    F.hist_fork(hist, off, parent, tok, ctx=ctx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, o = F.hist_fork(hist, off, parent, tok, ctx=ctx)
    assert out.numel() == 24 * 2 + 4
    for cut in ([0, 0, 24, 24, 24], [0, 24, 24, 24, 24], [0, 1, 2, 3, 4]):
        off.copy_(torch.tensor(cut))
        parent.copy_(torch.tensor([[1, 0], [1, 1]]))
        hist.add_(1)
        graph.replay()
        want = BU.fork([hist.tolist()[a:b] for a, b in zip(cut, cut[1:])], [0, 2, 4], parent.tolist(), tok.tolist())
        assert out[:int(o[-1])].tolist() == [x for h in want for x in h]


def test_fork_refuses_streams_without_beams():
    with pytest.raises(F.SamplerError):
        F.hist_fork(cuda(np.zeros(4, np.int32)), [0, 2, 4], np.zeros((2, 0), np.int32), row_off=[0, 1, 2])


# ------------------------------------------------------------------------------------------------ whole searches
@pytest.mark.parametrize("S,n,V,steps", [(3, 4, 211, 8), (1, 1, 50, 5), (2, 17, 131, 5)])
def test_steps_of_the_c_abi_on_two_buffers(S, n, V, steps):
    """The prompts' step and those behind it by the C calls, as a C++ program makes them: scores, histories and offsets change
    between two buffers after every step, the prompts' too; the first of them holds only the prompts' offsets."""
    model, rng = Model(S, V), np.random.default_rng(S)
    prompts = [rng.integers(1, V, int(rng.integers(1, 6))).tolist() for _ in range(S)]
    want = search(model, prompts, n, steps, 0)
    L, P, ctx = _lib.lib(), F.sampler._ptr, F.Context()
    i32 = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")
    parent, tok, done, done_parent, done_score = i32(S, n), i32(S, n), i32(S), i32(S, n), torch.zeros((S, n), device="cuda")
    score = [torch.full((S, n), float("nan"), device="cuda") for _ in range(2)]
    cap = S * n * (5 + steps)
    hist, hoff = [i32(cap) for _ in range(2)], [torch.full((S * n + 1,), -1, dtype=torch.int64, device="cuda") for _ in range(2)]
    lens = [len(p) for p in prompts]
    hist[0][:sum(lens)] = cuda(np.concatenate(prompts).astype(np.int32))
    hoff[0][:S + 1] = cuda(np.concatenate([[0], np.cumsum(lens)]))
    row_off1, prompt_len = cuda(np.arange(S + 1)), cuda(np.array(lens, np.int32))
    length = prompt_len.clone()
    pc = torch.zeros((S, 2, 32, model.dim // 2), device="cuda")
    for s, p in enumerate(prompts):
        pc[s, :, :len(p)] = model.dev[1][torch.tensor(p, device="cuda")].view(len(p), 2, -1).transpose(0, 1)
    cache = torch.full((S * n, 2, 32, model.dim // 2), float("nan"), device="cuda")
    opening, states = F.States([pc], [cache], pos_dim=2), F.States([cache], pos_dim=2)
    logits = model.device(torch.tensor([p[-1] for p in prompts], device="cuda"), pc, length)
    st, cur, ended = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), 0, [[] for _ in range(S)]
    for step in range(steps):
        x, ld, _, kind = F.sampler._typed_logits(logits, V)
        first = step == 0
        _lib.check(L.fs_beam_select(ctx.h, F.sampler._lptr(x), kind, ld, S, S if first else S * n, V,
                                    P(row_off1) if first else None, None if first else P(score[cur]), None, None, 0, n,
                                    F.BEAM_KEEP_SLOTS, P(parent), P(tok), P(score[cur ^ 1]), P(done), P(done_parent),
                                    P(done_score), st), "select")
        h, o = hist[cur].tolist(), hoff[cur].tolist()
        for s in range(S):
            for j in range(int(done[s])):
                r = s * (1 if first else n) + int(done_parent[s, j])
                ended[s].append(h[o[r]:o[r + 1]] + [0])
        _lib.check(L.fs_hist_fork(ctx.h, S, P(hist[cur]), P(hoff[cur]), P(row_off1) if first else None, n, P(parent), P(tok),
                                  P(hist[cur ^ 1]), cap, P(hoff[cur ^ 1]), st), "fork")
        _lib.check(L.fs_reorder_states(ctx.h, 1, opening.c if first else states.c, S, 1 if first else n, n, P(parent),
                                       None if first else P(prompt_len), P(length), st), "states")
        cur ^= 1
        rows = length.repeat_interleave(n).long()
        cache[torch.arange(S * n, device="cuda"), :, rows] = model.dev[1][tok.view(-1).long()].view(S * n, 2, -1)
        length += 1
        logits = model.device(tok.view(-1), cache, length.repeat_interleave(n))
    h, o = hist[cur].tolist(), hoff[cur].tolist()
    for s, (beams, done) in enumerate(want):
        got = score[cur][s].tolist()
        order = sorted(range(n), key=lambda j: (-got[j], j))
        assert [h[o[s * n + j]:o[s * n + j + 1]] for j in order] == [b[0] for b in beams], s
        assert ended[s] == [e[0] for e in done], s
