"""GPU: edited calls where they can go wrong - long bias lists, masks that leave the kernels' bounds without logits, capped
rows, ties, far offsets, contexts and streams side by side."""

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from ferro_amd._lib import check, lib  # noqa: E402
from tests import edit_util as U  # noqa: E402
from tests.test_gpu_edits import SETS, Batch, U_pack, check_rows, cuda, lp_tolerance  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


@pytest.mark.parametrize("nb", [1, 64, 65, 130, 256, 257, 1000, 20000])
@pytest.mark.parametrize("name", ["greedy", "small_k", "mid_k", "every", "large_k"])
def test_bias_lists_of_every_length(name, nb):
    """Lists that fit a wave, a workgroup, and neither; ids at the ends of segments, some twice, some outside the
    vocabulary (which do nothing)."""
    B, V = 3, 33001
    b = Batch(nb, B, V, ("most", "few"), nb=0, **SETS[name])
    for r in range(B):
        ids = np.sort(b.rng.integers(-2, V + 3, nb))
        ids[: min(nb, 3)] = np.sort(np.array([0, 4095, 4096][: min(nb, 3)]))
        ids = np.sort(ids)
        b.bias[r] = [(int(t), float(np.float32(b.rng.uniform(-5, 5)))) for t in ids]
    b.bias[1] = b.bias[1][: nb // 2]
    ed = F.Edits(mask=U_pack(b.allowed), mask_of=b.of, bias=U.csr(b.bias))
    out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=ed)
    assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) == 0
    rows = F.edit_batch(cuda(b.x), b.p, b.hist, b.off, edits=ed).cpu().numpy()
    tok = b.rng.integers(0, V, B)
    lp = F.logprobs(cuda(b.x), tok, 5, edits=ed)
    for r in range(B):
        np.testing.assert_array_equal(rows[r], U.edit_row(b.x[r], b.p[r], b.hs[r], b.bias[r], b.ok(r)))
        want = U.logprob_row(b.x[r], int(tok[r]), 5, bias=b.bias[r], allowed=b.ok(r))
        assert lp["ids"][r].tolist() == want[2].tolist() and int(lp["rank"][r]) == want[1]
        if np.isfinite(want[0]):
            assert abs(float(lp["lp"][r]) - want[0]) <= lp_tolerance(want[0])


def shaped(kind, V):
    t = np.arange(V)
    return {"run": (t >= 700) & (t < 5700), "low": t < 9000, "wave": (t // 256) % 4 == 0, "lanes": (t // 4) % 16 == 3,
            "one_in_500": t % 500 == 7, "ends": (t < 5) | (t >= V - 5)}[kind]


@pytest.mark.parametrize("kind", ["run", "low", "wave", "lanes", "one_in_500", "ends"])
@pytest.mark.parametrize("name", ["greedy_counts", "small_k", "mid_k", "every"])
def test_masks_that_leave_lanes_or_waves_empty(name, kind):
    B, V = 4, 70003
    b = Batch(3, B, V, "most", nb=6, H=300, **SETS[name])
    if name == "mid_k":
        b.p["top_k"] = [65, 300, 900, 70]
    b.allowed[:] = shaped(kind, V)
    b.ed = F.Edits(mask=U_pack(b.allowed), mask_of=b.of, bias=U.csr(b.bias))
    for x in (b.x, np.round(b.x).astype(np.float32)):            # and thousands of equal logits
        b.x = x
        out = F.sample_batch(cuda(x), b.p, b.u, b.hist, b.off, edits=b.ed)
        assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 1


@pytest.mark.parametrize("name", ["small_k", "mid_k", "every", "greedy"])
@pytest.mark.parametrize("nb", [0, 8])
def test_capped_rows(name, nb):
    """A softcap beside masks (fused) and beside biases (edited rows); capped -inf is a number, masked ones are not."""
    B, V = 5, 20011
    b = Batch(17 + nb, B, V, ("most", "few"), nb=nb, **dict(SETS[name], softcap=12.0))
    b.x[0, ::7] = -np.inf
    b.x[1, ::5] = np.nan
    for route in ("host", "device"):
        out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=b.ed, route=route)
        assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 1


def test_mixed_caps_in_a_batch():
    b = Batch(23, 6, 30000, ("most", "few"), nb=4, **SETS["mid_k"])
    b.p["softcap"][::2] = 9.0
    out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=b.ed)
    assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 1


@pytest.mark.parametrize("B,V", [(600, 1000), (2100, 257), (33, 300007)])
def test_other_batch_shapes(B, V):
    """Many short rows; rows longer than the mid-k kernel takes."""
    for name in ("greedy", "small_k", "mid_k", "every"):
        b = Batch(B, B, V, ("most", "few"), nb=2, H=5, **SETS[name])
        out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=b.ed)
        assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 3
        if B > 1000:
            break


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_past_32_bit_offsets(dtype):
    """Rows more than 2^31 logits apart, a mask table of more than 2^31 words apart."""
    V, ld = 5000, (1 << 30) + 64
    n = 2 * ld + V + 8
    buf = torch.empty(n, dtype=dtype, device="cuda")
    x = buf.as_strided((3, V), (ld, 1))
    vals = (torch.randn((3, V), device="cuda") * 3).to(dtype)
    x.copy_(vals)
    words = torch.empty(2 * ((1 << 30) + 3) + 200, dtype=torch.int32, device="cuda").as_strided((3, 157), ((1 << 30) + 3, 1))
    rng = np.random.default_rng(5)
    allowed = rng.random((3, V)) < 0.5
    words.copy_(cuda(F.Edits.pack(allowed)))
    ed = F.Edits(mask=words)
    assert ed.mask.data_ptr() == words.data_ptr()
    p = W.make_params(3, top_k=30, temperature=1.0, repetition_penalty=1.0)
    xs = vals.float().cpu().numpy()
    got = F.edit_batch(x, edits=ed).cpu().numpy()
    lp = F.logprobs(x, [1, 2, 3], 4, edits=ed)
    for r in range(3):
        np.testing.assert_array_equal(got[r], np.where(allowed[r], xs[r], -np.inf))
        assert lp["ids"][r].tolist() == U.logprob_row(xs[r], None, 4, allowed=allowed[r])[2].tolist()
    if dtype == torch.float32:
        u = np.array([0.1, 0.5, 0.9])
        tok = F.sample_batch(x, p, u, edits=ed)["tok"]
        for r in range(3):
            assert int(tok[r]) == U.sample_row(xs[r], p[r], [], u[r], allowed=allowed[r])["tok"]


@pytest.mark.parametrize("V", [1000, 65536, 200000])
@pytest.mark.parametrize("n", [1, 20, 64])
def test_largest_of_ordered_and_tied_rows(V, n):
    """Rows whose every chunk holds larger logits than the one before (each raises the bound), the reverse, few values,
    and all the largest in one place."""
    up = np.linspace(-8, 8, V).astype(np.float32)
    x = np.stack([up, up[::-1], np.round(up / 4), np.where(np.arange(V) % 97 == 5, 3.0, 0.0), np.zeros(V),
                  np.where((np.arange(V) >= V // 2) & (np.arange(V) < V // 2 + 200), up + 50, up)]).astype(np.float32)
    tok = np.array([0, V - 1, V // 2, 5, 7, V // 2], np.int32)
    for dtype in (torch.float32, torch.bfloat16):
        t = cuda(x).to(dtype)
        xs = t.float().cpu().numpy()
        out = F.logprobs(t, tok, min(n, V))
        for r in range(len(x)):
            lp, rank, ids, top = U.logprob_row(xs[r], int(tok[r]), min(n, V))
            assert out["ids"][r].tolist() == ids.tolist(), r
            assert int(out["rank"][r]) == rank
            assert np.all(np.abs(out["top"][r].cpu().numpy() - top) <= lp_tolerance(top))
            assert abs(float(out["lp"][r]) - lp) <= lp_tolerance(lp)


@pytest.mark.parametrize("B", [1, 7, 63, 1500])
def test_logprobs_of_many_rows(B):
    """One part per row and many; every row's ticket is left as it was found (the call is made twice)."""
    V = 20003
    g = torch.Generator("cuda").manual_seed(B)
    x = (torch.randn((B, V), device="cuda", generator=g) * 3).to(torch.bfloat16)
    tok = torch.randint(0, V, (B,), device="cuda", generator=g, dtype=torch.int32)
    ctx = F.Context()
    a = F.logprobs(x, tok, 8, ctx=ctx)
    b = F.logprobs(x, tok, 8, ctx=ctx)
    want = torch.log_softmax(x.double(), 1)
    lp = want.gather(1, tok.long()[:, None])[:, 0]
    assert torch.all((a["lp"].double() - lp).abs() <= 200 * 2.0 ** -24 + lp.abs() * 2.0 ** -24)
    v, i = torch.sort(x.float(), dim=1, descending=True, stable=True)
    assert torch.equal(a["ids"].long(), i[:, :8])
    assert torch.equal(a["rank"].long(), 1 + (x > x.gather(1, tok.long()[:, None])).sum(1))
    for k in a:
        assert torch.equal(a[k], b[k])


def test_extreme_temperatures_and_values():
    x = torch.randn((4, 3000), device="cuda") * 10
    x[1] *= 1e36
    x[2] = -3.0e38
    x[2, 7] = -3.4e38
    x[3, 5] = 3.4e38
    for T in (1e-6, 1.0, 1e6):
        p = W.make_params(4, temperature=T, repetition_penalty=1.0)
        out = F.logprobs(x, [5, 5, 7, 5], 3, params=p)
        for r in range(4):
            lp, rank, ids, top = U.logprob_row(x[r].cpu().numpy(), [5, 5, 7, 5][r], 3, T=float(np.float32(T)))
            assert out["ids"][r].tolist() == ids.tolist() and int(out["rank"][r]) == rank
            got = float(out["lp"][r])
            assert got == lp or abs(got - lp) <= lp_tolerance(lp) or (lp < -3.4e38 and got == float("-inf"))


def test_two_contexts_on_two_streams():
    """Edited calls of two contexts overlapping on two streams."""
    b = Batch(61, 12, 60000, ("most", "few"), nb=100, H=100, **SETS["small_k"])
    c = Batch(62, 9, 50000, ("most", "few"), nb=100, H=100, **SETS["mid_k"])
    work = []
    for w in (b, c):
        ctx, st = F.Context(), torch.cuda.Stream()
        args = [cuda(w.x), cuda(w.p.view(np.uint8)), cuda(w.u), cuda(w.hist), cuda(w.off)]
        work.append((ctx, st, args, w, F.sample_batch(args[0], w.p, args[2], args[3], args[4], edits=w.ed, ctx=ctx)["tok"].clone(),
                     F.logprobs(args[0], None, 7, edits=w.ed, ctx=ctx)["ids"].clone()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for ctx, st, a, w, tok, ids in work:
            with torch.cuda.stream(st):
                outs.append((F.sample_batch(a[0], w.p, a[2], a[3], a[4], edits=w.ed, ctx=ctx)["tok"], tok))
                outs.append((F.logprobs(a[0], None, 7, edits=w.ed, ctx=ctx)["ids"], ids))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)


def test_give_up_of_the_waiting_segments_is_exact():
    """A context whose waits give up at once: the rows' last segments select them alone, under the masks and biases."""
    for name in ("mid_k", "every"):
        b = Batch(71, 4, 40000, ("most", "few"), nb=12, **SETS[name])
        ctx = F.Context()
        ctx.set_wait_limit(0xFFFFFFFF)
        out = F.sample_batch(cuda(b.x), b.p, b.u, b.hist, b.off, edits=b.ed, ctx=ctx)
        assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 1
        assert F.device_error(ctx) & 2


def test_a_captured_window_and_step_replay():
    """A verification window and a decode step under edits in one graph, replayed: the draws advance, the workspaces are left
    as they were."""
    S, M, V = 3, 4, 30000
    rng = np.random.default_rng(9)
    x = cuda(W.mixture_logits(rng, S * M, V))
    p = cuda(W.make_params(S, **SETS["small_k"]).view(np.uint8))
    rows = cuda(rng.integers(0, V, S * M).astype(np.int32))
    row_off = cuda(np.arange(0, S * M + 1, M, dtype=np.int64))
    hist, off = cuda(rng.integers(0, V, 30).astype(np.int32)), cuda(np.array([0, 10, 10, 30], np.int64))
    u = cuda(rng.random(S * M))
    bias = U.csr(U.bias_lists(rng, S, V, 20))
    edw = F.Edits(mask=cuda(F.Edits.pack(U.masks(rng, "most", S * M, V))), bias=bias)
    eds = F.Edits(mask=cuda(F.Edits.pack(U.masks(rng, "most", S, V))), bias=bias)
    ctx = F.Context()
    outs = []
    for captured in (False, True):
        drng = F.DeviceRng([5, 6, 7])

        def step():
            tok, acc = F.verify(x, rows, row_off, p, u, hist, off, edits=edw, ctx=ctx)
            t, k, h, o = F.decode_step(x[:S], p, drng, hist, off, edits=eds, ctx=ctx)
            return tok, acc, t, k, h, o

        seq = []
        if not captured:
            for _ in range(4):
                seq.append([t.clone() for t in step()])
        else:
            warm = F.DeviceRng([1, 1, 1])
            drng, keep = warm, drng
            step()
            drng = keep
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = step()
            for _ in range(4):
                g.replay()
                torch.cuda.synchronize()
                seq.append([t.clone() for t in out])
                torch.randn(1000, device="cuda").sum()              # eager work in between
        outs.append(seq)
    for a, b in zip(*outs):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_one_context_through_many_layouts():
    """Calls of one context whose rows are cut into other numbers of parts, larger and smaller, with and without lists."""
    ctx = F.Context()
    g = torch.Generator("cuda").manual_seed(3)
    for B, V, n in ((1, 70000, 5), (3000, 40, 3), (40, 30000, 0), (2, 262144, 64), (20000, 64, 1), (7, 5000, 20), (1, 70000, 5)):
        x = torch.randn((B, V), device="cuda", generator=g) * 4
        tok = torch.randint(0, V, (B,), device="cuda", generator=g, dtype=torch.int32)
        out = F.logprobs(x, tok, n, ctx=ctx)
        lp = torch.log_softmax(x.double(), 1).gather(1, tok.long()[:, None])[:, 0]
        assert torch.all((out["lp"].double() - lp).abs() <= 200 * 2.0 ** -24 + lp.abs() * 2.0 ** -24), (B, V, n)
        if n:
            assert torch.equal(out["ids"].long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :n]), (B, V, n)


def test_edits_used_on_a_side_stream_may_go():
    """Edits dropped right after a call on another stream: their memory is not handed out while the call runs."""
    B, V = 4, 200000
    b = Batch(81, B, V, "most", nb=0, **SETS["small_k"])
    x, st = cuda(b.x), torch.cuda.Stream()
    want = F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=b.ed)["tok"]
    words, of = U_pack(b.allowed), b.of
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        ed = F.Edits(mask=cuda(words), mask_of=cuda(of))
        big = [torch.empty_like(x).copy_(x) for _ in range(4)]
        got.append(F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=ed, stream=st)["tok"])
        del ed, big
        torch.zeros((b.allowed.shape[0], words.shape[1]), dtype=torch.int32, device="cuda")      # takes freed memory
    torch.cuda.synchronize()
    for t in got:
        assert torch.equal(t, want)


@pytest.mark.parametrize("name", ["greedy", "small_k", "mid_k", "every", "large_k"])
def test_a_step_without_masks_biases_and_histories(name):
    """A table of no masks, empty bias lists and empty histories do what no edits do, in every call."""
    B, V = 3, 9001
    b = Batch(91, B, V, "none", nb=0, **SETS[name])
    x, off = cuda(b.x), np.zeros(B + 1, np.int64)
    words = torch.zeros((0, (V + 31) // 32), dtype=torch.int32, device="cuda")
    ed = F.Edits(mask=words, mask_of=np.full(B, -1), bias=[{}] * B)
    want = F.sample_batch(x, b.p, b.u)["tok"]
    assert torch.equal(F.sample_batch(x, b.p, b.u, edits=ed)["tok"], want)
    assert torch.equal(F.sample_batch(x, b.p, b.u, np.zeros(0, np.int32), off, edits=ed)["tok"], want)
    assert torch.equal(F.argmax_batch(x, edits=ed), F.argmax_batch(x))
    assert torch.equal(F.edit_batch(x, edits=ed), x)
    for got, plain in zip(F.logprobs(x, want, 4, edits=ed).values(), F.logprobs(x, want, 4).values()):
        assert torch.equal(got, plain)


@pytest.mark.parametrize("B", [520, 700, 1100])
def test_logprobs_of_rows_in_parts_past_the_first_round(B):
    """More rows than workgroups run at once, or more than half as many: parts that fill a last round (3, 1 and 2 of 15
    chunks)."""
    V = 60011
    g = torch.Generator("cuda").manual_seed(B)
    x = torch.randn((B, V + 1), device="cuda", generator=g)[:, :V] * 4
    tok = torch.randint(0, V, (B,), device="cuda", generator=g, dtype=torch.int32)
    ctx = F.Context()
    a = F.logprobs(x, tok, 3, ctx=ctx)
    b = F.logprobs(x, tok, 3, ctx=ctx)
    for r in range(0, B, 37):                          # (the reference a few rows at a time)
        s = slice(r, min(r + 37, B))
        want = torch.log_softmax(x[s].double(), 1)
        lp = want.gather(1, tok[s].long()[:, None])[:, 0]
        assert torch.all((a["lp"][s].double() - lp).abs() <= 200 * 2.0 ** -24 + lp.abs() * 2.0 ** -24)
        assert torch.equal(a["rank"][s].long(), 1 + (x[s] > x[s].gather(1, tok[s].long()[:, None])).sum(1))
        v, i = torch.sort(x[s], dim=1, descending=True, stable=True)
        assert torch.equal(a["ids"][s].long(), i[:, :3])
    for k in a:
        assert torch.equal(a[k], b[k])


@pytest.mark.parametrize("B,V", [(60, 70001), (20, 140003)])
def test_large_k_on_more_segments_than_run_at_once(B, V):
    """k up to 2048 on rows too short for the largest segments: smaller ones, more of them than run at once; the same tokens
    as from rows written out first (device parameters)."""
    b = Batch(B, B, V, ("most", "few", "block"), nb=40, **dict(SETS["mid_k"], frequency_penalty=0.2))
    b.p["top_k"] = np.exp(b.rng.uniform(0.0, np.log(2048.0), B)).astype(np.int32).clip(1, 2048)
    b.p["top_k"][:2] = 2048
    x = cuda(b.x)
    out = F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=b.ed)
    assert check_rows(b, out["tok"].cpu().numpy(), out["keep"].cpu().numpy()) <= 3
    other = F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=b.ed, route="device")
    assert torch.equal(out["tok"], other["tok"]) and torch.equal(out["keep"], other["keep"])


@pytest.mark.parametrize("B,V", [(2, 65536), (7, 131072), (24, 65540), (40, 131072), (90, 40000), (130, 16384)])
@pytest.mark.parametrize("name", ["greedy", "small_k"])
def test_batches_on_every_segment_size(name, B, V):
    """Segments of 4096, 8192 and 16384 logits, full ones and a last one of four; a context warmed up with greedy rows
    records sampled ones, and the other way round."""
    other = "small_k" if name == "greedy" else "greedy"
    b = Batch(B, B, V, ("most", "few", "block"), nb=9, **SETS[name])
    w = Batch(B, B, V, ("most", "few", "block"), nb=9, **SETS[other])
    x, ctx = cuda(b.x), F.Context()
    F.sample_batch(x, w.p, b.u, edits=b.ed, ctx=ctx)
    p, u = b.p, cuda(b.u)
    hist, off = cuda(b.hist), cuda(b.off)
    torch.cuda.synchronize()
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    dev = torch.from_numpy(p.view(np.uint8).copy()).cuda()
    tok = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    keep = torch.zeros(B, dtype=torch.int32, device="cuda")
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    with torch.cuda.graph(g, stream=st):
        check(lib().fs_sample_edited(ctx.h, ptr(x), x.stride(0), B, V, ptr(hist), ptr(off),
                                     ptr(dev), p.ctypes.data_as(ctypes.c_void_p), b.ed._ref(B, B, V, x.device), ptr(u),
                                     ptr(tok), 0, None, None, ptr(keep), ctypes.c_void_p(st.cuda_stream)), "edited")
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert check_rows(b, tok.cpu().numpy(), keep.cpu().numpy()) <= 3
        again = F.sample_batch(x, b.p, b.u, b.hist, b.off, edits=b.ed)
        assert torch.equal(again["tok"], tok) and torch.equal(again["keep"], keep)
        tok.fill_(-7)
