"""GPU: edited calls recorded into graphs on contexts that were warmed up with other calls - those that are refused leave
nothing behind, the others replay like the eager call."""
import ctypes
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from ferro_amd._lib import check, lib  # noqa: E402
from oracle import oracle as O  # noqa: E402
from tests import edit_util as U  # noqa: E402
from tests.test_gpu_edits import U_pack, cuda  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


# a softcap beside biases: the rows are edited into the workspace and sampled there
COMPOSED = dict(temperature=0.8, top_k=40, repetition_penalty=1.0, softcap=20.0)


class Step:
    """B streams' decode steps of V logits, with everything on the device."""

    def __init__(self, seed, B, V, **params):
        rng = np.random.default_rng(seed)
        self.x = cuda(W.mixture_logits(rng, B, V))
        self.p = W.make_params(B, **params)
        self.dev = cuda(self.p.view(np.uint8))
        self.ed = F.Edits(mask=cuda(U_pack(U.masks(rng, "most", B, V))), bias=U.csr(U.bias_lists(rng, B, V, 6)))
        self.seeds = np.arange(1, B + 1, dtype=np.uint64) * 31

    def run(self, ctx, drng, host):
        p = self.p if host else self.dev
        tok, keep, hist, off = F.decode_step(self.x, p, drng, edits=self.ed, ctx=ctx)
        return tok, keep, hist, off


def test_a_refused_step_leaves_the_graph_and_the_draws():
    """The edited rows of the recorded step fit what the context holds, the fused kernel's workspace does not: the call is
    refused before anything is launched, so a replay neither draws nor edits."""
    ctx = F.Context()
    warm = Step(1, 64, 28672, **COMPOSED)          # 448 slots of the fused kernel, 64 * 28672 edited logits
    warm.run(ctx, F.DeviceRng(warm.seeds), host=True)
    s = Step(2, 7, 262144, **COMPOSED)             # 512 slots, as many logits
    drng = F.DeviceRng(s.seeds)
    y = torch.zeros(2, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(F.SamplerError, match="allocation"):
            s.run(ctx, drng, host=False)
        y.add_(1.0)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
    assert y.tolist() == [3.0, 3.0]
    peeked = drng.draw(s.dev, peek=True).tolist()
    assert peeked == [O.canonical(O.MT64(int(seed)).next()) for seed in s.seeds]
    # the refused step, made eagerly, takes those draws
    got = s.run(ctx, drng, host=False)
    want = s.run(F.Context(), F.DeviceRng(s.seeds), host=False)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("first", [True, False])
def test_a_shape_warmed_up_with_one_kind_of_parameters_records_the_other(first):
    """Host parameters (the edited rows go to the small-k kernel) and device parameters (the fused one): a context that has
    made either call records the other, with the same tokens and draws as eager steps."""
    s = Step(3, 5, 30011, **COMPOSED)
    ctx = F.Context()
    s.run(ctx, F.DeviceRng(s.seeds), host=first)
    torch.cuda.synchronize()
    drng = F.DeviceRng(s.seeds)
    hp = s.p.copy()
    if not first:                                  # (the wrapper would copy host parameters to the device while recording)
        B, V = s.x.shape
        tok = torch.zeros(B, dtype=torch.int32, device="cuda")
        keep, hist = torch.zeros_like(tok), torch.zeros(B, dtype=torch.int32, device="cuda")
        off = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
        x = torch.zeros((B, V + (-V) % 4), device="cuda")
        x[:, :V] = s.x
        ptr = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
        torch.cuda.synchronize()

        def step():
            check(lib().fs_decode_step_edited(ctx.h, drng.h, ptr(x), x.stride(0), B, V, None, None, ptr(s.dev),
                                              hp.ctypes.data_as(ctypes.c_void_p), s.ed._ref(B, B, V, x.device), ptr(tok),
                                              ptr(keep), ptr(hist), ptr(off), B,
                                              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "step")
            return tok, keep, hist, off
    else:
        step = lambda: s.run(ctx, drng, host=False)        # noqa: E731
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    eager, other = F.DeviceRng(s.seeds), F.Context()
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = s.run(other, eager, host=not first)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_threads_on_one_context_and_stream():
    """Host calls that overlap on one context, their work in the order of one stream: composed calls of two threads, each
    with rows, masks and biases of its own, do not take each other's edited rows."""
    ctx = F.Context()
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())              # noqa: E731

    def worker(seed):
        """Calls of growing sizes (the workspaces are replaced under the other thread) and what they have to give."""
        work = []
        for i, (B, V) in enumerate(((3, 4000), (9, 8000), (20, 12000), (40, 16000))):
            s = Step(seed + i, B, V, **dict(COMPOSED, top_k=40 if i % 2 else 0))
            u = cuda(np.random.default_rng(seed + i).random(B))
            want = F.sample_batch(s.x, s.p, u, edits=s.ed, ctx=F.Context())["tok"]
            work.append((s, u, want))

        def run(out):
            for s, u, want in work:
                B, V = s.x.shape
                for _ in range(10):
                    tok = torch.full((B,), -7, dtype=torch.int32, device="cuda")
                    rc = lib().fs_sample_edited(ctx.h, ptr(s.x), V, B, V, None, None, ptr(s.dev), s.p.ctypes.data_as(ctypes.c_void_p),
                                                s.ed._ref(B, B, V, s.x.device), ptr(u), ptr(tok), 0, None, None, None, st)
                    out.append((rc, tok, want))
        return run

    runs, outs = [worker(100), worker(200)], ([], [])
    torch.cuda.synchronize()
    threads = [threading.Thread(target=r, args=(o,)) for r, o in zip(runs, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for out in outs:
        assert len(out) == 40
        for rc, tok, want in out:
            assert rc == 0 and torch.equal(tok, want)
