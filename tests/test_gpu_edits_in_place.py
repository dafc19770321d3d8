"""GPU: what a program writes into the tensors it gave an Edits is what the next call samples under, whatever their types
and strides."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from tests import edit_util as U  # noqa: E402
from tests.test_gpu_edits import cuda  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


B, V = 4, 1000
WORDS = (V + 31) // 32


def mask_buffers(kind):
    """(a buffer, its view of B + 1 masks)"""
    if kind == "packed":
        t = torch.zeros((B + 1, WORDS), dtype=torch.int32, device="cuda")
        return t, t
    if kind == "wide":
        t = torch.zeros((B + 1, WORDS + 9), dtype=torch.int32, device="cuda")
        return t, t[:, :WORDS]
    if kind == "columns":
        t = torch.zeros((WORDS, B + 1), dtype=torch.int32, device="cuda")
        return t, t.t()
    if kind == "every_other":
        t = torch.zeros((B + 1, 2 * WORDS), dtype=torch.int32, device="cuda")
        return t, t[:, ::2]
    t = torch.zeros((B + 1, WORDS), dtype=torch.uint32, device="cuda")
    return t.view(torch.int32), t


@pytest.mark.parametrize("types", [(torch.int32, torch.int32, torch.float32, torch.int64),
                                   (torch.int64, torch.int64, torch.float64, torch.int32)])
@pytest.mark.parametrize("kind", ["packed", "wide", "columns", "every_other", "uint32"])
@pytest.mark.parametrize("other_stream", [False, True])
def test_what_is_written_is_what_the_next_call_reads(kind, types, other_stream):
    t_of, t_ids, t_val, t_off = types
    rng = np.random.default_rng(7)
    buf, view = mask_buffers(kind)
    words = buf if kind == "uint32" else view
    of = torch.zeros(B, dtype=t_of, device="cuda")
    ids = torch.zeros(2 * B, dtype=t_ids, device="cuda")
    val = torch.zeros(2 * B, dtype=t_val, device="cuda")
    off = torch.zeros(B + 1, dtype=t_off, device="cuda")
    ed = F.Edits(mask=view, mask_of=of, bias=(ids, val, off))
    x = W.mixture_logits(rng, B, V)
    d = cuda(x)
    p = W.make_params(B, temperature=0.0, repetition_penalty=1.0)
    rows = torch.arange(B + 1, dtype=torch.int64, device="cuda")
    stream = torch.cuda.Stream() if other_stream else None
    for step in range(3):
        allowed = rng.random((B + 1, V)) < 0.3
        m = rng.integers(-1, B + 1, B)
        o = np.array([0, 2, 2, 5, 8]) if step % 2 else np.array([0, 1, 4, 6, 8])
        i = np.concatenate([np.sort(rng.choice(V, n, replace=False)) for n in np.diff(o)])
        b = rng.uniform(-8, 8, 8).astype(np.float32)
        words.copy_(cuda(F.Edits.pack(allowed)))
        of.copy_(cuda(m))
        ids.copy_(cuda(i))
        val.copy_(cuda(b))
        off.copy_(cuda(o))
        bias = [[(int(t), float(v)) for t, v in zip(i[o[r]:o[r + 1]], b[o[r]:o[r + 1]])] for r in range(B)]
        ok = [None if m[r] < 0 else allowed[m[r]] for r in range(B)]
        want = [U.sample_row(x[r], p[r], [], 0.0, bias[r], ok[r])["tok"] for r in range(B)]
        got = F.sample_batch(d, p, np.zeros(B), edits=ed, stream=stream)["tok"]
        win, _ = F.verify(d, np.zeros(B, np.int32), rows, p, edits=ed, stream=stream)
        lp = F.logprobs(d, np.array(want, np.int32), 1, edits=ed, stream=stream)
        edited = F.edit_batch(d, edits=ed, stream=stream)
        drng = F.DeviceRng(np.arange(1, B + 1))
        torch.cuda.synchronize()
        tok, _, _, _ = F.decode_step(d, p, drng, edits=ed, stream=stream)
        torch.cuda.synchronize()
        assert got.tolist() == want and win.tolist() == want and tok.tolist() == want, step
        assert lp["ids"][:, 0].tolist() == want and lp["rank"].tolist() == [1] * B
        for r in range(B):
            np.testing.assert_array_equal(edited[r].cpu().numpy(), U.edit_row(x[r], None, [], bias[r], ok[r]))


def test_a_captured_call_reads_them_too():
    rng = np.random.default_rng(8)
    of = torch.zeros(B, dtype=torch.int64, device="cuda")
    table = torch.zeros((WORDS, B), dtype=torch.int32, device="cuda")
    ed = F.Edits(mask=table.t(), mask_of=of)
    x, u = cuda(W.mixture_logits(rng, B, V)), torch.zeros(B, dtype=torch.float64, device="cuda")
    p = W.make_params(B, temperature=0.0, repetition_penalty=1.0)
    dev, ctx = cuda(p.view(np.uint8)), F.Context()
    F.sample_batch(x, dev, u, edits=ed, ctx=ctx)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok = F.sample_batch(x, dev, u, edits=ed, ctx=ctx)["tok"]
    for _ in range(3):
        allowed = rng.random((B, V)) < 0.2
        m = rng.permutation(B)
        table.t().copy_(cuda(F.Edits.pack(allowed)))
        of.copy_(cuda(m))
        g.replay()
        torch.cuda.synchronize()
        xs = x.cpu().numpy()
        assert tok.tolist() == [U.sample_row(xs[r], p[r], [], 0.0, allowed=allowed[m[r]])["tok"] for r in range(B)]
        assert torch.equal(F.sample_batch(x, p, u, edits=ed, ctx=ctx)["tok"], tok)
