"""GPU: calls of the beam search that a long run, a captured one or an unusual program makes (tests/beam_util.py)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from tests import beam_util as BU  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


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
