"""CPU: what the beam search's Python wrappers work out on the host, and calls they refuse."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import _lib  # noqa: E402

P = ctypes.c_void_p


@pytest.fixture()
def ctx():
    h = P()
    assert _lib.lib().fs_create(ctypes.byref(h)) == _lib.FS_OK
    yield h
    _lib.lib().fs_destroy(h)


@pytest.mark.parametrize("out", ["parent", "tok", "out", "done", "dp", "ds"])
def test_select_refuses_outputs_over_its_inputs(ctx, out):
    """Two streams of two rows, four beams: an output that begins or ends inside the scores, offsets or records. (Calls it
    takes go on to the device, so those that only touch are the GPU tests'.)"""
    MB = 1 << 20
    good = dict(ctx=ctx, logits=P(MB), type=0, ld=8, S=2, R=4, V=8, off=P(2 * MB), score=P(3 * MB), params=P(4 * MB), edits=None,
                eos=-1, n=4, flags=0, parent=P(5 * MB), tok=P(6 * MB), out=P(7 * MB), done=P(8 * MB), dp=P(9 * MB), ds=P(10 * MB),
                stream=None)
    size = 8 if out == "done" else 32
    for name, n in (("off", 24), ("score", 16), ("params", 2 * _lib.PARAMS_DTYPE.itemsize)):
        at = good[name].value
        for to in (at, at + n - 4, at - size + 4):
            assert _lib.lib().fs_beam_select(*dict(good, **{out: P(to)}).values()) == _lib.FS_E_INVALID, (name, to - at)


@pytest.mark.parametrize("seed", range(30))
def test_room_of_new_histories(seed):
    """Never less than what the parents that take most of it need, and no more."""
    rng = np.random.default_rng(seed)
    S, n = int(rng.integers(0, 7)), int(rng.integers(1, 5))
    counts = [n] * S if seed % 3 == 0 else rng.integers(0, 6, S)
    row_off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    lens = rng.integers(0, 9, row_off[-1])
    off = 4 + np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    want = sum(n * int(max(lens[a:b], default=0)) for a, b in zip(row_off, row_off[1:]))
    assert F.sampler._fork_ids(off, None if seed % 3 == 0 else row_off, S, n) == want


def fields(z):
    return {n: getattr(z, n) for n, _ in z._fields_ if n not in ("d_src", "d_dst")}


def test_states_refuse_buffers_that_overlap_themselves(ctx):
    t = torch.zeros((6, 3, 10, 4))
    one = torch.zeros((1, 3, 10, 4))
    windows = torch.zeros(200).as_strided((6, 3, 10, 4), (4, 40, 4, 1))    # row r's position p is row r + 1's p - 1
    for bad, pos in ((one.expand(6, 3, 10, 4), 2), (one.expand(6, 3, 10, 4), None), (t[:, :1].expand(6, 3, 10, 4), 2),
                     (t[:, :, :1].expand(6, 3, 10, 4), 2), (windows, 2), (t[:, :1].expand(6, 3, 10, 4), 1)):
        with pytest.raises(F.SamplerError, match="overlap"):
            F.States([bad], pos_dim=pos)
        with pytest.raises(F.SamplerError, match="overlap"):
            F.States([t], [bad], pos_dim=pos)
    # (read alone they are fine: one prompt's cache as every stream's; and so are sizes of one with any stride)
    F.States([one.expand(6, 3, 10, 4)], [t], pos_dim=2)
    F.States([one.expand(1, 3, 10, 4)], pos_dim=2)
    F.States([torch.zeros((6, 0, 10, 4)).expand(6, 0, 10, 4)], pos_dim=2)
    F.States([torch.zeros((1, 3, 10, 0)).expand(6, 3, 10, 0)], pos_dim=2)
    F.States([torch.zeros((13, 6, 3, 8)).transpose(0, 1)], pos_dim=1)      # rows between positions and heads
    F.States([torch.zeros((5, 6)).t()])                        # rows innermost
    good = dict(d_src=1 << 20, d_dst=2 << 20, src_row=64, src_block=32, src_pos=8, dst_row=64, dst_block=32, dst_pos=8, pos_bytes=8,
                blocks=2, positions=4)
    for bad in (dict(dst_row=0), dict(dst_row=7), dict(dst_block=0), dict(dst_block=7), dict(dst_pos=0), dict(dst_pos=7)):
        for src in (2 << 20, 1 << 20):                         # in place, and not
            z = dict(good, **bad)
            z.update(d_src=src, **({f"src_{k}": z[f"dst_{k}"] for k in ("row", "block", "pos")} if src == 2 << 20 else {}))
            rec = (_lib.FsState * 1)(_lib.FsState(**z))
            assert _lib.lib().fs_reorder_states(ctx, 1, rec, 2, 4, 4, P(3 << 20), None, None, None) == _lib.FS_E_INVALID, (bad, src)


def test_states_past_the_records_counts():
    """Blocks and positions that 32 bits do not hold (they were cut: no block, or a state without positions)."""
    meta = lambda *shape: torch.empty(shape, dtype=torch.uint8, device="meta")
    for t, pos in ((meta(2, 1 << 16, 1 << 16, 3)[..., :2], None), (meta(2, (1 << 32) + 7, 2), 1), (meta(2, 1 << 32, 2), 1),
                   (meta(2, 1 << 20, 1 << 20, 8), 2)):
        with pytest.raises(F.SamplerError, match="2\\^31"):
            F.States([t], pos_dim=pos)
    z = fields(F.States([meta(2, 3, (1 << 29) + 1, 4)], pos_dim=2).c[0])
    assert (z["blocks"], z["positions"], z["pos_bytes"]) == (3, (1 << 29) + 1, 4)
    z = fields(F.States([meta(2, (1 << 31) + 8)]).c[0])        # (one run of bytes: the call refuses it)
    assert (z["blocks"], z["pos_bytes"]) == (1, (1 << 31) + 8)
