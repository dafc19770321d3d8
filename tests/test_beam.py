"""CPU: refusals of the beam search's entry points before they touch the device, the records of state buffers, and the plain
implementations themselves."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import _lib  # noqa: E402
from tests import beam_util as BU  # noqa: E402

P = ctypes.c_void_p


@pytest.fixture()
def ctx():
    h = P()
    assert _lib.lib().fs_create(ctypes.byref(h)) == _lib.FS_OK
    yield h
    _lib.lib().fs_destroy(h)


def refused(fn, good, **changes):
    """The call with one argument changed is FS_E_INVALID, for each change."""
    for name, values in changes.items():
        for v in values if isinstance(values, list) else [values]:
            args = dict(good)
            args[name] = v
            assert fn(*args.values()) == _lib.FS_E_INVALID, (name, v)


def test_select_refusals(ctx):
    f = P(1 << 20)                                             # never read: the checks come first
    good = dict(ctx=ctx, logits=f, type=0, ld=8, S=2, R=4, V=8, off=None, score=f, params=None, edits=None, eos=-1, n=4, flags=0,
                parent=f, tok=f, out=f, done=f, dp=f, ds=f, stream=None)
    ed = _lib.FsEdits(d_mask=1 << 20, mask_ld=0, n_masks=4)
    few = _lib.FsEdits(d_mask=1 << 20, mask_ld=1, n_masks=3)
    refused(_lib.lib().fs_beam_select, good, ctx=None, logits=[None, P(8)], type=[3, -1], ld=[7, 10, 4], S=[-1, 3], R=-1, V=[0, -1],
            n=[0, -1, 65], flags=[2, -1], parent=None, tok=None, out=None, edits=[ctypes.byref(ed), ctypes.byref(few)])
    none = dict(good, S=0, R=0)
    assert _lib.lib().fs_beam_select(*none.values()) == _lib.FS_OK


def test_fork_refusals(ctx):
    f = [P((i + 1) << 20) for i in range(8)]
    good = dict(ctx=ctx, S=2, hist=f[0], off=f[1], row_off=None, n=4, parent=f[2], tok=f[3], out=f[4], cap=9, out_off=f[5],
                stream=None)
    refused(_lib.lib().fs_hist_fork, good, ctx=None, S=[-1, 1 << 30], off=None, n=[0, -4], parent=None, out=[None, f[0], f[2], f[3]],
            cap=-1, out_off=[None, f[1]])


def state(**kw):
    z = dict(d_src=1 << 20, d_dst=1 << 20, src_row=64, src_block=32, src_pos=8, dst_row=64, dst_block=32, dst_pos=8, pos_bytes=8,
             blocks=2, positions=4)
    z.update(kw)
    return (_lib.FsState * 1)(_lib.FsState(**z))


def test_state_refusals(ctx):
    f = P(1 << 20)
    good = dict(ctx=ctx, k=1, z=state(), S=2, n_src=4, n=4, parent=f, start=None, length=None, stream=None)
    bad = [state(**{k: -1}) for k in ("src_row", "src_block", "src_pos", "dst_row", "dst_block", "dst_pos", "pos_bytes", "blocks",
                                      "positions")]
    bad += [state(d_src=0), state(d_dst=0), state(d_dst=(1 << 20) + 8), state(dst_row=128), state(src_row=1 << 50, dst_row=1 << 50),
            state(pos_bytes=1 << 32), state(blocks=1 << 20, positions=1 << 20), state(blocks=1 << 15, positions=1 << 15, pos_bytes=64)]
    refused(_lib.lib().fs_reorder_states, good, ctx=None, k=-1, z=[None] + bad, S=-1, n_src=[0, 65, 3], n=[0, 65, 5], parent=None)
    twice = (_lib.FsState * 2)(state()[0], state(src_row=128, dst_row=128)[0])
    chain = (_lib.FsState * 2)(state(d_dst=2 << 20)[0], state(d_src=2 << 20, d_dst=3 << 20)[0])
    refused(_lib.lib().fs_reorder_states, dict(good, k=2), z=[twice, chain])
    apart = dict(good, z=state(d_dst=(1 << 20) + 512), S=0)
    assert _lib.lib().fs_reorder_states(*apart.values()) == _lib.FS_OK
    assert _lib.lib().fs_reorder_states(*dict(good, k=0, z=None).values()) == _lib.FS_OK


def fields(z):
    return {n: getattr(z, n) for n, _ in z._fields_ if n not in ("d_src", "d_dst")}


def test_state_records():
    t = torch.zeros((6, 3, 10, 4), dtype=torch.bfloat16)
    assert fields(F.States([t], pos_dim=2).c[0]) == dict(src_row=240, src_block=80, src_pos=8, dst_row=240, dst_block=80, dst_pos=8,
                                                         pos_bytes=8, blocks=3, positions=10)
    z = fields(F.States([t], pos_dim=1).c[0])
    assert (z["pos_bytes"], z["blocks"], z["positions"], z["src_pos"]) == (80, 1, 3, 80)
    z = fields(F.States([t]).c[0])
    assert (z["pos_bytes"], z["blocks"], z["positions"]) == (240, 1, 0)
    z = fields(F.States([t[:, :, ::2]]).c[0])                  # blocks of one row: 3 and 5 fold
    assert (z["pos_bytes"], z["blocks"], z["src_block"]) == (8, 15, 16)
    z = fields(F.States([t[:, 1]], pos_dim=1).c[0])
    assert (z["src_row"], z["pos_bytes"], z["blocks"], z["positions"]) == (240, 8, 1, 10)
    z = fields(F.States([t[:, :, :0]], pos_dim=2).c[0])
    assert z["blocks"] == 0
    s = F.States([t, t], [torch.zeros((12, 3, 16, 4), dtype=torch.bfloat16)] * 2, pos_dim=-2)
    assert len(s) == 2 and (s.src_rows, s.dst_rows) == (6, 12)
    z = fields(s.c[1])
    assert (z["positions"], z["src_block"], z["dst_block"], z["dst_row"]) == (10, 80, 128, 384)
    for bad in (dict(tensors=[t], pos_dim=4), dict(tensors=[t], pos_dim=0), dict(tensors=[t, t], pos_dim=[2]),
                dict(tensors=[t], dst=[]), dict(tensors=[t], dst=[t.float()]), dict(tensors=[t, t[:3]]),
                dict(tensors=[t[:, :, :, ::2]], pos_dim=2), dict(tensors=[t[:, ::2, ::3]])):
        with pytest.raises(F.SamplerError):
            F.States(**bad)
    with pytest.raises(F.SamplerError):
        F.reorder_states([t], np.zeros((2, 3), np.int32))      # not on a GPU


def brute(step, s):
    """A stream's beams and ended hypotheses straight from the definition."""
    rows = range(int(step.off[s]), int(step.off[s + 1]))
    all_ = [(-step.c[r][t], t != step.eos, i, -step.x[r][t], t) for i, r in enumerate(rows) for t in range(len(step.c[r]))
            if step.c[r][t] > -np.inf]
    all_.sort()
    beams = [e for e in all_ if e[1]][:step.n]
    done = [e for j, e in enumerate(all_) if not e[1] and j < step.n]
    return beams, done


@pytest.mark.parametrize("seed", range(4))
def test_the_check_takes_the_definition_and_no_other(seed):
    rng = np.random.default_rng(seed)
    counts, n, V = [3, 0, 4], 5, 40
    off = np.concatenate([[0], np.cumsum(counts)])
    x = rng.integers(-3, 9, (7, V)).astype(np.float32) if seed % 2 else rng.normal(0, 2, (7, V)).astype(np.float32)
    eos = int(x[0].argmax())
    step = BU.Step(x, -rng.exponential(2.0, 7).astype(np.float32), off, n, eos)
    out = dict(parent=np.full((3, n), -1), tok=np.full((3, n), -1), score=np.full((3, n), -np.inf), done=np.zeros(3, int),
               done_parent=np.full((3, n), -1), done_score=np.full((3, n), -np.inf))
    for s in range(3):
        beams, done = brute(step, s)
        for j, (c, _, i, _, t) in enumerate(beams):
            out["parent"][s, j], out["tok"][s, j], out["score"][s, j] = i, t, np.float32(-c)
        out["done"][s] = len(done)
        for j, (c, _, i, _, _) in enumerate(done):
            out["done_parent"][s, j], out["done_score"][s, j] = i, np.float32(-c)
    as_tensors = lambda o: {k: torch.from_numpy(np.array(v)) for k, v in o.items()}
    step.check(as_tensors(out))
    for key, at, by in (("tok", (0, 1), 1), ("score", (0, 0), 1e-3), ("parent", (2, 4), 1), ("done", (0,), 1)):
        wrong = {k: v.copy() for k, v in out.items()}
        wrong[key][at] = (wrong[key][at] + by) % (V if key == "tok" else 4 if key == "parent" else 1e9)
        with pytest.raises((AssertionError, IndexError)):
            step.check(as_tensors(wrong))


def test_slots():
    assert BU.slots([2, 2, 0, 3], 4) == [2, 1, 0, 3]
    assert BU.slots([0, 0, 0], 3) == [0, 1, 2]
    assert BU.slots([7, 1, -1, -1], 4) == [0, 1, 2, 3]
