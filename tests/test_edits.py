"""CPU: refusals of the calls under edits (the C ABI's checks come before any device work) and the Edits handle."""
import ctypes

import numpy as np
import pytest

import ferro_amd as F
from ferro_amd import _lib
from ferro_amd._lib import FS_E_INVALID, FS_OK, FsEdits, SamplerError
from tests.edit_util import unpack

torch = pytest.importorskip("torch")
P = ctypes.c_void_p
FAKE = P(64)                                   # never dereferenced: argument checks fail first


@pytest.fixture()
def ctx():
    h = P()
    assert _lib.lib().fs_create(ctypes.byref(h)) == FS_OK
    yield h
    _lib.lib().fs_destroy(h)


def edits(**kw):
    e = FsEdits()
    for k, v in kw.items():
        setattr(e, k, v)
    return e


GOOD = edits(d_mask=64, mask_ld=1, n_masks=1)
BAD = [
    edits(d_mask=64, mask_ld=0, n_masks=1),                    # masks shorter than the vocabulary
    edits(d_mask=64, mask_ld=1, n_masks=-1),
    edits(d_mask=64, mask_ld=1, n_masks=0),                    # fewer masks than rows, no index
    edits(d_mask=66, mask_ld=1, n_masks=1),                    # words not aligned
    edits(n_masks=1), edits(d_mask_of=64),                     # masks described, none given
    edits(d_bias_ids=64, d_bias=64), edits(d_bias_off=64, d_bias=64), edits(d_bias_off=64, d_bias_ids=64),
]


def sample(h, e, x=FAKE, ld=8, B=1, V=8, params=FAKE, tok=FAKE, kcap=0, cand=None):
    return _lib.lib().fs_sample_edited(h, x, ld, B, V, None, None, params, None, e, None, tok, kcap, cand, None, None, None)


def edit(h, e, x=FAKE, kind=0, ld=8, B=1, V=8, out=P(1 << 20), out_ld=8):
    return _lib.lib().fs_edit_batch(h, x, kind, ld, B, V, None, None, None, e, out, out_ld, None)


def logprobs(h, e, x=FAKE, kind=0, ld=8, B=1, V=8, tok=FAKE, n=0, lp=FAKE, rank=FAKE, ids=None, top=None):
    return _lib.lib().fs_logprobs(h, x, kind, ld, B, V, None, e, tok, n, lp, rank, ids, top, None)


@pytest.mark.parametrize("i", range(len(BAD)))
def test_bad_edits_are_refused(ctx, i):
    e = ctypes.byref(BAD[i])
    L = _lib.lib()
    assert sample(ctx, e) == FS_E_INVALID
    assert edit(ctx, e) == FS_E_INVALID
    assert logprobs(ctx, e) == FS_E_INVALID
    assert L.fs_verify_edited(ctx, FAKE, 8, 1, 1, 8, FAKE, FAKE, None, None, FAKE, None, e, None, -1, FAKE, FAKE, None) \
        == FS_E_INVALID


def test_bad_arguments_are_refused(ctx):
    e = ctypes.byref(GOOD)
    L = _lib.lib()
    assert sample(None, e) == FS_E_INVALID and sample(ctx, None) == FS_E_INVALID
    assert sample(ctx, e, params=None) == FS_E_INVALID and sample(ctx, e, tok=None) == FS_E_INVALID
    assert sample(ctx, e, cand=FAKE) == FS_E_INVALID and sample(ctx, e, kcap=-1) == FS_E_INVALID
    for bad in (dict(x=None), dict(x=P(4)), dict(ld=6, V=6), dict(ld=4), dict(V=0), dict(B=-1)):
        assert sample(ctx, e, **bad) == FS_E_INVALID, bad
        assert edit(ctx, e, **bad) == FS_E_INVALID, bad
        assert logprobs(ctx, e, **bad) == FS_E_INVALID, bad
    assert sample(ctx, e, B=0) == FS_OK and edit(ctx, e, B=0) == FS_OK and logprobs(ctx, e, B=0) == FS_OK
    # 16-bit logits: four of them aligned; no other types
    assert edit(ctx, e, kind=1, x=P(68)) == FS_E_INVALID and edit(ctx, e, kind=3) == FS_E_INVALID
    assert logprobs(ctx, e, kind=2, x=P(68)) == FS_E_INVALID and logprobs(ctx, e, kind=-1) == FS_E_INVALID
    # outputs: aligned, long enough, not over the inputs unless in place
    assert edit(ctx, e, out=None) == FS_E_INVALID and edit(ctx, e, out=P(8)) == FS_E_INVALID
    assert edit(ctx, e, out_ld=4) == FS_E_INVALID and edit(ctx, e, out_ld=10) == FS_E_INVALID
    assert edit(ctx, e, out=P(80)) == FS_E_INVALID                      # 16 bytes into the logits
    assert edit(ctx, e, out=FAKE, kind=1) == FS_E_INVALID               # in place in another type
    assert edit(ctx, e, x=P(1 << 20), out=P(1 << 20), ld=8, out_ld=12, B=2) == FS_E_INVALID
    # log-probabilities
    assert logprobs(ctx, e, n=-1) == FS_E_INVALID and logprobs(ctx, e, n=65, ids=FAKE) == FS_E_INVALID
    assert logprobs(ctx, e, tok=None) == FS_E_INVALID and logprobs(ctx, e, ids=FAKE) == FS_E_INVALID
    # a decode step: no streams, no outputs
    assert L.fs_decode_step_edited(ctx, None, FAKE, 8, 1, 8, None, None, FAKE, None, e, FAKE, None, FAKE, FAKE, 4, None) \
        == FS_E_INVALID
    assert L.fs_verify_edited(ctx, FAKE, 8, -1, 1, 8, FAKE, FAKE, None, None, FAKE, None, e, None, -1, FAKE, FAKE, None) \
        == FS_E_INVALID


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100])
def test_pack_is_the_words_bit_order(V):
    a = np.random.default_rng(V).random((3, V)) < 0.5
    w = F.Edits.pack(a)
    assert w.shape == (3, (V + 31) // 32) and np.array_equal(unpack(w, V), a)
    assert np.array_equal(F.Edits.pack(torch.from_numpy(a)).numpy(), w)
    for t in range(V):
        assert ((int(w[0, t // 32]) >> (t % 32)) & 1) == int(a[0, t])


def test_edits_handle_checks():
    cpu = dict(device="cpu")
    with pytest.raises(SamplerError):
        F.Edits(mask=np.zeros((2, 1), np.int64), **cpu)
    with pytest.raises(SamplerError):
        F.Edits(mask_of=[0], **cpu)
    with pytest.raises(SamplerError, match="ascend"):
        F.Edits(bias=(np.array([5, 3]), np.zeros(2, np.float32), [0, 2]), **cpu)
    with pytest.raises(SamplerError):
        F.Edits(bias=(np.array([5, 7]), np.zeros(2, np.float32), [0, 3]), **cpu)
    with pytest.raises(SamplerError):
        F.Edits(bias=(np.array([5, 7]), np.zeros(1, np.float32), [0, 2]), **cpu)
    e = F.Edits(bias=(np.array([5, 7, 3, 3]), np.zeros(4, np.float32), [0, 2, 4]), **cpu)   # ascending in each record
    assert e.bias_off.tolist() == [0, 2, 4]
    e = F.Edits(bias=[{9: 1.0, 2: -1.0}, {}, None, {4: 0.5}], **cpu)
    assert e.bias_ids.tolist() == [2, 9, 4] and e.bias_off.tolist() == [0, 2, 2, 2, 3]
    assert F.Edits(bias=[{}, {}], **cpu).bias_off.tolist() == [0, 0, 0]
    e = F.Edits(mask=np.zeros((2, 3), np.uint32), **cpu)
    assert (e.c.n_masks, e.c.mask_ld) == (2, 3) and e.mask.dtype == torch.int32
    for rows, records, V in ((3, 3, 96), (2, 2, 97)):
        with pytest.raises(SamplerError):
            e._ref(rows, records, V, torch.device("cpu"))
    with pytest.raises(SamplerError):
        F.Edits(mask=np.zeros((2, 3), np.int32), mask_of=[0, 1, 0], **cpu)._ref(2, 2, 96, torch.device("cpu"))
    with pytest.raises(SamplerError):
        F.Edits(bias=[{}], **cpu)._ref(2, 2, 96, torch.device("cpu"))


def test_a_table_without_masks_is_a_valid_pointer():
    """A step in which no row has a grammar: a table of no masks, every row's index negative."""
    e = F.Edits(mask=np.zeros((0, 3), np.int32), mask_of=[-1, -1], device="cpu")
    assert e.c.d_mask and e.c.d_mask_of and (e.c.n_masks, e.c.mask_ld) == (0, 3)
    e._ref(2, 2, 96, torch.device("cpu"))
    with pytest.raises(SamplerError):
        e._ref(2, 2, 97, torch.device("cpu"))
    with pytest.raises(SamplerError, match="one mask per row"):
        F.Edits(mask=np.zeros((0, 3), np.int32), device="cpu")._ref(2, 2, 96, torch.device("cpu"))
