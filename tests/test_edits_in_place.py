"""CPU: the struct an Edits gives a call, over tensors that are used in place and tensors that are converted."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402

CPU = torch.device("cpu")


def words_at(ptr, n):
    return list((ctypes.c_int32 * n).from_address(ptr))


def test_packed_tensors_are_used_in_place():
    table = torch.zeros((3, 9), dtype=torch.int32)
    of = torch.zeros(2, dtype=torch.int32)
    bias = (torch.tensor([5, 7], dtype=torch.int32), torch.zeros(2), torch.tensor([0, 1, 2]))
    ed = F.Edits(mask=table[:, :4], mask_of=of, bias=bias, device="cpu")
    c = ed._now(2, 2, 128, CPU)
    assert (c.d_mask, c.mask_ld, c.n_masks) == (table.data_ptr(), 9, 3) and c.d_mask_of == of.data_ptr()
    assert (c.d_bias_ids, c.d_bias, c.d_bias_off) == tuple(t.data_ptr() for t in bias)


@pytest.mark.parametrize("made", [torch.int64, torch.int16])
def test_other_tensors_are_converted_by_each_call(made):
    table = torch.zeros((4, 3), dtype=torch.int32)
    of = torch.zeros(2, dtype=made)
    ids, val, off = torch.tensor([5, 7]), torch.zeros(2, dtype=torch.float64), torch.tensor([0, 1, 2], dtype=torch.int32)
    ed = F.Edits(mask=table.t(), mask_of=of, bias=(ids, val, off), device="cpu")
    for step in range(1, 4):
        table.fill_(step)
        of.fill_(step - 1)
        ids[1] = 7 + step
        val.fill_(0.5 * step)
        off[1] = step % 2
        c = ed._now(2, 2, 128, CPU)
        assert words_at(c.d_mask, 12) == [step] * 12 and (c.mask_ld, c.n_masks) == (4, 3)
        assert words_at(c.d_mask_of, 2) == [step - 1] * 2 and words_at(c.d_bias_ids, 2) == [5, 7 + step]
        assert list((ctypes.c_float * 2).from_address(c.d_bias)) == [0.5 * step] * 2
        assert list((ctypes.c_int64 * 3).from_address(c.d_bias_off)) == [0, step % 2, 2]


def test_arrays_are_taken_as_they_are_when_given():
    of = np.zeros(2, np.int64)
    ed = F.Edits(mask=np.ones((2, 3), np.uint32), mask_of=of, device="cpu")
    of[:] = 1
    assert words_at(ed._now(2, 2, 96, CPU).d_mask_of, 2) == [0, 0]


@pytest.mark.parametrize("made", [list, tuple, iter])
def test_one_dict_per_record_in_any_sequence(made):
    """Three records, too: they are no CSR lists."""
    for dicts in ([{9: 1.0, 2: -1.0}, None, {4: 0.5}], [{3: 1.0}], [{}, {}, {}], []):
        ed = F.Edits(bias=made(dicts), device="cpu")
        assert ed.bias_ids.tolist() == [t for d in dicts for t in sorted(d or {})]
        assert ed.bias_off.tolist() == [0, *np.cumsum([len(d or {}) for d in dicts]).tolist()]


def test_csr_lists_in_a_list_and_refusals():
    ed = F.Edits(bias=[np.array([5, 7]), np.ones(2, np.float32), [0, 2]], device="cpu")
    assert ed.bias_ids.tolist() == [5, 7] and ed.bias_off.tolist() == [0, 2]
    for bad in ([np.array([5])], (np.array([5]), np.ones(1)), [{}, [1], {}, {}]):
        with pytest.raises(F.SamplerError):
            F.Edits(bias=bad, device="cpu")
