"""CPU: what the beam search's Python wrappers work out on the host, and calls they refuse."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402


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
