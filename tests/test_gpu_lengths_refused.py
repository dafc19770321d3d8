"""GPU (nothing is launched): draws, fed tokens and windows that do not cover the rows are refused, with edits and without."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("edited", [False, True])
def test_lengths_are_refused(edited):
    x = torch.randn((6, 64), device="cuda")
    kw = dict(edits=F.Edits()) if edited else {}
    p6, p2 = W.make_params(6), W.make_params(2)
    with pytest.raises(F.SamplerError, match="one draw per row"):
        F.sample_batch(x, p6, np.zeros(5), **kw)
    fed, off = np.zeros(6, np.int32), [0, 2, 6]
    with pytest.raises(F.SamplerError, match="one draw per row"):
        F.verify(x, fed, off, p2, u=np.zeros(5), **kw)
    with pytest.raises(F.SamplerError, match="one fed token"):
        F.verify(x, fed[:5], off, p2, **kw)
    # rows behind the last window, before the first one, windows that run backwards
    for bad in ([0, 2, 5], [1, 2, 6], [0, 7, 6], [0, 2, 7]):
        with pytest.raises(F.SamplerError, match="ascend from 0"):
            F.verify(x, fed, bad, p2, **kw)
        with pytest.raises(F.SamplerError, match="ascend from 0"):
            F.verify(x, fed, torch.tensor(bad), p2, **kw)
    tok, acc = F.verify(x, fed, off, p2, **kw)
    assert tok.numel() == 6 and acc.numel() == 2
    torch.cuda.synchronize()
