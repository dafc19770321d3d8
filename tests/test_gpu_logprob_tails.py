"""GPU: log-probabilities where the sum is one term and very little else, and at the ends of the temperatures' range."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import ferro_amd as F  # noqa: E402
from ferro_amd import workloads as W  # noqa: E402
from tests.edit_util import logprob_row  # noqa: E402
from tests.test_gpu_edits import lp_tolerance  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.synchronize()
    assert F.device_error() == 0


def lp_of_largest(x, T=1.0):
    """-log sum exp((x - max) / T) in 64 bits, the terms below 1 added by themselves."""
    d = (np.sort(x.astype(np.float64))[::-1] - float(x.max())) / T
    ones = int((d == 0).sum())
    rest = math.fsum(np.exp(d[ones:]))
    return -(math.log(ones) + math.log1p(rest / ones))


def near_certain_tolerance(lp):
    """The terms below 1 are positive, and no fp32 sum holds a 1 beside them, so their sum is off by a relative amount alone: a
    difference, c = log2 e / T and their product rounded (u = 2^-24 each, relative to an argument of at most 90 where a term
    is a normal number), the exponential (an ulp, 2u), at most 10 fp32 additions: (3 * 90 + 2 + 10) u. The logarithm of 1 + r
    moves by no more, relatively, than r; the result is rounded to fp32. In fp64 every sum that holds the 1 is rounded by up
    to 2^-53: here (a part per chunk) 16 additions of a lane's terms, two more in the lane, six over the wave, up to four and
    six over the row's waves, 34 in all."""
    return (282 + 1) * U * abs(lp) + 34 * 2.0 ** -53


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [2, 70, 16384, 151936])
@pytest.mark.parametrize("gap", [9.0, 15.0, 17.0, 18.0, 24.0])
def test_near_certain_tokens(dtype, V, gap):
    """The largest token and the runner-up side by side (one lane adds both), apart by `gap`, anywhere in the row; also after
    smaller ones, twice, and alone."""
    rows, tok = [], []
    for at in sorted({0, V // 3, V - 2}):
        x = np.full(V, -200.0)
        x[at], x[at + 1] = 3.0, 3.0 - gap
        rows.append(x)
        tok.append(at)
        y = x.copy()
        y[at], y[at + 1] = 3.0 - gap, 3.0                      # the runner-up first
        y[:at:7] = -4.0 - gap                                  # smaller ones before both
        rows.append(y)
        tok.append(at + 1)
    both = rows[-1].copy()
    both[0] = both.max()                                       # two largest ones
    rows.append(both)
    tok.append(0)
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda().to(DTYPES[dtype])
    xs = x.float().cpu().numpy()
    for T in (1.0, 0.5):
        p = W.make_params(len(rows), temperature=T, repetition_penalty=1.0)
        out = F.logprobs(x, np.array(tok, np.int32), min(V, 2), params=p)
        for r in range(len(rows)):
            want = lp_of_largest(xs[r], T)
            assert abs(float(out["lp"][r]) - want) <= near_certain_tolerance(want), (r, T, float(out["lp"][r]), want)
            assert out["top"][r, 0] == out["lp"][r] and int(out["rank"][r]) == 1


def test_near_certain_tokens_among_noise():
    """A body of logits far below one that stands out: each chunk has a part of the small sum."""
    g = torch.Generator("cuda").manual_seed(2)
    for V in (5000, 262144):
        x = torch.randn((4, V), device="cuda", generator=g)
        at = torch.tensor([0, 1, V // 2, V - 1], device="cuda")
        for up in (20.0, 30.0):
            y = x.clone()
            y[torch.arange(4), at] = up
            out = F.logprobs(y, at.to(torch.int32), 1)
            for r in range(4):
                want = lp_of_largest(y[r].cpu().numpy())
                assert abs(float(out["lp"][r]) - want) <= near_certain_tolerance(want), (V, up, r, float(out["lp"][r]), want)


TINY = np.float32(2.0 ** -149)


@pytest.mark.parametrize("T", [float(TINY), 1e-42, 2.0 ** -127, 1e-33, 1e33, 3e38, math.inf])
@pytest.mark.parametrize("V", [5, 4096, 30011])
def test_log_probabilities_at_the_ends_of_the_temperatures(T, V):
    """Temperatures whose reciprocal, or whose share of the logits' differences, fp32 does not hold; infinite ones (every
    token that takes part is equally likely)."""
    T = float(np.float32(T))
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((7, V)) * 3).astype(np.float32)
    x[1, 2:] = x[1, 0]                                         # ties
    x[2] = np.where(np.arange(V) % 3 == 0, 3e38, -3e38)        # a difference that fp32 does not hold
    x[3, ::2] = np.nan
    x[4] = np.arange(V) * np.float32(1e-40)                    # and differences below its normal numbers
    x[5, ::2] = -np.inf
    x[6, 3] = np.inf
    allowed = rng.random((7, V)) < 0.8
    allowed[:, :4] = True
    ed = F.Edits(mask=F.Edits.pack(allowed))
    p = W.make_params(7, temperature=T, repetition_penalty=1.0)
    tok = np.array([1, 1, 1, 1, 2, 1, 3], np.int32)
    n = min(V, 4)
    for dtype in (torch.float32, torch.bfloat16):
        t = torch.from_numpy(x).cuda().to(dtype)
        xs = t.float().cpu().numpy()
        out = {k: v.cpu().numpy() for k, v in F.logprobs(t, tok, n, params=p, edits=ed).items()}
        for r in range(7):
            lp, rank, ids, top = logprob_row(xs[r], int(tok[r]), n, T=T, allowed=allowed[r])
            assert out["ids"][r].tolist() == ids.tolist() and int(out["rank"][r]) == rank, r
            for got, want in zip([out["lp"][r], *out["top"][r]], [lp, *top]):
                if want < -3.4028235e38:
                    assert got == -math.inf, (r, got, want)
                else:
                    assert abs(float(got) - want) <= lp_tolerance(want), (r, got, want)
