"""ptmi_sample_dev against a plain 64-bit restatement."""
import numpy as np
import pytest

import pitorch_amd as pa
from pitorch_amd._ffi import check
from tests import _paged as R

pytestmark = pytest.mark.gpu

# A weight is a multiple of 2^-44, half a step off, and V of them in a sum that is at least 1: a
# decision nearer to its border than V 2^-44 (and 64-bit roundings of the restatement) may fall either way.
NEAR = 2.0**-44


def dev(a):
    from pitorch_amd._hip import DeviceArray
    return DeviceArray.from_host(np.ascontiguousarray(a))


def run(x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, pad=0):
    rows, V = x.shape
    m = np.full((rows, V + pad), np.float32(1e30))           # what stands between rows is never looked at
    m[:, :V] = x
    f = lambda a, t: None if a is None else dev(np.asarray(a, t))  # noqa: E731
    d = [f(temperature, np.float32), f(top_k, np.int32), f(top_p, np.float32), f(min_p, np.float32), f(u, np.float32)]
    dx, dt = dev(m.astype(np.float32).reshape(-1)), dev(np.full(rows + 1, -99, np.int32))
    check(pa.load_ptmi().ptmi_sample_dev(dx.ptr, V + pad, rows, V, *[a.ptr if a else None for a in d], dt.ptr, None))
    check(pa.load_ptmi().ptmi_sync())
    got = dt.download()
    assert got[rows] == -99
    return got[:rows]


def compare(x, pad=0, **kw):
    got = run(x, pad=pad, **kw)
    near = 0
    for r in range(len(x)):
        args = {k: (np.float32(v[r]) if k != "top_k" else int(v[r])) for k, v in kw.items() if v is not None}
        want, margin = R.sample(x[r], **{k: (float(v) if k != "top_k" else v) for k, v in args.items()})
        if got[r] != want:
            assert margin < x.shape[1] * NEAR, (r, got[r], want, margin, args)
            near += 1
    assert near <= 1
    return got


def logits(rng, rows, V, kind):
    x = rng.standard_normal((rows, V)).astype(np.float32)
    if kind == "model":
        x = x * 2 + 9 * rng.random((rows, V)).astype(np.float32) ** 200
    elif kind == "flat":
        x[:] = 0.25
    elif kind == "ties":
        x = np.round(x * 2) / 2
    elif kind == "sharp":
        x *= 30
    elif kind == "masked":
        x[rng.random((rows, V)) < 0.97] = -np.inf
        x[:, -1] = 0.5
    elif kind == "outlier":
        x *= 1e-3
        x[:, V // 2] = 3e4
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1027, 4096, 32000, 32003, 32768, 32769, 50259, 131072])
@pytest.mark.parametrize("kind", ["model", "flat", "ties", "sharp", "masked", "outlier"])
def test_all_filters(V, kind):
    rows = 24 if V < 40000 else 8
    rng = np.random.default_rng(V * 7 + len(kind))
    x = logits(rng, rows, V, kind)
    compare(x, temperature=rng.choice([0.0, 0.7, 1.0, 1.0, 1.5, 0.05], rows), top_k=rng.choice([0, 0, 1, 5, 50, V, V + 3, 700], rows),
            top_p=rng.choice([1.0, 0.9, 0.5, 0.99, 1e-6], rows), min_p=rng.choice([0.0, 0.0, 0.05, 0.3], rows), u=rng.random(rows))


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p", "u", None])
def test_absent_parameters(only):
    rng = np.random.default_rng(3)
    x = logits(rng, 16, 3000, "model")
    kw = {} if only is None else {only: {"temperature": [0.6] * 16, "top_k": [3] * 16, "top_p": [0.8] * 16, "min_p": [0.2] * 16,
                                         "u": rng.random(16)}[only]}
    compare(x, pad=5, **kw)


@pytest.mark.parametrize("V", [5, 100, 32000, 40000])
def test_rows_with_nothing_to_choose(V):
    x = np.full((6, V), -np.inf, np.float32)
    x[1] = np.nan
    x[2, V - 1] = -3e38                                       # one choice
    x[3, 3] = np.inf
    x[4, 1] = x[4, 3] = np.inf
    x[5, 2] = np.finfo(np.float32).min
    x[5, 4] = np.nan
    for u in (0.0, 0.49, 0.51, 0.99999994):
        got = compare(x, temperature=[1.0] * 6, u=[u] * 6)
        assert got.tolist() == [-1, -1, V - 1, 3, 1 if u < 0.5 else 3, 2]
    assert run(x, temperature=[0.0] * 6).tolist() == [-1, -1, V - 1, 3, 1, 2]


def test_parameters_out_of_range():
    rng = np.random.default_rng(4)
    x = logits(rng, 12, 500, "model")
    nan = float("nan")
    compare(x, temperature=[-1, nan, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1e-30], top_k=[0, 0, -4, 2**31 - 1, 0, 0, 0, 0, 0, 0, 0, 0],
            top_p=[1, 1, 1, 1, 0, -1, nan, 2, 1, 1, 1, 1], min_p=[0, 0, 0, 0, 0, 0, 0, 0, 2, -1, nan, 0],
            u=[.5, .5, -1, 2, .3, .3, .3, .3, .3, nan, .7, .7])


def test_temperatures_that_choose():
    """Logits nearer to the maximum than a millionth of it, at temperatures that tell them apart all the same."""
    x = np.full((8, 300), -5.0, np.float32)
    x[:, 40:60] = np.float32(1000) + np.arange(20, dtype=np.float32) * np.float32(2.0**-14)
    x[:, 47] = x[:, 59]                                       # two maxima
    for t in (1e-38, 1e-30, 1e-9, 1e-5):
        got = compare(x, temperature=[t] * 8, u=np.linspace(0, 0.99, 8))
        if t < 1e-6:
            assert got.tolist() == [47] * 4 + [59] * 4
    compare(x, temperature=[1e30, 3e38] * 4, u=np.linspace(0, 0.99, 8))


@pytest.mark.parametrize("unit", [1.4e-45, 3e-42, 1e-36, 1e-25, 1e33])
def test_logits_of_any_size(unit):
    """Subnormal logits, and differences that overflow: the order is that of the values all the same."""
    rng = np.random.default_rng(6)
    with np.errstate(under="ignore"):
        x = (rng.integers(-300, 300, (6, 5000)).astype(np.float64) * unit).astype(np.float32)
    x[3:, 7] = 3.3e38
    x[3:, 8] = -3.3e38
    t = [1.0, unit * 1e3 if unit * 1e3 > 1e-37 else 1e-37, 1e35] * 2
    compare(x, temperature=t, top_k=[700, 5, 4000, 2, 700, 4999], u=rng.random(6))
    compare(x, temperature=t, top_p=[0.3, 0.8, 0.5, 0.5, 0.9, 0.99], u=rng.random(6))


@pytest.mark.parametrize("V", [1, 3, 255, 256, 257, 4100, 9000, 20001, 33000, 70001])
@pytest.mark.parametrize("step", [0.0, 0.25])
def test_how_many_stay(V, step):
    """top_k around the numbers of logits that are compared at once or looked at one by one, with equals (step) and
    without, and top_p behind it."""
    rng = np.random.default_rng(V)
    ks = [2, 17, 63, 64, 65, 255, 256, 257, 300, V // 32, V // 32 + 1, V - 1]
    x = (rng.standard_normal((len(ks), V)) * 2).astype(np.float32)
    if step:
        x = (np.round(x / step) * step).astype(np.float32)
    x[::3, : V // 2] = -np.inf
    u, t = rng.random(len(ks)), np.full(len(ks), 0.9)
    for p in (1.0, 0.97, 0.5):
        compare(x, pad=1, temperature=t, top_k=ks, top_p=np.full(len(ks), p), u=u)
    compare(x, temperature=t, top_k=ks, min_p=np.full(len(ks), 0.03), top_p=np.full(len(ks), 0.9), u=u)


@pytest.mark.parametrize("V", [1000, 32000])
def test_equal_logits(V):
    """Whole weights: every border is met exactly, and the first of equals counts."""
    x = np.zeros((4, V), np.float32)
    x[2, ::2] = -0.0
    got = run(x, top_k=[10, 10, 10, 0], top_p=[1.0, 0.5, 1.0, 0.25], u=[0.35, 0.9, 0.95, 0.0])
    assert got.tolist() == [3, 4, 9, 0]
    assert run(x, top_p=[0.25] * 4, u=[0.99999994] * 4).tolist() == [V // 4 - 1] * 4
    assert run(x, u=[0.5] * 4).tolist() == [V // 2] * 4


def test_frequencies():
    """Tokens come as often as their probabilities say: each count within six deviations of its mean."""
    x = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625], np.float32))
    n = 20000
    got = run(np.tile(x, (n, 1)), u=(np.arange(n) + 0.5) / n)
    for i, p in enumerate((0.5, 0.25, 0.125, 0.0625, 0.0625)):
        assert abs((got == i).sum() - n * p) <= 2              # equally spaced numbers: exact but for the ends
