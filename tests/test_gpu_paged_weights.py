"""The weights' bits in gv_paged_attention's second product: 16-bit results over a bf16 cache, where they go to the matrix cores
as two parts of 8 bits."""
import numpy as np
import pytest

from paged_ref import Filled, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _half_step(x):
    """half a bf16 step at x (a value in [2^e, 2^(e+1)): 2^(e - 8))"""
    return 2.0 ** (np.floor(np.log2(np.abs(x))) - 8)


def _hard_cases(n, hd):
    """scores s (bf16) and values v (bf16) of which v w / (1 + w), w = e^s, lies a little more than 2^-16 above the middle
    between two bf16 values: a weight that is off by up to 2^-16 still rounds as it should, one off by 2^-15 need not"""
    s = -np.arange(1 << 8, 6 << 8) / 256.0
    s = np.unique(round_to(s, "bf16"))
    v = 1.0 + np.arange(128) / 128.0
    out = v * (np.exp(s) / (1 + np.exp(s)))[:, None]
    step = 2 * _half_step(out)
    past = (out / step - np.floor(out / step) - 0.5) * step / out   # how far above the middle, relative
    hit = (past > 1.05 * 2.0 ** -16) & (past < 1.5 * 2.0 ** -16)
    rows = np.argsort(-hit.sum(1), kind="stable")[:n]
    values = np.ones((n, hd))
    for i, r in enumerate(rows):
        found = v[hit[r]][:hd]
        values[i, :found.size] = found
    return s[rows], values


@pytest.mark.parametrize("nh,hd", [(1, 64), (20, 64), (1, 128), (20, 128), (1, 256), (20, 256)])
def test_weights_of_16_bits(gv, nh, hd):
    """two positions a sequence, of weight 1 and value 0, and of weight w: the result is off by its own rounding and 2^-16 of
    it (the weight's parts: the second, below 2^-7 of the first, rounded to 8 bits), and what the exponential and the sum
    in fp32 add (2^-20 is far more)"""
    n = 300
    s, v = _hard_cases(n, hd)
    f = Filled(60, "bf16", [1] * n, [2] * n, 16, 1, hd, spare=0)
    k, val = (np.zeros((n, 1, 16, hd)) for _ in range(2))
    for i in range(n):
        p, at = f.place(i, 0)
        k[p, 0, at, 0] = s[i]
        val[p, 0, at] = v[i]
    f.cache.write("k", k)
    f.cache.write("v", val)
    q = np.zeros((n, nh, hd))
    q[..., 0] = 1.0
    out, _ = gv.paged_attention(f.cache, f.batch, q, type_=gv.BF16, scale=1.0)
    w = np.exp(s)[:, None]
    want = v * w / (1 + w)
    tol = _half_step(want) + want * (2.0 ** -16 + 2.0 ** -20)
    err = np.abs(out - want[:, None])
    assert (err <= tol[:, None]).all(), f"{int((err > tol[:, None]).sum())} results are off"
