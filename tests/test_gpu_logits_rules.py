"""gv_process_logits on the GPU against its definition in 64 bits: penalties from histories, biases, masks, odd sizes,
16-bit logits, in place."""
import numpy as np
import pytest

from paged_ref import TYPES, U32, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _rules(seed, rows, V, history, biases=0, masks=0, hot=50):
    r = np.random.default_rng(seed)
    lens = r.integers(0, history + 1, rows)
    begin = np.concatenate([[0], np.cumsum(lens)[:-1]])
    tokens = np.where(r.random(int(lens.sum())) < 0.5, r.integers(0, V, int(lens.sum())), r.integers(0, min(V, hot), int(lens.sum())))
    a = dict(tokens=tokens, begin=begin, end=begin + lens, generated=begin + lens // 3,
             repetition=r.uniform(0.8, 1.5, rows), frequency=r.uniform(-0.2, 0.5, rows), presence=r.uniform(0, 1, rows))
    a = {k: v.astype(np.float32) if v.dtype == np.float64 else v.astype(np.int32) for k, v in a.items()}
    if biases:
        a.update(bias_token=r.integers(0, min(V, 3 * biases), rows * biases).astype(np.int32),
                 bias_value=r.uniform(-5, 5, rows * biases).astype(np.float32),
                 bias_begin=(np.arange(rows) * biases).astype(np.int32), bias_end=(np.arange(1, rows + 1) * biases).astype(np.int32))
    if masks:
        a.update(masks=r.integers(0, 2 ** 32, (masks, (V + 31) // 32 + 1), dtype=np.uint64).astype(np.uint32),
                 mask_of=r.integers(-1, masks, rows).astype(np.int32))
        a["masks"][0] = 0   # a mask that leaves nothing
    return a


def _want(x, a):
    """(values, bound): a division or product, a product and two differences, the biases' sum and its addition, each off by
    half a step of what it gives at most"""
    x = x.astype(np.float64).copy()
    tol = np.zeros_like(x)
    rows, V = x.shape
    for r in range(rows):
        if a.get("tokens") is not None:
            t = a["tokens"][a["begin"][r]:a["end"][r]]
            t = t[(t >= 0) & (t < V)]
            u = np.unique(t)
            rep = float(a["repetition"][r]) if a.get("repetition") is not None else 1.0
            x[r, u] = np.where(x[r, u] > 0, x[r, u] / rep, x[r, u] * rep)
            g = a["begin"][r] if a.get("generated") is None else max(a["begin"][r], a["generated"][r])
            t = a["tokens"][g:a["end"][r]]
            c = np.bincount(t[(t >= 0) & (t < V)], minlength=V)
            fr = float(a["frequency"][r]) if a.get("frequency") is not None else 0.0
            pr = float(a["presence"][r]) if a.get("presence") is not None else 0.0
            size = np.abs(x[r]) + np.abs(fr * c) + abs(pr) * (c > 0)
            x[r] -= fr * c + pr * (c > 0)
            tol[r, u] = 4 * U32 * size[u]
        if a.get("bias_token") is not None:
            at = slice(a["bias_begin"][r], a["bias_end"][r])
            for v, b in zip(a["bias_token"][at], a["bias_value"][at]):
                if 0 <= v < V:
                    x[r, v] += float(b)
                    tol[r, v] += U32 * (abs(x[r, v]) + 20 * abs(float(b)) + 40)
        if a.get("masks") is not None and a["mask_of"][r] >= 0:
            w = a["masks"][a["mask_of"][r]]
            bit = (w[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1
            x[r, bit == 0] = -np.inf
    return x, tol


def _check(gv, x, a, kind="f32", in_place=False):
    x = round_to(x, kind).astype(np.float32)
    got = gv.process_logits(x, type_=TYPES[kind], in_place=in_place, **a)
    want, tol = _want(x, a)
    gone = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), gone)
    assert (np.abs(got[~gone] - want[~gone]) <= tol[~gone]).all()
    return got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 3, 31, 33, 2048, 2051, 4099, 50000, 151936])
def test_everything_at_once(gv, kind, V):
    r = np.random.default_rng(50)
    _check(gv, r.standard_normal((5, V)) * 3, _rules(51, 5, V, 600, biases=9, masks=3), kind)


@pytest.mark.parametrize("rows,V", [(1, 151936), (7, 32000), (70, 20001), (300, 4096)])
@pytest.mark.parametrize("parts", ["penalties", "biases", "masks", "none"])
def test_each_rule_alone(gv, rows, V, parts):
    r = np.random.default_rng(52)
    a = _rules(53, rows, V, 100, biases=5, masks=2)
    names = {"penalties": ("tokens", "begin", "end", "generated", "repetition", "frequency", "presence"),
             "biases": ("bias_token", "bias_value", "bias_begin", "bias_end"), "masks": ("masks", "mask_of"), "none": ()}[parts]
    x = r.standard_normal((rows, V)) * 3
    got = _check(gv, x, {k: a[k] for k in names})
    if parts == "none":
        assert np.array_equal(got, x.astype(np.float32))


@pytest.mark.parametrize("which", ["repetition", "frequency", "presence"])
def test_one_penalty(gv, which):
    a = _rules(54, 4, 5000, 300)
    a = {k: v for k, v in a.items() if k not in ("repetition", "frequency", "presence") or k == which}
    del a["generated"]   # (the whole history is generated)
    _check(gv, np.random.default_rng(55).standard_normal((4, 5000)), a)


@pytest.mark.parametrize("V", [5000, 5001])
def test_in_place(gv, V):
    """the same bits as out of place, what no rule changes left alone"""
    r = np.random.default_rng(56)
    x = (r.standard_normal((6, V)) * 3).astype(np.float32)
    x[0, 3] = np.nan
    a = _rules(57, 6, V, 80, biases=4, masks=2)
    a["mask_of"][0] = -1
    a["end"][0] = a["begin"][0]
    a["bias_end"][0] = a["bias_begin"][0]
    one, two = gv.process_logits(x, **a), gv.process_logits(x, in_place=True, **a)
    assert np.array_equal(one.view(np.uint32), two.view(np.uint32))


def test_biases_of_one_token_add_up_in_order(gv):
    """many biases of the same few tokens, over several batches of the list: the fp32 sum in the list's order, bit for bit"""
    r = np.random.default_rng(58)
    V, n = 9000, 700
    tok = np.where(r.random(n) < 0.7, r.integers(0, 5, n), r.integers(0, V, n)).astype(np.int32)
    val = (r.standard_normal(n) * 10.0 ** r.integers(-3, 4, n)).astype(np.float32)
    got = gv.process_logits(np.zeros((1, V), np.float32), bias_token=tok, bias_value=val, bias_begin=[0], bias_end=[n])
    want = np.zeros(V, np.float32)
    for t, b in zip(tok, val):
        want[t] = np.float32(want[t] + b)
    assert np.array_equal(got[0], want)


def test_tokens_outside_the_vocabulary_and_infinite_logits(gv):
    V = 3000
    a = dict(tokens=np.array([-1, V, 2 ** 30, 7, -2 ** 31, 9, 9], np.int32), begin=np.array([0], np.int32),
             end=np.array([7], np.int32), repetition=np.array([1.25], np.float32), frequency=np.array([0.5], np.float32),
             bias_token=np.array([-5, V, 8], np.int32), bias_value=np.array([1, 1, 2], np.float32),
             bias_begin=np.array([0], np.int32), bias_end=np.array([3], np.int32))
    x = np.ones((1, V), np.float32)
    x[0, 7], x[0, 9], x[0, 20] = -np.inf, np.inf, np.nan
    got = gv.process_logits(x, **a)
    assert np.isneginf(got[0, 7]) and np.isposinf(got[0, 9]) and np.isnan(got[0, 20]) and got[0, 8] == 3.0
    rest = np.ones(V, bool)
    rest[[7, 8, 9, 20]] = False
    assert (got[0, rest] == 1.0).all()


def test_shared_histories_of_a_chain(gv):
    """row i of a draft chain sees the conversation and the i drafts before it (ranges over the same tokens)"""
    r = np.random.default_rng(59)
    V, n = 4000, 500
    tokens = r.integers(0, 60, n + 4).astype(np.int32)
    a = dict(tokens=tokens, begin=np.zeros(5, np.int32), end=(n + np.arange(5)).astype(np.int32),
             generated=np.full(5, 200, np.int32), presence=np.full(5, 0.7, np.float32), frequency=np.full(5, 0.1, np.float32),
             repetition=np.full(5, 1.1, np.float32))
    _check(gv, r.standard_normal((5, V)), a)


def test_long_histories_of_one_token(gv):
    """100,000 times one token: counted exactly"""
    a = dict(tokens=np.full(100000, 17, np.int32), begin=[0], end=[100000], frequency=np.array([2.0 ** -10], np.float32))
    a["begin"], a["end"] = np.array([0], np.int32), np.array([100000], np.int32)
    got = gv.process_logits(np.zeros((1, 300), np.float32), **a)
    assert got[0, 17] == -100000 * 2.0 ** -10 and np.count_nonzero(got) == 1


def test_faults_in_device_memory(gv):
    """ranges and masks outside their arrays: reported, the other rows as without them"""
    r = np.random.default_rng(60)
    x = r.standard_normal((4, 3000)).astype(np.float32)
    a = _rules(61, 4, 3000, 50, biases=3, masks=2)
    base = gv.process_logits(x, **a)
    for name, row, val in (("end", 1, len(a["tokens"]) + 1), ("begin", 1, -1), ("begin", 1, int(a["end"][1]) + 1),
                           ("bias_end", 2, 100), ("bias_begin", 2, -3), ("mask_of", 3, 2)):
        b = {k: np.array(v) for k, v in a.items()}
        b[name][row] = val
        with pytest.raises(gv.GeodeError, match="range"):
            gv.process_logits(x, **b)
        gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    assert np.array_equal(gv.process_logits(x, **a), base)


def test_then_sampled(gv):
    """the processed rows into the sampler, as a host uses them: greedy picks are the processed rows' first maxima, and a
    mask that leaves one token gives that token"""
    r = np.random.default_rng(62)
    V = 20000
    x = (r.standard_normal((4, V)) * 3).astype(np.float32)
    a = _rules(63, 4, V, 200, biases=4, masks=2)
    a["masks"][1] = 0
    a["masks"][1, 77 // 32] = 1 << (77 % 32)
    a["mask_of"] = np.array([-1, -1, 1, 1], np.int32)
    y = gv.process_logits(x, **a)
    pick = gv.sample_rows(y, 0.0)
    assert list(pick) == [int(np.argmax(row)) for row in y] and pick[2] == pick[3] == 77
    assert list(gv.sample_rows(y, 0.7, 0.95, 0, 1024, np.full(4, 0.6)))[2:] == [77, 77]
