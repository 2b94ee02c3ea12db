"""gv_paged_attention over an int8 cache whose value scales span far beyond fp16's range: what a position adds is its weight
times its scale, so neither a huge scale of no weight nor the strong positions' tiny scales may cost the others' bits."""
import numpy as np
import pytest

from paged_ref import TYPES, Filled, attention, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _spanned(f, seed, scores, log2_scales, reach):
    """an int8 Filled's codes and scales rewritten: position p of sequence i has the key value scores[i][p] / reach in
    dim 0 (at most 0) and none elsewhere, and the value scale 2^log2_scales[i][p] x a little"""
    r = np.random.default_rng(seed)
    nkv, hd = f.cache.desc.n_kv_heads, f.cache.desc.head_dim
    pool = f.cache.desc.n_pages
    k, v = np.zeros((pool, nkv, f.page, hd)), r.integers(-127, 128, (pool, nkv, f.page, hd))
    ks, vs = (np.full((pool, nkv, f.page), np.nan, np.float32) for _ in range(2))
    for i, n in enumerate(f.lens):
        for pos in range(n):
            p, s = f.place(i, pos)
            k[p, :, s, 0] = -127
            ks[p, :, s] = -scores[i][pos] / reach / 127.0
            vs[p, :, s] = 2.0 ** log2_scales[i][pos] * r.uniform(1.0, 1.9, nkv)
    for name, codes, scales in (("k", k, ks), ("v", v, vs)):
        f.cache.write(name, codes, scales)
        f.host[name] = codes * scales[..., None].astype(np.float64)
    return vs


def _check(gv, f, kind, nh, reach, vs):
    T, hd = f.batch.desc.n_rows, f.cache.desc.head_dim
    q = np.zeros((T, nh, hd))
    q[..., 0] = reach
    q = round_to(q, kind)
    out, lse = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind], scale=1.0)
    want, want_lse, tol, tol_lse = attention(f, q, 1.0, kind)
    # Beside paged_ref's bound: a weight x scale goes to the products in steps of 2^-24 of a power of two of which the largest
    # has at least 2^13, so it is off by 2^-37 of the largest at most, with codes of 127; its exponential's argument is off by
    # |s - m| 2^-24 also where p itself is below what paged_ref looks at (|s - m| at most 90 here).
    for i, n in enumerate(f.lens):
        for r in range(f.start[i], f.start[i + 1]):
            for h in range(nh):
                g = h // (nh // f.cache.desc.n_kv_heads)
                seen = n - f.rows[i] + r - f.start[i] + 1
                s = f.sequence("k", i)[g, :seen, 0] * q[r, h, 0]
                w = np.exp(s - s.max()) / np.exp(s - s.max()).sum()
                scale = np.array([vs[f.place(i, p)[0], g, f.place(i, p)[1]] for p in range(seen)], np.float64)
                tol[r, h] += seen * 2.0 ** -36 * 127 * (w * scale).max()
                tol[r, h] += 2 * 90 * 2.0 ** -24 * (w @ np.abs(f.sequence("v", i)[g, :seen]))
    own = np.zeros(T, bool)
    for i in range(len(f.lens)):
        own[f.start[i]:f.start[i + 1]] = True
    err = np.abs(out - want)[own]
    assert np.isfinite(out[own]).all()
    assert (err <= tol[own]).all(), f"out off by {np.max(err / np.maximum(tol[own], 1e-30)):.3g} of its bound"
    assert (np.abs(lse - want_lse)[own] <= tol_lse[own]).all()


SHAPES = [(2, 2, 64), (4, 2, 128), (3, 1, 192), (8, 2, 256)]
ROWS = [[1, 1], [13, 2]]   # few and many columns a KV head


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("span", [20, 28, 34, 40, 80])
def test_a_huge_scale_of_no_weight(gv, nh, nkv, hd, rows, span):
    """one position of a score 60 below the others' whose scale is 2^span times theirs, early, late, and in the one chunk
    or one of several"""
    lens = [90, 700]
    f = Filled(70, "i8", rows, lens, 32, nkv, hd)
    r = np.random.default_rng(71)
    scores, scales = [], []
    for n, at in zip(lens, (5, 400)):
        s = r.uniform(-1.0, 0.0, n)
        e = np.full(n, -6.0)
        s[at], e[at] = -60.0, span - 6.0
        scores.append(s)
        scales.append(e)
    vs = _spanned(f, 72, scores, scales, 8.0)
    _check(gv, f, "f32", nh, 8.0, vs)


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rise", ["up", "down", "any"])
def test_scores_and_scales_of_any_kind(gv, nh, nkv, hd, rows, kind, rise):
    """scores between -90 and 0 with scales of 2^-60 to 2^60: rising, falling or in any order, the larger scale now at the
    stronger, now at the weaker position"""
    lens = [260, 1300]
    f = Filled(73, "i8", rows, lens, 64, nkv, hd)
    r = np.random.default_rng(74)
    scores, scales = [], []
    for i, n in enumerate(lens):
        s = r.uniform(-90.0, 0.0, n)
        s = np.sort(s) if rise == "up" else np.sort(s)[::-1] if rise == "down" else s
        e = -s * 0.9 / np.log(2.0) - 60.0 if i == 0 else r.uniform(-60.0, 60.0, n)
        scores.append(s)
        scales.append(e)
    vs = _spanned(f, 75, scores, scales, 8.0)
    _check(gv, f, kind, nh, 8.0, vs)


@pytest.mark.parametrize("nh,hd,rows", [(4, 64, 3), (4, 256, 3), (16, 64, 5), (16, 128, 5), (16, 256, 5), (6, 192, 5)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_row_that_is_not_finite_is_not_made_finite(gv, nh, hd, rows, which, value):
    """a NaN or an infinity in a new row's key or value shows in what the cache then holds of that (position, KV head), and a
    NaN in the results of the rows that see it; other positions, KV heads and rows are as without it"""
    nkv = 2
    r = np.random.default_rng(76)
    q, k, v = (round_to(r.standard_normal((rows, h, hd)), "f32") for h in (nh, nkv, nkv))
    got = {}
    for bad in (False, True):
        f = Filled(77, "i8", [rows], [400], 32, nkv, hd)
        x = {"k": k.copy(), "v": v.copy()}
        if bad:
            x[which][1, 1, hd // 2 + 1] = value
        gv.paged_append(f.cache, f.batch, None, x["k"], x["v"])
        got[bad] = (f.cache.read("k"), f.cache.read("v"), *gv.paged_attention(f.cache, f.batch, q))
    p, s = f.place(0, 400 - rows + 1)
    n = "kv".index(which)
    assert not np.isfinite(got[True][n][p, 1, s]).any()
    for i in (0, 1):
        a, b = got[False][i].copy(), got[True][i].copy()
        if i == n:
            a[p, 1, s] = b[p, 1, s] = 0
        assert np.array_equal(a, b, equal_nan=True)
    half = nh // 2
    for i in (2, 3):
        assert np.array_equal(got[True][i][0], got[False][i][0])
        assert np.array_equal(got[True][i][:, :half], got[False][i][:, :half])
    if np.isnan(value):
        assert np.isnan(got[True][2][1:, half:]).all()
        assert np.isfinite(got[False][2]).all()


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("score", [3e7, 1e9, -1e9, 1e15])
def test_large_equal_scores(gv, nh, nkv, hd, rows, score):
    """positions of one and the same key, whatever the score's size: the plain mean of their values, of scales 1 to 2^20"""
    lens = [90, 700]
    f = Filled(78, "i8", rows, lens, 32, nkv, hd)
    r = np.random.default_rng(79)
    # (_spanned gives keys of at most 0 in dim 0: the query's sign makes the score's)
    vs = _spanned(f, 80, [np.full(n, -1.0) for n in lens], [r.uniform(0.0, 20.0, n) for n in lens], 1.0)
    T = f.batch.desc.n_rows
    q = np.zeros((T, nh, hd))
    q[..., 0] = -score
    out, lse = gv.paged_attention(f.cache, f.batch, round_to(q, "f32"), scale=1.0)
    for i, n in enumerate(lens):
        for t in range(f.start[i], f.start[i + 1]):
            seen = n - f.rows[i] + t - f.start[i] + 1
            for h in range(nh):
                v = f.sequence("v", i)[h // (nh // nkv), :seen]
                # every weight is 1: the scales' 22 bits (2^-21), the sums' roundings (fewer than 64 of 2^-24)
                tol = np.abs(v).mean(0) * 2.0 ** -17 + vs[np.isfinite(vs)].max() * 127 * 2.0 ** -36
                assert (np.abs(out[t, h] - v.mean(0)) <= tol).all(), (i, t, h)
    assert np.isfinite(lse).all()
