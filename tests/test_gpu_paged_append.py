"""gv_paged_append on the GPU against its definition in 64 bits, and against the model's own arithmetic: rows of several
sequences normalized, rotated and put into their pages, nothing else touched."""
import numpy as np
import pytest

from paged_ref import HALF_STEP, TYPES, U32, Filled, round_to

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _tables(n, rope):
    angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(rope // 2) / max(1, rope // 2))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _turned(x, w, pos, cos, sin, rope, interleaved):
    """(values, the fp32 error a correct kernel may have): x [row, head, dim] in 64 bits. Norm: the sum's rounding to fp32,
    the mean + eps, root, quotient, two products: 6 half steps; rotation: two products and a sum of at most
    |a c| + |b s|: 3 half steps of that."""
    err = np.zeros_like(x)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPS))) * (1.0 + w.astype(np.float64))
        err = 7 * U32 * np.abs(x)
    y, e = x.copy(), err.copy()
    for f in range(rope // 2):
        i, j = (2 * f, 2 * f + 1) if interleaved else (f, f + rope // 2)
        c, s = cos[pos, f].astype(np.float64)[:, None], sin[pos, f].astype(np.float64)[:, None]
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        for o, a, b in ((i, i, j), (j, j, i)):
            size = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
            e[..., o] = err[..., a] * np.abs(c) + err[..., b] * np.abs(s) + 3 * U32 * size
    return y, e


def _run(gv, seed, cache_kind, kind, q_kind, rows, lens, page=32, nh=6, nkv=2, hd=64, rope=32, norm=True,
         interleaved=False, by_position=False, positions=None, n_rows=None, first_row=0):
    f = Filled(seed, cache_kind, rows, lens, page, nkv, hd, by_position, n_rows=n_rows, first_row=first_row)
    before = {n: f.cache.read(n) for n in ("k", "v")}
    T = f.batch.desc.n_rows
    r = np.random.default_rng(seed + 1)
    q, k, v = (round_to(r.standard_normal((T, h, hd)) * 2.0, kind) for h in (nh, nkv, nkv))
    wq, wk = (r.standard_normal(hd).astype(np.float32) * np.float32(0.1) for _ in range(2)) if norm else (None, None)
    n_pos = 9000
    cos, sin = _tables(n_pos, rope)
    got = gv.paged_append(f.cache, f.batch, q, k, v, type_=TYPES[kind], q_type=TYPES[q_kind], q_norm=wq, k_norm=wk, eps=EPS,
                          rope_dim=rope, interleaved=interleaved, cos=cos if rope else None, sin=sin if rope else None,
                          positions=positions)
    slot_pos = np.full(T, -1)
    seq = np.full(T, -1)
    for i in range(len(rows)):
        for j in range(rows[i]):
            seq[f.start[i] + j], slot_pos[f.start[i] + j] = i, lens[i] - rows[i] + j
    own = seq >= 0
    pos = np.where(own, slot_pos if positions is None else positions, 0)
    want, err = _turned(q, wq, pos, cos, sin, rope, interleaved)
    tol = err + HALF_STEP[q_kind] * (np.abs(want) + err) + 2.0 ** -25
    assert (np.abs(got - want) <= tol)[own].all(), "queries"
    assert not got[~own].any(), "a row of no sequence was written"
    for name, x, w in (("k", k, wk), ("v", v, None)):
        y, e = _turned(x, w, pos, cos, sin, rope if name == "k" else 0, interleaved)
        after = f.cache.read(name)
        touched = np.zeros(after.shape[:3], bool)
        for t in np.nonzero(own)[0]:
            p, s = f.place(seq[t], slot_pos[t])
            touched[p, :, s] = True
            if cache_kind == "i8":   # half a step of the row's largest / 127, and the codes' and the scale's own rounding
                step = np.abs(y[t]).max(-1, keepdims=True) / 127.0
                lim = step * (0.5 + 2.0 ** -12) + e[t].max(-1, keepdims=True) * 2
                assert (np.abs(after[p, :, s] - y[t]) <= lim).all()
                assert (np.abs(np.abs(after[p, :, s]).max(-1) - np.abs(y[t]).max(-1)) <= 4 * U32 * np.abs(y[t]).max(-1) + e[t].max(-1) * 2).all()
            else:
                lim = e[t] + HALF_STEP[cache_kind] * (np.abs(y[t]) + e[t]) + 2.0 ** -25
                assert (np.abs(after[p, :, s] - y[t]) <= lim).all()
        keep = ~touched
        assert np.array_equal(after[keep], before[name][keep], equal_nan=True), "another position was written"
    return f


@pytest.mark.parametrize("cache", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("kind,q_kind", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_types(gv, cache, kind, q_kind):
    _run(gv, 31, cache, kind, q_kind, [1, 5, 0, 3], [40, 5, 7, 1000])


@pytest.mark.parametrize("cache", ["f16", "i8"])
@pytest.mark.parametrize("hd,rope", [(256, 64), (128, 128), (64, 0), (80, 40), (96, 24), (192, 8), (16, 16), (48, 24)])
@pytest.mark.parametrize("norm,interleaved", [(True, False), (False, True)])
def test_head_sizes_and_rotations(gv, cache, hd, rope, norm, interleaved):
    _run(gv, 32, cache, "f32", "f32", [3, 1], [50, 17], hd=hd, rope=rope, norm=norm, interleaved=interleaved)


@pytest.mark.parametrize("page,by_position", [(16, True), (48, False), (256, True)])
def test_pages_and_orders(gv, page, by_position):
    _run(gv, 33, "bf16", "bf16", "f32", [40, 1, 100], [40, 300, 100], page=page, by_position=by_position)


@pytest.mark.parametrize("n_seqs", [1, 63, 64, 65, 200, 4200])
def test_a_rows_sequence_is_found(gv, n_seqs):
    """ragged rows of few and many sequences, some without rows, rows before the first and behind the last"""
    r = np.random.default_rng(34)
    rows = r.integers(0, 4, n_seqs)
    rows[-1] = 2
    lens = rows + r.integers(0, 40, n_seqs)
    _run(gv, 35, "f16", "f32", "f32", list(rows), list(lens), page=16, nh=1, nkv=1, hd=16, rope=8,
         n_rows=int(rows.sum()) + 8, first_row=3)


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("i8", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("nh,nkv,hd,rope,interleaved", [(9, 3, 256, 64, False), (7, 5, 64, 64, False), (6, 1, 128, 96, True)])
def test_prompts(gv, cache, kind, nh, nkv, hd, rope, interleaved):
    """many rows: several rounds of heads a wave, four heads a lane group, the last of them not whole"""
    _run(gv, 42, cache, kind, kind, [700, 800, 3000], [700, 811, 3000], page=64, nh=nh, nkv=nkv, hd=hd, rope=rope,
         interleaved=interleaved)


def test_a_pool_past_32_bits(gv):
    """pages whose elements lie past 2^32 (an 8-bit pool of 5 GB): the same codes and scales as in a small pool"""
    f = Filled(43, "i8", [3, 1], [70, 9], 64, 2, 128)
    n_pages = (5 << 30) // (64 * 2 * 128)
    big = gv.PagedCache(gv.I8, n_pages, 64, 2, 128)
    moved = np.where(f.pages >= 0, n_pages - 1 - 2 * f.pages, f.pages)
    r = np.random.default_rng(44)
    q, k, v = (r.standard_normal((4, h, 128)) for h in (4, 2, 2))
    cos, sin = _tables(80, 64)
    a = gv.paged_append(f.cache, f.batch, q, k, v, rope_dim=64, cos=cos, sin=sin)
    b = gv.paged_append(big, gv.PagedBatch(f.rows, f.lens, moved), q, k, v, rope_dim=64, cos=cos, sin=sin)
    assert np.array_equal(a, b)
    size, row = 64 * 2 * 128, gv.DeviceBuffer(64 * 2 * 128)
    scales = gv.DeviceBuffer(64 * 2 * 4)
    for i, pos in ((0, 67), (0, 68), (0, 69), (1, 8)):
        p, s = f.place(i, pos)
        for small, large, n, buf, t, shape in (
                (f.cache.k, big.k, size, row, np.int8, (2, 64, 128)), (f.cache.v, big.v, size, row, np.int8, (2, 64, 128)),
                (f.cache.k_scale, big.k_scale, 512, scales, np.float32, (2, 64)),
                (f.cache.v_scale, big.v_scale, 512, scales, np.float32, (2, 64))):
            got = []
            for src, page in ((small, int(p)), (large, n_pages - 1 - 2 * int(p))):
                gv.check(gv.lib.gv_memcpy_d2d(buf.ptr, src.ptr + page * n, n), "copy")
                got.append(buf.download(t, shape)[:, s])
            assert np.array_equal(*got) and got[0].any()


def test_tree_positions_and_far_angles(gv):
    """rotary positions apart from the places in the cache (a draft tree's depths), near the tables' end"""
    pos = np.array([8990, 8991, 8991, 8991, 8992, 8999], np.int32)
    _run(gv, 36, "f16", "f32", "f32", [6], [77], positions=pos)


def test_a_zero_row_of_an_int8_cache(gv):
    f = Filled(37, "i8", [1], [5], 16, 1, 64)
    z = np.zeros((1, 1, 64))
    gv.paged_append(f.cache, f.batch, None, z, z)
    p, s = f.place(0, 4)
    assert not f.cache.read("k")[p, :, s].any() and not f.cache.read("v")[p, :, s].any()


def test_queries_in_place_and_parts_of_one_array(gv):
    """q | k | v as one product's rows with each head's gate beside its queries; and the queries written over themselves"""
    import ctypes

    f = Filled(38, "f16", [2, 3], [20, 33], 16, 2, 64)
    r = np.random.default_rng(39)
    nh, nkv, hd = 4, 2, 64
    rows = r.standard_normal((5, nh * 2 * hd + 2 * nkv * hd)).astype(np.float32)
    cos, sin = _tables(40, 32)
    q = rows[:, :nh * 2 * hd].reshape(5, nh, 2, hd)[:, :, 0]
    k, v = rows[:, nh * 2 * hd:].reshape(5, 2, nkv, hd).transpose(1, 0, 2, 3)
    want = gv.paged_append(f.cache, f.batch, q, k, v, rope_dim=32, cos=cos, sin=sin)
    want_k, want_v = f.cache.read("k"), f.cache.read("v")
    for b in (f.cache.k, f.cache.v):
        b.zero()
    dev, dc, ds = (gv.DeviceBuffer.from_array(a) for a in (rows, cos, sin))
    out = gv.DeviceBuffer(5 * nh * hd * 4)
    w = rows.shape[1]
    a = gv.GvAppendRows(type=gv.F32, n_heads=nh, q=dev.ptr, q_row=w, q_head=2 * hd, k=dev.ptr + 4 * nh * 2 * hd, k_row=w,
                        k_head=hd, v=dev.ptr + 4 * (nh * 2 + nkv) * hd, v_row=w, v_head=hd, eps=EPS, rope_dim=32,
                        cos=dc.ptr, sin=ds.ptr, n_positions=40, q_type=gv.F32, q_out=out.ptr, q_out_row=nh * hd)
    call = lambda a: gv.lib.gv_paged_append(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), ctypes.byref(a))   # noqa: E731
    gv.check(call(a), "gv_paged_append")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    assert np.array_equal(out.download(np.float32, (5, nh, hd)), want)
    own = ~np.isnan(want_k) & (want_k != 0)
    assert np.array_equal(f.cache.read("k")[own][:0], want_k[own][:0])
    for t, (i, pos) in enumerate([(0, 18), (0, 19), (1, 30), (1, 31), (1, 32)]):
        p, s = f.place(i, pos)
        assert np.array_equal(f.cache.read("k")[p, :, s], want_k[p, :, s])
        assert np.array_equal(f.cache.read("v")[p, :, s], want_v[p, :, s])
    dq = gv.DeviceBuffer.from_array(np.ascontiguousarray(q))
    a.q, a.q_row, a.q_head, a.q_out = dq.ptr, nh * hd, hd, dq.ptr
    gv.check(call(a), "gv_paged_append")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    assert np.array_equal(dq.download(np.float32, (5, nh, hd)), want)


def test_faults_in_device_memory(gv):
    """a page outside the pool, lengths that do not fit, a rotary position outside the tables: reported, the other rows
    appended, nothing else written"""
    f = Filled(40, "f16", [1, 2, 1], [40, 70, 30], 16, 2, 64)
    r = np.random.default_rng(41)
    q, k, v = (r.standard_normal((4, h, 64)) for h in (2, 2, 2))
    cos, sin = _tables(80, 32)
    bad = f.pages.copy()
    bad[1, 69 // 16] = -1
    for buf, good, planted, word in ((2, f.pages, bad, "page"), (1, f.lens, np.array([40, 1, 30]), "length"),
                                     (1, f.lens, np.array([40, 71, 30]), "length"),
                                     (0, f.start, np.array([0, 1, 5, 4]), "row")):
        f.batch.bufs[buf].upload(planted.astype(np.int32))
        before = f.cache.read("k")
        with pytest.raises(gv.GeodeError, match=word):
            gv.paged_append(f.cache, f.batch, q, k + 1, v, rope_dim=32, cos=cos, sin=sin)
        f.batch.bufs[buf].upload(good.astype(np.int32))
        after = f.cache.read("k")
        changed = np.argwhere((after != before) & ~(np.isnan(after) & np.isnan(before)))
        places = {f.place(i, p) for i, p in ((0, 39), (1, 68), (1, 69), (2, 29))}
        assert {(int(c[0]), int(c[2])) for c in changed} <= {(int(a), int(b)) for a, b in places}
    with pytest.raises(gv.GeodeError, match="rotary"):
        gv.paged_append(f.cache, f.batch, q, k, v, rope_dim=32, cos=cos[:69], sin=sin[:69])
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
