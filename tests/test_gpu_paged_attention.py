"""gv_paged_attention on the GPU against its definition in 64 bits: types, head layouts, lengths around tiles and chunks,
pages that end inside them, both orders of a page, chains and trees, rows that see nothing, values that a row must not see."""
import numpy as np
import pytest

from paged_ref import HALF_STEP, TYPES, Filled, attention, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _queries(seed, T, nh, hd, kind, sigma=1.5):
    return round_to(np.random.default_rng(seed).standard_normal((T, nh, hd)) * sigma, kind)


def _check(gv, f, q, kind, scale=None, visible=None):
    scale = float(np.float32(q.shape[2] ** -0.5 if scale is None else scale))
    out, lse = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind], scale=scale, visible=visible)
    want, want_lse, tol, tol_lse = attention(f, q, scale, kind, visible)
    own = np.zeros(q.shape[0], bool)
    for i in range(len(f.rows)):
        own[f.start[i]:f.start[i + 1]] = True
    assert not out[~own].any() and not lse[~own].any(), "a row of no sequence was written"
    assert np.isfinite(out[own]).all()
    err = np.abs(out - want)[own]
    assert (err <= tol[own]).all(), f"out off by {np.max(err / np.maximum(tol[own], 1e-30)):.2f} of its bound"
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(lse)[own], empty[own])
    some = own[:, None] & ~empty
    assert (np.abs(lse[some] - want_lse[some]) <= tol_lse[some]).all(), "log-sum-exp"
    return out, lse


COMBOS = [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("i8", "f16"), ("i8", "bf16"), ("i8", "f32")]


@pytest.mark.parametrize("cache,kind", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 256), (8, 8, 64), (6, 2, 128), (3, 1, 80), (5, 5, 16), (4, 2, 192)])
def test_one_token(gv, cache, kind, nh, nkv, hd):
    f = Filled(1, cache, [1] * 7, [1, 16, 17, 33, 128, 129, 300], 32, nkv, hd)
    _check(gv, f, _queries(2, 7, nh, hd, kind), kind)


@pytest.mark.parametrize("cache,kind", COMBOS)
@pytest.mark.parametrize("page,by_position", [(16, False), (48, True), (64, False), (256, True)])
def test_pages_and_orders(gv, cache, kind, page, by_position):
    f = Filled(3, cache, [1, 3, 0, 5], [257, 40, 9, 511], page, 2, 64, by_position, n_rows=12)
    _check(gv, f, _queries(4, 12, 8, 64, kind), kind)


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("lens", [[4097], [512, 513, 1024, 1025], [1, 2000], [31, 5, 700, 2049, 1]])
def test_lengths_around_chunks(gv, cache, kind, lens):
    f = Filled(5, cache, [1] * len(lens), lens, 64, 2, 128)
    _check(gv, f, _queries(6, len(lens), 4, 128, kind), kind)


@pytest.mark.parametrize("cache,kind", [("f16", "f16"), ("f16", "f32"), ("bf16", "f32"), ("i8", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("rows", [2, 5, 17, 32])
def test_chains(gv, cache, kind, rows):
    f = Filled(7, cache, [rows, 1, rows - 1], [rows + 200, 150, rows - 1], 32, 2, 256)
    _check(gv, f, _queries(8, 2 * rows, 16, 256, kind), kind)


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f16")])
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_tree_and_rows_that_see_nothing(gv, cache, kind, hd):
    """a row's own bits alone decide what it sees of its sequence's rows: a tree, a row that does not see itself, and in a
    sequence without context rows that see nothing"""
    f = Filled(9, cache, [6, 4, 32], [100, 4, 300], 16, 2, hd)
    r = np.random.default_rng(10)
    vis = np.concatenate([[1, 3, 5, 9, 0, 35], [1, 0, 4, 0], r.integers(0, 2 ** 32, 32, dtype=np.uint64)]).astype(np.uint32)
    out, lse = _check(gv, f, _queries(11, 42, 8, hd, kind), kind, visible=vis)
    assert not out[7].any() and not out[9].any() and np.isneginf(lse[[7, 9]]).all()


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("nh,nkv,hd", [(2, 2, 64), (8, 2, 64), (2, 2, 256), (8, 2, 128), (16, 2, 256), (6, 2, 192)])
def test_trees_across_chunks(gv, cache, kind, nh, nkv, hd):
    """a sequence's own rows on both sides of a chunk's end, chunks of which a row sees nothing but single positions"""
    f = Filled(51, cache, [32, 5, 12, 1], [650, 900, 1029, 641], 48, nkv, hd)
    r = np.random.default_rng(52)
    vis = r.integers(0, 2 ** 32, 50, dtype=np.uint64).astype(np.uint32)
    vis[[3, 33, 40]] = 0
    _check(gv, f, _queries(53, 50, nh, hd, kind), kind, visible=vis)


@pytest.mark.parametrize("cache,kind", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("nh,hd", [(4, 64), (16, 64), (4, 128), (16, 128), (16, 96), (4, 256), (16, 256), (16, 192)])
def test_values_a_row_does_not_see(gv, cache, kind, nh, hd):
    """NaNs and infinities in later rows' keys and values reach the rows that see them and no others (few and many columns
    a KV head)"""
    f = Filled(12, cache, [6, 5], [70, 5], 16, 2, hd)
    clean = {n: f.host[n].copy() for n in ("k", "v")}
    q = _queries(13, 11, nh, hd, kind)
    scale = float(np.float32(hd ** -0.5))
    base, _ = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind], scale=scale)
    for name, val in (("v", np.nan), ("v", np.inf), ("k", np.nan), ("v", -np.inf)):
        f.host[name] = clean[name].copy()
        for i, pos in ((0, 67), (1, 3)):   # the sequences' rows 3 and 3
            p, slot = f.place(i, pos)
            f.host[name][p, 1, slot, 5] = val
        f.rewrite()
        got, _ = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind], scale=scale)
        blind = np.array([0, 1, 2, 6, 7, 8])        # rows before it
        assert np.array_equal(got[blind], base[blind]), (name, val)
        sees = np.array([3, 4, 5, 9, 10])
        assert np.array_equal(got[sees][:, :nh // 2], base[sees][:, :nh // 2])     # the other KV head's query heads
        if name == "v":
            others = np.arange(hd) != 5
            a, b = got[sees][:, nh // 2:, others], base[sees][:, nh // 2:, others]
            assert (np.abs(a - b) <= 2.0 ** -16 + 2 * HALF_STEP[kind] * np.abs(b)).all()   # (added up in another order)
            assert not np.isfinite(got[sees][:, nh // 2:, 5]).any()
        else:
            assert np.isnan(got[sees][:, nh // 2:]).all()
        f.host[name] = clean[name]
    f.rewrite()


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("nh,hd", [(4, 64), (16, 64), (4, 128), (16, 128), (4, 256), (16, 256)])
def test_nan_keys_everywhere_in_a_chunk(gv, cache, kind, nh, hd):
    """positions whose keys are all NaN, a whole chunk of them or every one a row sees: the rows that see them get NaNs, also
    where the chunks are joined"""
    f = Filled(45, cache, [3, 3, 3], [2000, 2000, 300], 16, 2, hd)
    for i, lo, hi in ((0, 512, 1536), (2, 0, 300)):
        for pos in range(lo, hi):
            p, s = f.place(i, pos)
            f.host["k"][p, 0, s] = np.nan
    f.rewrite()
    out, lse = gv.paged_attention(f.cache, f.batch, _queries(46, 9, nh, hd, kind), type_=TYPES[kind])
    half = nh // 2
    for rows, finite in ((slice(0, 3), False), (slice(3, 6), True), (slice(6, 9), False)):
        for x in (out[rows][:, :half], lse[rows][:, :half]):
            assert np.isfinite(x).all() if finite else np.isnan(x).all()
        assert np.isfinite(out[rows][:, half:]).all() and np.isfinite(lse[rows][:, half:]).all()


@pytest.mark.parametrize("cache,kind", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 256), (12, 1, 128), (9, 3, 96), (10, 2, 192), (8, 2, 64), (3, 1, 16)])
def test_many_columns(gv, cache, kind, nh, nkv, hd):
    """chains of up to 13 rows: columns that fill one, two and several column tiles, ragged; several chunks"""
    f = Filled(30, cache, [13, 4, 0, 7, 1], [900, 4, 0, 77, 130], 48, nkv, hd, n_rows=26)
    _check(gv, f, _queries(31, 26, nh, hd, kind), kind)


@pytest.mark.parametrize("n_seqs,by_position", [(9, False), (70, False), (300, False), (9, True), (70, True)])
@pytest.mark.parametrize("cache,kind,rows,nh,nkv,hd", [
    ("f16", "f32", 1, 8, 4, 64), ("bf16", "bf16", 1, 4, 4, 128), ("i8", "f16", 1, 4, 4, 256), ("f16", "f16", 2, 4, 4, 80),
    ("bf16", "f32", 1, 4, 4, 192), ("f16", "f32", 6, 16, 4, 64), ("i8", "f32", 6, 16, 4, 16)])
def test_far_longer_cache_than_sequences(gv, n_seqs, by_position, cache, kind, rows, nh, nkv, hd):
    """a page table for many positions of which most sequences hold few: far more chunks by max_len than there are"""
    r = np.random.default_rng(32)
    rows = np.minimum(r.integers(0, rows + 1, n_seqs), rows)
    lens = np.maximum(rows, r.integers(1, 40, n_seqs))
    rows[n_seqs // 2], lens[n_seqs // 2] = 1, 700
    f = Filled(33, cache, rows, lens, 16, nkv, hd, by_position)
    top = 3 * (1 << 20) // n_seqs
    f.pages = np.concatenate([f.pages, np.full((n_seqs, -(-top // 16) - f.pages.shape[1]), -9, np.int32)], 1)
    f.batch = gv.PagedBatch(rows, lens, f.pages, max_len=top)
    q = _queries(34, int(f.start[-1]), nh, hd, kind)
    _check(gv, f, q, kind)
    lens = lens.copy()
    lens[n_seqs - 1] = top + 1
    f.batch.bufs[1].upload(lens.astype(np.int32))
    with pytest.raises(gv.GeodeError, match="length"):
        gv.paged_attention(f.cache, f.batch, q)


@pytest.mark.parametrize("nh,hd", [(4, 64), (4, 128), (8, 128), (8, 256)])
def test_an_int8_scale_a_row_does_not_see(gv, nh, hd):
    """a draft's NaN, infinite or huge scale leaves the rows that do not see it as they were"""
    f = Filled(14, "i8", [4], [40], 16, 1, hd)
    q = _queries(15, 4, nh, hd, "f32")
    base, _ = gv.paged_attention(f.cache, f.batch, q)
    sc = f.cache.v_scale.download(np.float32, f.cache.scale_shape)
    p, slot = f.place(0, 38)
    for val in (np.nan, np.inf, 1e30):
        bad = sc.copy()
        bad[p, 0, slot] = val
        f.cache.v_scale.upload(bad)
        got, _ = gv.paged_attention(f.cache, f.batch, q)
        assert np.array_equal(got[:2], base[:2]), val


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "f32"), ("i8", "f32"), ("f16", "f16")])
def test_large_scores(gv, cache, kind):
    """scores of thousands: the weights stay those of the scores' differences"""
    f = Filled(16, cache, [2, 1], [90, 700], 32, 1, 128)
    _check(gv, f, _queries(17, 3, 4, 128, kind, sigma=200.0), kind, scale=1.0)


@pytest.mark.parametrize("factor", [1e-6, 1.0, 1e6])
def test_queries_of_any_size(gv, factor):
    """fp32 queries far outside fp16's range over an fp16 and an int8 cache, the score's factor making up for it"""
    for cache in ("f16", "i8"):
        f = Filled(18, cache, [1, 2], [50, 260], 32, 1, 64)
        q = _queries(19, 3, 2, 64, "f32") * np.float64(np.float32(factor))
        q = round_to(q, "f32")
        _check(gv, f, q, "f32", scale=0.125 / factor)


def test_many_weak_positions(gv):
    """one strong position and thousands of weak ones that together weigh as much"""
    f = Filled(20, "f16", [1], [6000], 64, 1, 64)
    k = f.host["k"]
    k[~np.isnan(k)] = 0.0
    p, slot = f.place(0, 1234)
    k[p, 0, slot, 0] = 8.0
    f.rewrite()
    q = np.zeros((1, 2, 64))
    q[0, :, 0] = np.log(6000.0) / 8.0
    _check(gv, f, round_to(q, "f32"), "f32", scale=1.0)


def test_equal_calls_give_equal_bits(gv):
    f = Filled(21, "bf16", [3, 1, 5], [1500, 9, 640], 64, 2, 128)
    q = _queries(22, 9, 16, 128, "f32")
    a = gv.paged_attention(f.cache, f.batch, q)
    for _ in range(3):
        b = gv.paged_attention(f.cache, f.batch, q)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_calls_share_a_workspace(gv):
    """one call after the other in one workspace, nothing waited for in between: what each gives alone; and nothing behind
    the bytes that were asked for is written"""
    import ctypes

    nh, hd = 16, 128
    todo = []
    for seed, lens, rows in ((40, [3000], [1]), (41, [900, 20, 700], [4, 3, 1]), (42, [5000, 1], [2, 1])):
        f = Filled(seed, "f16", rows, lens, 32, 2, hd)
        q = _queries(seed, sum(rows), nh, hd, "f32")
        todo.append((f, q, gv.paged_attention(f.cache, f.batch, q)))
    need = [gv.lib.gv_paged_attention_workspace_bytes(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), nh)
            for f, _, _ in todo]
    most = max(need)
    ws = gv.DeviceBuffer(most + 4096)
    ws.upload(np.full(most + 4096, 0x5A, np.uint8))
    runs = []
    for f, q, _ in todo * 2:
        dq = gv.DeviceBuffer.from_array(q.astype(np.float32))
        out, lse = gv.DeviceBuffer(q.size * 4), gv.DeviceBuffer(q.shape[0] * nh * 4)
        runs.append((dq, out, lse))
        a = gv.GvAttentionRows(type=gv.F32, n_heads=nh, q=dq.ptr, q_row=nh * hd, out=out.ptr, out_row=nh * hd, lse=lse.ptr,
                               scale=hd ** -0.5)
        gv.check(gv.lib.gv_paged_attention(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), ctypes.byref(a), ws.ptr,
                                           most), "gv_paged_attention")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    for (f, q, (want, want_lse)), (_, out, lse) in zip(todo * 2, runs):
        assert np.array_equal(out.download(np.float32, want.shape), want)
        assert np.array_equal(lse.download(np.float32, want_lse.shape), want_lse)
    assert (ws.download(np.uint8, (most + 4096,))[most:] == 0x5A).all()


def test_calls_of_several_threads(gv):
    """calls of several host threads on data and workspaces of their own"""
    from concurrent.futures import ThreadPoolExecutor

    todo = []
    for seed, cache, hd in ((47, "f16", 64), (48, "bf16", 128), (49, "i8", 256), (50, "f16", 80)):
        f = Filled(seed, cache, [1, 7], [1500, 300], 32, 2, hd)
        q = _queries(seed, 8, 16, hd, "f32")
        todo.append((f, q, gv.paged_attention(f.cache, f.batch, q)))
    with ThreadPoolExecutor(4) as pool:
        for got, (_, _, want) in zip(pool.map(lambda t: gv.paged_attention(t[0].cache, t[0].batch, t[1]), todo * 6), todo * 6):
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_rows_before_and_behind_the_sequences(gv):
    f = Filled(23, "f16", [2, 1], [30, 600], 32, 2, 64, n_rows=9, first_row=2)
    _check(gv, f, _queries(24, 9, 4, 64, "f32"), "f32")


def test_faults_in_device_memory(gv):
    """a page outside the pool, a length past max_len, descending row starts: reported by the next synchronize, the other
    sequences as without them"""
    f = Filled(25, "f16", [1, 2, 1], [40, 70, 300], 16, 2, 64)
    q = _queries(26, 4, 4, 64, "f32")
    base, _ = gv.paged_attention(f.cache, f.batch, q)
    bad = f.pages.copy()
    bad[1, 2] = f.cache.desc.n_pages
    for buf, good, planted, word in ((2, f.pages, bad, "page"), (1, f.lens, np.array([40, 70, 301]), "length"),
                                     (1, f.lens, np.array([0, 70, 300]), "length"),
                                     (0, f.start, np.array([0, 1, 0, 4]), "row")):
        f.batch.bufs[buf].upload(planted.astype(np.int32))
        with pytest.raises(gv.GeodeError, match=word):
            gv.paged_attention(f.cache, f.batch, q)
        f.batch.bufs[buf].upload(good.astype(np.int32))
        gv.check(gv.lib.gv_synchronize(), "gv_synchronize")   # (reported once)
    f.batch.bufs[2].upload(bad)
    try:
        gv.paged_attention(f.cache, f.batch, q)
    except gv.GeodeError:
        pass
    f.batch.bufs[2].upload(f.pages)
    got, _ = gv.paged_attention(f.cache, f.batch, q)
    assert np.array_equal(got, base)


def test_a_pool_past_32_bits(gv):
    """pages whose elements lie past 2^32 (an 8-bit pool of 5 GB): the same results as from a small pool"""
    f = Filled(27, "i8", [1, 2], [100, 200], 64, 2, 128)
    page_elems = 64 * 2 * 128
    n_pages = (5 << 30) // page_elems
    big = gv.PagedCache(gv.I8, n_pages, 64, 2, 128)
    moved = f.pages.copy()
    for i in range(2):
        for p in range(-(-int(f.lens[i]) // 64)):
            old, new = int(f.pages[i, p]), n_pages - 1 - 2 * int(f.pages[i, p])
            moved[i, p] = new
            for a, b, size in ((f.cache.k, big.k, page_elems), (f.cache.v, big.v, page_elems),
                               (f.cache.k_scale, big.k_scale, 2 * 64 * 4), (f.cache.v_scale, big.v_scale, 2 * 64 * 4)):
                gv.check(gv.lib.gv_memcpy_d2d(b.ptr + new * size, a.ptr + old * size, size), "copy")
    q = _queries(28, 3, 8, 128, "f32")
    base = gv.paged_attention(f.cache, f.batch, q)
    got = gv.paged_attention(big, gv.PagedBatch(f.rows, f.lens, moved), q)
    assert np.array_equal(base[0], got[0]) and np.array_equal(base[1], got[1])
