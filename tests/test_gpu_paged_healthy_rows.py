"""A sequence or row whose page, length, position, range or mask does not fit leaves the others as they would be: outputs read
back after the call that failed, not after a later one."""
import ctypes

import numpy as np
import pytest

from paged_ref import TYPES, Filled, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _attend(gv, f, dq, nh, hd, kind, ok):
    """out and lse (first filled with a pattern) of one call, whether it was told as in order or not"""
    T = f.batch.desc.n_rows
    size = 4 if kind == "f32" else 2
    out, lse = gv.DeviceBuffer.from_array(np.full(T * nh * hd * size, 0x5A, np.uint8)), \
        gv.DeviceBuffer.from_array(np.full(T * nh * 4, 0x5A, np.uint8))
    n = gv.lib.gv_paged_attention_workspace_bytes(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), nh)
    ws = gv.DeviceBuffer.from_array(np.full(max(1, n), 0xFF, np.uint8))   # (NaNs: what is not written must not be read)
    a = gv.GvAttentionRows(type=TYPES[kind], n_heads=nh, q=dq.ptr, q_row=nh * hd, out=out.ptr, out_row=nh * hd, lse=lse.ptr,
                           scale=hd ** -0.5)
    gv.check(gv.lib.gv_paged_attention(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), ctypes.byref(a), ws.ptr, n),
             "gv_paged_attention")
    assert gv.lib.gv_synchronize() == (0 if ok else -1)
    return out.download(np.uint8, (T, nh * hd * size)), lse.download(np.uint8, (T, nh * 4))


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f16")])
@pytest.mark.parametrize("nh,hd,rows,lens", [
    (2, 64, [1, 2, 1], [40, 70, 300]),            # few columns, one chunk and several
    (16, 64, [4, 9, 3], [40, 700, 300]),          # many columns in the same kernel
    (16, 128, [4, 9, 3], [1500, 900, 30]), (16, 256, [4, 9, 3], [1500, 900, 30])])
def test_attention(gv, cache, kind, nh, hd, rows, lens):
    f = Filled(90, cache, rows, lens, 16, 2, hd, n_rows=sum(rows) + 2)
    T = sum(rows) + 2
    q = round_to(np.random.default_rng(91).standard_normal((T, nh, hd)), kind)
    dq = gv._typed(q, TYPES[kind])
    base = _attend(gv, f, dq, nh, hd, kind, True)
    behind = slice(sum(rows), T)
    assert (base[0][behind] == 0x5A).all() and (base[1][behind] == 0x5A).all()
    bad_page, bad_first = f.pages.copy(), f.pages.copy()
    bad_page[1, (lens[1] - 1) // 16] = f.cache.desc.n_pages
    bad_first[1, 0] = -1
    long, short = np.array(lens), np.array(lens)
    long[1], short[1] = f.batch.desc.max_len + 1, rows[1] - 1
    past = f.start.copy()
    past[3] = T + 1
    for buf, good, planted, seq in ((2, f.pages, bad_page, 1), (2, f.pages, bad_first, 1), (1, f.lens, long, 1),
                                    (1, f.lens, short, 1), (0, f.start, past, 2)):
        f.batch.bufs[buf].upload(planted.astype(np.int32))
        got = _attend(gv, f, dq, nh, hd, kind, False)
        f.batch.bufs[buf].upload(good.astype(np.int32))
        for i in range(3):
            if i != seq:
                at = slice(f.start[i], f.start[i + 1])
                assert np.array_equal(got[0][at], base[0][at]) and np.array_equal(got[1][at], base[1][at]), (buf, i)
        if seq != 2:   # (rows behind the last sequence are its own where its end is past them)
            assert (got[0][behind] == 0x5A).all() and (got[1][behind] == 0x5A).all()
    again = _attend(gv, f, dq, nh, hd, kind, True)
    assert all(np.array_equal(x, y) for x, y in zip(again, base))


def test_attention_far_more_chunks_than_there_are(gv):
    """the units counted from the lengths: one sequence's length past max_len, one's page outside the pool"""
    n = 9
    rows, lens = np.ones(n, int), np.array([30, 17, 700, 1, 16, 33, 5, 99, 20])
    f = Filled(92, "f16", rows, lens, 16, 4, 64)
    top = 3 * (1 << 20) // n
    f.pages = np.concatenate([f.pages, np.full((n, -(-top // 16) - f.pages.shape[1]), -9, np.int32)], 1)
    f.batch = gv.PagedBatch(rows, lens, f.pages, max_len=top)
    q = np.random.default_rng(93).standard_normal((n, 8, 64)).astype(np.float32)
    dq = gv.DeviceBuffer.from_array(q)
    base = _attend(gv, f, dq, 8, 64, "f32", True)
    long = lens.copy()
    long[4] = top + 1
    pages = f.pages.copy()
    pages[2, 3] = 1 << 30
    for buf, good, planted, seq in ((1, lens, long, 4), (2, f.pages, pages, 2)):
        f.batch.bufs[buf].upload(planted.astype(np.int32))
        got = _attend(gv, f, dq, 8, 64, "f32", False)
        f.batch.bufs[buf].upload(good.astype(np.int32))
        others = np.arange(n) != seq
        assert np.array_equal(got[0][others], base[0][others]) and np.array_equal(got[1][others], base[1][others])


@pytest.mark.parametrize("cache", ["f16", "i8"])
@pytest.mark.parametrize("big", [False, True])
def test_append(gv, cache, big):
    """each call's own fresh rows: the healthy ones' keys, values (scales) and queries as from a call in order, nothing else
    of the cache written (few rows, and so many that a workgroup takes a whole row)"""
    rows, lens = ([700, 900, 3000], [700, 911, 3000]) if big else ([1, 2, 1], [40, 70, 30])
    nh, nkv, hd = 3, 2, 64
    T = sum(rows)
    f = Filled(94, cache, rows, lens, 16, nkv, hd)
    names = ("k", "v") + (("k_scale", "v_scale") if cache == "i8" else ())
    raw = lambda n: getattr(f.cache, n).download(np.uint8, (getattr(f.cache, n).nbytes,))   # noqa: E731
    clean = {n: raw(n) for n in names}
    angle = np.arange(3100)[:, None] * 1e4 ** (-np.arange(16) / 16)
    cos, sin = (gv.DeviceBuffer.from_array(g(angle).astype(np.float32)) for g in (np.cos, np.sin))
    seq = np.repeat(np.arange(3), rows)
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
    out = gv.DeviceBuffer(T * nh * hd * 4)

    def call(seed, n_positions, positions, ok):
        r = np.random.default_rng(seed)
        dev = [gv.DeviceBuffer.from_array(r.standard_normal((T, h, hd)).astype(np.float32)) for h in (nh, nkv, nkv)]
        for n in names:
            getattr(f.cache, n).upload(clean[n])
        out.upload(np.full(T * nh * hd, 7.0, np.float32))
        q, k, v = dev
        a = gv.GvAppendRows(type=gv.F32, n_heads=nh, q=q.ptr, q_row=nh * hd, q_head=hd, k=k.ptr, k_row=nkv * hd, k_head=hd,
                            v=v.ptr, v_row=nkv * hd, v_head=hd, eps=1e-6, rope_dim=32, cos=cos.ptr, sin=sin.ptr,
                            n_positions=n_positions, positions=positions.ptr if positions else None, q_type=gv.F32,
                            q_out=out.ptr, q_out_row=nh * hd)
        gv.check(gv.lib.gv_paged_append(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), ctypes.byref(a)), "gv_paged_append")
        assert gv.lib.gv_synchronize() == (0 if ok else -1)
        return {n: raw(n) for n in names}, out.download(np.float32, (T, nh, hd))

    def place(c, n, t):   # row t's bytes in array n of a cache's contents
        p, s = f.place(seq[t], pos[t])
        x = c[n].view(np.float32) if "scale" in n else c[n] if cache == "i8" else c[n].view(np.uint16)
        x = x.reshape((-1, nkv, 16) if "scale" in n else (-1, nkv, 16, hd))
        return x[p, :, s]

    pages = f.pages.copy()
    pages[1, (lens[1] - 1) // 16] = -1
    lost = (seq == 1) & (pos // 16 == (lens[1] - 1) // 16)
    short, long = np.array(lens), np.array(lens)
    short[1], long[0] = rows[1] - 1, max(lens) + 1
    past = f.start.copy()
    past[3] = T + 1
    far = gv.DeviceBuffer.from_array(np.where(seq == 2, 5000, pos).astype(np.int32))
    for i, (buf, planted, bad) in enumerate(((2, pages, lost), (1, short, seq == 1), (1, long, seq == 0), (0, past, seq == 2),
                                             (None, far, seq == 2))):
        want, want_q = call(100 + i, 3100, None, True)
        good = {0: f.start, 1: f.lens, 2: f.pages}.get(buf)
        if buf is not None:
            f.batch.bufs[buf].upload(planted.astype(np.int32))
        got, got_q = call(100 + i, 3100, far if buf is None else None, False)
        if buf is not None:
            f.batch.bufs[buf].upload(good.astype(np.int32))
        assert np.array_equal(got_q[~bad], want_q[~bad]) and (want_q[~bad] != 7.0).any(-1).all()
        for n in names:
            back = got[n].copy()
            for t in range(T):
                if not bad[t]:
                    assert np.array_equal(place(got, n, t), place(want, n, t)), (i, n, t)
                    assert not np.array_equal(place(got, n, t), place(clean, n, t)), (i, n, t)
            state = {n: back}
            for t in range(T):   # what is left once the rows' own places are put back is the cache as it was
                place(state, n, t)[...] = place(clean, n, t)
            assert np.array_equal(back, clean[n]), (i, n)


@pytest.mark.parametrize("rows,V", [(4, 3000), (40, 50000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_logits(gv, rows, V, in_place):
    """ranges and masks outside their arrays: the other rows' logits as from a call in order"""
    r = np.random.default_rng(95)
    x = r.standard_normal((rows, V)).astype(np.float32)
    lens = r.integers(1, 50, rows)
    begin = np.concatenate([[0], np.cumsum(lens)[:-1]])
    a = dict(tokens=r.integers(0, V, int(lens.sum())), begin=begin, end=begin + lens, generated=begin + lens // 3,
             bias_token=r.integers(0, V, 3 * rows), bias_begin=3 * np.arange(rows), bias_end=3 * np.arange(1, rows + 1),
             mask_of=r.integers(-1, 2, rows))
    a = {k: v.astype(np.int32) for k, v in a.items()}
    a.update({k: r.uniform(0.5, 1.5, rows).astype(np.float32) for k in ("repetition", "frequency", "presence")})
    a["bias_value"] = r.uniform(-5, 5, 3 * rows).astype(np.float32)
    a["masks"] = r.integers(0, 2 ** 32, (2, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)

    def call(b, ok):
        dev = {n: gv.DeviceBuffer.from_array(v) for n, v in b.items()}
        src = gv.DeviceBuffer.from_array(x)
        out = src if in_place else gv.DeviceBuffer.from_array(np.full((rows, V), 9.0, np.float32))
        rules = gv.GvLogitsRules(**{n: d.ptr for n, d in dev.items()}, n_tokens=len(b["tokens"]), n_biases=3 * rows, n_masks=2,
                                 ld_mask=(V + 31) // 32)
        gv.check(gv.lib.gv_process_logits(ctypes.byref(rules), src.ptr, gv.F32, V, rows, V, out.ptr, V), "gv_process_logits")
        assert gv.lib.gv_synchronize() == (0 if ok else -1)
        return out.download(np.float32, (rows, V))

    base = call(a, True)
    assert (base != x).any(1).all()
    for name, row, val in (("end", 1, len(a["tokens"]) + 1), ("begin", 1, -1), ("begin", 1, int(a["end"][1]) + 1),
                           ("bias_end", 2, 3 * rows + 1), ("bias_begin", 2, -3), ("mask_of", 3, 2)):
        b = {k: np.array(v) for k, v in a.items()}
        b[name][row] = val
        others = np.arange(rows) != row
        assert np.array_equal(call(b, False)[others], base[others]), name
