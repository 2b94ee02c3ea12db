"""The strides that the paged calls' descriptions allow beside dense arrays, and the joining of few, some and many chunks."""
import ctypes

import numpy as np
import pytest

from paged_ref import TYPES, Filled, attention, round_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _strided(gv, f, page_stride, head_stride, pos_stride, v_at):
    """a copy of a Filled's dense cache [page][head][position][dim] in one allocation of other strides (elements), values
    v_at elements behind the keys, poison between: (description, buffer, its bytes, the index of every element)"""
    d, kind = f.cache.desc, f.kind
    es = 1 if kind == "i8" else 2
    p, h, s, x = np.ix_(range(d.n_pages), range(d.n_kv_heads), range(d.page_size), range(d.head_dim))
    at = p * page_stride + h * head_stride + s * pos_stride + x
    raw = np.full(int(at.max()) + 1 + v_at, -1, np.int8 if es == 1 else np.int16)   # (0xFFFF: a NaN)
    for name, off in (("k", 0), ("v", v_at)):
        raw[at + off] = getattr(f.cache, name).download(raw.dtype, at.shape)
    buf = gv.DeviceBuffer.from_array(raw)
    kv = gv.GvPagedKv(d.type, d.n_kv_heads, d.head_dim, d.page_size, d.n_pages, buf.ptr, buf.ptr + v_at * es, d.k_scale, d.v_scale,
                      page_stride, head_stride, pos_stride)
    return kv, buf, raw, at


def _layouts(nkv, page, hd):
    n = nkv * page * hd
    return {
        "values behind their page's keys": (2 * n, page * hd, hd, n),
        "the same by position": (2 * n, hd, nkv * hd, n),
        "a head's keys beside its values": (2 * n, 2 * page * hd, hd, page * hd),
        "a position's keys beside its values": (2 * n, hd, 2 * nkv * hd, nkv * hd),
        "everything padded": (nkv * (page * (hd + 16) + 48) + 112, page * (hd + 16) + 48, hd + 16, 1 << 22),
    }


@pytest.mark.parametrize("layout", list(_layouts(1, 16, 16)))
@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f16")])
@pytest.mark.parametrize("nh,nkv,hd,rows,lens", [(6, 3, 64, [1, 3, 2], [70, 300, 2]), (16, 2, 128, [5, 1, 13], [300, 40, 700]),
                                                 (3, 3, 80, [1, 1, 1], [129, 1, 50]), (16, 2, 256, [5, 1, 13], [300, 40, 700])])
def test_strides(gv, layout, cache, kind, nh, nkv, hd, rows, lens):
    """the dense cache's bits from other layouts, with wider rows of queries and results; then rows appended to both"""
    page, T, pad = 32, sum(rows), 24
    f = Filled(110, cache, rows, lens, page, nkv, hd)
    kv, buf, raw, at = _strided(gv, f, *_layouts(nkv, page, hd)[layout])
    q = round_to(np.random.default_rng(111).standard_normal((T, nh, hd)), kind)
    want = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind])
    n = gv.lib.gv_paged_attention_workspace_bytes(ctypes.byref(kv), ctypes.byref(f.batch.desc), nh)
    ws = gv.DeviceBuffer(n)
    wide = np.full((T, nh * hd + pad), np.nan, np.float32)
    wide[:, :nh * hd] = q.reshape(T, -1)
    dq, out = gv._typed(wide, TYPES[kind]), gv._typed(np.full(wide.shape, 5.0), TYPES[kind])
    a = gv.GvAttentionRows(type=TYPES[kind], n_heads=nh, q=dq.ptr, q_row=nh * hd + pad, out=out.ptr, out_row=nh * hd + pad,
                           scale=hd ** -0.5)
    gv.check(gv.lib.gv_paged_attention(ctypes.byref(kv), ctypes.byref(f.batch.desc), ctypes.byref(a), ws.ptr, n), "gv_paged_attention")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    got = gv._from_bits(out.download(gv._NP_TYPE[TYPES[kind]], wide.shape), TYPES[kind])
    assert np.array_equal(got[:, :nh * hd].reshape(T, nh, hd), want[0]) and (got[:, nh * hd:] == 5.0).all()

    r = np.random.default_rng(112)
    k, v = (r.standard_normal((T, nkv, hd)).astype(np.float32) for _ in range(2))
    scales = [(s, s.download(np.uint8, (s.nbytes,))) for s in (f.cache.k_scale, f.cache.v_scale) if s is not None]
    dense = gv.paged_append(f.cache, f.batch, np.zeros((T, 1, hd)), k, v)
    assert not dense.any()
    after = {n: getattr(f.cache, n).download(raw.dtype, at.shape) for n in ("k", "v")}
    new_scales = [s.download(np.uint8, b.shape) for s, b in scales]
    for s, b in scales:
        s.upload(b)
    rows_kv = np.full((T, nkv, 2, hd + 4), np.nan, np.float32)   # a head's key beside its value, padded
    rows_kv[:, :, 0, :hd], rows_kv[:, :, 1, :hd] = k, v
    dr, w = gv.DeviceBuffer.from_array(rows_kv), 2 * (hd + 4)
    a = gv.GvAppendRows(type=gv.F32, k=dr.ptr, k_row=nkv * w, k_head=w, v=dr.ptr + 4 * (hd + 4), v_row=nkv * w, v_head=w, eps=1e-6)
    gv.check(gv.lib.gv_paged_append(ctypes.byref(kv), ctypes.byref(f.batch.desc), ctypes.byref(a)), "gv_paged_append")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    for name, off in (("k", 0), ("v", _layouts(nkv, page, hd)[layout][3])):
        raw[at + off] = after[name]
    assert np.array_equal(buf.download(raw.dtype, raw.shape), raw)
    for (s, _), x in zip(scales, new_scales):
        assert np.array_equal(s.download(np.uint8, x.shape), x)


def test_positions_as_far_apart_as_allowed(gv):
    """strides of just below 2^24 elements between positions: a page's last position lies 480 MB behind its first"""
    nkv, page, hd = 2, 16, 64
    f = Filled(113, "f16", [2], [20], page, nkv, hd, spare=0)
    step = (1 << 24) - 16
    size = 2 * ((2 * page - 1) * step + nkv * hd)
    bufs = {n: gv.DeviceBuffer(size) for n in ("k", "v")}
    for n, b in bufs.items():
        x = getattr(f.cache, n).download(np.uint16, (2, nkv, page, hd))
        for p in range(2):
            for s in range(page):
                b.upload(np.ascontiguousarray(x[p, :, s]), 2 * (p * page + s) * step)
    kv = gv.GvPagedKv(gv.F16, nkv, hd, page, 2, bufs["k"].ptr, bufs["v"].ptr, None, None, page * step, hd, step)
    q = np.random.default_rng(114).standard_normal((2, 4, hd)).astype(np.float32)
    want, _ = gv.paged_attention(f.cache, f.batch, q)
    dq, out = gv.DeviceBuffer.from_array(q), gv.DeviceBuffer(q.nbytes)
    a = gv.GvAttentionRows(type=gv.F32, n_heads=4, q=dq.ptr, q_row=4 * hd, out=out.ptr, out_row=4 * hd, scale=hd ** -0.5)
    gv.check(gv.lib.gv_paged_attention(ctypes.byref(kv), ctypes.byref(f.batch.desc), ctypes.byref(a), None, 0), "gv_paged_attention")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    assert np.array_equal(out.download(np.float32, q.shape), want)
    rows = np.random.default_rng(115).standard_normal((2, 2, nkv, hd)).astype(np.float32)
    dr = gv.DeviceBuffer.from_array(rows)
    b = gv.GvAppendRows(type=gv.F32, k=dr.ptr, k_row=nkv * hd, k_head=hd, v=dr.ptr + rows[0].nbytes, v_row=nkv * hd, v_head=hd)
    gv.check(gv.lib.gv_paged_append(ctypes.byref(kv), ctypes.byref(f.batch.desc), ctypes.byref(b)), "gv_paged_append")
    for x, name in zip(rows, ("k", "v")):
        for t, pos in enumerate((18, 19)):
            p, s = f.place(0, pos)
            got = bufs[name].download(np.uint16, (nkv, hd), 2 * (int(p) * page + int(s)) * step)
            assert np.array_equal(got, x[t].astype(np.float16).view(np.uint16))


@pytest.mark.parametrize("cache,kind", [("f16", "f32"), ("bf16", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("nh,hd,rows", [(2, 64, [1, 1, 1, 1]), (2, 128, [1, 2, 1, 1]), (20, 64, [1, 1, 2, 1]), (20, 128, [2, 1, 1, 1])])
def test_few_some_and_many_chunks_joined(gv, cache, kind, nh, hd, rows):
    """sequences of two chunks to some hundred in one batch"""
    f = Filled(116, cache, rows, [40000, 9000, 3000, 600], 64, 1, hd)
    T = sum(rows)
    need = gv.lib.gv_paged_attention_workspace_bytes(ctypes.byref(f.cache.desc), ctypes.byref(f.batch.desc), nh)
    assert need // (T * nh * (hd + 2) * 4) > 64   # chunks of the longest
    q = round_to(np.random.default_rng(117).standard_normal((T, nh, hd)) * 1.5, kind)
    scale = float(np.float32(hd ** -0.5))
    out, lse = gv.paged_attention(f.cache, f.batch, q, type_=TYPES[kind], scale=scale)
    want, want_lse, tol, tol_lse = attention(f, q, scale, kind)
    assert (np.abs(out - want) <= tol).all() and (np.abs(lse - want_lse) <= tol_lse).all()
