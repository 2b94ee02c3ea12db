"""A step over several conversations as a host composes it: norm and quantize, q | k | v's products, keys and values
appended to the conversations' pages, attention over them (one call after the other, nothing waited for), the gate (on the
host here), the output product onto the residual stream; then the head's products, the logits' rules, the tokens. Each
conversation's rows are held to what the model gives for them alone (gv_model_layer at its position), over two steps of
which the first's last rows are not kept."""
import ctypes

import numpy as np
import pytest

import pyoracle as po
from model_helpers import SMALL, SMALL_ROUTER_SIGMA, adopt_oracle_model, rel_err

pytestmark = pytest.mark.gpu

CTX = 140
H, NH, NKV, HD, V = (SMALL[k] for k in ("hidden", "n_heads", "n_kv_heads", "head_dim", "vocab"))
QROW = NH * 2 * HD + 2 * NKV * HD   # a row of q (each head's gate beside its queries) | k | v
PAGE = 16


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


@pytest.fixture(scope="module", params=[0, 1], ids=["f16", "i8"])
def pair(request, gv):
    cfg = dict(SMALL, kv_int8=request.param)
    om = po.Model(cfg, seed=7, router_sigma=SMALL_ROUTER_SIGMA, ctx=CTX)
    gm = gv.VerifyModel(cfg)
    yield om, gm
    gm.close()


class Layer:
    """one layer's matrices and norms on the device"""

    def __init__(self, gv, om, l):
        self.products = [gv.Q4Matrix(om.tensor(kind, l)[0], rows, cols, float(om.tensor(kind, l)[1][0]))
                         for kind, rows, cols in ((po.Q, NH * 2 * HD, H), (po.K, NKV * HD, H), (po.V, NKV * HD, H))]
        self.o = gv.Q4Matrix(om.tensor(po.O, l)[0], H, NH * HD, float(om.tensor(po.O, l)[1][0]))
        self.norms = {k: gv.DeviceBuffer.from_array(om.tensor(k, l)[0].view(np.float32))
                      for k in (po.IN_NORM, po.Q_NORM, po.K_NORM)}


def _cache(gv, om, l, pages, lens, pool):
    """the layer's cached positions, each conversation's to pages of its own"""
    kind = gv.I8 if om.cfg["kv_int8"] else gv.F16
    c = gv.PagedCache(kind, pool, PAGE, NKV, HD)
    if kind == gv.I8:
        x = om.tensor(po.KV8, l)[0].view(np.int8).reshape(2, -1, NKV, HD)
        s = om.tensor(po.KVS, l)[0].view(np.float32).reshape(2, -1, NKV)
    else:
        x = om.tensor(po.KV, l)[0].view(np.float16).reshape(2, -1, NKV, HD).astype(np.float32)
    for which, name in enumerate(("k", "v")):
        w, ws = np.zeros((pool, NKV, PAGE, HD), np.float32), np.zeros((pool, NKV, PAGE), np.float32)
        for i, n in enumerate(lens):
            for p in range(n):
                w[pages[i, p // PAGE], :, p % PAGE] = x[which, p]
                if kind == gv.I8:
                    ws[pages[i, p // PAGE], :, p % PAGE] = s[which, p]
        c.write(name, w, ws)
    return c


def _attend(gv, layer, cache, batch, x, T, rope):
    """x (device, [T][H]) += the layer's attention, as a host enqueues it; the gate alone is made on the host"""
    lib, chk = gv.lib, gv.check
    act = gv.DeviceBuffer(T * gv.act_bytes(H))
    qkv, q, out = (gv.DeviceBuffer(T * n * 4) for n in (QROW, NH * HD, NH * HD))
    chk(lib.gv_quantize(x.ptr, H, T, H, layer.norms[po.IN_NORM].ptr, SMALL["eps"], act.ptr, None), "gv_quantize")
    at = 0
    for w in layer.products:
        chk(lib.gv_gemv_q4(w.ref(), act.ptr, T, qkv.ptr + 4 * at, QROW, 0), "gv_gemv_q4")
        at += w.rows
    cos, sin = rope
    a = gv.GvAppendRows(type=gv.F32, n_heads=NH, q=qkv.ptr, q_row=QROW, q_head=2 * HD, k=qkv.ptr + 4 * NH * 2 * HD, k_row=QROW,
                        k_head=HD, v=qkv.ptr + 4 * (NH * 2 + NKV) * HD, v_row=QROW, v_head=HD,
                        q_norm=layer.norms[po.Q_NORM].ptr, k_norm=layer.norms[po.K_NORM].ptr, eps=SMALL["eps"],
                        rope_dim=SMALL["rope_dim"], cos=cos.ptr, sin=sin.ptr, n_positions=SMALL["max_ctx"], q_type=gv.F32,
                        q_out=q.ptr, q_out_row=NH * HD)
    kv, b = ctypes.byref(cache.desc), ctypes.byref(batch.desc)
    chk(lib.gv_paged_append(kv, b, ctypes.byref(a)), "gv_paged_append")
    n = lib.gv_paged_attention_workspace_bytes(kv, b, NH)
    ws = gv.DeviceBuffer(n)
    r = gv.GvAttentionRows(type=gv.F32, n_heads=NH, q=q.ptr, q_row=NH * HD, out=out.ptr, out_row=NH * HD, scale=HD ** -0.5)
    chk(lib.gv_paged_attention(kv, b, ctypes.byref(r), ws.ptr, n), "gv_paged_attention")
    chk(lib.gv_synchronize(), "gv_synchronize")
    gate = qkv.download(np.float32, (T, QROW))[:, :NH * 2 * HD].reshape(T, NH, 2, HD)[:, :, 1]
    y = out.download(np.float32, (T, NH, HD)) / (1.0 + np.exp(-gate))
    out.upload(np.ascontiguousarray(y, np.float32))
    chk(lib.gv_quantize(out.ptr, NH * HD, T, NH * HD, None, 0.0, act.ptr, None), "gv_quantize")
    chk(lib.gv_gemv_q4(layer.o.ref(), act.ptr, T, x.ptr, H, 1), "gv_gemv_q4")
    chk(lib.gv_synchronize(), "gv_synchronize")


def test_steps_over_several_conversations(gv, pair):
    om, gm = pair
    adopt_oracle_model(gm, om, CTX)
    # the longest first: the model's rows of a conversation then lie behind the next one's context
    ctx, rows, kept = np.array([130, 97, 64, 31, 1]), np.array([5, 1, 7, 2, 4]), np.array([3, 1, 1, 2, 4])
    n_seqs, T, T2 = 5, int(rows.sum()), 5
    r = np.random.default_rng(3)
    wide = 10
    pages = r.permutation(n_seqs * wide).astype(np.int32).reshape(n_seqs, wide)
    half = SMALL["rope_dim"] // 2
    inv = (1.0 / np.float32(SMALL["rope_theta"]) ** (np.arange(half, dtype=np.float32) * 2 / SMALL["rope_dim"])).astype(np.float32)
    angle = np.arange(SMALL["max_ctx"], dtype=np.float32)[:, None] * inv
    rope = [gv.DeviceBuffer.from_array(f(angle).astype(np.float32)) for f in (np.cos, np.sin)]
    start = np.concatenate([[0], np.cumsum(rows)])
    for l in range(SMALL["n_layers"]):
        x1, x2 = (r.standard_normal((n, H)).astype(np.float32) for n in (T, T2))
        want1, want2 = np.empty_like(x1), np.empty_like(x2)
        for i in range(n_seqs):
            gm.position = int(ctx[i])
            want1[start[i]:start[i + 1]] = gm.layer(l, x1[start[i]:start[i + 1]])[0]
            gm.position = int(ctx[i] + kept[i])
            want2[i] = gm.layer(l, x2[i:i + 1])[0]
        layer, cache = Layer(gv, om, l), _cache(gv, om, l, pages, ctx, n_seqs * wide)
        for x, want, batch in ((x1, want1, gv.PagedBatch(rows, ctx + rows, pages)),
                               (x2, want2, gv.PagedBatch([1] * n_seqs, ctx + kept + 1, pages))):
            dev = gv.DeviceBuffer.from_array(x)
            _attend(gv, layer, cache, batch, dev, len(x), rope)
            got = dev.download(np.float32, x.shape)
            # A difference of some 1e-6 between two fp32 orders moves an activation's int8 code now and then, a 1/127th of
            # its block's largest each: with weights of 0.02 and gated values below 2, 3e-4 a code against streams of about 3
            assert rel_err(got, want) <= 1e-3, (l, rel_err(got, want))
        adopt_oracle_model(gm, om, CTX)   # (the cache as it was)


def test_tokens_under_the_rules(gv, pair):
    """the head's products, each conversation's rules, greedy tokens: chains of three rows whose history grows by a draft a row"""
    om = pair[0]
    lib, chk = gv.lib, gv.check
    r = np.random.default_rng(4)
    seqs, chain = 4, 3
    T = seqs * chain
    x = r.standard_normal((T, H)).astype(np.float32)
    head = gv.Q4Matrix(om.tensor(po.LM_HEAD)[0], V, H, float(om.tensor(po.LM_HEAD)[1][0]))
    norm = gv.DeviceBuffer.from_array(om.tensor(po.FINAL_NORM)[0].view(np.float32))
    hist = [r.integers(0, V, 40) for _ in range(seqs)]
    begin = np.concatenate([[np.full(chain, 40 * i)] for i in range(seqs)]).reshape(-1).astype(np.int32)
    end = (begin + 38 + np.tile(np.arange(chain), seqs)).astype(np.int32)
    masks = np.full((1, V // 32), 0xFFFFFFFF, np.uint32)
    masks[0, :V // 64] = 0x55555555
    a = {"tokens": np.concatenate(hist).astype(np.int32), "begin": begin, "generated": begin + 10, "end": end,
         "repetition": np.full(T, 1.3, np.float32), "frequency": np.full(T, 0.25, np.float32),
         "presence": np.full(T, 0.5, np.float32), "masks": masks, "mask_of": np.repeat([-1, 0, -1, 0], chain).astype(np.int32)}
    dev = {n: gv.DeviceBuffer.from_array(b) for n, b in a.items()}
    dx, act = gv.DeviceBuffer.from_array(x), gv.DeviceBuffer(T * gv.act_bytes(H))
    raw, done = gv.DeviceBuffer(T * V * 4), gv.DeviceBuffer(T * V * 4)
    rules = gv.GvLogitsRules(**{n: b.ptr for n, b in dev.items()}, n_tokens=a["tokens"].size, n_masks=1, ld_mask=V // 32)
    toks = np.empty(T, np.int32)
    u = np.zeros(T)
    chk(lib.gv_quantize(dx.ptr, H, T, H, norm.ptr, SMALL["eps"], act.ptr, None), "gv_quantize")
    chk(lib.gv_gemv_q4(head.ref(), act.ptr, T, raw.ptr, V, 0), "gv_gemv_q4")
    chk(lib.gv_process_logits(ctypes.byref(rules), raw.ptr, gv.F32, V, T, V, done.ptr, V), "gv_process_logits")
    chk(lib.gv_sample_rows(done.ptr, V, T, V, 0.0, 1.0, 0, 1024, u.ctypes.data, toks.ctypes.data), "gv_sample_rows")
    chk(lib.gv_synchronize(), "gv_synchronize")
    got, want = done.download(np.float32, (T, V)), raw.download(np.float32, (T, V)).astype(np.float64)
    for t in range(T):
        seen = np.unique(a["tokens"][begin[t]:end[t]])
        count = np.bincount(a["tokens"][begin[t] + 10:end[t]], minlength=V)
        rep = float(np.float32(1.3))
        want[t, seen] = np.where(want[t, seen] > 0, want[t, seen] / rep, want[t, seen] * rep)
        want[t] -= 0.25 * count + 0.5 * (count > 0)
        if a["mask_of"][t] == 0:
            want[t, (masks[0][np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin)
    assert (np.abs(got[fin] - want[fin]) <= 4 * 2.0 ** -24 * (np.abs(want[fin]) + 8)).all()   # (four roundings, penalties below 8)
    assert np.array_equal(toks, got.argmax(1))
    assert (toks != raw.download(np.float32, (T, V)).argmax(1)).any(), "the rules changed no token"
