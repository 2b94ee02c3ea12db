"""What gv_paged_append, gv_paged_attention and gv_process_logits refuse, each by one planted fault in arguments that are
else in order (CPU: every refusal comes before any device work)."""
import ctypes

import pytest

import geode_amd as g

MEM = 1 << 20   # an address of the right alignment: refused calls touch no memory


def _kv(**k):
    return g.GvPagedKv(**{**dict(type=g.F16, n_kv_heads=2, head_dim=64, page_size=32, n_pages=8, k=MEM, v=MEM, k_scale=MEM,
                                 v_scale=MEM, page_stride=4096, head_stride=2048, pos_stride=64), **k})


def _batch(**k):
    return g.GvPagedBatch(**{**dict(n_seqs=2, n_rows=4, max_rows=3, max_len=100, row_start=MEM, lens=MEM, pages=MEM,
                                    ld_pages=4), **k})


def _append(**k):
    return g.GvAppendRows(**{**dict(type=g.F32, n_heads=4, q=MEM, k=MEM, v=MEM, q_row=256, q_head=64, k_row=128, k_head=64,
                                    v_row=128, v_head=64, eps=1e-6, rope_dim=32, cos=MEM, sin=MEM, n_positions=100,
                                    q_type=g.F32, q_out=2 * MEM, q_out_row=256), **k})


def _rows(**k):
    return g.GvAttentionRows(**{**dict(type=g.F32, n_heads=4, q=MEM, q_row=256, out=2 * MEM, out_row=256, scale=0.125), **k})


def _refused(rc, *words):
    assert rc == -1
    msg = g.lib.gv_last_error().decode()
    for w in words:
        assert w in msg, msg


KV = [(dict(type=g.F32), "GV_F16"), (dict(type=7), "GV_F16"), (dict(n_kv_heads=0), "KV heads"), (dict(head_dim=0), "head_dim"),
      (dict(head_dim=72), "head_dim"), (dict(head_dim=272), "head_dim"), (dict(page_size=8), "page_size"),
      (dict(page_size=40), "page_size"), (dict(n_pages=0), "pages"), (dict(k=None), "aligned"), (dict(v=MEM + 8), "aligned"),
      (dict(type=g.I8, k_scale=None), "scale"), (dict(type=g.I8, v_scale=MEM + 4), "scale"), (dict(pos_stride=0), "strides"),
      (dict(pos_stride=72), "strides"), (dict(head_stride=-64), "strides"), (dict(pos_stride=1 << 24), "strides"),
      (dict(page_stride=8), "strides")]
BATCH = [(dict(n_seqs=0), "n_seqs"), (dict(n_rows=0), "n_rows"), (dict(max_rows=0), "max_rows"), (dict(row_start=None), "row_start"),
         (dict(lens=None), "lens"), (dict(pages=None), "pages"), (dict(ld_pages=0), "ld_pages"), (dict(max_len=0), "max_len"),
         (dict(max_len=129), "max_len")]


@pytest.mark.parametrize("kv,batch,word", [(k, {}, w) for k, w in KV] + [({}, b, w) for b, w in BATCH])
def test_cache_and_batch(kv, batch, word):
    c, b = _kv(**kv), _batch(**batch)
    r, a = ctypes.byref(_rows()), ctypes.byref(_append())
    _refused(g.lib.gv_paged_append(ctypes.byref(c), ctypes.byref(b), a), "gv_paged_append", word)
    _refused(g.lib.gv_paged_attention(ctypes.byref(c), ctypes.byref(b), r, MEM, 1 << 30), "gv_paged_attention", word)
    assert g.lib.gv_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 4) == 0


@pytest.mark.parametrize("rows,word", [
    (dict(type=g.I8), "rows are"), (dict(n_heads=-1), "n_heads"), (dict(k=None), "k and v"), (dict(v=MEM + 4), "k and v"),
    (dict(k_row=130), "k and v"), (dict(v_head=-64), "k and v"), (dict(rope_dim=12), "rope_dim"), (dict(rope_dim=72), "rope_dim"),
    (dict(rope_dim=-8), "rope_dim"), (dict(cos=None), "cos"), (dict(sin=MEM + 4), "cos"), (dict(n_positions=0), "cos"),
    (dict(q=None), "q:"), (dict(q_row=258), "q:"), (dict(q_type=g.I8), "q_out"), (dict(q_out=None), "q_out"),
    (dict(q_out_row=192), "q_out"), (dict(q_out=MEM, q_type=g.F16), "q_out is q"), (dict(q_out=MEM, q_head=128), "q_out is q")])
def test_append(rows, word):
    _refused(g.lib.gv_paged_append(ctypes.byref(_kv()), ctypes.byref(_batch()), ctypes.byref(_append(**rows))), "gv_paged_append", word)


@pytest.mark.parametrize("rows,kv,batch,ws,word", [
    (dict(type=g.BF16), {}, {}, MEM, "cache's type"), (dict(type=g.I8), dict(type=g.I8), {}, MEM, "cache's type"),
    (dict(n_heads=3), {}, {}, MEM, "n_heads"), (dict(n_heads=0), {}, {}, MEM, "n_heads"), (dict(q=None), {}, {}, MEM, "q and out"),
    (dict(out=MEM + 8), {}, {}, MEM, "q and out"), (dict(q_row=248), {}, {}, MEM, "q and out"), (dict(out_row=260), {}, {}, MEM, "q and out"),
    (dict(out=MEM), {}, {}, MEM, "out is not q"), (dict(scale=float("nan")), {}, {}, MEM, "scale"),
    ({}, {}, dict(max_rows=33), MEM, "32 rows"), ({}, {}, dict(max_len=2000, ld_pages=100), None, "workspace"),
    ({}, {}, dict(max_len=2000, ld_pages=100), MEM + 4, "workspace")])
def test_attention(rows, kv, batch, ws, word):
    _refused(g.lib.gv_paged_attention(ctypes.byref(_kv(**kv)), ctypes.byref(_batch(**batch)), ctypes.byref(_rows(**rows)), ws, 1 << 30),
             "gv_paged_attention", word)


def test_more_than_a_launch_can_count():
    """the threads of a launch's axis past 32 bits, partial results past any memory: refused, not wrapped around"""
    kv = _kv(n_kv_heads=8, head_dim=256, page_size=64, pos_stride=256, head_stride=16384, page_stride=131072)
    for b, heads in ((_batch(max_len=1 << 30, ld_pages=1 << 24), 8), (_batch(n_seqs=1 << 20, max_len=1 << 16, ld_pages=1024), 8),
                     (_batch(n_rows=(1 << 24) - 1, max_len=1 << 29, ld_pages=1 << 23), 4096)):
        r = _rows(n_heads=heads, q_row=1 << 20, out_row=1 << 20)
        assert g.lib.gv_paged_attention_workspace_bytes(ctypes.byref(kv), ctypes.byref(b), heads) == 0
        _refused(g.lib.gv_paged_attention(ctypes.byref(kv), ctypes.byref(b), ctypes.byref(r), MEM, 1 << 62), "too many")
    b = _batch(n_rows=1 << 24)
    _refused(g.lib.gv_paged_append(ctypes.byref(_kv()), ctypes.byref(b), ctypes.byref(_append())), "n_rows")
    rules = g.GvLogitsRules(tokens=MEM, begin=MEM, end=MEM, n_tokens=1 << 30)
    _refused(g.lib.gv_process_logits(ctypes.byref(rules), 2 * MEM, g.F32, 100, 2, 100, MEM, 100), "n_tokens")
    _refused(g.lib.gv_process_logits(ctypes.byref(g.GvLogitsRules()), 2 * MEM, g.F32, 1 << 24, 65536, 1 << 24, MEM, 1 << 24),
             "too many")


def test_attention_workspace_too_small():
    b = _batch(max_len=2000, ld_pages=100)
    n = g.lib.gv_paged_attention_workspace_bytes(ctypes.byref(_kv()), ctypes.byref(b), 4)
    assert n > 0
    _refused(g.lib.gv_paged_attention(ctypes.byref(_kv()), ctypes.byref(b), ctypes.byref(_rows()), MEM, n - 1), "workspace")


def test_null_descriptions():
    _refused(g.lib.gv_paged_append(None, None, None), "no cache")
    _refused(g.lib.gv_paged_append(ctypes.byref(_kv()), None, None), "no batch")
    _refused(g.lib.gv_paged_append(ctypes.byref(_kv()), ctypes.byref(_batch()), None), "no rows")
    _refused(g.lib.gv_paged_attention(ctypes.byref(_kv()), ctypes.byref(_batch()), None, None, 0), "no rows")
    _refused(g.lib.gv_process_logits(None, MEM, g.F32, 8, 1, 8, MEM, 8), "no rules")


@pytest.mark.parametrize("rules,args,word", [
    ({}, dict(type=g.I8), "logits are"), ({}, dict(rows=0), "rows"), ({}, dict(rows=65537), "rows"), ({}, dict(V=0), "V:"),
    ({}, dict(V=(1 << 24) + 1, ld=1 << 25, ldo=1 << 25), "V:"), ({}, dict(logits=None), "device memory"),
    ({}, dict(out=None), "device memory"), ({}, dict(out=MEM + 2), "device memory"), ({}, dict(ld=99), "ld and ldo"),
    ({}, dict(ldo=99), "ld and ldo"), ({}, dict(logits=MEM, out=MEM, type=g.F16), "out is logits"),
    ({}, dict(logits=MEM, out=MEM, ldo=200), "out is logits"), (dict(tokens=MEM, begin=MEM), {}, "tokens need"),
    (dict(presence=MEM), {}, "penalties need"), (dict(tokens=MEM, begin=MEM, end=MEM, n_tokens=-1), {}, "tokens need"),
    (dict(bias_token=MEM, bias_value=MEM), {}, "biases need"), (dict(masks=MEM, n_masks=1, ld_mask=4), {}, "masks need"),
    (dict(masks=MEM, mask_of=MEM, n_masks=0, ld_mask=4), {}, "masks need"),
    (dict(masks=MEM, mask_of=MEM, n_masks=1, ld_mask=3), {}, "masks need")])
def test_logits(rules, args, word):
    a = {**dict(logits=2 * MEM, type=g.F32, ld=100, rows=2, V=100, out=MEM, ldo=100), **args}
    _refused(g.lib.gv_process_logits(ctypes.byref(g.GvLogitsRules(**rules)), a["logits"], a["type"], a["ld"], a["rows"],
                                     a["V"], a["out"], a["ldo"]), "gv_process_logits", word)


def test_the_bindings_arrays():
    """arrays of other shapes than the batch's and the cache's are refused before anything is uploaded"""
    from types import SimpleNamespace

    import numpy as np

    cache, batch = SimpleNamespace(desc=_kv()), SimpleNamespace(desc=_batch())
    z = lambda *s: np.zeros(s, np.float32)   # noqa: E731
    good = dict(q=z(4, 4, 64), k=z(4, 2, 64), v=z(4, 2, 64))
    for bad in (dict(k=z(3, 2, 64)), dict(v=z(4, 1, 64)), dict(q=z(4, 4, 32)), dict(q_norm=z(32)), dict(positions=z(3)),
                dict(rope_dim=32, cos=z(9, 16), sin=z(9, 8)), dict(rope_dim=32, cos=z(9, 8), sin=z(9, 8))):
        with pytest.raises(g.GeodeError, match="paged_append"):
            g.paged_append(cache, batch, **{**good, **bad})
    for q, visible in ((z(3, 4, 64), None), (z(4, 4, 32), None), (z(4, 4, 64), z(3))):
        with pytest.raises(g.GeodeError, match="paged_attention"):
            g.paged_attention(cache, batch, q, visible=visible)
    for bad in (dict(begin=z(3)), dict(mask_of=z(1)), dict(repetition=z(2, 1)), dict(bias_token=z(3), bias_value=z(2))):
        with pytest.raises(g.GeodeError, match="process_logits"):
            g.process_logits(z(2, 10), **bad)
    for rows, lens, pages in (([1, 1], [2], z(2, 1)), ([1, 1], [2, 2], z(1, 2)), ([1], [2], z(1))):
        with pytest.raises(g.GeodeError, match="PagedBatch"):
            g.PagedBatch(rows, lens, pages)


def test_the_structures_are_the_headers():
    """the ctypes structures' sizes against the C compiler's"""
    import os
    import subprocess
    import tempfile

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"gv_paged_kv": g.GvPagedKv, "gv_paged_batch": g.GvPagedBatch, "gv_append_rows": g.GvAppendRows,
             "gv_attention_rows": g.GvAttentionRows, "gv_logits_rules": g.GvLogitsRules}
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        lines = []
        for n, s in names.items():
            lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
            lines += [f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for f in s._fields_]
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "geode_verify.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
        exe = os.path.join(d, "s")
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", exe], check=True)
        said = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, s in names.items():
        assert int(said[n]) == ctypes.sizeof(s)
        for f in s._fields_:
            assert int(said[f"{n}.{f[0]}"]) == getattr(s, f[0]).offset, f"{n}.{f[0]}"
