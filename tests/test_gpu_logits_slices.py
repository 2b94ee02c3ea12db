"""gv_process_logits where a workgroup takes two or four quads of logits a thread (many logits), in and out of place, with rows
wider than the vocabulary: bit for bit what calls of few rows give, which tests/test_gpu_logits_rules.py holds to the definition,
and that definition in 64 bits."""
import ctypes

import numpy as np
import pytest

from paged_ref import TYPES, round_to
from test_gpu_logits_rules import _rules, _want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


def _call(gv, x, kind, a, pad, in_place):
    """(the rows after the rules, what lies behind each row) of rows pad elements wider than the vocabulary"""
    rows, V = x.shape
    wide = np.full((rows, V + pad), 3.0, np.float32)
    wide[:, :V] = x
    src = gv._typed(wide, TYPES[kind])
    out = src if in_place else gv.DeviceBuffer.from_array(np.full((rows, V + 2 * pad), 4.0, np.float32))
    ldo = V + pad if in_place else V + 2 * pad
    dev = {n: gv.DeviceBuffer.from_array(v) for n, v in a.items()}
    r = gv.GvLogitsRules(**{n: b.ptr for n, b in dev.items()}, n_tokens=len(a["tokens"]), n_biases=len(a["bias_token"]),
                         n_masks=len(a["masks"]), ld_mask=a["masks"].shape[1])
    gv.check(gv.lib.gv_process_logits(ctypes.byref(r), src.ptr, TYPES[kind], V + pad, rows, V, out.ptr, ldo), "gv_process_logits")
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
    y = out.download(np.float32, (rows, ldo))
    return y[:, :V], y[:, V:]


# rows x vocabulary: two quads a thread where 1,024 workgroups of 2,048 logits are there, four where 1,024 of 4,096 are
@pytest.mark.parametrize("rows,V", [(300, 9001), (260, 16500), (300, 12291), (64, 80003), (1030, 5)])
@pytest.mark.parametrize("kind,in_place", [("f32", False), ("f32", True), ("f16", False), ("bf16", False)])
@pytest.mark.parametrize("pad", [0, 3])
def test_many_logits(gv, rows, V, kind, in_place, pad):
    a = _rules(120, rows, V, 200, biases=5, masks=3)
    x = round_to(np.random.default_rng(121).standard_normal((rows, V)) * 3, kind).astype(np.float32)
    got, behind = _call(gv, x, kind, a, pad, in_place)
    assert (behind == (3.0 if in_place else 4.0)).all()
    want, tol = _want(x, a)
    gone = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), gone) and (np.abs(got[~gone] - want[~gone]) <= tol[~gone]).all()
    for r in (0, rows // 2, rows - 1):   # a row alone
        one = {n: v if n in ("tokens", "bias_token", "bias_value", "masks") else v[r:r + 1] for n, v in a.items()}
        alone, _ = _call(gv, x[r:r + 1], kind, one, 0, False)
        assert np.array_equal(alone[0].view(np.uint32), got[r].view(np.uint32))
