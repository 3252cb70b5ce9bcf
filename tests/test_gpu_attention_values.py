"""Attention in flash mode on values at the edges of their types."""
import numpy as np
import pytest

from decoder_reference import check, decoder_attention
from emx_onnx_cgen_b200 import workloads as W
from emx_onnx_cgen_b200.runtime import Session
from gpu_util import plan_for, require_gpu

pytestmark = pytest.mark.gpu


def run(wl, x):
    return Session(plan_for(wl, attention_mode="flash")).run(x)["Y"]


@pytest.mark.parametrize("mask", ["f16", "f32"])
@pytest.mark.parametrize("kw", [
    dict(q_seq=3, kv_seq=150), dict(q_seq=40, kv_seq=150), dict(q_seq=200, kv_seq=150, head_dim=128),
    dict(q_seq=40, kv_seq=40, past=100, shared_past=False), dict(q_seq=3, kv_seq=3, past=100),
])
def test_additive_entries_of_causally_hidden_keys(kw, mask):
    """Whatever a mask holds for a key behind the token reaches nothing: NaN, infinities, the type's extremes."""
    require_gpu()
    tq, past = kw["q_seq"], kw.get("past", 0)
    t = past + kw["kv_seq"]
    kw = dict(batch=2, q_heads=2, kv_heads=2, causal=True, mask=mask, mask_shape=(2, 1, tq, t), **kw)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(32)
    m = x["mask"]
    big = np.finfo(m.dtype)
    for q in range(tq):
        at = np.arange(past + q + 1, t)
        m[:, 0, q, at] = np.array([np.nan, np.inf, -np.inf, big.max, big.min, 0], m.dtype)[at % 6]
    if mask == "f32":
        m[1, 0, tq // 2, :past + tq // 2 + 1] = big.min
    check(run(wl, x), *decoder_attention(wl, x), str(kw))


@pytest.mark.parametrize("mask", ["f16", "f32"])
@pytest.mark.parametrize("q_seq", [3, 40])
def test_additive_entries_behind_the_valid_count(q_seq, mask):
    require_gpu()
    kw = dict(batch=4, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=150, count=True, mask=mask, mask_shape=(4, 1, q_seq, 150))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(33)
    x["count"][:] = [150, 0, 63, 101]
    for b, n in enumerate(x["count"]):
        x["mask"][b, :, :, n:] = np.array([np.nan, np.inf, np.finfo(x["mask"].dtype).max], x["mask"].dtype)[np.arange(150 - n) % 3]
    check(run(wl, x), *decoder_attention(wl, x), str(kw))


@pytest.mark.parametrize("mask", ["f16", "f32"])
@pytest.mark.parametrize("q_seq", [3, 40])
def test_visible_infinite_and_nan_entries(q_seq, mask):
    """A visible +inf or NaN entry makes its row NaN, as the sum does, and no other row."""
    require_gpu()
    kw = dict(batch=2, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=150, mask=mask, mask_shape=(2, 1, q_seq, 150))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(34)
    want, tol = decoder_attention(wl, x)
    x["mask"][0, 0, 1, 77], x["mask"][1, 0, 2, 149] = np.inf, np.nan
    got = run(wl, x)
    assert np.isnan(got[0, :, 1]).all() and np.isnan(got[1, :, 2]).all()
    got[0, :, 1], got[1, :, 2] = want[0, :, 1], want[1, :, 2]
    check(got, want, tol, str(kw))
