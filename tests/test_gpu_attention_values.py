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


@pytest.mark.parametrize("kw", [
    dict(batch=3, q_heads=2, kv_heads=2, q_seq=2, kv_seq=200),                         # few-row pass
    dict(batch=2, q_heads=6, kv_heads=2, q_seq=5, kv_seq=333, head_dim=128),           # its 16-row form
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=3, kv_seq=4000),                        # split key ranges
    dict(batch=3, q_heads=2, kv_heads=2, q_seq=40, kv_seq=200),                        # 128-row pass
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=20, kv_seq=3000, head_dim=128),         # split
    dict(batch=2, q_heads=2, kv_heads=1, q_seq=150, kv_seq=190, causal=True),
    dict(batch=3, q_heads=4, kv_heads=2, q_seq=2, kv_seq=70, past=321),                # a shared past: merged
    dict(batch=40, q_heads=8, kv_heads=2, q_seq=1, kv_seq=70, past=700, head_dim=128),
    dict(batch=3, q_heads=4, kv_heads=2, q_seq=30, kv_seq=30, past=321, shared_past=False, causal=True),
])
def test_large_additive_entries_keep_their_order(kw):
    """fp32 entries beyond 2^24 of different sizes in one row: only the largest of them count, and among equal ones the
    scores decide (from 2^56 on a sum has none of its score's digits in 64 bits either)."""
    require_gpu()
    b, tq, t = kw["batch"], kw["q_seq"], kw["kv_seq"] + kw.get("past", 0)
    kw = dict(kw, mask="f32", mask_shape=(b, 1, tq, t))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(31)
    r = np.random.default_rng(7)
    levels = [(-1e9, -2e9), (-1e30, np.finfo(np.float32).min), (-2e9, -1e9, -3e7), (0.0, -1e9, -2e9), (1e9, 2e9, -1e9),
              (-1e30, -1e9), (1e30, 3e38), (-3e7, -4e7), (-1e9, -1e9 - 64, -1e9 - 128), (0.0, -1e9, np.finfo(np.float32).min),
              (np.finfo(np.float32).min, np.finfo(np.float32).max), (-16777216.0, -16777218.0, -16777220.0)]
    m = x["mask"]
    for i in range(b):
        for q in range(tq):
            lv = np.array(levels[(i * tq + q) % len(levels)], np.float32)
            row = lv[r.integers(0, len(lv), t)]
            if q % 3 == 1:  # the larger ones late, or early, in the row
                row = np.sort(row)
            elif q % 3 == 2:
                row = np.sort(row)[::-1]
            m[i, 0, q] = row
    check(run(wl, x), *decoder_attention(wl, x), str(kw))


@pytest.mark.parametrize("mask", ["none", "bool", "f16", "f32"])
@pytest.mark.parametrize("scale", [0.125, -0.125, 0.5])
@pytest.mark.parametrize("kw", [
    dict(q_seq=1, kv_seq=300), dict(q_seq=9, kv_seq=300, head_dim=128), dict(q_seq=40, kv_seq=300),
    dict(q_seq=40, kv_seq=300, head_dim=128), dict(q_seq=300, kv_seq=300), dict(q_seq=300, kv_seq=300, head_dim=128),
    dict(q_seq=1, kv_seq=3000), dict(q_seq=2, kv_seq=60, past=240),
])
def test_scores_far_apart_pick_one_key(kw, scale, mask):
    """Scores of 2^17 to 2^33, further apart than any rounding of them: all the weight is on the largest, and its value
    comes out, within half a step for the weight (a pass may round it for the product but not for the sum) and half a
    step for the result."""
    require_gpu()
    past = kw.get("past", 0)
    t = kw["kv_seq"] + past
    kw = dict(batch=2, q_heads=2, kv_heads=2, scale=scale, **kw)
    if mask != "none":
        kw.update(mask=mask, mask_shape=(2, 1, kw["q_seq"], t))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(35)
    if mask == "bool":
        x["mask"][:] = True
    r = np.random.default_rng(8)
    for size in (37.0, 8192.0, 60000.0):
        x["Q"][:] = size
        # D times whole numbers, each key its own: scores are at least size * D * |scale| apart
        level = np.stack([r.permutation(2047)[:t] - 1023 if t < 2000 else r.permutation(t) - t // 2 for _ in range(4)]).reshape(2, 2, t).astype(np.float16)
        if past:
            level[1, :, :past] = level[0, :, :past]
            x["PK"][:] = level[:1, :, :past, None]
        x["K"][:] = level[:, :, past:, None]
        top = np.sort(level if scale > 0 else -level, axis=2)
        assert (top[..., -1] > top[..., -2]).all()
        best = level.argmax(2) if scale > 0 else level.argmin(2)
        got = run(wl, x)
        for b in range(2):
            for h in range(2):
                k = best[b, h]
                want = x["PV"][0, h, k] if k < past else x["V"][b, h, k - past]
                want = np.broadcast_to(want, got[b, h].shape).astype(np.float64)
                check(got[b, h], want, (2.0 ** -10 + 2.0 ** -20) * np.abs(want) + 2.0 ** -25, f"{size} {b} {h}")


@pytest.mark.parametrize("mask", ["f16", "f32"])
@pytest.mark.parametrize("q_seq", [1, 9, 40, 150])
def test_scores_of_keys_hidden_by_an_entry(q_seq, mask):
    """-inf hides its key whatever the key's score is, beside entries of any size."""
    require_gpu()
    kw = dict(batch=2, q_heads=2, kv_heads=2, q_seq=q_seq, kv_seq=260, mask=mask, mask_shape=(2, 1, q_seq, 260))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(38)
    hidden = [0, 3, 70, 128, 259]
    x["mask"][1] -= 60000 if mask == "f16" else np.float32(1e9)
    x["mask"][..., hidden] = -np.inf
    want = decoder_attention(wl, x)
    x["K"][:, :, hidden] = np.array([np.inf, np.nan, -np.inf, np.nan, np.inf], np.float16)[:, None]
    check(run(wl, x), *want, str(kw))


@pytest.mark.parametrize("kw", [
    dict(q_seq=1, kv_seq=16384), dict(q_seq=9, kv_seq=16384, head_dim=128), dict(q_seq=40, kv_seq=16384),
    dict(q_seq=300, kv_seq=16384), dict(q_seq=300, kv_seq=16384, head_dim=128),
])
@pytest.mark.parametrize("log2", [-14.5, -16.4, -18.6])
def test_weights_below_fp16s_normal_range(kw, log2):
    """One key of weight 1 and thousands far below 2^-14, which together matter: each is within half a step of fp16
    (2^-25 there), whichever of the passes' sums it enters, rounded or not."""
    require_gpu()
    kw = dict(batch=1, q_heads=2, kv_heads=2, scale=1.0, **kw)
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(37)
    x["Q"][:], x["K"][:] = 0, 0
    x["Q"][..., 0] = 1
    x["K"][..., 0] = log2 * np.log(2)
    x["K"][:, :, 700, 0] = 0
    x["V"][:] = 1 + 0.25 * x["V"]
    x["V"][:, :, 700] = 0
    check(run(wl, x), *decoder_attention(wl, x), str(kw))


def _marked(t, d, n):
    """Values [n, t, d] of which each column holds one key's mark, t, so that equal weights 1/t give 1 for a key that
    counts once, 0 for one that is lost and 2 for one that counts twice; n columns sets share the keys."""
    v = np.zeros((n, t, d), np.float16)
    keys = np.arange(n * d) % t if n * d >= t else np.linspace(0, t - 1, n * d).round().astype(int)
    if n * d < t:  # both sides of the tiles' edges rather than an even grid
        edge = np.unique(np.concatenate([np.arange(0, t, 64), np.arange(63, t, 64), np.arange(15, t, 16)[:n * d], [0, t - 1]]))
        keys[:min(len(edge), n * d)] = edge[:n * d]
    v[np.arange(n * d) // d, keys, np.arange(n * d) % d] = t
    return v


@pytest.mark.parametrize("kw", [
    dict(batch=1, q_heads=2, kv_heads=2, q_seq=1, kv_seq=5000, head_dim=128),
    dict(batch=2, q_heads=32, kv_heads=16, q_seq=1, kv_seq=4096, head_dim=128),
    dict(batch=3, q_heads=16, kv_heads=8, q_seq=3, kv_seq=4104, head_dim=64),
    dict(batch=1, q_heads=48, kv_heads=24, q_seq=5, kv_seq=3000, head_dim=128),
    dict(batch=1, q_heads=24, kv_heads=24, q_seq=40, kv_seq=3000, head_dim=128),            # 128-row pass
    dict(batch=1, q_heads=16, kv_heads=16, q_seq=40, kv_seq=1000, head_dim=64, mask="f16"),
    dict(batch=2, q_heads=24, kv_heads=12, q_seq=40, kv_seq=2000, head_dim=96, mask="f32"),
    dict(batch=1, q_heads=32, kv_heads=32, q_seq=300, kv_seq=2000, head_dim=64),            # 256-row pass
    dict(batch=2, q_heads=16, kv_heads=16, q_seq=150, kv_seq=3000, head_dim=128, mask="bool"),
    dict(batch=2, q_heads=32, kv_heads=16, q_seq=1, kv_seq=3000, head_dim=128, mask="bool"),
    dict(batch=3, q_heads=32, kv_heads=16, q_seq=1, kv_seq=24, past=9000, head_dim=128),    # a shared past in ranges
    dict(batch=128, q_heads=16, kv_heads=16, q_seq=1, kv_seq=300, past=700, head_dim=64),
    dict(batch=130, q_heads=64, kv_heads=16, q_seq=1, kv_seq=104, past=2000, head_dim=128, mask="bool"),
    dict(batch=3, q_heads=16, kv_heads=16, q_seq=60, kv_seq=60, past=1940, head_dim=64),
    dict(batch=2, q_heads=16, kv_heads=16, q_seq=2, kv_seq=40, past=1000, head_dim=64, shared_past=False),
])
def test_every_key_of_a_range_counts_once(kw):
    require_gpu()
    b, h, past, own, d = kw["batch"], kw["kv_heads"], kw.get("past", 0), kw["kv_seq"], kw["head_dim"]
    t = past + own
    assert t % 8 == 0 and t < 16384  # a mark is a whole fp16 number
    if "mask" in kw:
        kw = dict(kw, mask_shape=(b, 1, kw["q_seq"], t))
    wl = W.decoder_attention(**kw)
    x = wl.make_inputs(36)
    x["Q"][:] = 0
    if "mask" in x:
        x["mask"][:] = x["mask"].dtype == bool
    shared = past and kw.get("shared_past", True)
    v = np.zeros((b, h, t, d), np.float16)
    if shared:  # a sequence marks its own keys in half of the columns, all the past's in the others
        v[:, :, :past, :d // 2] = _marked(past, d // 2, h) / np.float16(past) * np.float16(t)
        v[:, :, past:, d // 2:] = (_marked(own, d - d // 2, b * h) / np.float16(own) * np.float16(t)).reshape(b, h, own, -1)
        x["PV"][:] = v[:1, :, :past]
        x["V"][:] = v[:, :, past:]
    else:
        v[:] = _marked(t, d, b * h).reshape(b, h, t, d)
        if past:
            x["PV"][:], x["V"][:] = v[:, :, :past], v[:, :, past:]
        else:
            x["V"][:] = v
    got = run(wl, x).astype(np.float64)
    want = (v != 0).sum(2, dtype=np.int64)  # [b, h, d]: 0 or 1
    assert set(np.unique(want)) <= {0, 1} and want.any()
    want = np.repeat(want, kw["q_heads"] // h, axis=1)[:, :, None]
    # one mark times an exact weight over an exact sum (whole numbers below 2^24), and the roundings of the division,
    # the merge's factors of 1 and the result
    assert np.abs(got - want).max() <= 2.0 ** -10
